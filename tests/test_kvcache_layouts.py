"""CPU tests of the cache layouts that an append refuses: rows that share memory."""

import pytest

from fa2 import _kvlib, _lib
from test_kvcache_host import append, attn, read

APART = [
    dict(),
    dict(k_stride=(8192, 256, 128), v_stride=(8192, 256, 128)),            # page, row, head
    dict(k_stride=(128, 1280 * 2, 1280), ks_stride=(1, 20, 10)),           # the page runs fastest
    dict(k_stride=(1 << 20, 144, 1 << 14), vs_stride=(999, 3, 97)),        # gaps
    dict(heads_kv=1, k_stride=(4096, 128, 0), ks_stride=(32, 1, 0)),       # the stride of a single entry
    dict(num_pages=1, v_stride=(0, 128, 4096)),
]
SHARED = [
    dict(k_stride=(8192, 128, 0)),                                         # one head's rows for all
    dict(v_stride=(0, 128, 4096)),                                         # one page
    dict(ks_stride=(64, 0, 32)),
    dict(vs_stride=(64, 1, 0)),
    dict(k_stride=(8192, 112, 4096)),                                      # rows reach into the next
    dict(v_stride=(8192 - 16, 128, 4096)),                                 # pages do
    dict(ks_stride=(63, 1, 32)),
    dict(vs_stride=(64, 1, 31)),
]


@pytest.mark.parametrize("kw", APART)
def test_rows_that_lie_apart_are_taken(kw):
    L = _kvlib.lib()
    assert L.fa2_kv8_append_sm100_check(append(**kw)) == _lib.FA2_OK


@pytest.mark.parametrize("kw", SHARED)
def test_shared_rows_are_read_but_not_written(kw):
    L = _kvlib.lib()
    assert L.fa2_kv8_append_sm100_check(append(**kw)) == _lib.FA2_ERR_LAYOUT
    assert L.fa2_kv8_append_sm100(append(**kw), None) == _lib.FA2_ERR_LAYOUT
    assert L.fa2_kv8_read_sm100_check(read(**kw)) == _lib.FA2_OK
    assert L.fa2_kv8_attn_sm100_check(attn(**kw)) == _lib.FA2_OK
