"""CPU tests of the host side of fa2.rotary and fa2.kvcache: the library exports what its header
declares, the struct packing matches the C layout, the host checks refuse what the kernels do not
take, and the Python entry points refuse wrong arguments before anything is launched."""

import os
import re

import pytest
import torch

from fa2 import _kvlib, _lib
from fa2.kvcache import (KVCacheFP8, alloc_kvcache_fp8, attention_kvcache_fp8, kvcache_append_fp8,
                         kvcache_read_fp8)
from fa2.rotary import rotary, rotary_inv_freq

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "fa2_kvcache_sm100.h")


# ------------------------------------------------------------------------------------ the library
def test_library_exports_every_declared_symbol():
    declared = set(re.findall(r"FA2_API\s+[\w\s\*]+?\b(fa2_\w+)\s*\(", open(HEADER).read()))
    assert declared == set(_kvlib.EXPORTED)
    for name in declared:
        assert hasattr(_kvlib.lib(), name), name


def test_abi_version_and_struct_sizes():
    L = _kvlib.lib()
    assert L.fa2_kvcache_sm100_abi_version() == _kvlib.ABI_VERSION
    assert [L.fa2_kvcache_sm100_params_size(i) for i in range(4)] == [s.size for s in _kvlib.STRUCTS]
    assert L.fa2_kvcache_sm100_params_size(4) == -1
    assert _lib.strerror(_lib.FA2_ERR_PAGE) != _lib.strerror(999)


def test_packing_follows_the_header_field_by_field():
    """The names of each struct in the header, in order, are the names that are packed."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    structs = dict(re.findall(r"typedef struct (\w+) \{(.*?)\} \w+;", text, flags=re.S))
    sizes = {"int32_t": "i", "int64_t": "q", "float": "f"}

    def fields(body):
        out = []
        for line in filter(None, (part.strip() for part in body.split(";"))):
            kind, name = re.match(r"(.*?)(\w+(?:\[\d+\])?)$", line).groups()
            count = re.search(r"\[(\d+)\]", name)
            if kind.strip() == "Fa2Kv8Cache":
                out += fields(structs["Fa2Kv8Cache"])
            else:
                code = "P" if "*" in kind else sizes[kind.strip()]
                out.append((name.split("[")[0], (count.group(1) if count else "") + code))
        return out

    for name, layout in zip(("Fa2RotaryParams", "Fa2Kv8AppendParams", "Fa2Kv8ReadParams", "Fa2Kv8AttnParams"), _kvlib.STRUCTS):
        short = {"k_in": "k", "v_in": "v"} if "Append" in name else {}
        declared, packed = fields(structs[name]), layout.fields
        assert [code for _, code in declared] == [code for _, code in packed], name
        assert [n for n, _ in declared] == [short.get(n, n) for n, _ in packed], name


def test_c_header_compiles_as_c99(tmp_path):
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    src = tmp_path / "caller.c"
    src.write_text('#include "fa2_kvcache_sm100.h"\n'
                   "int main(void) { Fa2Kv8AttnParams p = {0};\n"
                   "  if (fa2_kv8_attn_sm100_check(&p) != FA2_ERR_NULL) return 1;\n"
                   "  if (fa2_kvcache_sm100_params_size(3) != (int64_t)sizeof p) return 2;\n"
                   "  return fa2_kvcache_sm100_abi_version() == FA2_KVCACHE_ABI_VERSION ? 0 : 3; }\n")
    where = os.path.dirname(_kvlib.LIB_PATH)
    exe = str(tmp_path / "caller")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Wextra", "-Werror", "-I", os.path.dirname(HEADER), str(src), "-o", exe,
                    "-L", where, "-l:libfa2_kvcache_sm100.so", f"-Wl,-rpath,{where}"], check=True)
    assert subprocess.run([exe], timeout=120).returncode == 0


# ------------------------------------------------------------------------------------ host checks
def pack(layout, values):
    flat = []
    for name, _ in layout.fields:
        v = values[name]
        flat += list(v) if isinstance(v, (tuple, list)) else [v]
    return layout.pack(*flat)


CACHE = dict(k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, k_stride=(8192, 128, 4096), v_stride=(8192, 128, 4096),
             ks_stride=(64, 1, 32), vs_stride=(64, 1, 32), num_pages=10, page_size=32, heads_kv=2, head_dim=128)
TABLE = dict(block_table=0x50000, cu_seqlens=0, err_flag=0, block_table_stride=5, pages_per_seq=5, batch=3, dtype=1)


def append(**kw):
    return pack(_kvlib.APPEND, {**CACHE, **TABLE, "k_in": 0x100, "v_in": 0x200, "k_in_stride": (256, 128, 256, 1),
                                "v_in_stride": (256, 128, 256, 1), "cache_seqlens": 0x60000, "seqlen": 1, **kw})


def read(**kw):
    return pack(_kvlib.READ, {**CACHE, **TABLE, "cu_seqlens": 0x600, "k_out": 0x100, "v_out": 0x200, "total": 100, **kw})


def attn(**kw):
    return pack(_kvlib.ATTN, {**CACHE, **TABLE, "q": 0x100, "o": 0x200, "q_stride": (1024, 128, 128, 1),
                              "o_stride": (1024, 128, 128, 1), "cache_seqlens": 0x60000, "cu_seqlens_q": 0, "workspace": 0x1000,
                              "workspace_bytes": 1 << 40, "timeout_cycles": 0, "heads_q": 8, "seqlen_q": 1, "total_q": 0,
                              "max_seqlen_k": 160, "causal": 1, "causal_align": 1, "num_splits": 0, "qk_scale": 0.1,
                              "reserved": 0, **kw})


def rotation(**kw):
    return pack(_kvlib.ROTARY, {**dict(q=0x100, k=0x200, q_out=0x300, k_out=0x400, q_stride=(1, 1, 1, 1), k_stride=(1, 1, 1, 1),
                                       q_out_stride=(1, 1, 1, 1), k_out_stride=(1, 1, 1, 1), positions=0x500, pos_stride=(0, 1),
                                       inv_freq=0x600, pos_is_64=0, batch=1, seqlen=4, heads_q=8, heads_kv=2, head_dim=80,
                                       rotary_dim=64, dtype=1, interleaved=0, inverse=0, magnitude=1.0, reserved=0), **kw})


BAD_CACHE = [
    (dict(k_scale=0), _lib.FA2_ERR_NULL),
    (dict(num_pages=0), _lib.FA2_ERR_SHAPE),
    (dict(heads_kv=0), _lib.FA2_ERR_SHAPE),
    (dict(heads_kv=-1), _lib.FA2_ERR_SHAPE),
    (dict(page_size=0), _lib.FA2_ERR_SHAPE),
    (dict(page_size=48), _lib.FA2_ERR_SHAPE),
    (dict(page_size=192), _lib.FA2_ERR_SHAPE),
    (dict(head_dim=96), _lib.FA2_ERR_HEAD_DIM),
    (dict(k=0x10008), _lib.FA2_ERR_LAYOUT),               # codes start on 16 bytes
    (dict(v_scale=0x40002), _lib.FA2_ERR_LAYOUT),
    (dict(v_stride=(8192, 136, 4096)), _lib.FA2_ERR_LAYOUT),
    (dict(k_stride=(-8192, 128, 4096)), _lib.FA2_ERR_LAYOUT),
    (dict(k_stride=(8192, 1 << 31, 4096)), _lib.FA2_ERR_LAYOUT),
    (dict(block_table=0), _lib.FA2_ERR_NULL),
    (dict(batch=0), _lib.FA2_ERR_SHAPE),
    (dict(pages_per_seq=0), _lib.FA2_ERR_SHAPE),
    (dict(dtype=2), _lib.FA2_ERR_DTYPE),
]


@pytest.mark.parametrize("kw,status", BAD_CACHE)
def test_every_cache_operator_refuses(kw, status):
    L = _kvlib.lib()
    for entry, packed in ((L.fa2_kv8_append_sm100, append(**kw)), (L.fa2_kv8_read_sm100, read(**kw)), (L.fa2_kv8_attn_sm100, attn(**kw))):
        assert getattr(L, entry.__name__ + "_check")(packed) == status
        assert entry(packed, None) == status  # before any CUDA call
    assert L.fa2_kv8_attn_sm100_workspace_bytes(attn(**kw)) == -1


@pytest.mark.parametrize("make,check,kw,status", [
    (append, "fa2_kv8_append_sm100_check", dict(), _lib.FA2_OK),
    (append, "fa2_kv8_append_sm100_check", dict(seqlen=0), _lib.FA2_OK),
    (append, "fa2_kv8_append_sm100_check", dict(num_pages=1, k_stride=(3, 128, 4096)), _lib.FA2_OK),  # never used
    (append, "fa2_kv8_append_sm100_check", dict(k_in=0), _lib.FA2_ERR_NULL),
    (append, "fa2_kv8_append_sm100_check", dict(cache_seqlens=0), _lib.FA2_ERR_NULL),
    (append, "fa2_kv8_append_sm100_check", dict(seqlen=-1), _lib.FA2_ERR_SHAPE),
    (append, "fa2_kv8_append_sm100_check", dict(seqlen=1 << 29), _lib.FA2_ERR_SHAPE),  # rows beyond 31 bits
    (read, "fa2_kv8_read_sm100_check", dict(), _lib.FA2_OK),
    (read, "fa2_kv8_read_sm100_check", dict(cu_seqlens=0), _lib.FA2_ERR_NULL),
    (read, "fa2_kv8_read_sm100_check", dict(total=-1), _lib.FA2_ERR_SHAPE),
    (read, "fa2_kv8_read_sm100_check", dict(total=1 << 30), _lib.FA2_ERR_SHAPE),
    (read, "fa2_kv8_read_sm100_check", dict(k_out=0x108), _lib.FA2_ERR_LAYOUT),
    (attn, "fa2_kv8_attn_sm100_check", dict(), _lib.FA2_OK),
    (attn, "fa2_kv8_attn_sm100_check", dict(o=0), _lib.FA2_ERR_NULL),
    (attn, "fa2_kv8_attn_sm100_check", dict(heads_q=7), _lib.FA2_ERR_GQA),
    (attn, "fa2_kv8_attn_sm100_check", dict(heads_q=0), _lib.FA2_ERR_SHAPE),
    (attn, "fa2_kv8_attn_sm100_check", dict(seqlen_q=-1), _lib.FA2_ERR_SHAPE),
    (attn, "fa2_kv8_attn_sm100_check", dict(cu_seqlens_q=0x10, total_q=-1), _lib.FA2_ERR_SHAPE),
    (attn, "fa2_kv8_attn_sm100_check", dict(causal_align=2), _lib.FA2_ERR_SHAPE),
    (attn, "fa2_kv8_attn_sm100_check", dict(causal_align=2, causal=0), _lib.FA2_OK),
    (attn, "fa2_kv8_attn_sm100_check", dict(num_splits=257), _lib.FA2_ERR_SHAPE),
    (attn, "fa2_kv8_attn_sm100_check", dict(num_splits=-1), _lib.FA2_ERR_SHAPE),
    (attn, "fa2_kv8_attn_sm100_check", dict(qk_scale=0.0), _lib.FA2_ERR_SCALE),
    (attn, "fa2_kv8_attn_sm100_check", dict(qk_scale=float("nan")), _lib.FA2_ERR_SCALE),
    (attn, "fa2_kv8_attn_sm100_check", dict(q=0x108), _lib.FA2_ERR_LAYOUT),
    (attn, "fa2_kv8_attn_sm100_check", dict(o_stride=(1024, 131, 128, 1)), _lib.FA2_ERR_LAYOUT),
    (attn, "fa2_kv8_attn_sm100_check", dict(q_stride=(1024, 128, 128, 2)), _lib.FA2_ERR_LAYOUT),
    (attn, "fa2_kv8_attn_sm100_check", dict(seqlen_q=1 << 20, max_seqlen_k=1 << 30), _lib.FA2_ERR_SHAPE),  # the line of tiles
    (attn, "fa2_kv8_attn_sm100_check", dict(workspace=0), _lib.FA2_ERR_WORKSPACE),
    (attn, "fa2_kv8_attn_sm100_check", dict(workspace_bytes=16), _lib.FA2_ERR_WORKSPACE),
    (rotation, "fa2_rotary_sm100_check", dict(), _lib.FA2_OK),
    (rotation, "fa2_rotary_sm100_check", dict(k=0, k_out=0, heads_kv=0), _lib.FA2_OK),
    (rotation, "fa2_rotary_sm100_check", dict(k=0), _lib.FA2_ERR_NULL),
    (rotation, "fa2_rotary_sm100_check", dict(inv_freq=0), _lib.FA2_ERR_NULL),
    (rotation, "fa2_rotary_sm100_check", dict(seqlen=0), _lib.FA2_ERR_SHAPE),
    (rotation, "fa2_rotary_sm100_check", dict(rotary_dim=63), _lib.FA2_ERR_HEAD_DIM),
    (rotation, "fa2_rotary_sm100_check", dict(rotary_dim=82), _lib.FA2_ERR_HEAD_DIM),
    (rotation, "fa2_rotary_sm100_check", dict(dtype=2), _lib.FA2_ERR_DTYPE),
    (rotation, "fa2_rotary_sm100_check", dict(magnitude=0.0), _lib.FA2_ERR_SCALE),
])
def test_check_statuses(make, check, kw, status):
    assert getattr(_kvlib.lib(), check)(make(**kw)) == status


def test_workspace_follows_the_sizes():
    size = lambda **kw: _kvlib.lib().fa2_kv8_attn_sm100_workspace_bytes(attn(**kw))  # noqa: E731
    assert size(workspace=0, workspace_bytes=0) == size() > 0 and size() % 16 == 0
    # No more CTAs than 128-key tiles: 160 keys have two.
    assert size(num_splits=5) == size(num_splits=2) > size(num_splits=1)
    assert size(num_splits=5, max_seqlen_k=2048) > size(num_splits=2, max_seqlen_k=2048) == size(num_splits=2)
    # Its size is bounded by the GPU's, not by the batch: two partial results for each CTA.
    assert size(batch=4096, seqlen_q=1, max_seqlen_k=160) <= 2 * 148 * 3 * (8 * (128 * 4 + 4) + 32)
    assert size(batch=4096, seqlen_q=512, max_seqlen_k=160) <= 2 * 148 * (256 * (128 * 4 + 4) + 32)


# ------------------------------------------------------------------------------------ Python
def arguments(D=64, H_kv=2, B=2, N=1, pages=4, page_size=32, dtype=torch.bfloat16):
    cache = alloc_kvcache_fp8(pages, page_size, H_kv, D, "cpu")
    q, k = torch.zeros(B, 2 * H_kv, N, D, dtype=dtype), torch.zeros(B, H_kv, N, D, dtype=dtype)
    table = torch.zeros(B, 2, dtype=torch.int32)
    return cache, q, k, table, torch.ones(B, dtype=torch.int32)


def test_alloc_layout():
    cache = alloc_kvcache_fp8(3, 16, 5, 32, "cpu")
    assert cache.k.shape == cache.v.shape == (3, 16, 5, 32) and cache.k.dtype == torch.float8_e4m3fn
    assert cache.k_scale.shape == (3, 16, 5) and cache.k_scale.dtype == torch.float32
    assert cache.k.stride() == (16 * 5 * 32, 32, 16 * 32, 1)  # a head's rows are adjacent
    assert all((t.float() == 0).all() for t in cache)


def test_no_cpu_path():
    cache, q, k, table, lens = arguments()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    freq, _ = rotary_inv_freq(64)
    for call in (lambda: attention_kvcache_fp8(q, cache, table, lens), lambda: kvcache_append_fp8(k, k, cache, table, lens),
                 lambda: kvcache_read_fp8(cache, table, cu, 2), lambda: rotary(q, k, torch.zeros(1, dtype=torch.int64), freq)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_append_and_read_refuse():
    cache, q, k, table, lens = arguments()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    for bad in (lambda: kvcache_append_fp8(k, k[..., :32], cache, table, lens),            # shapes differ
                lambda: kvcache_append_fp8(k.float(), k.float(), cache, table, lens),
                lambda: kvcache_append_fp8(k, k.half(), cache, table, lens),
                lambda: kvcache_append_fp8(q, q, cache, table, lens),                       # not the cache's heads
                lambda: kvcache_append_fp8(k[:, :, 0], k[:, :, 0], cache, table, lens),     # packed without sums
                lambda: kvcache_append_fp8(k[:1], k[:1], cache, table, lens),               # not the table's batch
                lambda: kvcache_append_fp8(k, k, cache, table, lens.long()),
                lambda: kvcache_append_fp8(k, k, cache, table.long(), lens),
                lambda: kvcache_append_fp8(k, k, cache, table[0], lens),
                lambda: kvcache_append_fp8(k[:, :, 0], k[:, :, 0], cache, table, lens, cu_seqlens=cu[:2]),
                lambda: kvcache_append_fp8(k, k, cache[:3], table, lens),
                lambda: kvcache_append_fp8(k, k, (cache.k.view(torch.uint8), *cache[1:]), table, lens),
                lambda: kvcache_append_fp8(k, k, (*cache[:2], cache.k_scale.double(), cache.v_scale), table, lens),
                lambda: kvcache_append_fp8(k, k, (*cache[:3], cache.v_scale[:3]), table, lens),
                lambda: kvcache_read_fp8(cache, table, cu[:2], 2),
                lambda: kvcache_read_fp8(cache, table, cu, -1),
                lambda: kvcache_read_fp8(cache, table, cu, 2, dtype=torch.float32)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(_lib.Fa2Error):  # rows of codes that are not adjacent values
        turned = torch.zeros(4, 32, 64, 2, dtype=torch.uint8).view(torch.float8_e4m3fn).transpose(2, 3)
        kvcache_append_fp8(k, k, (turned, turned, cache.k_scale, cache.v_scale), table, lens)


@pytest.mark.parametrize("D,page_size", [(96, 32), (64, 24), (64, 192), (256, 32), (8, 32)])
def test_caches_of_other_sizes_are_refused(D, page_size):
    cache, q, k, table, lens = arguments(D=D, page_size=page_size)
    with pytest.raises(AssertionError):
        attention_kvcache_fp8(q, cache, table, lens)


def test_attention_refuses():
    cache, q, k, table, lens = arguments()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    for bad in (lambda: attention_kvcache_fp8(q[..., :32], cache, table, lens),
                lambda: attention_kvcache_fp8(q.float(), cache, table, lens),
                lambda: attention_kvcache_fp8(q[:, :3], cache, table, lens),                # 3 heads over 2
                lambda: attention_kvcache_fp8(q[:1], cache, table, lens),
                lambda: attention_kvcache_fp8(q, cache, table, lens, causal_align="left"),
                lambda: attention_kvcache_fp8(q[:, :, 0], cache, table, lens),              # packed without sums
                lambda: attention_kvcache_fp8(q[:, :, 0], cache, table, lens, cu_seqlens_q=cu),  # or the longest
                lambda: attention_kvcache_fp8(q, cache, table, lens[:1])):
        with pytest.raises(AssertionError):
            bad()


def test_rotary_refuses():
    cache, q, k, _, _ = arguments()
    freq, _ = rotary_inv_freq(64)
    pos = torch.zeros(2, 1, dtype=torch.int64)
    for bad in (lambda: rotary(q[0, 0], None, pos, freq), lambda: rotary(q.float(), None, pos, freq),
                lambda: rotary(q, k.half(), pos, freq), lambda: rotary(q, k[..., :32], pos, freq),
                lambda: rotary(q, k, pos[:1], freq), lambda: rotary(q, k, pos.float(), freq),
                lambda: rotary(q, k, pos, freq.float()), lambda: rotary(q, k, pos, rotary_inv_freq(66)[0]),
                lambda: rotary(q, k, pos, freq[:0])):
        with pytest.raises(AssertionError):
            bad()
    for magnitude in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            rotary(q, k, pos, freq, magnitude=magnitude)


def test_inv_freq():
    f, m = rotary_inv_freq(8)
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-12)
    assert torch.allclose(rotary_inv_freq(8, scaling="linear", factor=4.0)[0], f / 4, rtol=1e-12)
    ntk = rotary_inv_freq(8, scaling="ntk", factor=4.0)[0]
    assert ntk[0] == 1.0 and abs(ntk[3].item() * 4 / f[3].item() - 1) < 1e-12
    long, base = rotary_inv_freq(128, scaling="yarn", factor=8.0, original_max_position=4096)[0], rotary_inv_freq(128)[0]
    turns = 4096 * base / (2 * torch.pi)
    assert torch.equal(long[turns > 40], base[turns > 40])  # fast pairs as they are, slow ones stretched
    assert torch.allclose(long[turns < 0.8], base[turns < 0.8] / 8, rtol=1e-12)
    assert (long <= base).all() and (long >= base / 8 * (1 - 1e-12)).all()
    assert abs(rotary_inv_freq(128, scaling="yarn", factor=8.0)[1] - 1.2079441541679836) < 1e-12
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="cubic"), dict(rotary_dim=8, base=1.0),
                dict(rotary_dim=8, factor=0.5)):
        with pytest.raises(ValueError):
            rotary_inv_freq(**bad)


def test_cache_is_any_sequence_of_four():
    cache, q, k, table, lens = arguments()
    assert isinstance(cache, KVCacheFP8)
    with pytest.raises(RuntimeError, match="no CPU path"):  # past the checks of the arguments
        attention_kvcache_fp8(q, list(cache), table, lens)
