"""CPU tests of fa2.rotary's host side: which tensors a rotation in place refuses, and the frequencies."""

import random

import pytest
import torch

from fa2.rotary import _share_memory, rotary, rotary_inv_freq


def addresses(t):
    at = torch.full(t.shape, t.storage_offset(), dtype=torch.int64)
    for d, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s).view([-1 if i == d else 1 for i in range(t.dim())])
    return at.flatten()


def test_share_memory_against_every_address():
    """Random sizes and strides, nested and not, against the addresses written out."""
    rng = random.Random(1)
    store, seen = torch.zeros(4000), set()
    for _ in range(3000):
        made = []
        for _ in range(2):
            shape = [rng.choice([1, 1, 2, 3, 5]) for _ in range(4)]
            stride = [rng.choice([0, 1, 1, 2, 3, 5, 8, 15, 16, 40, 64, 120]) for _ in range(4)]
            if rng.random() < 0.5:  # a dense order of the dimensions, now and then with gaps
                step = 1
                for d in rng.sample(range(4), 4):
                    stride[d], step = step, step * shape[d] + rng.choice([0, 0, 7])
            made.append(store.as_strided(shape, stride, rng.randrange(300)))
        a, b = made
        dims = [tuple(zip(t.shape, t.stride())) for t in made]
        for t, d in zip(made, dims):
            want = addresses(t).unique().numel() < t.numel()
            assert _share_memory(d) == want
            seen.add(("one", want))
        want = bool(torch.isin(addresses(a), addresses(b)).any())
        assert _share_memory(dims[0], dims[1], b.storage_offset() - a.storage_offset()) == want
        seen.add(("two", want))
    assert len(seen) == 4


def test_rotation_in_place_refuses_shared_values():
    freq, _ = rotary_inv_freq(64)
    pos = torch.arange(6)
    qkv = torch.zeros(2, 6, 3, 4, 64, dtype=torch.float16)
    x = qkv[:, :, 0].transpose(1, 2)
    flat = torch.zeros(2000, dtype=torch.float16)
    packed = torch.zeros(6, 12, 64, dtype=torch.float16)
    bad = [(x, x), (x, x[:, 1:3]), (x, qkv.view(2, 6, 12, 64)[:, :, 3:5].transpose(1, 2)), (x[:, :1].expand(2, 4, 6, 64), None),
           (flat.as_strided((1, 4, 6, 64), (0, 64, 64, 1)), None), (packed[:, :8], packed[:, 7:]),
           (flat.as_strided((1, 2, 6, 64), (0, 384, 64, 1)), flat.as_strided((1, 2, 6, 64), (0, 384, 64, 1), 700))]
    for q, k in bad:
        with pytest.raises(ValueError, match="share memory"):
            rotary(q, k, pos, freq, inplace=True)
    good = [(x, qkv[:, :, 1].transpose(1, 2)), (x, None), (packed[:, :8], packed[:, 8:]), (x.clone(), x),
            (qkv[:, :, 0, :3].transpose(1, 2), qkv[:, :, 0, 3:].transpose(1, 2)), (qkv[:1, :, 0].transpose(1, 2), qkv[1:, :, 0].transpose(1, 2))]
    for q, k in good:
        with pytest.raises(RuntimeError, match="no CPU path"):  # past the check
            rotary(q, k, pos, freq, inplace=True)
    with pytest.raises(RuntimeError, match="no CPU path"):  # into new tensors: inputs may share
        rotary(x, x, pos, freq)


@pytest.mark.parametrize("base,original,rd,low,high", [
    (10000.0, 65536, 128, 40, 65),    # the slowest pair still turns 1.2 times: the ramp ends behind it
    (10000.0, 131072, 64, 22, 35),
    (10000.0, 4096, 128, 20, 46),     # the ramp ends at pair 45.03, before the last one
    (500000.0, 8192, 128, 18, 35),
    (10.0, 10 ** 9, 8, 7, 7),         # every pair turns often: nothing is stretched
])
def test_yarn_ramp(base, original, rd, low, high):
    """The ramp's ends, worked out by hand as rd ln(original / (2 pi turns)) / (2 ln base), rounded down for 32
    turns and up for one, and kept within [0, rd - 1]; between them a linear share of f / factor."""
    factor = 8.0
    f = rotary_inv_freq(rd, base=base)[0]
    got, _ = rotary_inv_freq(rd, base=base, scaling="yarn", factor=factor, original_max_position=original)
    for i in range(rd // 2):
        share = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
        want = f[i].item() * (1 - share) + f[i].item() / factor * share
        assert abs(got[i].item() - want) <= 1e-12 * want
    turns = original * f / (2 * torch.pi)
    assert (got[turns > 1.001] > f[turns > 1.001] / factor * (1 + 1e-9)).all()  # none of these is stretched all the way
