"""Attention over a cache in 8 bits where keys, values and queries are near the ends of their types: what 64 bits give, as far as it
is a number of bf16.  Tolerances are those of tests/test_kv8_gpu.py: bounds relative to sum w |v|, which powers of two do not
change."""
import math

import pytest
import torch

from mxllm.ops import kv8

from .test_kv8_gpu import HALF, _exact, _i32, _random_pages

pytestmark = pytest.mark.gpu


def _near(got, want, size):
    assert bool(got.isfinite().all())
    assert bool(((got.double().cpu() - want).abs() <= (HALF + 2.0 ** -11) * size + HALF * want.abs()).all())


# (whole rows of 8 and of 4 waves, cut rows, rows that share a workgroup)
LAYOUTS = [([2000] * 50, 4, 2), ([2000] * 70, 4, 2), ([20000, 1, 3000], 4, 2), ([5000, *range(0, 260, 2)], 2, 1)]


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("lens,Hq,Hkv", LAYOUTS)
def test_sums_of_the_largest_values(gpu, D, lens, Hq, Hkv):
    """Many keys of like weight, values of one sign up to 448 * 2 ** 112: their sum is past f32, their mean is not."""
    p = _random_pages(gpu, lens, Hkv, 256, D)
    there = p.v_exp < 200
    p.v_exp.copy_(torch.where(there, p.v_exp + 119, p.v_exp))  # 118 .. 120 -> 237 .. 239
    p.v_exp[0] = torch.where(there[0], p.v_exp[0] - 119, p.v_exp[0])  # some page among them as it was
    p.v.bitwise_and_(0x7F)
    q = (0.1 * torch.randn(len(lens), Hq, D, device=gpu, generator=torch.Generator(gpu).manual_seed(1))).bfloat16()
    pos = [n - 1 for n in lens]
    got = kv8.decode_attention(q, p, _i32(pos, gpu), None, max(lens)).view(len(lens), Hq, D)
    want, size = _exact(q, p, pos, list(range(len(lens))), max(lens), D ** -0.5)
    assert float(size.max()) * max(lens) > 2.0 ** 128
    _near(got, want, size)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("late", [False, True])
def test_large_values_first_or_last(gpu, D, late):
    """A wave that has small values behind it when the first large ones come, and the other way round; and rows of small ones
    alone, which stay as exact as they are."""
    lens, Hq, Hkv = [1000, 30000, 17, 900], 4, 2
    p = _random_pages(gpu, lens, Hkv, 256, D)
    for b in (0, 1):
        n = lens[b]
        pages = p.table[b, :-(-n // 256)].long()
        half = len(pages) // 2
        p.v_exp[pages[half:] if late else pages[:half]] += 100
    p.v_exp[p.table[3, :4].long()] -= 80
    q = (0.1 * torch.randn(4, Hq, D, device=gpu, generator=torch.Generator(gpu).manual_seed(1))).bfloat16()
    pos = [n - 1 for n in lens]
    got = kv8.decode_attention(q, p, _i32(pos, gpu), None, 30000).view(4, Hq, D)
    want, size = _exact(q, p, pos, [0, 1, 2, 3], 30000, D ** -0.5)
    _near(got, want, size)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("size", [2.0 ** 95, 2.0 ** 104, 2.0 ** 118, 2.0 ** 125])
@pytest.mark.parametrize("lens,Hq,Hkv", LAYOUTS[::2])
def test_large_queries(gpu, D, lens, Hq, Hkv, size):
    """Scores are of ordinary size by the keys' exponents, or by the scale; heads of ordinary and of large queries share keys."""
    p = _random_pages(gpu, lens, Hkv, 256, D)
    q = torch.randn(len(lens), Hq, D, device=gpu, generator=torch.Generator(gpu).manual_seed(1)).bfloat16()
    q[:, 0, 0] = 3
    q[:, -1] = 0
    pos = [n - 1 for n in lens]
    want, total = _exact(q, p, pos, list(range(len(lens))), max(lens), D ** -0.5)
    args = (_i32(pos, gpu), None, max(lens))
    if size < 2.0 ** 118:  # (scales under 2^-126 have fewer bits)
        by_scale = kv8.decode_attention(q * size, p, *args, D ** -0.5 / size).view(len(lens), Hq, D)
        _near(by_scale, want, total)
    down = int(math.log2(size))
    small = p._replace(k_exp=torch.where(p.k_exp < 200, p.k_exp - min(down, 110), p.k_exp))
    by_keys = kv8.decode_attention(q * size, small, *args, D ** -0.5 * 2.0 ** -max(down - 110, 0)).view(len(lens), Hq, D)
    _near(by_keys, want, total)
    mixed = q.clone()
    mixed[:, 0] *= size  # one of a group's heads
    got = kv8.decode_attention(mixed, p, *args).view(len(lens), Hq, D)
    assert bool(got.isfinite().all())
    _near(got[:, 1:], want[:, 1:], total[:, 1:])
