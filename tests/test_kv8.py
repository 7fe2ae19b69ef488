"""The key/value cache in 8 bits (mxllm/ops/kv8.py), on the CPU: its number format, what appending does to groups of positions, and
its refusals; the kernels are compared with it in tests/test_kv8_gpu.py."""
import itertools
import math

import pytest
import torch

from mxllm.ops import kv8
from mxllm.ops import reference as ref


def _pages(slots, per, pool, Hkv, block, D, seed=0, fill=True):
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(pool, generator=g)[:slots * per].to(torch.int32).view(slots, per)
    p = kv8.Pages.empty(pool, Hkv, block, D, table)
    if fill:  # what earlier owners of the pages left
        for t, hi in ((p.k, 256), (p.v, 256), (p.k_exp, 140), (p.v_exp, 140)):
            t.copy_(torch.randint(0, hi, t.shape, generator=g, dtype=torch.uint8))
    return p


def _rows(T, Hq, Hkv, D, seed=0):
    g = torch.Generator().manual_seed(seed + 77)
    x = torch.randn(T, Hq + 2 * Hkv, D, generator=g) * torch.exp(torch.randn(T, Hq + 2 * Hkv, 1, generator=g))
    return x.reshape(T, -1).bfloat16()


def _tables(n, D):
    return ref.rope_tables(n, D, 500000.0, None)


def test_exponents_are_the_least_that_fit():
    x = torch.tensor([0.0, 1e-45, 448.0, 448.00003, 224.0, 1.0, 1.75, 1.7500001, 3.3e38, 2.0 ** -126])
    e = kv8.exponents(x)
    top = 448.0 * torch.exp2(e.double() - 127)
    assert bool((top >= x.double()).all())
    assert bool(((top / 2 < x.double()) | (e == 1)).all()) and e.tolist()[:5] == [1, 1, 127, 128, 126]


def test_every_code_is_exact_in_bf16_and_comes_back():
    """A code's last bit is at least 2^-9, so a value's is 2^(e - 136); bf16's smallest number is 2^-133: exact from e = 3 on, below
    that off by up to half of it."""
    codes = torch.arange(256, dtype=torch.uint8)
    for e in (1, 3, 60, 127, 200, 247):
        v = kv8.decode(codes, torch.tensor(e))
        held = v[v.isfinite()]  # (f32 ends inside the last byte that amax can give)
        off = (held.bfloat16().double() - held.double()).abs().max()
        assert off <= (0 if e >= 3 else 2.0 ** -134) and v.isnan().sum() == 2
        if e > 10:
            back = kv8.encode(held, torch.tensor(e))
            assert torch.equal(back, codes[v.isfinite()])


def test_codes_are_nearest():
    x = torch.randn(4000)
    e = kv8.exponents(x.abs().amax())
    x = x.double()
    every = kv8.decode(torch.arange(256, dtype=torch.uint8), e).double()
    every = every[~every.isnan()]
    best = (every[:, None] - x).abs().amin(0)
    got = kv8.decode(kv8.encode(x, e), e).double()
    assert bool(((got - x).abs() <= best).all())


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("block,start,n", [(16, 0, 40), (48, 5, 33), (256, 250, 20), (32, 31, 1)])
def test_tokens_one_by_one_are_the_prompt(block, start, n, norm):
    """Exponents alike, values apart by no more than the roundings of a growing group: half a step of the
    smallest numbers each time its exponent grew, from what a first rounding gave."""
    Hq, Hkv, D, per = 4, 2, 32, 8
    w = (torch.rand(2, D) + 0.5).bfloat16() if norm else (None, None)
    cos, sin = _tables(start + n, D)
    qkv = _rows(n, Hq, Hkv, D)
    a, b = (_pages(3, max(1, -(-(start + n) // block)), 60, Hkv, block, D, seed=4) for _ in range(2))
    q, k, v = kv8.append_prompts(qkv, cos, sin, kv8.prompt_runs([start], [n], [1]), a, Hq, *w)
    for i in range(n):
        qi = kv8.append_tokens(qkv[i:i + 1], cos, sin, torch.tensor([start + i], dtype=torch.int32),
                               torch.tensor([1], dtype=torch.int32), b, Hq, *w)
        assert torch.equal(qi[0], q[:, i])
    assert torch.equal(a.k_exp, b.k_exp) and torch.equal(a.v_exp, b.v_exp)
    span = [torch.tensor([x], dtype=torch.int32) for x in (1, start, start + n)]
    for one, two, exps in zip(kv8.read(a, *span, n), kv8.read(b, *span, n), (a.k_exp, a.v_exp)):
        smallest = 2.0 ** (int(exps.max()) - 127 - 9)  # a step of the smallest numbers of the widest group
        assert float((one.double() - two.double()).abs().max()) <= 8 * smallest
    whole = kv8.read(a, *span, n)
    for got, want in zip(whole, (k, v)):  # e4m3 of what the prompt's attention has, which is rounded to bf16
        big = want.double().abs().amax((1, 2))
        err = (got[0].double() - want.double()).abs()
        assert bool((err <= (2.0 ** -4 + 2.0 ** -8) * want.double().abs() + 2.0 ** -9 * 2.0 ** -8 * 2 * big[:, None, None]).all())


def test_what_a_page_held_before_does_not_matter_to_a_new_group():
    Hq = Hkv = 1
    cos, sin = _tables(64, 32)
    qkv = _rows(20, Hq, Hkv, 32)
    out = []
    for seed in (1, 2):
        p = _pages(2, 2, 9, Hkv, 32, 32, seed=3)
        p.k.copy_(torch.randint(0, 256, p.k.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(seed)))
        p.k_exp.fill_(100 * seed)
        kv8.append_prompts(qkv, cos, sin, kv8.prompt_runs([0], [20], [0]), p, Hq)
        out.append(kv8.read(p, *(torch.tensor([x], dtype=torch.int32) for x in (0, 0, 20)), 24))
    assert all(torch.equal(a, b) for a, b in zip(*out)) and not out[0][0][:, :, 20:].any()


def test_rows_that_are_no_numbers():
    Hq, Hkv, D = 1, 1, 32
    cos, sin = _tables(4, D)
    qkv = _rows(2, Hq, Hkv, D)
    qkv[0, 2 * D] = float("inf")
    qkv[0, 2 * D + 1] = float("nan")
    qkv[0, 2 * D + 2] = 5.0
    qkv[0, 2 * D + 3:] = 0.5
    p = _pages(1, 1, 2, Hkv, 16, D)
    kv8.append_prompts(qkv[:1], cos, sin, kv8.prompt_runs([0], [1], [0]), p, Hq)
    _, v = kv8.read(p, *(torch.tensor([x], dtype=torch.int32) for x in (0, 0, 1)), 1)
    assert v[0, 0, 0, :2].isnan().all() and v[0, 0, 0, 2] == 5.0 and v[0, 0, 0, 3] == 0.5


def test_places_that_are_none():
    Hq, Hkv, D = 2, 1, 32
    cos, sin = _tables(100, D)
    p = _pages(2, 2, 6, Hkv, 16, D)
    p.table[1, 1] = 6
    before = [t.clone() for t in p[:4]]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    q = kv8.append_tokens(_rows(5, Hq, Hkv, D), cos, sin, i32(-1, 32, 3, 3, 17), i32(0, 0, -1, 2, 1), p, Hq)
    assert all(torch.equal(a, b) for a, b in zip(before, p[:4]))
    assert not q[:4].any() and q[4].any()  # the last has a place, but its page is none of the pool
    k, v = kv8.read(p, i32(1, 0, 5), i32(15, 30, 0), i32(18, 40, 5), 4)
    assert k[0, 0, 1].isnan().all() and not k[0, 0, 3].any() and not k[1, :, 2:].any() and not k[2].any()
    o = kv8.decode_attention(_rows(4, Hq, 0, D).view(4, Hq, D), p, i32(17, -1, 3, 3), i32(1, 0, -1, 2), 32)
    assert o[0].isnan().all() and not o[1:].any()


def test_refusals():
    Hq, Hkv, D = 2, 1, 32
    cos, sin = _tables(40, D)
    p = _pages(2, 2, 6, Hkv, 16, D)
    rows, i32 = _rows(2, Hq, Hkv, D), torch.tensor([0, 1], dtype=torch.int32)
    for bad in [dict(qkv=rows[:, 1:]), dict(pos=i32.long()), dict(pos=i32[:1]), dict(slots=i32.float()), dict(Hq=3), dict(cos=cos[:, :8]),
                dict(q_norm=torch.ones(D)), dict(pages=p._replace(k=p.k.float())), dict(pages=p._replace(k_exp=p.k_exp[:, :, :0])),
                dict(pages=p._replace(table=p.table.long())), dict(pages=p._replace(v=p.v[:5]))]:
        a = dict(qkv=rows, cos=cos, sin=sin, pos=i32, slots=i32, pages=p, Hq=Hq) | bad
        with pytest.raises((ValueError, RuntimeError)):
            kv8.append_tokens(**a)
    with pytest.raises(ValueError):
        kv8.append_prompts(rows, cos, sin, i32, p, Hq)
    with pytest.raises(ValueError):
        kv8.decode_attention(torch.zeros(2, 2, D), p, i32, i32, 0)
    with pytest.raises(ValueError):
        kv8.decode_attention(torch.zeros(2, 2, 64), p, i32, i32, 8)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            kv8.decode_attention(torch.zeros(2, 2, D), p, i32, i32, 8, scale)
    with pytest.raises(ValueError):
        kv8.Pages.empty(2, 1, 24, D, p.table)
    for starts, lens, slots in [([0], [1, 2], [0]), ([0, 4], [1, 2], [3, 3]), ([-1], [2], [0]), ([0], [-2], [0])]:
        with pytest.raises(ValueError):
            kv8.prompt_runs(starts, lens, slots)


def test_prompt_runs_cut_at_groups():
    runs = kv8.prompt_runs([0, 30, 7], [17, 3, 0], [2, 0, 1]).tolist()
    assert runs == [[0, 16, 2, 0], [16, 1, 2, 16], [17, 2, 0, 30], [19, 1, 0, 32]]
    assert kv8.prompt_runs([], [], []).shape == (0, 4)


def test_decode_attention_reads_what_was_appended():
    Hq, Hkv, D, n = 4, 2, 32, 50
    cos, sin = _tables(n, D)
    p = _pages(2, 4, 9, Hkv, 16, D)
    kv8.append_prompts(_rows(n, Hq, Hkv, D), cos, sin, kv8.prompt_runs([0], [n], [1]), p, Hq)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    k, v = (x[0].double() for x in kv8.read(p, i32(1), i32(0), i32(n), n))
    q = torch.randn(1, Hq, D).bfloat16()
    for pos, bound in itertools.product((0, 15, 16, n - 1), (1, 17, 1000)):
        m = min(pos + 1, bound)
        s = q[0].double().view(Hkv, 2, D) @ k[:, :m].transpose(1, 2) / math.sqrt(D)
        want = (torch.softmax(s, -1) @ v[:, :m]).reshape(1, -1)
        got = kv8.decode_attention(q, p, i32(pos), i32(1), bound).double()
        assert float((got - want).abs().max()) <= 2.0 ** -8 * float(v.abs().max())
