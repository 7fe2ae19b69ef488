"""The kernels of the key/value cache in 8 bits (csrc/kernels/kv8.hip, kv8_attn.hip): the cache bit for bit what the plain form on the
CPU makes of the same rows (both form keys in 64 bits), attention against 64 bits over the values that the cache holds.

Tolerances.  Queries: a rounding to bf16 (2^-8 of the value) and f32 in between (2^-19 of the summands, 16 of its roundings).
Attention: a weight is rounded to bf16 once, 2^-8 of it, so an output is off by 2^-8 of sum w |v|, and as much of itself
by its own rounding; scores of up to 128 products in f32, of summands that together are below 2^4, leave 2^-24 * 128 * 2^4 =
2^-13 of a weight, and f32 sums less: 2^-11 of sum w |v| for both."""
import math

import pytest
import torch

from mxllm import ops
from mxllm.ops import kv8
from mxllm.ops import reference as ref

from .test_kv8 import _pages, _rows, _tables

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8
HEADS = [(32, 8, 2), (64, 4, 4), (128, 16, 1), (128, 6, 2), (64, 32, 8)]


def _i32(x, dev="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _to(pages, dev):
    return kv8.Pages(*(t.to(dev) for t in pages))


def _same(a, b):
    """The same bytes; of the codes 0x7f and 0xff, both of which are NaN, either (a conversion's NaN has no meaning in its sign)."""
    def bits(i, t):
        t = t.cpu()
        return torch.where(t == 0xFF, 0x7F, t) if i < 2 else t

    return all(torch.equal(bits(i, x), bits(i, y)) for i, (x, y) in enumerate(zip(a, b)))


def _near_rows(got, want, qkv, cos):
    """bf16 queries or keys, and the plain form's."""
    want = want.double()
    assert bool(((got.double().cpu() - want).abs() <= 2 * HALF * want.abs() + 2.0 ** -19 * 2 * float(want.abs().max())).all())


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("block", [16, 48, 256])
@pytest.mark.parametrize("D,Hq,Hkv", HEADS)
def test_tokens(gpu, D, Hq, Hkv, block, norm):
    """Rows at the edges of groups and pages, two of one group, three of one position, and rows without a place."""
    pos = [0, 15, 16, 17, 33, 47, 48, 255, 256, 90, 91, 90, 90, 5, -1, 600, 3]
    slots = [3, 1, 0, 2, 4, 5, 6, 7, 8, 9, 9, 9, 9, 10, 1, 2, 12]
    cos, sin = _tables(300, D)
    per = -(-300 // block)
    cpu = _pages(12, per, 12 * per + 3, Hkv, block, D, seed=D + block)
    dev = _to(cpu, gpu)
    w = [(torch.rand(D) + 0.5).bfloat16() for _ in range(2)] if norm else [None, None]
    qkv = _rows(len(pos), Hq, Hkv, D)
    for i in range(2):  # the second time over what the first one left
        want = kv8.append_tokens(qkv, cos, sin, _i32(pos), _i32(slots), cpu, Hq, *w)
        got = kv8.append_tokens(qkv.to(gpu), cos.to(gpu), sin.to(gpu), _i32(pos, gpu), _i32(slots, gpu), dev, Hq,
                                *(t.to(gpu) if t is not None else None for t in w))
        assert _same(cpu, dev) and not got[14:].any()
        _near_rows(got, want, qkv, cos)
        qkv = (qkv.float() * 5).bfloat16()


def test_many_tokens_share_a_group_across_chunks_of_rows(gpu):
    """150 rows, the positions of one group spread over them: the first of them writes the group."""
    D, Hq, Hkv, n = 64, 2, 2, 150
    cos, sin = _tables(32, D)
    slots = [i % 149 for i in range(n)]
    pos = [3] * n
    for i, p in ((70, 1), (149, 2), (10, 0), (5, 4)):
        slots[i], pos[i] = 5, p
    cpu = _pages(150, 1, 150, Hkv, 32, D)
    dev = _to(cpu, gpu)
    qkv = _rows(n, Hq, Hkv, D)
    kv8.append_tokens(qkv, cos, sin, _i32(pos), _i32(slots), cpu, Hq)
    kv8.append_tokens(qkv.to(gpu), cos.to(gpu), sin.to(gpu), _i32(pos, gpu), _i32(slots, gpu), dev, Hq)
    assert _same(cpu, dev)


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("block,starts,lens", [(256, [0], [1]), (16, [0, 0, 0], [17, 1, 40]), (48, [5, 0, 31], [11, 100, 33]),
                                               (256, [250, 1003], [20, 300])])
@pytest.mark.parametrize("D,Hq,Hkv", HEADS)
def test_prompts(gpu, D, Hq, Hkv, block, starts, lens, norm):
    top = max(a + n for a, n in zip(starts, lens))
    cos, sin = _tables(top, D)
    per, slots = -(-top // block), [4, 0, 2][:len(lens)]
    cpu = _pages(5, per, 5 * per + 2, Hkv, block, D, seed=D)
    dev = _to(cpu, gpu)
    w = [(torch.rand(D) + 0.5).bfloat16() for _ in range(2)] if norm else [None, None]
    qkv = _rows(sum(lens), Hq, Hkv, D)
    runs = kv8.prompt_runs(starts, lens, slots)
    want = kv8.append_prompts(qkv, cos, sin, runs, cpu, Hq, *w)
    wide = torch.full((sum(lens), qkv.shape[1] + 8), float("nan"), device=gpu, dtype=torch.bfloat16)
    wide[:, :-8] = qkv.to(gpu)
    got = kv8.append_prompts(wide[:, :-8], cos.to(gpu), sin.to(gpu), runs.to(gpu), dev, Hq,
                             *(t.to(gpu) if t is not None else None for t in w))
    assert _same(cpu, dev)
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[2].cpu(), want[2])
    _near_rows(got[0], want[0], qkv, cos)
    args = (_i32(slots), _i32([max(0, a - 9) for a in starts]), _i32([a + n for a, n in zip(starts, lens)]))
    a, b = kv8.read(cpu, *args, max(lens) + 20), kv8.read(dev, *(t.to(gpu) for t in args), max(lens) + 20)
    assert all(torch.equal(x.view(torch.int16), y.cpu().view(torch.int16)) | bool(x.isnan().any()) for x, y in zip(a, b))
    assert all(torch.equal(torch.nan_to_num(x, 7.0), torch.nan_to_num(y.cpu(), 7.0)) for x, y in zip(a, b))


def test_runs_without_a_place_are_left_out(gpu):
    D, Hq, Hkv = 32, 2, 1
    cos, sin = _tables(64, D)
    cpu = _pages(3, 2, 8, Hkv, 32, D)
    cpu.table[1, 0] = -1
    dev = _to(cpu, gpu)
    runs = _i32([[0, 3, 0, 0], [3, 2, 3, 0], [5, 17, 0, 16], [5, 2, 0, 15], [-1, 2, 2, 0], [38, 3, 2, 0], [7, 0, 2, 0],
                 [8, 4, 2, 61], [8, 4, 1, 0], [12, 3, 2, -2], [20, 5, 2, 40]])
    qkv = _rows(40, Hq, Hkv, D)
    want = kv8.append_prompts(qkv, cos, sin, runs, cpu, Hq)
    got = kv8.append_prompts(qkv.to(gpu), cos.to(gpu), sin.to(gpu), runs.to(gpu), dev, Hq)
    assert _same(cpu, dev)
    for t in (0, 1, 2, 8, 9, 10, 11, 20, 24):
        assert torch.equal(got[1][:, t].cpu(), want[1][:, t])


def test_no_numbers_and_extremes_reach_the_cache_alike(gpu):
    D, Hq, Hkv = 64, 1, 1
    cos, sin = _tables(8, D)
    qkv = _rows(8, Hq, Hkv, D)
    qkv[1, D + 3], qkv[1, 2 * D] = float("nan"), float("inf")
    qkv[2, 2 * D:] = 1e-38
    qkv[3] = 0
    qkv[4, 2 * D] = 3.3e38
    qkv[5, D:] = float("-inf")
    qkv[6, D:] = 448.0
    for order in (range(8), [3, 2, 6, 0, 4, 7, 1, 5]):
        cpu = _pages(1, 1, 1, Hkv, 16, D)
        dev = _to(cpu, gpu)
        for i, t in enumerate(order):
            kv8.append_tokens(qkv[t:t + 1], cos, sin, _i32([i]), _i32([0]), cpu, Hq)
            kv8.append_tokens(qkv[t:t + 1].to(gpu), cos.to(gpu), sin.to(gpu), _i32([i], gpu), _i32([0], gpu), dev, Hq)
            a, b = (kv8.read(p, *(_i32([x], p.k.device) for x in (0, 0, 8)), 8) for p in (cpu, dev))
            for x, y in zip(a, b):
                assert torch.equal(x.isnan(), y.cpu().isnan()) and torch.equal(torch.nan_to_num(x), torch.nan_to_num(y.cpu()))


# ---------------------------------------------------------------------------------------------------- attention
def _random_pages(dev, lens, Hkv, block, D, seed=0, extra=3):
    """A pool dealt out in no order: codes of all kinds in the rows that are there, NaN and wide exponents elsewhere."""
    g = torch.Generator(dev).manual_seed(seed)
    need = [max(1, -(-n // block)) for n in lens]
    pool = sum(need) + extra
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), pool + 5, dtype=torch.int32, device=dev)
    p = kv8.Pages.empty(pool, Hkv, block, D, table)
    for t in (p.k, p.v):
        t.fill_(0x7F)  # NaN
    p.k_exp.fill_(255)
    p.v_exp.fill_(255)
    at = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]]
        for j in range(need[b]):
            page, m = int(order[at + j]), min(block, n - j * block)
            for codes, exps in ((p.k, p.k_exp), (p.v, p.v_exp)):
                e = torch.randint(118, 121, (Hkv, block // 16), generator=g, device=dev)
                c = kv8.encode(torch.randn(Hkv, block, D, generator=g, device=dev).mul_(90).clamp_(-448, 448),
                               torch.tensor(127, device=dev))
                codes[page, :, :m] = c[:, :m]
                exps[page, :, :-(-m // 16)] = e[:, :-(-m // 16)].to(torch.uint8)
        at += need[b]
    return p


def _exact(q, p, pos, slots, bound, scale):
    """f64 outputs [B, Hq, D], and sum of w |v|."""
    B, Hq, D = q.shape
    Hkv, block = p.k.shape[1], p.k.shape[2]
    out, size = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
    for b in range(B):
        n = min(pos[b] + 1, bound)
        if n <= 0:
            continue
        pages = p.table[slots[b], :-(-n // block)].long()

        def whole(codes, exps):
            x = kv8.decode(codes[pages], exps[pages].repeat_interleave(16, 2)[..., None]).double()
            return x.transpose(0, 1).reshape(Hkv, -1, D)[:, :n]

        k, v = whole(p.k, p.k_exp), whole(p.v, p.v_exp)
        w = torch.softmax((q[b].double().view(Hkv, -1, D) @ k.transpose(1, 2).contiguous()) * scale, -1)
        out[b], size[b] = (w @ v).reshape(Hq, D).cpu(), (w @ v.abs()).reshape(Hq, D).cpu()
    return out, size


def _check_attention(dev, lens, Hq, Hkv, block, D, seed=0, bound=None, order=None, scale=None):
    p = _random_pages(dev, lens, Hkv, block, D, seed)
    order = list(range(len(lens))) if order is None else order
    q = torch.randn(len(order), Hq, D, device=dev, generator=torch.Generator(dev).manual_seed(seed + 1)).bfloat16()
    pos = [lens[s] - 1 for s in order]
    bound = bound or max(max(lens), 1)
    got = kv8.decode_attention(q, p, _i32(pos, dev), _i32(order, dev), bound, scale).view(len(order), Hq, D)
    want, size = _exact(q, p, pos, order, bound, scale or D ** -0.5)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= (HALF + 2.0 ** -11) * size + HALF * want.abs()).all()), float((err / (size + 1e-30)).max())
    return p, q, got


@pytest.mark.parametrize("block", [16, 48, 256])
@pytest.mark.parametrize("D,Hq,Hkv", HEADS)
def test_attention_of_short_rows(gpu, D, Hq, Hkv, block):
    _check_attention(gpu, [0, 1, 15, 16, 17, 31, 33, 63, 65, 128, 255, 256, 257, 511, 512], Hq, Hkv, block, D)


@pytest.mark.parametrize("lens", [[513], [1, 4000, 0, 17, 700], [2048] * 9, [0, 0, 1000], [30000, 1, 16], list(range(1, 900, 13)), [4096] * 2,
                                  [4500, *range(1, 900, 13)], [5000, 0, 3000, *range(0, 260, 2)]])
@pytest.mark.parametrize("D,Hq,Hkv", HEADS[:4])
def test_attention_of_long_and_uneven_rows(gpu, D, Hq, Hkv, lens):
    _check_attention(gpu, lens, Hq, Hkv, 256, D, seed=len(lens))


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("B,hi", [(64, 700), (64, 2100), (20, 900), (130, 1000), (16, 4096), (16, 4200), (4, 1024), (7, 1800)])
def test_attention_of_whole_rows_of_4_and_8_waves(gpu, B, hi, D):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, hi, (B,), generator=g).tolist()
    _check_attention(gpu, lens + [hi], 16, 8, 256, D, seed=B)


@pytest.mark.parametrize("size", [2.0 ** -60, 1.0, 2.0 ** 60])
def test_queries_of_unlike_sizes(gpu, size):
    """Channels of a query from 2^-14 of its largest on, whose low codes end, and queries far from one."""
    D, Hq, Hkv = 128, 8, 2
    p = _random_pages(gpu, [600, 2000], Hkv, 256, D)
    q = (torch.randn(2, Hq, D, device=gpu) * 2.0 ** torch.randint(-14, 1, (2, Hq, D), device=gpu).float()).bfloat16()
    q[0, 3] = 0
    got = kv8.decode_attention(q * size, p, _i32([599, 1999], gpu), None, 2000, D ** -0.5 / size).view(2, Hq, D)
    want, total = _exact(q, p, [599, 1999], [0, 1], 2000, D ** -0.5)
    assert bool(((got.double().cpu() - want).abs() <= (HALF + 2.0 ** -11) * total + HALF * want.abs()).all())


def test_attention_of_many_rows_one_slot_and_small_pages(gpu):
    _check_attention(gpu, [700, 33, 2100], 32, 8, 16, 64, order=[0, 1, 2, 2, 0, 1, 0] * 40)


def test_rows_of_no_keys_at_all(gpu):
    _, _, o = _check_attention(gpu, [0, 0, 0], 8, 2, 256, 128, bound=5000)
    assert not o.any()


@pytest.mark.parametrize("bound", [1, 16, 100, 512, 513, 1999])
def test_bound_hides_what_lies_behind(gpu, bound):
    _check_attention(gpu, [2000, 40, 700], 8, 2, 256, 64, bound=bound)


def test_scale_and_heads_of_one_group(gpu):
    for Hq in (1, 3, 16):
        _check_attention(gpu, [600, 90], Hq, 1, 64, 128, scale=0.05)


def test_bad_pages_and_slots(gpu):
    p, q, good = _check_attention(gpu, [900, 900, 300], 8, 2, 256, 64, bound=1024)
    p.table[1, 2] = p.k.shape[0]
    pos, slots = _i32([899, 899, 299, 299], gpu), _i32([0, 1, -1, 3], gpu)
    for bound, broken in ((1024, True), (300, False)):
        o = kv8.decode_attention(torch.cat([q, q[:1]]), p, pos, slots, bound).view(4, 8, 64)
        assert bool(o[1].isnan().all()) == broken and not o[2:].any() and not o[0].isnan().any()
    p.table[1].fill_(-1)  # no page of a row is there
    o = kv8.decode_attention(torch.cat([q, q[:1]]), p, pos, slots, 1024).view(4, 8, 64)
    assert o[1].isnan().all() and torch.equal(o[0], good[0])


def test_nan_keys_of_one_row_stay_with_it(gpu):
    p, q, good = _check_attention(gpu, [700, 700, 700], 4, 2, 256, 64)
    p.k[int(p.table[1, 1]), 0, 7, 5] = 0x7F
    o = kv8.decode_attention(q, p, _i32([699] * 3, gpu), None, 700).view(3, 4, 64)
    assert o[1, :2].isnan().all() and torch.equal(o[1, 2:], good[1, 2:]) and torch.equal(o[0], good[0]) and torch.equal(o[2], good[2])


@pytest.mark.parametrize("lens", [[40, 40], [5000, 40]])
def test_scores_that_are_all_minus_infinity_have_no_softmax(gpu, lens):
    D, Hq, Hkv = 64, 4, 2
    p, q, good = _check_attention(gpu, lens, Hq, Hkv, 256, D)
    for x in (p.k, p.v):
        x.fill_(0x38)  # 1
    p.k_exp.fill_(127)
    p.v_exp.fill_(127)
    q[:, 1, 7] = -torch.inf
    args = (_i32([n - 1 for n in lens], gpu), None, max(lens))
    o = kv8.decode_attention(q, p, *args).view(2, Hq, D)
    assert o[:, 1].isnan().all() and bool((o[:, [0, 2, 3]] == 1).all())
    plain = kv8.decode_attention(q.cpu(), kv8.Pages(*(t.cpu() for t in p)), _i32([n - 1 for n in lens]), None, max(lens))
    assert torch.equal(plain.view(2, Hq, D).isnan(), o.isnan().cpu())


def test_the_same_call_has_the_same_bits_captured_and_on_another_stream(gpu):
    """Two captured graphs, replayed in turn beside eager calls: neither shares a workspace with the other."""
    D, Hq, Hkv, block = 128, 8, 2, 256
    cos, sin = (t.to(gpu) for t in _tables(1200, D))
    lens = [900, 5, 1100]
    p = _random_pages(gpu, [n + 60 for n in lens], Hkv, block, D)
    p = p._replace(table=p.table.clamp_max(p.k.shape[0] - 1))
    qkv, pos, slots = _rows(3, Hq, Hkv, D).to(gpu), _i32(lens, gpu), _i32([0, 1, 2], gpu)

    def step(pages, x, at):
        q = kv8.append_tokens(x, cos, sin, at, slots, pages, Hq)
        return kv8.decode_attention(q, pages, at, slots, 1200)

    mine = kv8.Pages(*(t.clone() for t in p))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kv8.Pages(*(t.clone() for t in p)), qkv, pos)
    torch.cuda.current_stream().wait_stream(side)
    buf, at = qkv.clone(), pos.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="thread_local"):
            out = step(mine, buf, at)
        graphs.append((graph, out))
    eager = kv8.Pages(*(t.clone() for t in p))
    mine = [t.copy_(s) for t, s in zip(mine, p)]
    for i in range(6):
        buf.copy_(qkv * (1 + i % 3))
        at.copy_(pos + i)
        graphs[i % 2][0].replay()
        want = step(eager, qkv * (1 + i % 3), pos + i)
        torch.cuda.synchronize()
        assert torch.equal(graphs[i % 2][1], want) and _same(mine, eager)


def test_pages_past_32_bits(gpu):
    """A pool whose last pages lie more than 4 GiB behind its first gives what a small one does."""
    D, Hq, Hkv, block, n = 128, 16, 8, 256, 300
    cos, sin = (t.to(gpu) for t in _tables(n + 2, D))
    qkv, more = _rows(n, Hq, Hkv, D).to(gpu), _rows(1, Hq, Hkv, D, seed=5).to(gpu)
    runs, pos, slots = kv8.prompt_runs([0], [n], [0], gpu), _i32([n], gpu), _i32([0], gpu)
    out = []
    for pages, table in ((3, [[2, 0]]), (17000, [[16999, 16500]])):
        k, v = (torch.empty(pages, Hkv, block, D, dtype=torch.uint8, device=gpu) for _ in range(2))
        ke, ve = (torch.zeros(pages, Hkv, block // 16, dtype=torch.uint8, device=gpu) for _ in range(2))
        p = kv8.Pages(k, v, ke, ve, _i32(table, gpu))
        kv8.append_prompts(qkv, cos, sin, runs, p, Hq)
        q = kv8.append_tokens(more, cos, sin, pos, slots, p, Hq)
        out.append([q, *kv8.read(p, slots, _i32([0], gpu), pos + 1, n + 1), kv8.decode_attention(q, p, pos, slots, n + 1),
                    kv8.decode_attention(q, p, pos, slots, 4096)])
        del p, k, v
    assert 16500 * Hkv * block * D > 2 ** 32 and all(torch.equal(a, b) for a, b in zip(*out))


def test_prompt_then_tokens_is_attention_over_all(gpu):
    """What serving does: a prompt with normed heads appended, then token after token; each token's attention against 64 bits over
    what was appended.  Half a step of e4m3 (2^-4 of a value, or 2^-10 of the power of two that its group has) in keys moves a
    score by less than 2^-4 |q| |k| scale: held to a third of a typical output here, and exactly by the tests above."""
    D, Hq, Hkv, S, more = 64, 8, 2, 333, 20
    torch.manual_seed(0)
    cos, sin = (t.to(gpu) for t in _tables(S + more, D))
    qkv = torch.randn(S + more, (Hq + 2 * Hkv) * D, device=gpu).bfloat16()
    wq, wk = ((torch.rand(D, device=gpu) + 0.5).bfloat16() for _ in range(2))
    p = kv8.Pages.empty(5, Hkv, 256, D, _i32([[3, 1], [4, 0]], gpu))
    q, k, v = kv8.append_prompts(qkv[:S], cos, sin, kv8.prompt_runs([0], [S], [1], gpu), p, Hq, wq, wk)
    full = ops.qk_norm_rope(qkv, wq, wk, cos, sin, 1, S + more, Hq, Hkv, D)
    assert (q.float() - full[0][0, :, :S].float()).abs().max() <= 2 * HALF * q.abs().max().float()
    want = ref.attention(*(t.transpose(1, 2).cpu() for t in full))[0]
    for i in range(S, S + more):
        qi = kv8.append_tokens(qkv[i:i + 1], cos, sin, _i32([i], gpu), _i32([1], gpu), p, Hq, wq, wk)
        o = kv8.decode_attention(qi, p, _i32([i], gpu), _i32([1], gpu), S + more)
        w = want[i].reshape(-1).double()
        assert float((o[0].double().cpu() - w).norm() / w.norm()) < 1 / 3
        assert torch.equal(o, kv8.decode_attention(qi, p, _i32([i], gpu), _i32([1], gpu), i + 1)) or i + 1 > 512


def test_the_plain_forms_on_the_gpu_are_those_on_the_cpu(gpu, monkeypatch):
    """MXLLM_REFERENCE_OPS=1, which turns the kernels off."""
    D, Hq, Hkv = 32, 4, 2
    cos, sin = (t.to(gpu) for t in _tables(60, D))
    qkv = _rows(50, Hq, Hkv, D).to(gpu)
    out = []
    for plain in (False, True):
        if plain:
            monkeypatch.setenv("MXLLM_REFERENCE_OPS", "1")
        p = _to(_pages(2, 4, 9, Hkv, 16, D, fill=False), gpu)  # (positions 0 .. 2 hold zeros)
        q, k, v = kv8.append_prompts(qkv[:49], cos, sin, kv8.prompt_runs([3], [49], [1], gpu), p, Hq)
        q1 = kv8.append_tokens(qkv[49:], cos, sin, _i32([52], gpu), _i32([1], gpu), p, Hq)
        o = kv8.decode_attention(q1, p, _i32([52], gpu), _i32([1], gpu), 64)
        out.append((p, k, v, *kv8.read(p, _i32([1], gpu), _i32([3], gpu), _i32([53], gpu), 50), o))
    a, b = out
    assert _same(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[1:5], b[1:5]))
    assert float((a[5].double() - b[5].double()).norm() / b[5].double().norm()) < 2 * HALF


def test_refusals(gpu):
    Hq, Hkv, D = 4, 2, 64
    cos, sin = (t.to(gpu) for t in _tables(40, D))
    p = _to(_pages(2, 2, 6, Hkv, 16, D), gpu)
    rows, i32 = _rows(2, Hq, Hkv, D).to(gpu), _i32([0, 1], gpu)
    base = dict(qkv=rows, cos=cos, sin=sin, pos=i32, slots=i32, pages=p, Hq=Hq)
    norm = torch.ones(D, device=gpu, dtype=torch.bfloat16)
    for bad in [dict(qkv=rows[:, 64:]), dict(qkv=rows.float()), dict(pos=i32.long()), dict(pos=i32[:1]), dict(pos=i32.cpu()), dict(slots=i32[:1]),
                dict(Hq=3), dict(cos=cos[:, :8]), dict(sin=sin[:4]), dict(cos=cos.double(), sin=sin.double()), dict(q_norm=norm),
                dict(q_norm=norm.float(), k_norm=norm.float()), dict(q_norm=norm[:8], k_norm=norm[:8]), dict(pages=p._replace(k=p.k.float())),
                dict(pages=p._replace(k=p.k[:, :, :8].contiguous(), v=p.v[:, :, :8].contiguous())), dict(pages=p._replace(k_exp=p.k_exp[:1])),
                dict(pages=p._replace(table=p.table.long())), dict(pages=p._replace(table=p.table.cpu())), dict(pages=p._replace(v=p.v.transpose(0, 1)))]:
        with pytest.raises(RuntimeError):
            kv8.append_tokens(**(base | bad))
    before = [t.clone() for t in p]
    for runs in (i32, torch.zeros(2, 4, device=gpu), _i32([[0, 1, 0]], gpu), _i32([[0, 1, 0, 0]])):
        with pytest.raises(RuntimeError):
            kv8.append_prompts(rows, cos, sin, runs, p, Hq)
    q = torch.zeros(2, Hq, D, device=gpu, dtype=torch.bfloat16)
    for args in [(q.float(), p, i32, i32, 8), (q, p, i32, i32, 0), (q[:, :3], p, i32, i32, 8), (q[..., :32], p, i32, i32, 8), (q[:1], p, i32, i32, 8),
                 (torch.zeros(2, 34, D, device=gpu, dtype=torch.bfloat16), p, i32, i32, 8), (q, p, i32.long(), i32, 8),
                 (q, p, i32, i32, 8, 0.0), (q, p, i32, i32, 8, -0.1), (q, p, i32, i32, 8, math.nan), (q, p, i32, i32, 8, math.inf)]:
        with pytest.raises(RuntimeError):
            kv8.decode_attention(*args)
    with pytest.raises(RuntimeError):
        kv8.read(p, i32, i32, i32[:1], 4)
    with pytest.raises(RuntimeError):
        kv8.read(p, i32, i32, i32, -1)
    assert _same(before, p)


def test_weights_tables_and_runs_at_odd_places(gpu):
    """Copied, as rows there are: 16 bytes at a time is how they are read."""
    D, Hq, Hkv, block = 64, 4, 2, 32
    cos, sin = (t.to(gpu) for t in _tables(40, D))
    qkv = _rows(33, Hq, Hkv, D).to(gpu)
    wq, wk = ((1 + 0.1 * torch.randn(D)).bfloat16().to(gpu) for _ in range(2))
    runs = kv8.prompt_runs([0], [33], [0], gpu)

    def odd(t):
        return torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape)

    got = []
    for place in (lambda t: t, odd):
        p = kv8.Pages.empty(2, Hkv, block, D, _i32([[0, 1]], gpu))
        got.append([*kv8.append_prompts(qkv, place(cos), place(sin), place(runs), p, Hq, place(wq), place(wk)), *p[:4]])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_no_rows(gpu):
    Hq, Hkv, D = 4, 2, 64
    cos, sin = (t.to(gpu) for t in _tables(4, D))
    p = _to(_pages(2, 2, 6, Hkv, 16, D), gpu)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    rows = torch.zeros(0, (Hq + 2 * Hkv) * D, device=gpu, dtype=torch.bfloat16)
    assert kv8.append_tokens(rows, cos, sin, none, none, p, Hq).shape == (0, Hq, D)
    assert kv8.append_prompts(rows, cos, sin, none.view(0, 4), p, Hq)[1].shape == (Hkv, 0, D)
    assert kv8.decode_attention(rows[:, :Hq * D].view(0, Hq, D), p, none, none, 700).shape == (0, Hq * D)
    assert kv8.read(p, none, none, none, 5)[0].shape == (0, Hkv, 5, D)
    assert kv8.read(p, _i32([0], gpu), _i32([0], gpu), _i32([5], gpu), 0)[0].shape == (1, Hkv, 0, D)
