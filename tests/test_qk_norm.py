"""RMS norm of query and key heads with the rotation (mxllm/ops/attention.py ``qk_norm_rope``, csrc/kernels/qk_norm.hip): against the
formulas in 64 bits, their gradients and differences.

A rounding to bf16 is off by up to 2^-8 of the value (HALF).  What f32 adds is at most a few of its own roundings of the largest
summand: F32 = 2^-19 of the sum of the summands' sizes (16 roundings of 2^-24 and the reductions of 128 channels,
which a tree of depth 7 forms)."""
import pytest
import torch

from mxllm import ops
from mxllm.ops import reference as ref

HALF, F32, EPS = 2.0 ** -8, 2.0 ** -19, 1e-5


def _inputs(dev, B, S, Hq, Hkv, D, seed=0, table=None):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B * S, (Hq + 2 * Hkv) * D, generator=g) * torch.exp(0.5 * torch.randn(B * S, 1, generator=g))
    wq, wk = (1 + 0.3 * torch.randn(D, generator=g) for _ in range(2))
    grads = [torch.randn(B, h, S, D, generator=g) for h in (Hq, Hkv, Hkv)]
    cos, sin = ref.rope_tables(table or max(S, 1), D, 500000.0, None)
    return [t.to(torch.bfloat16).to(dev) for t in (qkv, wq, wk, *grads)], cos.to(dev), sin.to(dev)


def _exact(qkv, wq, wk, cos, sin, B, S, Hq, Hkv, D, pos=None):
    """f64 outputs, and the sizes of the two summands of each turned value."""
    x = qkv.view(B, S, -1, D)
    pos = torch.arange(S, device=x.device).expand(B, S) if pos is None else pos.view(B, S).long()
    c, s = cos[pos].double()[:, :, None], sin[pos].double()[:, :, None]

    def one(h, w):
        n = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * w
        a, b = n.split(D // 2, -1)
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
        size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
        return y.transpose(1, 2), size.transpose(1, 2)

    q, qs = one(x[:, :, :Hq], wq)
    k, ks = one(x[:, :, Hq:Hq + Hkv], wk)
    v = x[:, :, Hq + Hkv:].transpose(1, 2)
    return (q, k, v), (qs, ks, v.abs())


def _near(got, want, size):
    err = (got.double() - want).abs()
    assert bool((err <= HALF * want.abs() + F32 * size + 1e-30).all()), float((err - HALF * want.abs()).max())


CASES = [(1, 1, 4, 2, 32), (3, 5, 8, 8, 64), (2, 129, 12, 2, 64), (1, 33, 6, 1, 128), (5, 17, 32, 8, 128), (1, 700, 3, 3, 32)]


def _check(dev, B, S, Hq, Hkv, D, packed, run=ops.qk_norm_rope):
    (qkv, wq, wk, *grads), cos, sin = _inputs(dev, B, S, Hq, Hkv, D)
    pos = torch.randint(0, S, (B * S,), dtype=torch.int32, generator=torch.Generator().manual_seed(9)).to(dev) if packed else None
    leaves = [t.clone().requires_grad_() for t in (qkv, wq, wk)]
    out = run(*leaves, cos, sin, B, S, Hq, Hkv, D, EPS, pos)
    got = torch.autograd.grad(out, leaves, grads)
    exact = [t.double().requires_grad_() for t in (qkv, wq, wk)]
    want, sizes = _exact(*exact, cos, sin, B, S, Hq, Hkv, D, pos)
    for o, w, s in zip(out, want, sizes):
        assert o.dtype == torch.bfloat16 and o.is_contiguous() and o.shape == w.shape
        _near(o, w, s)
    wg = torch.autograd.grad(want, exact, [g.double() for g in grads], retain_graph=True)
    # sizes of the summands of the gradients: the formulas with every term at its size
    x = qkv.double().view(B, S, -1, D)
    p = torch.arange(S, device=dev).expand(B, S) if pos is None else pos.view(B, S).long()
    c, s = cos[p].double().abs()[:, :, None], sin[p].double().abs()[:, :, None]
    dx_size, dw_size = [], []
    for h, w, g in ((x[:, :, :Hq], wq, grads[0]), (x[:, :, Hq:Hq + Hkv], wk, grads[1])):
        ga, gb = g.double().abs().transpose(1, 2).split(D // 2, -1)
        dn = torch.cat([ga * c + gb * s, gb * c + ga * s], -1)
        r = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
        gw = dn * w.double().abs()
        dx_size.append(r * (gw + h.abs() * r * r * (gw * h.abs()).mean(-1, keepdim=True)))
        dw_size.append((dn * h.abs() * r).sum((0, 1, 2)))
    dv = grads[2].double().abs().transpose(1, 2)
    _near(got[0], wg[0], torch.cat([*dx_size, dv], 2).reshape(B * S, -1))
    _near(got[1], wg[1], dw_size[0])
    _near(got[2], wg[2], dw_size[1])
    # the gradient of the formula against a difference of it, along one direction
    step = [torch.randn_like(t) for t in exact]
    h = 1e-5

    def loss(sign):
        o, _ = _exact(*[t.detach() + sign * h * d for t, d in zip(exact, step)], cos, sin, B, S, Hq, Hkv, D, pos)
        return sum((a * g.double()).sum() for a, g in zip(o, grads))

    slope = sum((a * d).sum() for a, d in zip(wg, step))
    size = sum((a * d).abs().sum() for a, d in zip(wg, step))
    assert abs(float((loss(1) - loss(-1)) / (2 * h) - slope)) < 1e-6 * float(size)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("B,S,Hq,Hkv,D", CASES[:4])
def test_plain_against_64_bits(B, S, Hq, Hkv, D, packed):
    _check("cpu", B, S, Hq, Hkv, D, packed)


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("B,S,Hq,Hkv,D", CASES)
def test_kernel_against_64_bits(gpu, B, S, Hq, Hkv, D, packed):
    _check(gpu, B, S, Hq, Hkv, D, packed)


@pytest.mark.gpu
def test_many_rows_and_workgroups(gpu):
    """More heads than one turn of the backward's workgroups takes."""
    _check(gpu, 2, 1500, 32, 8, 128, False)


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hq,Hkv", [(32, 4, 2), (128, 8, 2)])
def test_rows_of_a_wider_buffer_and_broadcast_gradients(gpu, D, Hq, Hkv):
    B, S = 2, 19
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, B, S, Hq, Hkv, D, table=40)
    wide = torch.full((B * S, qkv.shape[1] + 24), float("nan"), device=gpu, dtype=torch.bfloat16)
    wide[:, :qkv.shape[1]] = qkv
    one = torch.ones((), device=gpu, dtype=torch.bfloat16)
    res = []
    for rows in (wide[:, :qkv.shape[1]], qkv):
        leaves = [t.detach().requires_grad_() for t in (rows, wq, wk)]
        out = ops.qk_norm_rope(*leaves, cos, sin, B, S, Hq, Hkv, D)
        res.append([*out, *torch.autograd.grad(out, leaves, [one.expand(o.shape) for o in out])])
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.gpu
def test_rows_past_32_bits(gpu):
    """351 copies of 1,000 rows, 2^31 numbers and more: the last copy comes out, and goes back, as the rows alone do."""
    B, S, Hq, Hkv, D, n = 8, 43875, 32, 8, 128, 1000
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, 1, n, Hq, Hkv, D)
    pos = torch.randint(0, n, (n,), generator=torch.Generator().manual_seed(3)).int().to(gpu)
    ends = []
    for b, s in ((1, n), (B, S)):
        rows = qkv.repeat(b * s // n, 1)
        at = pos.repeat(b * s // n)
        rows.requires_grad_()
        out = ops.qk_norm_rope(rows, wq, wk, cos, sin, b, s, Hq, Hkv, D, EPS, at)
        back = torch.autograd.grad(out, rows, [o.detach() for o in out])[0]
        ends.append([*(o.detach()[-1, :, -n:].clone() for o in out), back[-n:].clone()])
        assert b == 1 or rows.numel() > 2 ** 31
        del rows, out, back
    assert all(torch.equal(x, y) for x, y in zip(*ends))


@pytest.mark.gpu
def test_unused_outputs_and_frozen_weights(gpu):
    B, S, Hq, Hkv, D = 1, 21, 4, 2, 64
    (qkv, wq, wk, gq, gk, gv), cos, sin = _inputs(gpu, B, S, Hq, Hkv, D)
    x = qkv.clone().requires_grad_()
    q, k, v = ops.qk_norm_rope(x, wq, wk, cos, sin, B, S, Hq, Hkv, D)
    (dx,) = torch.autograd.grad(q, x, gq)
    assert not dx[:, Hq * D:].any() and dx[:, :Hq * D].any()
    w = wk.clone().requires_grad_()
    q, k, v = ops.qk_norm_rope(qkv, wq, w, cos, sin, B, S, Hq, Hkv, D)
    k.backward(gk)
    full = [t.clone().requires_grad_() for t in (qkv, wq, wk)]
    out = ops.qk_norm_rope(*full, cos, sin, B, S, Hq, Hkv, D)
    dw = torch.autograd.grad(out[1], full, gk)[2]
    assert torch.equal(w.grad, dw)
    first = w.grad.clone()
    q, k, v = ops.qk_norm_rope(qkv, wq, w, cos, sin, B, S, Hq, Hkv, D)
    k.backward(gk)
    assert torch.equal(w.grad, first + dw)
    with pytest.raises(RuntimeError):  # differentiable once
        out = ops.qk_norm_rope(*full, cos, sin, B, S, Hq, Hkv, D)
        g = torch.autograd.grad(out[0], full[0], gq, create_graph=True)[0]
        g.sum().backward()


def _outside(dev):
    Hq, Hkv, D = 4, 2, 64
    (qkv, wq, wk, *_), cos, sin = _inputs(dev, 1, 4, Hq, Hkv, D)
    pos = torch.tensor([0, -1, 3, 4], dtype=torch.int32, device=dev)
    q, k, v = ops.qk_norm_rope(qkv, wq, wk, cos, sin, 1, 4, Hq, Hkv, D, EPS, pos)
    bad = torch.isnan(q[0, :, :, 0]).all(0).tolist()
    assert bad == [False, True, False, True] and torch.isnan(k[0, :, 1]).all() and not torch.isnan(v).any()


def test_positions_outside_the_table_plain():
    _outside("cpu")


@pytest.mark.gpu
def test_one_weight_for_both_norms_and_rows_at_odd_places(gpu):
    """A weight that is both norms' has the sum of their gradients; rows that start between pieces of 16 bytes are copied."""
    B, S, Hq, Hkv, D = 1, 9, 4, 2, 64
    (qkv, w, _, gq, gk, gv), cos, sin = _inputs(gpu, B, S, Hq, Hkv, D)
    p, a, b = (w.clone().requires_grad_() for _ in range(3))
    one = torch.autograd.grad(ops.qk_norm_rope(qkv, p, p, cos, sin, B, S, Hq, Hkv, D), p, (gq, gk, gv))[0]
    two = torch.autograd.grad(ops.qk_norm_rope(qkv, a, b, cos, sin, B, S, Hq, Hkv, D), (a, b), (gq, gk, gv))
    assert torch.equal(one, two[0] + two[1])
    wide = torch.zeros(S, qkv.shape[1] + 8, device=gpu, dtype=torch.bfloat16)
    wide[:, 3:3 + qkv.shape[1]] = qkv
    out = ops.qk_norm_rope(wide[:, 3:3 + qkv.shape[1]], w, w, cos, sin, B, S, Hq, Hkv, D)
    assert all(torch.equal(x, y) for x, y in zip(out, ops.qk_norm_rope(qkv, w, w, cos, sin, B, S, Hq, Hkv, D)))


@pytest.mark.gpu
def test_weights_tables_and_gradients_at_odd_places(gpu):
    B, S, Hq, Hkv, D = 2, 9, 4, 2, 64
    (qkv, *rest), cos, sin = _inputs(gpu, B, S, Hq, Hkv, D)

    def odd(t):
        return torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape)

    got = []
    for place in (lambda t: t, odd):
        wq, wk, *grads = map(place, rest)
        leaves = [t.detach().requires_grad_() for t in (qkv, wq, wk)]
        out = ops.qk_norm_rope(*leaves, place(cos), place(sin), B, S, Hq, Hkv, D)
        got.append([*out, *torch.autograd.grad(out, leaves, grads)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
def test_no_rows_and_positions_outside_the_table(gpu):
    Hq, Hkv, D = 4, 2, 64
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, 0, 5, Hq, Hkv, D, table=4)
    leaves = [t.clone().requires_grad_() for t in (qkv, wq, wk)]
    out = ops.qk_norm_rope(*leaves, cos, sin, 0, 5, Hq, Hkv, D, EPS, torch.zeros(0, dtype=torch.int32, device=gpu))
    grads = torch.autograd.grad(out, leaves, [torch.zeros_like(o) for o in out])
    assert out[0].shape == (0, Hq, 5, D) and not grads[1].any() and not grads[2].any()
    _outside(gpu)


@pytest.mark.gpu
def test_captured_and_on_another_stream(gpu):
    B, S, Hq, Hkv, D = 2, 65, 8, 2, 64
    (qkv, wq, wk, *grads), cos, sin = _inputs(gpu, B, S, Hq, Hkv, D)

    def step(x):
        leaves = [t.detach().requires_grad_() for t in (x, wq, wk)]
        out = ops.qk_norm_rope(*leaves, cos, sin, B, S, Hq, Hkv, D)
        return [*out, *torch.autograd.grad(out, leaves, grads)]

    buf = qkv.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(buf)
        step(buf)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, step(qkv)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        got = step(buf)
    for i in range(4):
        buf.copy_(qkv * (i + 1))
        graph.replay()
        want = step(qkv * (i + 1))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_forward_mode_is_refused(gpu):
    B, S, Hq, Hkv, D = 1, 6, 4, 2, 64
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, B, S, Hq, Hkv, D)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(qkv, torch.ones_like(qkv))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                ops.qk_norm_rope(dual, wq, wk, cos, sin, B, S, Hq, Hkv, D)


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
@pytest.mark.parametrize("block", [False, True])
def test_a_capture_beside_a_living_graph_of_the_same_leaves_is_refused(gpu, block):
    B, S, Hq, Hkv, D = 1, 40, 4, 2, 64
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, B, S, Hq, Hkv, D)
    leaves = [t.detach().requires_grad_() for t in (qkv, wq, wk)]

    def step():
        if block:
            return ops.attention_block(leaves[0], cos, sin, B, S, Hq, Hkv, D, norms=(*leaves[1:], EPS))
        return ops.qk_norm_rope(*leaves, cos, sin, B, S, Hq, Hkv, D)

    alive = step()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), capture_error_mode="thread_local"):
            step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"), torch.no_grad():
        got = step()  # (without a backward there is nothing to refuse)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*((x,) if block else x for x in (alive, got))))


@pytest.mark.gpu
@pytest.mark.parametrize("D,Hq,Hkv,S", [(32, 4, 2, 33), (64, 8, 2, 100), (128, 4, 1, 130)])
def test_attention_block_with_norms(gpu, D, Hq, Hkv, S):
    """Norm, rotation and attention as one node against 64 bits: outputs and every gradient by their whole error; the attention
    kernels' own roundings (inputs, weights and dS in bf16) make up to four of 2^-8 along the way to a gradient."""
    B = 2
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, B, S, Hq, Hkv, D, seed=3)
    do = torch.randn(B * S, Hq * D, device=gpu).bfloat16()
    leaves = [t.clone().requires_grad_() for t in (qkv, wq, wk)]
    o = ops.attention_block(leaves[0], cos, sin, B, S, Hq, Hkv, D, norms=(leaves[1], leaves[2], EPS), grad_pad=64)
    got = torch.autograd.grad(o, leaves, do)
    exact = [t.double().cpu().requires_grad_() for t in (qkv, wq, wk)]
    (q, k, v), _ = _exact(*exact, cos.cpu(), sin.cpu(), B, S, Hq, Hkv, D)
    k, v = (t.repeat_interleave(Hq // Hkv, 1) for t in (k, v))
    s = (q @ k.transpose(2, 3)) * D ** -0.5
    s = s.masked_fill(torch.ones(S, S).triu(1).bool(), float("-inf"))
    want = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B * S, -1)
    wg = torch.autograd.grad(want, exact, do.double().cpu())

    def rel(a, b):
        return float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm())

    assert rel(o, want) < 2 * HALF
    assert all(rel(a, b) < 4 * HALF for a, b in zip(got, wg))


@pytest.mark.gpu
def test_owned_weight_gradients_go_to_their_owner(gpu):
    """A weight whose owner keeps its gradient in f32 (a trainer's flat buffer) gets the f32 sums there, overwritten where the
    buffer is fresh and added to afterwards."""
    B, S, Hq, Hkv, D = 1, 40, 4, 2, 64
    (qkv, wq, wk, gq, gk, gv), cos, sin = _inputs(gpu, B, S, Hq, Hkv, D)
    w = torch.nn.Parameter(wq.clone())
    w._mx_grad32, w._mx_grad_fresh = torch.full((D,), 7.0, device=gpu), True
    for n in (1, 2):
        q, _, _ = ops.qk_norm_rope(qkv, w, wk, cos, sin, B, S, Hq, Hkv, D)
        q.backward(gq)
        p = torch.nn.Parameter(wq.clone())
        torch.autograd.backward(ops.qk_norm_rope(qkv, p, wk, cos, sin, B, S, Hq, Hkv, D)[0], gq)
        assert w.grad is None and torch.allclose(w._mx_grad32, n * p.grad.float(), rtol=2 * HALF, atol=1e-3)


@pytest.mark.gpu
def test_refusals(gpu):
    B, S, Hq, Hkv, D = 1, 6, 4, 2, 64
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, B, S, Hq, Hkv, D)
    args = (cos, sin, B, S, Hq, Hkv, D)
    for bad in [(qkv.float(), wq, wk, *args), (qkv[:, :-64], wq, wk, *args), (qkv, wq[:32], wk, *args), (qkv, wq.float(), wk, *args),
                (qkv, wq, wk.cpu(), *args), (qkv, wq, wk, cos[:5], sin[:5], *args[2:]), (qkv, wq, wk, cos, sin[:5], *args[2:]),
                (qkv, wq, wk, cos, sin, 2, *args[3:]), (qkv, wq, wk, cos, sin, B, S, 3, 2, D), (qkv, wq, wk, cos, sin, B, S, 2, 1, 96),
                (qkv, wq, wk, *args, EPS, torch.zeros(S, device=gpu)), (qkv, wq, wk, *args, EPS, torch.zeros(S + 1, dtype=torch.int32, device=gpu)),
                (qkv, wq, wk, *args, EPS, torch.zeros(S, dtype=torch.int32))]:
        with pytest.raises(RuntimeError):
            ops.qk_norm_rope(*bad)
