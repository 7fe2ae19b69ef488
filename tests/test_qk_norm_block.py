"""``attention_block(norms=)``: its weights' gradients where an owner keeps them, and its backward in every form of the attention's.

Tolerances: whole errors as in tests/test_qk_norm.py (the attention kernels' roundings of 2^-8 along the way, two to an output and four
to a gradient); what an owner gets in f32 against autograd's bf16 of the same sums: its rounding, 2^-8 of the value."""
import pytest
import torch

from mxllm import ops
from mxllm.ops import attention

from .test_qk_norm import EPS, HALF, _exact, _inputs

pytestmark = pytest.mark.gpu


def _run(block, x, wq, wk, tables, dims):
    if block:
        return ops.attention_block(x, *tables, *dims, norms=(wq, wk, EPS))
    return torch.cat([t.flatten(2).flatten() for t in ops.qk_norm_rope(x, wq, wk, *tables, *dims, EPS)])


def _owner(w, fresh):
    """A parameter whose gradient a trainer keeps, and the calls that tell it so."""
    p, told = torch.nn.Parameter(w.clone()), []
    p._mx_grad32 = torch.full(w.shape, 7.0, device=w.device)
    p._mx_grad_fresh = fresh
    p._mx_on_grad_ready = lambda q: told.append(q._mx_grad32.clone())
    return p, told


@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("fresh", [False, True])
@pytest.mark.parametrize("who", ["both", "queries", "keys", "one"])
def test_owned_weights(gpu, block, fresh, who):
    """Owners of both weights, of either, and of one weight that both norms have: the f32 sums, once, and the owner hears of them
    when they are whole."""
    dims = (2, 40, 8, 2, 64)
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, *dims)
    if who == "one":
        wk = wq
    base = 0.0 if fresh else 7.0
    leaves = [t.clone().requires_grad_() for t in (qkv, wq, wk)]
    out = _run(block, *leaves, (cos, sin), dims)
    do = torch.randn(out.shape, device=gpu, generator=torch.Generator(gpu).manual_seed(2)).bfloat16()
    want = torch.autograd.grad(out, leaves, do)
    a, told_a = _owner(wq, fresh)
    b, told_b = (a, told_a) if who == "one" else _owner(wk, fresh)
    if who == "queries":
        b, told_b = leaves[2], None
    if who == "keys":
        a, told_a = leaves[1], None
    x = qkv.clone().requires_grad_()
    _run(block, x, a, b, (cos, sin), dims).backward(do)
    assert torch.equal(x.grad, want[0])
    if who == "one":
        sums = [(a, told_a, want[1].float() + want[2].float(), want[1].float().abs() + want[2].float().abs())]
    else:
        sums = [(p, t, w.float(), w.float().abs()) for p, t, w in ((a, told_a, want[1]), (b, told_b, want[2]))]
    for p, told, w, size in sums:
        if told is None:
            assert torch.equal(p.grad.float(), w)
            continue
        assert p.grad is None and not p._mx_grad_fresh
        assert bool(((p._mx_grad32 - base - w).abs() <= HALF * size + 2.0 ** -20).all())
        assert len(told) == 1 and torch.equal(told[0], p._mx_grad32)


@pytest.mark.parametrize("mode,budget", [(1, None), (2, None), (3, None), (3, 0)])
@pytest.mark.parametrize("D,Hq,Hkv,S", [(32, 8, 2, 600), (64, 8, 2, 700), (128, 8, 1, 513), (128, 16, 2, 1030)])
def test_longer_rows_in_every_form_of_the_backward(gpu, monkeypatch, D, Hq, Hkv, S, mode, budget):
    """Sums of dQ by atomics, by ordered parts, by an image of dS, and that in chunks of heads; several partials of a key head."""
    monkeypatch.setenv("MXLLM_ATTN_DQ_MODE", str(mode))
    if budget is not None:
        monkeypatch.setattr(attention, "_DS_BUDGET", budget)
    dims = (2, S, Hq, Hkv, D)
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, *dims, seed=S)
    do = torch.randn(2 * S, Hq * D, device=gpu, generator=torch.Generator(gpu).manual_seed(2)).bfloat16()
    leaves = [t.clone().requires_grad_() for t in (qkv, wq, wk)]
    out = ops.attention_block(leaves[0], cos, sin, *dims, norms=(*leaves[1:], EPS))
    got = torch.autograd.grad(out, leaves, do)
    exact = [t.double().cpu().requires_grad_() for t in (qkv, wq, wk)]
    (q, k, v), _ = _exact(*exact, cos.cpu(), sin.cpu(), *dims)
    k, v = (t.repeat_interleave(Hq // Hkv, 1) for t in (k, v))
    s = (q @ k.transpose(2, 3)) * D ** -0.5
    s = s.masked_fill(torch.ones(S, S).triu(1).bool(), float("-inf"))
    want = (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(2 * S, -1)
    grads = torch.autograd.grad(want, exact, do.double().cpu())

    def rel(a, b):
        return float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm())

    assert rel(out, want) < 2 * HALF
    assert all(rel(a, b) < 4 * HALF for a, b in zip(got, grads)), [rel(a, b) for a, b in zip(got, grads)]
