"""``qk_norm_rope`` under what records, batches or stands in for calls: such a tool has to meet the op itself, forward and backward,
and not the allocations inside it."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from mxllm import ops

from .test_qk_norm import EPS, _inputs

pytestmark = pytest.mark.gpu
DIMS = (2, 19, 4, 2, 64)
FORWARD, BACKWARD = "mxllm::qk_norm_rope", "mxllm::qk_norm_rope_bwd"


class Calls(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func._schema.name)
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("grad", [False, True])
def test_a_trace_records_the_op_and_replays_it(gpu, grad):
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, *DIMS)
    other, _, _ = _inputs(gpu, *DIMS, seed=5)

    def forward(x, a, b):
        return ops.qk_norm_rope(x, a, b, cos, sin, *DIMS, EPS)

    def both(x, a, b):
        leaves = [t.detach().requires_grad_() for t in (x, a, b)]
        out = forward(*leaves)
        return [*(o.detach() for o in out), *torch.autograd.grad(out, leaves, [2 * o.detach() for o in out])]

    run = both if grad else forward
    traced = make_fx(run, tracing_mode="real")(qkv, wq, wk)
    names = [n.target._schema.name for n in traced.graph.nodes if isinstance(n.target, torch._ops.OpOverload)]
    assert names.count(FORWARD) == 1 and names.count(BACKWARD) == grad
    for given in ((qkv, wq, wk), other[:3]):
        assert all(torch.equal(x, y) for x, y in zip(traced(*given), run(*given)))


@pytest.mark.parametrize("grad", [False, True])
def test_dispatch_modes_see_the_op(gpu, grad):
    (qkv, wq, wk, *grads), cos, sin = _inputs(gpu, *DIMS)
    leaves = [t.clone().requires_grad_(grad) for t in (qkv, wq, wk)]
    with Calls() as seen:
        out = ops.qk_norm_rope(*leaves, cos, sin, *DIMS, EPS)
    assert seen.names.count(FORWARD) == 1
    if grad:
        with Calls() as seen:
            got = torch.autograd.grad(out, leaves, grads)
        assert seen.names.count(BACKWARD) == 1
        again = torch.autograd.grad(ops.qk_norm_rope(*leaves, cos, sin, *DIMS, EPS), leaves, grads)
        assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize("packed", [False, True])
def test_many_backwards_at_once(gpu, packed):
    """``is_grads_batched`` runs the backward once for each of them."""
    B, S = DIMS[:2]
    (qkv, wq, wk, *grads), cos, sin = _inputs(gpu, *DIMS)
    pos = torch.randint(0, S, (B * S,), dtype=torch.int32, generator=torch.Generator().manual_seed(1)).to(gpu) if packed else None
    leaves = [t.clone().requires_grad_() for t in (qkv, wq, wk)]
    out = ops.qk_norm_rope(*leaves, cos, sin, *DIMS, EPS, pos)
    got = torch.autograd.grad(out, leaves, [torch.stack([g, -3 * g]) for g in grads], is_grads_batched=True, retain_graph=True)
    for i, f in enumerate((1, -3)):
        want = torch.autograd.grad(out, leaves, [f * g for g in grads], retain_graph=True)
        assert all(torch.equal(x[i], y) for x, y in zip(got, want))


def test_many_rows_at_once(gpu):
    """``torch.vmap`` over rows, without gradients."""
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, *DIMS)
    many = torch.stack([qkv, 3 * qkv])
    got = torch.vmap(lambda x: ops.qk_norm_rope(x, wq, wk, cos, sin, *DIMS, EPS))(many)
    for i, x in enumerate(many):
        assert all(torch.equal(a[i], b) for a, b in zip(got, ops.qk_norm_rope(x, wq, wk, cos, sin, *DIMS, EPS)))


def test_rows_at_odd_places_have_gradients(gpu):
    """Rows that the kernels cannot read as they lie are copied by both ops: the same gradients, in the rows' own places."""
    (qkv, wq, wk, *grads), cos, sin = _inputs(gpu, *DIMS)
    got = []
    for shift in (0, 3):
        wide = torch.zeros(qkv.shape[0], qkv.shape[1] + 8, device=gpu, dtype=torch.bfloat16)
        wide[:, shift:shift + qkv.shape[1]] = qkv
        wide.requires_grad_()
        out = ops.qk_norm_rope(wide[:, shift:shift + qkv.shape[1]], wq, wk, cos, sin, *DIMS, EPS)
        back = torch.autograd.grad(out, wide, grads)[0]
        assert not back[:, :shift].any() and not back[:, shift + qkv.shape[1]:].any()
        got.append([*out, back[:, shift:shift + qkv.shape[1]]])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_attention_block_with_norms(gpu):
    """The block's own autograd: a trace has its ops, and many backwards at once are those one by one."""
    (qkv, wq, wk, *_), cos, sin = _inputs(gpu, *DIMS)

    def run(x, a, b):
        return ops.attention_block(x, cos, sin, *DIMS, norms=(a, b, EPS))

    traced = make_fx(run, tracing_mode="real")(qkv, wq, wk)
    names = [n.target._schema.name for n in traced.graph.nodes if isinstance(n.target, torch._ops.OpOverload)]
    assert names.count(FORWARD) == 1
    other, _, _ = _inputs(gpu, *DIMS, seed=5)
    for given in ((qkv, wq, wk), other[:3]):
        assert torch.equal(traced(*given), run(*given))
    leaves = [t.clone().requires_grad_() for t in (qkv, wq, wk)]
    out = run(*leaves)
    do = torch.randn(2, *out.shape, device=gpu, generator=torch.Generator(gpu).manual_seed(1)).bfloat16()
    got = torch.autograd.grad(out, leaves, do, is_grads_batched=True, retain_graph=True)
    for i in range(2):
        want = torch.autograd.grad(out, leaves, do[i], retain_graph=True)
        assert all(torch.equal(x[i], y) for x, y in zip(got, want))
