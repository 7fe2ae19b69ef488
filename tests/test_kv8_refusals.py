"""Calls over a cache in 8 bits, and of the norms of heads, that are refused by the kernels' bindings and the plain forms alike."""
import pytest
import torch

from mxllm import ops
from mxllm.ops import kv8

from .test_kv8 import _pages, _rows, _tables
from .test_qk_norm import _inputs

Hq, Hkv, D = 4, 2, 64
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
REFUSED = (ValueError, RuntimeError)


def _i32(*x, dev="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cache(dev):
    return kv8.Pages(*(t.to(dev) for t in _pages(2, 2, 6, Hkv, 16, D)))


def _calls(dev, pages, dim=D):
    """Every operator over ``pages``, by name, with operands of heads of ``dim`` channels."""
    cos, sin = (t.to(dev) for t in _tables(40, D))
    cos, sin = cos[:, :dim // 2].contiguous(), sin[:, :dim // 2].contiguous()
    rows = _rows(2, Hq, Hkv, D).view(2, -1, D)[..., :dim].reshape(2, (Hq + 2 * Hkv) * dim).to(dev)
    at = _i32(0, 1, dev=dev)
    return {
        "tokens": lambda: kv8.append_tokens(rows, cos, sin, at, at, pages, Hq),
        "prompts": lambda: kv8.append_prompts(rows, cos, sin, kv8.prompt_runs([0], [2], [0], dev), pages, Hq),
        "read": lambda: kv8.read(pages, at, at, at + 2, 2),
        "attention": lambda: kv8.decode_attention(rows[:, :Hq * dim].reshape(2, Hq, dim), pages, at, at, 8, 0.1),
    }


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name", ["tokens", "prompts", "read", "attention"])
def test_caches_of_nothing(dev, name):
    """No pages, no heads, heads of no channels: an error (the last divided by zero)."""
    good = _cache(dev)
    _calls(dev, good)[name]()
    for cut in (lambda t: t[:0], lambda t: t[:, :0]):
        with pytest.raises(REFUSED):
            _calls(dev, kv8.Pages(*(cut(t) for t in good[:4]), good.table))[name]()
    with pytest.raises(REFUSED):
        _calls(dev, good._replace(k=good.k[..., :0], v=good.v[..., :0]), 0)[name]()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name", ["tokens", "prompts", "read", "attention"])
def test_tables_of_nothing(dev, name):
    good = _cache(dev)
    for table in (good.table[:0], good.table[:, :0]):
        with pytest.raises(REFUSED):
            _calls(dev, good._replace(table=table))[name]()


@pytest.mark.parametrize("dev", DEVICES)
def test_more_sequences_than_slots_are_read_as_slots_that_are_none(dev):
    """Without ``slots`` a row's number is its slot: rows past the table have nothing, as rows of a slot named that there is not."""
    p = _cache(dev)
    at = _i32(0, 0, 0, 0, dev=dev)
    q = torch.ones(4, Hq, D, device=dev).bfloat16()
    for slots in (None, _i32(0, 1, 2, 3, dev=dev)):
        k, v = kv8.read(p, slots, at, at + 5, 5)
        assert not k[2:].any() and not v[2:].any() and k[:2].any()
        o = kv8.decode_attention(q, p, at + 4, slots, 5)
        assert not o[2:].any() and o[:2].any()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("block", [False, True])
def test_norms_of_rows_that_the_operands_do_not_fit(dev, block):
    """Sequences longer than the rotation's table, and operands of other shapes: refused, where ``positions`` names no rows of it NaN."""
    B, S = 2, 6
    (qkv, wq, wk, *_), cos, sin = _inputs(dev, B, S, Hq, Hkv, D)

    def call(x=qkv, a=wq, b=wk, c=cos, s=sin, S=S, Hq=Hq, positions=None):
        if block:
            return ops.attention_block(x, c, s, B, S, Hq, Hkv, D, norms=(a, b, 1e-5))
        return ops.qk_norm_rope(x, a, b, c, s, B, S, Hq, Hkv, D, 1e-5, positions)

    call()
    bad = [dict(c=cos[:5], s=sin[:5]), dict(s=sin[:5]), dict(c=cos[:, :8], s=sin[:, :8]), dict(c=cos[:0], s=sin[:0]), dict(a=wq[:1]),
           dict(b=wk[:32]), dict(b=wk[None]), dict(x=qkv[:11]), dict(x=qkv[:, 64:]), dict(x=qkv[None]), dict(S=5), dict(Hq=3)]
    if not block:
        at = torch.zeros(B * S, dtype=torch.int32, device=dev)
        bad += [dict(positions=at.long()), dict(positions=at[1:]), dict(positions=at.view(B, S))]
        q, k, _ = call(c=cos[:5], s=sin[:5], positions=at + 5)
        assert q.isnan().all() and k.isnan().all()
    for args in bad:
        with pytest.raises(REFUSED):
            call(**args)
