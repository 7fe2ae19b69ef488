"""Calls over a cache in 8 bits that are refused, by the kernels' bindings and the plain forms alike."""
import pytest
import torch

from mxllm.ops import kv8

from .test_kv8 import _pages, _rows, _tables

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
