"""``kv8.prompt_attention``: causal attention of several prompts to themselves, by itself (tests/test_kv8_engine.py has it in a model).
Against 64 bits with the tolerance of tests/test_kv8_gpu.py: a weight and the output rounded to bf16, 2^-11 for what f32 adds."""
import pytest
import torch

from mxllm import ops
from mxllm.ops import kv8
from mxllm.ops.hybrid import PromptRows

HALF = 2.0 ** -8
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
LENS = [[1], [128], [129, 1, 17], [300, 0, 65, 128, 3, 0]]
HEADS = [(32, 4, 2), (64, 8, 8), (128, 8, 1)]


def _inputs(dev, T, Hq, Hkv, D):
    g = torch.Generator().manual_seed(T + D)
    return [torch.randn(h, T, D, generator=g).bfloat16().to(dev) for h in (Hq, Hkv, Hkv)]


def _exact(q, k, v, lens):
    out, size, at = [], [], 0
    q, k, v = (t.double().cpu() for t in (q, k, v))
    for n in lens:
        a, b, c = (t[:, at:at + n] for t in (q, *(t.repeat_interleave(q.shape[0] // k.shape[0], 0) for t in (k, v))))
        s = (a @ b.transpose(1, 2)) * q.shape[2] ** -0.5
        w = torch.softmax(s.masked_fill(torch.ones(n, n).triu(1).bool(), -torch.inf), -1)
        out.append((w @ c).transpose(0, 1).flatten(1))
        size.append((w @ c.abs()).transpose(0, 1).flatten(1))
        at += n
    return torch.cat(out), torch.cat(size)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("D,Hq,Hkv", HEADS)
def test_against_64_bits(dev, D, Hq, Hkv, lens):
    q, k, v = _inputs(dev, sum(lens), Hq, Hkv, D)
    got = kv8.prompt_attention(q, k, v, lens)
    want, size = _exact(q, k, v, lens)
    assert got.shape == want.shape and got.dtype == q.dtype
    assert bool(((got.double().cpu() - want).abs() <= (HALF + 2.0 ** -11) * size + HALF * want.abs()).all())
    blocks = PromptRows([n for n in lens if n], dev).attn_blocks(max(lens))
    assert torch.equal(got, kv8.prompt_attention(q, k, v, lens, blocks))
    odd = [torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape) for t in (q, k, v)]
    strided = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    for others in (odd, strided):
        assert torch.equal(got, kv8.prompt_attention(*others, lens))


@pytest.mark.parametrize("dev", DEVICES)
def test_no_rows(dev):
    q, k, v = _inputs(dev, 0, 4, 2, 64)
    for lens in ([], [0, 0]):
        assert kv8.prompt_attention(q, k, v, lens).shape == (0, 256)


@pytest.mark.parametrize("dev", DEVICES)
def test_lengths_and_blocks_that_are_not_the_rows(dev):
    lens = [130, 20]
    q, k, v = _inputs(dev, 150, 4, 2, 64)
    for bad in ([130], [130, 21], [150, 20], [160, -10], []):
        with pytest.raises(ValueError):
            kv8.prompt_attention(q, k, v, bad)
    with pytest.raises((ValueError, RuntimeError)):
        kv8.prompt_attention(q, k[:, :149], v[:, :149], lens)
    with pytest.raises((ValueError, RuntimeError)):
        kv8.prompt_attention(q[:3], k, v, lens)
    if dev == "cuda":
        for other in ([130], [300, 20]):
            with pytest.raises(ValueError):
                kv8.prompt_attention(q, k, v, lens, PromptRows(other, dev).attn_blocks(max(other)))


@pytest.mark.gpu
def test_blocks_of_rows_that_are_none_are_left_out(gpu):
    """In a table of blocks, those of other rows than the call has neither read nor write."""
    T, lens = 150, [130, 20]
    q, k, v = _inputs(gpu, T, 4, 2, 64)
    blocks = PromptRows(lens, gpu).attn_blocks(130)
    bad = [[-1, 5, 0, 0], [148, 3, 0, 0], [0, 0, 0, 0], [0, -4, 0, 0], [0, 128, 1, 0], [0, 150, -1, 0], [150, 1, 0, 0], [2 ** 31 - 1, 9, 0, 0]]
    both = torch.cat([torch.tensor(bad, dtype=torch.int32, device=gpu), blocks])
    got = ops.native().prompt_rows_attention(q, k, v, both, 0.125)
    assert torch.equal(got, kv8.prompt_attention(q, k, v, lens, blocks))
