"""How near attention over a cache in 8 bits is to 64 bits over the same codes: its output's own rounding, and what f32 leaves.

A weight is the sum of two numbers of bf16: the first is off by 2^-8 of it, the second by 2^-8 of that, 2^-16 of the weight.  Scores
leave 2^-13 of a weight and f32 sums less (tests/test_kv8_gpu.py), 2^-11 of sum w |v| for both; the output is rounded once."""
import pytest
import torch

from mxllm.ops import kv8

from .test_kv8_gpu import HALF, HEADS, _exact, _i32, _random_pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[1, 17, 256, 700], [900] * 40, [300] * 80, [16384, 40, 5000]])
@pytest.mark.parametrize("D,Hq,Hkv", HEADS)
def test_weights_are_not_rounded_to_bf16(gpu, D, Hq, Hkv, lens):
    p = _random_pages(gpu, lens, Hkv, 256, D)
    q = torch.randn(len(lens), Hq, D, device=gpu, generator=torch.Generator(gpu).manual_seed(3)).bfloat16()
    pos = [n - 1 for n in lens]
    got = kv8.decode_attention(q, p, _i32(pos, gpu), None, max(lens)).view(len(lens), Hq, D).double().cpu()
    want, size = _exact(q, p, pos, list(range(len(lens))), max(lens), D ** -0.5)
    assert bool(((got - want).abs() <= (2.0 ** -16 + 2.0 ** -11) * size + HALF * want.abs()).all())
