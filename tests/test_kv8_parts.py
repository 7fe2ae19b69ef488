"""The parts of rows that attention over a cache in 8 bits cuts: the memory that they take, and the forms that join them."""
import pytest
import torch

from mxllm.ops import kv8

from .test_kv8_gpu import _check_attention, _i32, _random_pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Hq,Hkv,D,max_len", [(1024, 16, 1, 128, 32768), (256, 64, 8, 128, 8192), (4000, 8, 2, 32, 300000)])
def test_the_workspace_does_not_grow_with_rows_or_lengths(gpu, B, Hq, Hkv, D, max_len):
    """Two parts for each of 256 shares (rounded up to whole ones a key head) of every query head of a group, whatever B and
    ``max_len`` are: 512 rep (D + 2) numbers and the output, doubled for what the allocator rounds."""
    lens = [300, 17, 1, 40]
    p = _random_pages(gpu, lens, Hkv, 256, D)
    table = torch.zeros(4, -(-max_len // 256), dtype=torch.int32, device=gpu)
    table[:, :2] = p.table[:, :2].clamp_max(p.k.shape[0] - 1)
    p = p._replace(table=table)
    slots = torch.arange(B, device=gpu, dtype=torch.int32) % 4
    pos = _i32(lens, gpu)[slots.long()] - 1
    q = torch.randn(B, Hq, D, device=gpu).bfloat16()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = kv8.decode_attention(q, p, pos, slots, max_len)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= 2 * (4 * 512 * (Hq // Hkv) * (D + 2) + 2 * q.numel()) + 2 ** 21
    want = kv8.decode_attention(q, p, pos, slots, 301)  # (other forms)
    assert float((got.double() - want.double()).norm() / want.double().norm()) < 2.0 ** -7


@pytest.mark.parametrize("Hq,Hkv", [(16, 1), (64, 4)])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_a_row_of_many_parts_beside_many_rows(gpu, D, Hq, Hkv):
    """Over 512 query rows, one of them in more than 64 parts (of one key head, whose 256 shares they are)."""
    lens = [*range(1, 30), 30000, *range(30, 60), 0]
    _check_attention(gpu, lens, Hq, Hkv, 256, D, seed=D)
    _check_attention(gpu, [30000, 29000, *lens], Hq, Hkv, 256, D, seed=D + 1)


def test_two_graphs_and_eager_calls_have_workspaces_of_their_own(gpu):
    p = _random_pages(gpu, [9000, 500, 20000], 2, 256, 64)
    qs = [torch.randn(3, 8, 64, device=gpu).bfloat16() for _ in range(2)]
    pos = _i32([8999, 499, 19999], gpu)
    want = [kv8.decode_attention(q, p, pos, None, 20000) for q in qs]
    graphs = []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            out = kv8.decode_attention(q, p, pos, None, 20000)
        graphs.append((g, out))
    for i in range(6):
        graphs[i % 2][0].replay()
        eager = kv8.decode_attention(qs[1 - i % 2], p, pos, None, 20000)
        torch.cuda.synchronize()
        assert torch.equal(graphs[i % 2][1], want[i % 2]) and torch.equal(eager, want[1 - i % 2])
