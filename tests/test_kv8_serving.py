"""``Engine(kv_dtype="e4m3")`` beside the engine's other choices: tensor parallelism, e4m3 projection weights, the server's loop."""
import os

import pytest
import torch
import torch.multiprocessing as mp

from mxllm.models import Llama, get_config
from mxllm.serve.engine import Engine
from mxllm.serve.kvcache import KV8Cache

from .test_kv8_engine import _logits
from .test_tensor_parallel import PROMPTS, _model, _port

STEPS = 6


def _steps(engine):
    slots = list(range(len(PROMPTS)))
    out = [engine.prefill_batch(slots, PROMPTS)]
    for i in range(STEPS):
        out.append(engine.decode(slots, torch.tensor([p[i % 3] for p in PROMPTS])).float())
    return torch.stack(out)


def _worker(rank, world, port, out_q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), MXLLM_FORCE_CPU="1")
    torch.set_num_threads(1)
    import torch.distributed as dist

    from mxllm.parallel import runtime
    from mxllm.parallel.tensor import shard_llama

    runtime.init(rank=rank, world_size=world)
    engine = Engine(shard_llama(_model(), rank, world), max_batch=4, max_seq=64, tp_group=dist.group.WORLD, kv_dtype="e4m3")
    logits = _steps(engine)
    everyone = [torch.zeros_like(logits) for _ in range(world)]
    dist.all_gather(everyone, logits)
    if rank == 0:
        out_q.put((logits.numpy(), all(torch.equal(logits, x) for x in everyone), tuple(engine.kv.k_exp[0].shape)))
    runtime.cleanup()


@pytest.mark.parametrize("world", [2, 4])
def test_tensor_parallel_shards_keep_their_heads(world):
    """Every rank has the keys and values of its own heads, with exponents of their own.  Sums over ranks are f32 in another order, so a
    code of some thousands may fall the other way: one of a few keys by 2^-3, the logits of a step by much less than half
    of 2^-5.5, what rounding all of them does (tests/test_kv8_engine.py)."""
    want = _steps(Engine(_model(), max_batch=4, max_seq=64, kv_dtype="e4m3"))
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    got, same, exps = q.get(timeout=240)
    got = torch.from_numpy(got)  # (a tensor would be shared, and its process is gone)
    for p in procs:
        p.join(60)
        assert p.exitcode == 0
    assert same and exps[1] == 4 // world
    assert torch.allclose(got[0], want[0], atol=1e-4, rtol=1e-4)  # (prompts attend to what is not rounded)
    assert float((got - want).norm() / want.norm()) < 2.0 ** -6.5


def test_server_loop():
    """Requests through the engine's own thread, more than it has slots, get what ``generate`` gives."""
    from mxllm.serve.engine import SamplingParams

    want = Engine(_model(), max_batch=2, max_seq=64, kv_dtype="e4m3").generate(PROMPTS, max_new_tokens=5)
    engine = Engine(_model(), max_batch=2, max_seq=64, kv_dtype="e4m3", kv_pool_tokens=512)
    assert isinstance(engine.kv, KV8Cache)
    engine.start()
    requests = [engine.submit(p, SamplingParams(max_new_tokens=5)) for p in PROMPTS]
    for r in requests:
        assert r.done.wait(120)
    engine.stop()
    assert [r.output for r in requests] == want


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiny", "tiny-d128"])
def test_fp8_weights(gpu, name):
    """e4m3 projections with either cache: logits as far apart as with bf16 projections (tests/test_kv8_engine.py: 3 * 2^-5.5 of them),
    prompts' by bf16's roundings alone; steps replayed as graphs are the eager ones."""
    from mxllm.serve.quant import W8Linear, quantize_model_fp8_

    m = Llama(get_config(name), device=gpu, seed=0).eval()
    assert quantize_model_fp8_(m) > 0 and isinstance(m.layers[0].wqkv, W8Linear)
    prompts = [list(range(1, n)) for n in (20, 130, 400)]

    def logits(**kw):
        return _logits(Engine(m, max_batch=3, max_seq=1024, **kw), prompts, 8)

    wide, narrow, eager = logits(kv_dtype="bf16"), logits(kv_dtype="e4m3"), logits(kv_dtype="e4m3", use_graphs=False)
    assert torch.allclose(wide[0], narrow[0], rtol=0, atol=2.0 ** -7 * float(wide[0].abs().max()))
    assert float((wide[1:] - narrow[1:]).norm() / wide[1:].norm()) < 3 * 2.0 ** -5.5
    assert float((eager - narrow).norm() / narrow.norm()) < 2.0 ** -6


@pytest.mark.gpu
def test_server_loop_over_graphs(gpu):
    """The engine's thread beside this one, steps of growing and shrinking batches replayed as graphs: requests end, with as many
    tokens as they asked for, and their blocks come back."""
    from mxllm.serve.engine import SamplingParams

    m = Llama(get_config("tiny-d128"), device=gpu, seed=0).eval()
    engine = Engine(m, max_batch=4, max_seq=1024, kv_pool_tokens=4096, kv_dtype="e4m3")
    free = engine.kv.free_blocks
    engine.start()
    requests = [engine.submit(list(range(1, 5 + 37 * i)), SamplingParams(max_new_tokens=3 + 5 * (i % 4))) for i in range(11)]
    for r in requests:
        assert r.done.wait(100)
    engine.stop()
    assert [len(r.output) for r in requests] == [3 + 5 * (i % 4) for i in range(11)] and engine.kv.free_blocks == free
