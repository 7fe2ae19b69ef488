"""The serving engine over a key/value cache in 8 bits (``Engine(kv_dtype="e4m3")``): the same schedule as over bf16, a cache of half
the size that holds what prompts and tokens appended, and logits near those of the bf16 cache."""
import pytest
import torch

from mxllm.models import Llama, get_config
from mxllm.ops import kv8
from mxllm.serve.engine import Engine
from mxllm.serve.kvcache import KV8Cache, KVCache


def _prompts():
    return [[i, i + 3, i + 7, 11] * (1 + 5 * (i % 3)) for i in range(1, 8)]


def _model(device="cpu", name="tiny"):
    return Llama(get_config(name), device=device, seed=0).eval()


def test_paged_engine_matches_static():
    m = _model()
    static = Engine(m, max_batch=4, max_seq=512, kv_dtype="e4m3")
    paged = Engine(m, max_batch=4, max_seq=512, kv_pool_tokens=1024, kv_dtype="e4m3")
    a, b = (e.generate(_prompts(), max_new_tokens=6) for e in (static, paged))
    assert a == b and paged.kv.free_blocks == 4 and isinstance(paged.kv, KV8Cache)


def test_cache_takes_half_and_reads_back():
    m = _model()
    a, b = (Engine(m, max_batch=2, max_seq=512, kv_dtype=d) for d in ("bf16", "e4m3"))
    size = a.kv.nbytes() / 2
    assert size <= b.kv.nbytes() <= size * (1 + 1 / (16 * 32)) + 1
    for e in (a, b):
        e.prefill(1, list(range(1, 40)))
    for x, y in zip(a.kv.gather(0, 1, 39), b.kv.gather(0, 1, 39)):
        err = (x.double() - y.double()).abs()  # half a step of e4m3, or of its smallest numbers, and bf16's of x itself
        assert bool((err <= (2.0 ** -4 + 2.0 ** -8) * x.double().abs() + 2.0 ** -17 * 2 * float(x.abs().max())).all())
    with pytest.raises(NotImplementedError):
        b.kv.write(0, 0, torch.zeros(2, 4, 32), torch.zeros(2, 4, 32))


def test_a_slot_is_used_again():
    """A second request in a slot sees nothing of the first one's groups."""
    m = _model()
    e = Engine(m, max_batch=1, max_seq=512, kv_dtype="e4m3")
    first = e.generate([[5, 6, 7] * 9], max_new_tokens=5)
    e.generate([[500, 400, 300, 200] * 20], max_new_tokens=9)
    assert e.generate([[5, 6, 7] * 9], max_new_tokens=5) == first


def test_choice_of_type(monkeypatch):
    m = _model()
    assert type(Engine(m, max_batch=1, max_seq=256).kv) is KVCache
    monkeypatch.setenv("MXLLM_KV_DTYPE", "e4m3")
    e = Engine(m, max_batch=1, max_seq=256)
    assert type(e.kv) is KV8Cache and e.model_steps.cached_bytes(16) == 2 * 2 * 2 * (16 * 32 + 1)
    assert type(Engine(m, max_batch=1, max_seq=256, kv_dtype="bf16").kv) is KVCache
    with pytest.raises(ValueError):
        Engine(m, max_batch=1, kv_dtype="int8")
    from mxllm.models.revesun import Revesun

    with pytest.raises(ValueError):
        Engine(Revesun(get_config("revesun-tiny")), max_batch=1, max_seq=256)


def _logits(engine, prompts, steps):
    slots = list(range(len(prompts)))
    for s, p in zip(slots, prompts):
        engine.reserve(s, len(p) + steps + 1)
    out = [engine.prefill_batch(slots, prompts)]
    tokens = torch.tensor([p[0] for p in prompts])
    for i in range(steps):
        out.append(engine.decode(slots, tokens + i).float())
    return torch.stack(out).double().cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiny", "tiny-d128"])
def test_graphed_steps_are_the_eager_ones(gpu, name):
    m = _model(gpu, name)
    eager, graphed = (Engine(m, max_batch=5, max_seq=2048, use_graphs=g, kv_pool_tokens=4096, kv_dtype="e4m3") for g in (False, True))
    prompts = [list(range(1, n)) for n in (2, 17, 40, 300, 511)]
    a, b = (_logits(e, prompts, 20) for e in (eager, graphed))
    # (steps padded to other batches take other GEMM tiles: near, not equal)
    assert float((a - b).norm() / a.norm()) < 2.0 ** -7
    for i in range(2):
        for j, p in enumerate(prompts):
            x, y = (e.kv.gather(0, j, len(p) + 20)[i].double() for e in (eager, graphed))
            assert float((x - y).norm() / x.norm()) < 2.0 ** -7


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiny", "tiny-d128"])
def test_logits_near_those_over_bf16(gpu, name):
    """Keys and values off by up to 2^-4, about 2^-5.5 of them on average (uniform over half a step, of values spread over an octave),
    at random: the attention's outputs, sums of many, by less, and the logits of two layers by a few 2^-5.5 of themselves."""
    m = _model(gpu, name)
    a, b = (_logits(Engine(m, max_batch=3, max_seq=1024, kv_dtype=d), [list(range(1, n)) for n in (20, 130, 400)], 8) for d in ("bf16", "e4m3"))
    assert torch.allclose(a[0], b[0], rtol=0, atol=2.0 ** -7 * float(a[0].abs().max()))  # a prompt attends to what is not rounded
    assert float((a[1:] - b[1:]).norm() / a[1:].norm()) < 3 * 2.0 ** -5.5


@pytest.mark.gpu
def test_a_full_group_of_slots_and_prompts(gpu):
    m = _model(gpu, "tiny-d128")
    e = Engine(m, max_batch=8, max_seq=1024, kv_pool_tokens=8192, kv_dtype="e4m3")
    one = Engine(m, max_batch=1, max_seq=1024, kv_dtype="e4m3", use_graphs=False)
    prompts = [list(range(3, 3 + n)) for n in (1, 15, 16, 17, 255, 256, 257, 400)]
    slots = list(range(8))
    for s, p in zip(slots, prompts):
        e.reserve(s, len(p) + 4)
    e.prefill_batch(slots, prompts)
    for s, p in zip(slots, prompts):
        one.prefill(0, p)
        for x, y in zip(e.kv.gather(1, s, len(p)), one.kv.gather(1, 0, len(p))):
            assert float((x.double() - y.double()).norm() / y.double().norm()) < 2.0 ** -7
    assert e.kv.pages(0).nbytes() == kv8.Pages.empty(*e.kv.k[0].shape, e.kv.bt).nbytes()
