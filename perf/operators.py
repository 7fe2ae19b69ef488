"""The operators around a key/value cache that is held in 8 bits, as cases that can be timed and compared.

Kinds of case:
  * ``norm``: RMS norm of every query and key head with the position rotation in the same pass, from the rows of
    the qkv projection to the head-major layout of attention; with ``grad`` the gradients of rows and weights too;
  * ``tokens``: one token of each of ``batch`` sequences appended to the paged 8-bit cache (rotated on the way,
    normed first where ``norm`` says so), its group of cached rows read back;
  * ``prompts``: ``seqs`` runs of ``lo`` to ``hi`` tokens appended at once, from position 0 or further on
    (``start``), read back;
  * ``attend``: attention of one token of each of ``batch`` sequences of ``lo`` to ``hi`` cached tokens.

The cache: pages of ``block`` positions of every key/value head, e4m3 codes with one power of two for each group of
16 positions of a head, keys and values apart.  A group's exponent byte e stands for 2 ** (e - 127); a token alone
would take the least e of 1 to 254 with amax <= 448 * 2 ** (e - 127) (values that are no numbers do not count), and a
group takes the largest of its tokens'.  Rows of a group that were held before are rounded again where it grows.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

GROUP, TOP, EPS, BASE = 16, 448.0, 1e-5, 500000.0
BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
E4M3 = torch.float8_e4m3fn
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------- cases
def _norm(name, batch, seq, hq, hkv, d, grad, packed=False):
    return {"name": name, "kind": "norm", "batch": batch, "seq": seq, "hq": hq, "hkv": hkv, "d": d, "grad": grad,
            "packed": packed}


def _tokens(name, batch, lo, hi, hq, hkv, d, norm, block=256):
    return {"name": name, "kind": "tokens", "batch": batch, "lo": lo, "hi": hi, "hq": hq, "hkv": hkv, "d": d,
            "norm": norm, "block": block}


def _prompts(name, seqs, lo, hi, start, hq, hkv, d, norm, block=256):
    return {"name": name, "kind": "prompts", "seqs": seqs, "lo": lo, "hi": hi, "start": start, "hq": hq, "hkv": hkv,
            "d": d, "norm": norm, "block": block}


def _attend(name, batch, lo, hi, hq, hkv, d, block=256):
    return {"name": name, "kind": "attend", "batch": batch, "lo": lo, "hi": hi, "hq": hq, "hkv": hkv, "d": d,
            "block": block}


def listed():
    return [
        # a short prompt of a small model, nothing to train: the latency of a launch
        _norm("norm_short_prompt", 1, 17, 32, 8, 64, False),
        # a training step's two sequences at the 8B head layout
        _norm("norm_train_2x2048", 2, 2048, 32, 8, 128, True),
        # an odd batch of heads of 64, rows packed from documents of their own positions
        _norm("norm_train_packed", 3, 1001, 32, 8, 64, True, True),
        # the widest head layout over one long sequence
        _norm("norm_train_long", 1, 8192, 64, 8, 128, True),
        # one user of a small model
        _tokens("tokens_b1", 1, 700, 700, 32, 8, 64, False),
        # a full batch of a large model with normed heads
        _tokens("tokens_b64", 64, 100, 4000, 64, 8, 128, True),
        # a handful of short requests admitted together
        _prompts("prompts_ragged", 6, 17, 901, 0, 32, 8, 64, False),
        # one long document that goes on where an earlier part ended, inside a group
        _prompts("prompt_goes_on", 1, 4096, 4096, 1003, 32, 8, 128, True),
        # one user, small heads: latency
        _attend("attend_b1_d64", 1, 700, 700, 32, 8, 64),
        # a busy server: requests of unlike lengths
        _attend("attend_b32_ragged", 32, 100, 2000, 32, 8, 128),
        # few users with long documents
        _attend("attend_b8_16384", 8, 16384, 16384, 32, 8, 128),
        # a full batch of a large model
        _attend("attend_b64_4096", 64, 2048, 4096, 64, 8, 128),
    ]


_HEADS = [(32, 8, 128), (64, 8, 128), (32, 8, 64), (8, 2, 32), (4, 2, 128), (12, 12, 64), (28, 4, 128), (40, 5, 64)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["norm", "tokens", "prompts", "attend"], [3, 2, 2, 4])[0]
    hq, hkv, d = rng.choice(_HEADS)
    block = rng.choice([256, 256, 512, 64, 16])
    if kind == "norm":
        rows = _log(rng, 1, 8192)
        batch = min(rows, rng.choice([1, 1, 2, 3, 5]))
        return _drawn(_norm("", batch, max(1, rows // batch), hq, hkv, d, rng.random() < 0.7, rng.random() < 0.3))
    if kind == "tokens":
        hi = _log(rng, 1, 4000)
        return _drawn(_tokens("", _log(rng, 1, 96), _log(rng, 1, hi), hi, hq, hkv, d, rng.random() < 0.5, block))
    if kind == "prompts":
        seqs = rng.choice([1, 1, 2, 3, 6])
        hi = _log(rng, 1, 6000 // seqs)
        start = rng.choice([0, 0, rng.randrange(1, 2000)])
        return _drawn(_prompts("", seqs, _log(rng, 1, hi), hi, start, hq, hkv, d, rng.random() < 0.5, block))
    batch = _log(rng, 1, 64)
    hi = _log(rng, 1, min(65536, 180000 // batch))
    return _drawn(_attend("", batch, _log(rng, 1, hi), hi, hq, hkv, d, block))


def _drawn(case):
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=F32)


def _rows(g, n, heads, d):
    """Rows of a qkv projection: channels and tokens of unlike size."""
    x = _normal(g, n, heads, d) * torch.exp(0.5 * _normal(g, 1, heads, d)) * torch.exp(0.5 * _normal(g, n, 1, 1))
    return x.to(BF).reshape(n, heads * d)


def _tables(n, d):
    ang = torch.outer(torch.arange(n, dtype=F64, device=DEV),
                      BASE ** (-torch.arange(0, d, 2, dtype=F64, device=DEV) / d))
    return ang.cos().to(F32), ang.sin().to(F32)


def _lengths(case, count, seed):
    r = np.random.RandomState(seed % (1 << 31))
    return r.randint(case["lo"], case["hi"] + 1, count)


def _counts(case):
    """Tokens of each run of ``prompts``: the case's own, as the sizes of what a pass returns go by them."""
    r = np.random.RandomState(1009 * case["hi"] + 31 * case["lo"] + case["seqs"])
    return r.randint(case["lo"], case["hi"] + 1, case["seqs"])


def _up(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).to(DEV)


def _fill(g, pool, hkv, block, d):
    """Codes and exponents of a pool that sequences have been appended to, page by page: random bits of sane sizes."""
    n = pool * hkv * (block // GROUP)
    codes = torch.empty(n, GROUP, d, dtype=torch.uint8, device=DEV)
    exps = torch.empty(n, dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 25) // (GROUP * d))
    size = torch.exp(0.5 * _normal(g, d))
    for a in range(0, n, step):  # (a part at a time: the f32 values of a large pool are many times its size)
        m = min(step, n - a)
        x = (_normal(g, m, GROUP, d) * size).to(BF).to(F32)
        e = _exponent(x.abs().amax((1, 2)))
        exps[a:a + m] = e.to(torch.uint8)
        codes[a:a + m] = _codes(x, e[:, None, None])
    return codes.view(pool, hkv, block, d), exps.view(pool, hkv, block // GROUP)


def _cache(g, caps, hkv, block, d):
    """Pages for sequences that hold up to ``caps`` positions each, dealt out of a pool in no order."""
    pages = [max(1, -(-int(c) // block)) for c in caps]
    pool, width = sum(pages) + 1, max(pages)
    order = torch.randperm(pool, generator=g, device=DEV).to(I32)
    table = torch.zeros(len(caps), width, dtype=I32, device=DEV)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        table[i, n:] = order[at + n - 1]
        at += n
    k, ke = _fill(g, pool, hkv, block, d)
    v, ve = _fill(g, pool, hkv, block, d)
    return {"k": k, "v": v, "ke": ke, "ve": ve, "table": table}


def prepare(case, seed):
    g = torch.Generator(DEV)
    g.manual_seed(int(seed))
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    nh, kind = hq + 2 * hkv, case["kind"]
    s = {"case": case}
    if kind == "norm" or case.get("norm"):
        s["wq"] = (1 + 0.2 * _normal(g, d)).to(BF)
        s["wk"] = (1 + 0.2 * _normal(g, d)).to(BF)
    if kind == "norm":
        b, n = case["batch"], case["seq"]
        s["qkv"] = _rows(g, b * n, nh, d)
        s["cos"], s["sin"] = _tables(n, d)
        if case["packed"]:  # documents of random lengths, each from position 0
            new = torch.rand(b * n, generator=g, device=DEV) < 4.0 / n
            new[::n] = True
            at = torch.arange(b * n, device=DEV)
            s["positions"] = (at - torch.cummax(torch.where(new, at, 0), 0).values).to(I32)
        if case["grad"]:
            s["gq"] = _normal(g, b, hq, n, d).to(BF)
            s["gk"] = _normal(g, b, hkv, n, d).to(BF)
            s["gv"] = _normal(g, b, hkv, n, d).to(BF)
        return s
    if kind == "attend":
        lens = _lengths(case, case["batch"], seed)
        s.update(_cache(g, lens, hkv, case["block"], d))
        s["q"] = _normal(g, case["batch"], hq, d).to(BF)
        s["pos"], s["slots"], s["max_len"] = _up(lens - 1), _up(np.arange(len(lens))), int(lens.max())
        return s
    if kind == "tokens":
        lens = _lengths(case, case["batch"], seed)
        pos = lens - 1
        s["pos"] = _up(pos)
        starts, ends, n = pos // GROUP * GROUP, lens, GROUP
        s["qkv"] = _rows(g, len(lens), nh, d)
    else:
        counts = np.random.RandomState(seed % (1 << 31)).permutation(_counts(case))
        ends = case["start"] + counts
        lens, starts, n = ends, np.full(len(counts), case["start"]), int(counts.max())
        runs, row = [], 0  # (first row, rows, slot, first position): what lies in one group of positions
        for slot, end in enumerate(ends):
            p = case["start"]
            while p < end:
                m = min(int(end), (p // GROUP + 1) * GROUP) - p
                runs.append((row, m, slot, p))
                row, p = row + m, p + m
        s["runs"] = _up(np.array(runs).reshape(-1, 4))
        s["qkv"] = _rows(g, row, nh, d)
    s.update(_cache(g, lens, hkv, case["block"], d))
    s["cos"], s["sin"] = _tables(int(max(ends)), d)
    s["slots"], s["starts"], s["ends"], s["n"] = _up(np.arange(len(lens))), _up(starts), _up(ends), n
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _exponent(amax):
    """The least exponent byte under which amax fits e4m3 (f32 in, int32 out)."""
    m, x = torch.frexp(amax)
    e = (x - 1) - 8 + (m > 0.875).to(I32) + 127
    return torch.where(amax > 0, e, 1).clamp(1, 254).to(I32)


def _codes(x, e):
    """e4m3 codes (uint8) of f32 values under exponent bytes e."""
    return torch.ldexp(x, 127 - e).to(E4M3).view(torch.uint8)


def _values(codes, e):
    return torch.ldexp(codes.view(E4M3).to(F32), e.to(I32) - 127)


def _rotated(x, w, cos, sin):
    """x [rows, heads, d] f32 -> the heads normed (where w is given) and rotated; cos, sin [rows, 1, d / 2]."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(F32)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _heads(s, positions):
    c = s["case"]
    x = s["qkv"].view(-1, c["hq"] + 2 * c["hkv"], c["d"]).to(F32)
    q, k, v = x.split([c["hq"], c["hkv"], c["hkv"]], 1)
    cos, sin = s["cos"][positions][:, None], s["sin"][positions][:, None]
    return q, k, v, cos, sin


def _plain_norm(s):
    c = s["case"]
    b, n, hq, hkv, d = c["batch"], c["seq"], c["hq"], c["hkv"], c["d"]
    pos = s["positions"].long() if c["packed"] else torch.arange(n, device=DEV).repeat(b)
    q, k, v, cos, sin = _heads(s, pos)

    def out(x):
        return x.view(b, n, -1, d).transpose(1, 2).contiguous().to(BF)

    got = [out(_rotated(q, s["wq"], cos, sin)), out(_rotated(k, s["wk"], cos, sin)), out(v)]
    if not c["grad"]:
        return got

    def back(x, w, g):
        g = g.transpose(1, 2).reshape(b * n, -1, d).to(F32)
        ga, gb = g.chunk(2, -1)
        g = torch.cat([ga * cos + gb * sin, gb * cos - ga * sin], -1)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        dw = (g * x * r).sum((0, 1))
        g = g * w.to(F32)
        return r * (g - x * (r * r) * (g * x).mean(-1, keepdim=True)), dw.to(BF)

    dq, dwq = back(q, s["wq"], s["gq"])
    dk, dwk = back(k, s["wk"], s["gk"])
    dv = s["gv"].transpose(1, 2).reshape(b * n, hkv, d).to(F32)
    return got + [torch.cat([dq, dk, dv], 1).reshape(b * n, -1).to(BF), dwq, dwk]


def _plain_store(s, name, x, rows, slot, group, block):
    """Rows x [tokens, hkv, d] f32 into the cache: rows [n, 16] say which token a group's row gets (-1: none)."""
    codes, exps = s[name], s[name + "e"]
    page = s["table"][slot.long(), (group * GROUP // block).long()].long()
    sub = (group % (block // GROUP)).long()
    paged = codes.view(*codes.shape[:2], block // GROUP, GROUP, codes.shape[3])
    old, old_e = paged[page, :, sub], exps[page, :, sub].to(I32)  # [n, hkv, 16, d], [n, hkv]
    new = rows >= 0
    x = x[rows.clamp_min(0).long()].transpose(1, 2)  # [n, hkv, 16, d]
    amax = torch.where(new[:, None, :, None] & torch.isfinite(x), x.abs(), 0.0).amax((2, 3))
    last = torch.where(new, torch.arange(GROUP, device=DEV), -1).amax(1, keepdim=True)
    kept = ~new & (torch.arange(GROUP, device=DEV) < last)  # held before, ahead of the newest row
    e = _exponent(amax)
    e = torch.where(kept.any(1)[:, None], torch.maximum(e, old_e), e)
    wide = e[:, :, None, None]
    again = _codes(_values(old, old_e[:, :, None, None]), wide)
    put = torch.where(new[:, None, :, None], _codes(x, wide), torch.where(kept[:, None, :, None], again, old))
    paged[page, :, sub] = put
    exps[page, :, sub] = e.to(torch.uint8)


def _plain_read(s, name):
    """Positions starts .. ends of every sequence as bf16 [batch, hkv, n, d], zero behind the end."""
    block = s["case"]["block"]
    at = s["starts"][:, None].long() + torch.arange(s["n"], device=DEV)
    there = at < s["ends"][:, None]
    at = torch.where(there, at, s["starts"][:, None].long())
    page = torch.gather(s["table"][s["slots"].long()].long(), 1, at // block)
    row = at % block
    x = _values(s[name][page, :, row], s[name + "e"][page, :, row // GROUP][..., None])  # [batch, n, hkv, d]
    return torch.where(there[:, :, None, None], x, 0.0).transpose(1, 2).contiguous().to(BF)


def _plain_append(s):
    c = s["case"]
    if c["kind"] == "tokens":
        pos, slot = s["pos"].long(), s["slots"]
        group = pos // GROUP
        rows = torch.where(torch.arange(GROUP, device=DEV) == (pos % GROUP)[:, None],
                           torch.arange(len(pos), device=DEV)[:, None], -1)
    else:
        row, count, slot, first = s["runs"].long().unbind(1)
        group, at = first // GROUP, torch.arange(GROUP, device=DEV) - (first % GROUP)[:, None]
        rows = torch.where((at >= 0) & (at < count[:, None]), row[:, None] + at, -1)
        pos = torch.zeros(s["qkv"].shape[0] + 1, dtype=torch.long, device=DEV)
        pos[rows] = group[:, None] * GROUP + torch.arange(GROUP, device=DEV)  # (-1: the spare row)
        pos = pos[:-1]
    q, k, v, cos, sin = _heads(s, pos)
    q, k = _rotated(q, s.get("wq"), cos, sin), _rotated(k, s.get("wk"), cos, sin)
    _plain_store(s, "k", k, rows, slot, group, c["block"])
    _plain_store(s, "v", v, rows, slot, group, c["block"])
    got = [q.to(BF)] if c["kind"] == "tokens" else [x.transpose(0, 1).contiguous().to(BF) for x in (q, k, v)]
    return got + [_plain_read(s, "k"), _plain_read(s, "v")]


def _plain_attend(s):
    c = s["case"]
    b, hkv, d, block = c["batch"], c["hkv"], c["d"], c["block"]
    pages = s["table"][s["slots"].long(), :-(-s["max_len"] // block)].long()

    def whole(name):  # [b, hkv, positions, d] f32
        x = s[name][pages].view(b, -1, hkv, block // GROUP, GROUP, d)
        x = _values(x, s[name + "e"][pages].view(b, -1, hkv, block // GROUP, 1, 1))
        return x.transpose(1, 2).reshape(b, hkv, -1, d)

    q = s["q"].to(F32).view(b, hkv, -1, d)
    k = whole("k")
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(d)
    there = torch.arange(k.shape[2], device=DEV) <= s["pos"][:, None]
    score = score.masked_fill(~there[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(p, whole("v") * there[:, None, :, None]) / p.sum(-1, keepdim=True)
    return o.reshape(b, -1).to(BF)


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    c = state["case"]
    if own:
        return _own(state)
    if c["kind"] == "norm":
        return _plain_norm(state)
    return _plain_attend(state) if c["kind"] == "attend" else _plain_append(state)


def _own(s):
    from mxllm.ops import kv8, qk_norm_rope

    c = s["case"]
    if c["kind"] == "norm":
        args = (s["cos"], s["sin"], c["batch"], c["seq"], c["hq"], c["hkv"], c["d"], EPS, s.get("positions"))
        if not c["grad"]:
            return list(qk_norm_rope(s["qkv"], s["wq"], s["wk"], *args))
        leaves = [s[n].detach().requires_grad_() for n in ("qkv", "wq", "wk")]
        out = qk_norm_rope(*leaves, *args)
        return [x.detach() for x in out] + list(torch.autograd.grad(out, leaves, (s["gq"], s["gk"], s["gv"])))
    pages = kv8.Pages(s["k"], s["v"], s["ke"], s["ve"], s["table"])
    if c["kind"] == "attend":
        return kv8.decode_attention(s["q"], pages, s["pos"], s["slots"], s["max_len"])
    norms = (s.get("wq"), s.get("wk"), EPS)
    if c["kind"] == "tokens":
        got = [kv8.append_tokens(s["qkv"], s["cos"], s["sin"], s["pos"], s["slots"], pages, c["hq"], *norms)]
    else:
        got = list(kv8.append_prompts(s["qkv"], s["cos"], s["sin"], s["runs"], pages, c["hq"], *norms))
    return got + list(kv8.read(pages, s["slots"], s["starts"], s["ends"], s["n"]))


def work(case):
    hq, hkv, d, kind = case["hq"], case["hkv"], case["d"], case["kind"]
    nh = hq + 2 * hkv
    if kind == "norm":
        rows = case["batch"] * case["seq"]
        table = case["seq"] * d * 4
        move = 2 * rows * nh * d * 2 + table  # rows in, heads out
        if case["grad"]:  # the gradients in, the rows' gradient out
            move += 2 * rows * nh * d * 2
        return {"bytes": move, "flops": rows * nh * d * (30 if case["grad"] else 10)}
    mean = (case["lo"] + case["hi"]) / 2
    if kind == "attend":
        keys = case["batch"] * mean
        return {"bytes": keys * hkv * 2 * (d + 1 / GROUP) + case["batch"] * hq * d * 4, "flops": 4 * keys * hq * d}
    if kind == "tokens":  # rows in, q out; codes out, the groups' codes in and their values out
        b = case["batch"]
        return {"bytes": b * (nh * d * 2 + hq * d * 2 + 2 * hkv * d * (1 + GROUP * 3) + 4 * d), "flops": b * nh * d * 10}
    rows = int(_counts(case).sum())  # rows in, heads out; codes out and in, values out
    return {"bytes": rows * (2 * nh * d * 2 + 2 * hkv * d * 4 + 4 * d), "flops": rows * nh * d * 10}


# ---------------------------------------------------------------------------------------------------- 64 bits
def _e4m3(x):
    """x (f64) at the nearest value of e4m3, ties to even, as f64; what is no number as NaN."""
    size = x.abs()
    ulp = torch.exp2(torch.floor(torch.log2(size.clamp_min(2.0 ** -6))).clamp(-6, 8) - 3)
    return torch.where(torch.isfinite(x), torch.round(x / ulp) * ulp, math.nan)


def _power(amax):
    """The least power of two p of 2^-126 .. 2^127 with amax <= 448 p (f64)."""
    e = torch.ceil(torch.log2((amax / TOP).clamp_min(2.0 ** -140)))
    e = torch.where(torch.ldexp(torch.full_like(e, TOP / 2), e.to(I32)) >= amax, e - 1, e)  # (the logarithm's rounding)
    return torch.exp2(torch.where(torch.exp2(e) * TOP < amax, e + 1, e).clamp(-126, 127))


def _exact_heads(rows, heads, d, w, cos, sin):
    """Heads of f64 rows normed and turned, as products of complex numbers."""
    x = rows.to(F64).view(-1, heads, d)
    if w is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + EPS) * w.to(F64)
    z = torch.complex(x[..., :d // 2], x[..., d // 2:]) * torch.complex(cos.to(F64), sin.to(F64))[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_norm(s):
    c = s["case"]
    b, n, hq, hkv, d = c["batch"], c["seq"], c["hq"], c["hkv"], c["d"]
    pos = (s["positions"].view(b, n) if c["packed"] else torch.arange(n, device=DEV).expand(b, n)).long()
    x = s["qkv"].to(F64).view(b * n, -1, d)
    leaves = [x.requires_grad_(), s["wq"].to(F64).requires_grad_(), s["wk"].to(F64).requires_grad_()]
    cos, sin = s["cos"][pos].view(b * n, -1), s["sin"][pos].view(b * n, -1)
    with torch.enable_grad():
        parts = [_exact_heads(leaves[0][:, :hq], hq, d, leaves[1], cos, sin),
                 _exact_heads(leaves[0][:, hq:hq + hkv], hkv, d, leaves[2], cos, sin), leaves[0][:, hq + hkv:]]
        out = [p.reshape(b, n, -1, d).permute(0, 2, 1, 3) for p in parts]
        if c["grad"]:
            grads = torch.autograd.grad(out, leaves, [s[k].to(F64) for k in ("gq", "gk", "gv")])
    out = [o.detach().contiguous() for o in out]
    return out if not c["grad"] else out + [grads[0].reshape(b * n, -1), grads[1], grads[2]]


def _exact_append(s):
    c = s["case"]
    hq, hkv, d, block = c["hq"], c["hkv"], c["d"], c["block"]
    starts, ends = s["starts"].tolist(), s["ends"].tolist()
    if c["kind"] == "tokens":
        spans = [(i, p, p + 1) for i, p in enumerate(s["pos"].tolist())]
    else:
        spans = [(i, a, e) for i, (a, e) in enumerate(zip(starts, ends))]
    qs, ks, vs = [], [], []
    kept = {"k": torch.zeros(len(spans), hkv, s["n"], d, dtype=F64, device=DEV)}
    kept["v"] = torch.zeros_like(kept["k"])
    row = 0
    for slot, a, e in spans:
        x = s["qkv"][row:row + e - a].view(e - a, -1, d)
        row += e - a
        cos, sin = s["cos"][a:e], s["sin"][a:e]
        qs.append(_exact_heads(x[:, :hq], hq, d, s.get("wq"), cos, sin))
        ks.append(_exact_heads(x[:, hq:hq + hkv], hkv, d, s.get("wk"), cos, sin))
        vs.append(x[:, hq + hkv:].to(F64))
        g0, g1 = a // GROUP, -(-e // GROUP)
        for name, new in (("k", ks[-1]), ("v", vs[-1])):
            whole = torch.zeros(g1 - g0, GROUP, hkv, d, dtype=F64, device=DEV)
            flat = whole.view(-1, hkv, d)
            flat[a - g0 * GROUP:e - g0 * GROUP] = new
            size = torch.where(torch.isfinite(whole), whole.abs(), 0.0).amax((1, 3))
            power = _power(size)
            ahead = a - g0 * GROUP
            if ahead:  # rows held before, in the first group
                page, at = int(s["table"][slot, g0 * GROUP // block]), g0 * GROUP % block
                was = torch.exp2(s[name + "e"][page, :, at // GROUP].to(F64) - 127)
                power[0] = torch.maximum(power[0], was)
                flat[:ahead] = (s[name][page, :, at:at + ahead].view(E4M3).to(F64) * was[:, None, None]).transpose(0, 1)
            got = (_e4m3(whole / power[:, None, :, None]) * power[:, None, :, None]).view(-1, hkv, d)
            lo = starts[slot] - g0 * GROUP
            kept[name][slot, :, :e - starts[slot]] = got[lo:e - g0 * GROUP].transpose(0, 1)
    if c["kind"] == "tokens":
        return [torch.cat(qs), kept["k"], kept["v"]]
    return [torch.cat(x).transpose(0, 1).contiguous() for x in (qs, ks, vs)] + [kept["k"], kept["v"]]


def _exact_attend(s):
    c = s["case"]
    hkv, d, block = c["hkv"], c["d"], c["block"]
    out = []
    for i, p in enumerate(s["pos"].tolist()):
        pages = s["table"][i, :p // block + 1].long()

        def whole(name):  # [hkv, positions, d]
            e = s[name + "e"][pages].to(F64).repeat_interleave(GROUP, 2)[..., None]
            x = s[name][pages].view(E4M3).to(F64) * torch.exp2(e - 127)
            return x.permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :p + 1]

        q = s["q"][i].to(F64).view(hkv, -1, d)
        w = torch.softmax(q @ whole("k").transpose(1, 2) / math.sqrt(d), -1)
        out.append((w @ whole("v")).reshape(-1))
    return torch.stack(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(s)
    return _exact_attend(s) if case["kind"] == "attend" else _exact_append(s)
