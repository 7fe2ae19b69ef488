"""Keys and values held in 8 bits: appending to a paged cache, attention over it, reading it back.

Per layer the cache is ``Pages``: e4m3 codes [pages, Hkv, block, D] and exponent bytes [pages, Hkv, block / 16], keys and
values apart, and the block table of the sequences' slots.  The 16 positions of a group of one head share a power of two:
a code c under exponent byte e stands for c * 2 ** (e - 127).  One token alone would take the least e of 1 .. 254 with
amax <= 448 * 2 ** (e - 127); a group takes the largest of its tokens'.  The codes have exponents of their own, so a
power of two more costs no precision but for values 2 ** -14 of the group's largest and smaller, and rows that are rounded
again as their group grows keep their values down to there.  Values that are no numbers are held as NaN and do not count in amax.

A position written starts its group afresh where it is the group's first; else the rows ahead of it are kept.  Rows behind the
newest position are nobody's: their codes stay, and mean something else once the group grows.

GPU: csrc/kernels/kv8.hip, kv8_attn.hip (heads of 32, 64, 128; blocks of any multiple of 16 positions; up to 16 query
heads a key head).  CPU: the same in plain PyTorch.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import reference as ref
from ._ext import native, use_native
from .hybrid import PromptRows

GROUP = 16  # positions that share an exponent
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0


class Pages(NamedTuple):
    """One layer's cache and the block table: position p of slot s lies in page ``table[s, p // block]`` at row
    ``p % block``.  Kernels look at no page outside the pool: what a sequence has there is not written, and comes
    back, from a read or through attention, as NaN.  Slots may share pages that they read; a group of positions that two of them
    append to in one call is the callers' to prevent."""

    k: torch.Tensor  # uint8 [pages, Hkv, block, D]
    v: torch.Tensor
    k_exp: torch.Tensor  # uint8 [pages, Hkv, block / 16]
    v_exp: torch.Tensor
    table: torch.Tensor  # int32 [slots, max_pages]

    @staticmethod
    def empty(pages: int, heads: int, block: int, dim: int, table: torch.Tensor) -> "Pages":
        """A pool of zeros on the table's device."""
        if block % GROUP or block < GROUP:
            raise ValueError(f"blocks of a multiple of {GROUP} positions, got {block}")
        k, v = (torch.zeros(pages, heads, block, dim, dtype=torch.uint8, device=table.device) for _ in range(2))
        ke, ve = (torch.zeros(pages, heads, block // GROUP, dtype=torch.uint8, device=table.device) for _ in range(2))
        return Pages(k, v, ke, ve, table)

    def nbytes(self) -> int:
        return sum(t.numel() for t in self[:4])


def exponents(amax: torch.Tensor) -> torch.Tensor:
    """The exponent bytes (int32) of tokens or groups of these largest values (>= 0, finite)."""
    m, x = torch.frexp(amax.float())
    e = x + 118 + (m > 0.875).to(torch.int32)  # amax = 2 m 2^(x - 1), 448 = 1.75 * 2^8
    return torch.where(amax > 0, e, 1).clamp(1, 254).to(torch.int32)


def encode(x: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """uint8 codes of values under exponent bytes ``e`` (broadcast)."""
    return torch.ldexp(x.float(), 127 - e.to(torch.int32)).to(E4M3).view(torch.uint8)


def decode(codes: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """f32 values of uint8 codes under exponent bytes ``e`` (broadcast)."""
    return torch.ldexp(codes.view(E4M3).float(), e.to(torch.int32) - 127)


def prompt_runs(starts, lens, slots, device=None) -> torch.Tensor:
    """The table that ``append_prompts`` takes, int32 [n, 4] = (first row, rows, slot, first position): sequences of ``lens``
    tokens one after another in the rows, from position ``starts`` of slot ``slots`` on, cut where groups of positions end."""
    if not len(starts) == len(lens) == len(slots):
        raise ValueError("a start, a length and a slot for each sequence")
    if len(set(slots)) < len(slots):
        raise ValueError("a slot is named twice: what two runs of one group would write depends on their order")
    if any(n < 0 or p < 0 or s < 0 for p, n, s in zip(starts, lens, slots)):
        raise ValueError("starts, lengths and slots must not be negative")
    out, row = [], 0
    for p, n, s in zip(starts, lens, slots):
        end = p + n
        while p < end:
            m = min(end, (p // GROUP + 1) * GROUP) - p
            out.append((row, m, s, p))
            row, p = row + m, p + m
    return torch.tensor(out, dtype=torch.int32).reshape(-1, 4).to(device or "cpu")


def append_tokens(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, slots: torch.Tensor | None,
                  pages: Pages, Hq: int, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                  eps: float = 1e-5) -> torch.Tensor:
    """One token a row: qkv [B, (Hq + 2 Hkv) D] at positions ``pos`` int32 [B] of ``slots`` int32 [B] (None: the rows' numbers).
    Queries and keys are normed (where weights [D] are given) and rotated, keys and values go into the cache; returns
    the queries [B, Hq, D].  Rows may share a sequence, and a position (the last row then stays).  A row without a place
    (a negative position or slot, or one past the block table or the rotation table) is not kept, and its query is zero."""
    if use_native(qkv):
        return native().kv8_append_tokens(qkv, cos, sin, pos, slots, *pages, Hq, q_norm, k_norm, eps)
    T, Hkv, D = _check_rows(qkv, cos, sin, pages, Hq, q_norm, k_norm)
    _check_ints(pos, (T,), "pos")
    where = _slots(slots, T)
    cap = min(pages.table.shape[1] * pages.k.shape[2], cos.shape[0])
    ok = [(0 <= p < cap and 0 <= s < pages.table.shape[0]) for p, s in zip(pos.tolist(), where)]
    q, k, v = _heads(qkv, cos, sin, pos.clamp(0, cap - 1).long(), Hq, Hkv, D, q_norm, k_norm, eps)
    groups: dict = {}
    for t, (p, s) in enumerate(zip(pos.tolist(), where)):
        if ok[t]:
            groups.setdefault((s, p // GROUP), {})[p % GROUP] = t
    for (s, g), rows in groups.items():
        _store(pages, s, g, rows, k, v)
    q[~torch.tensor(ok, dtype=torch.bool, device=q.device)] = 0
    return q.to(qkv.dtype)


def append_prompts(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, runs: torch.Tensor, pages: Pages, Hq: int,
                   q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-5):
    """Rows of several sequences: qkv [T, (Hq + 2 Hkv) D], ``runs`` int32 [n, 4] = (first row, rows, slot, first position) on the
    same device, each within one group of positions (``prompt_runs``); every row in one run, and no group in two.  Returns
    q [Hq, T, D] and k, v [Hkv, T, D], normed and rotated but not rounded to 8 bits, for the attention of the prompt.  A run
    without a place is left out, its rows' outputs with it."""
    if use_native(qkv):
        return native().kv8_append_prompts(qkv, cos, sin, runs, *pages, Hq, q_norm, k_norm, eps)
    T, Hkv, D = _check_rows(qkv, cos, sin, pages, Hq, q_norm, k_norm)
    _check_ints(runs, (runs.shape[0] if runs.dim() else -1, 4), "runs")
    cap = min(pages.table.shape[1] * pages.k.shape[2], cos.shape[0])
    table = [r for r in runs.tolist() if r[0] >= 0 and 1 <= r[1] <= GROUP and r[0] + r[1] <= T and r[3] >= 0 and
             r[3] + r[1] <= cap and r[3] % GROUP + r[1] <= GROUP and 0 <= r[2] < pages.table.shape[0]]
    pos = torch.zeros(T, dtype=torch.long, device=qkv.device)
    for t0, n, _, p0 in table:
        pos[t0:t0 + n] = torch.arange(p0, p0 + n, device=qkv.device)
    q, k, v = _heads(qkv, cos, sin, pos, Hq, Hkv, D, q_norm, k_norm, eps)
    for t0, n, s, p0 in table:
        _store(pages, s, p0 // GROUP, {p0 % GROUP + i: t0 + i for i in range(n)}, k, v)
    return tuple(x.transpose(0, 1).contiguous().to(qkv.dtype) for x in (q, k, v))


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: list[int],
                     blocks: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of each of several prompts to itself: q [Hq, T, D], k, v [Hkv, T, D] of sequences of ``lens`` rows one
    after another, T in all (``append_prompts`` from position 0) -> [T, Hq * D].  ``blocks``: the table of 128-row blocks that the
    GPU takes, made here (and sent there) if it is not given; for many layers it is made once:
    ``PromptRows(lens, device).attn_blocks(max(lens))``."""
    if q.dim() != 3 or k.dim() != 3 or sum(lens) != q.shape[1] or any(n < 0 for n in lens):
        raise ValueError(f"lens of q's rows, got {lens} of {list(q.shape)}")
    if use_native(q):
        if blocks is None:
            blocks = PromptRows([n for n in lens if n], q.device).attn_blocks(max(lens)) if sum(lens) else q.new_zeros(0, 4).int()
        if blocks.shape[0] != sum(-(-n // 128) for n in lens):
            raise ValueError(f"blocks of 128 rows of {lens}, got {blocks.shape[0]}")
        return native().prompt_rows_attention(q, k, v, blocks, 1.0 / math.sqrt(q.shape[-1]))
    if q.shape[0] % max(k.shape[0], 1) or k.shape[0] == 0 or k.shape[1:] != q.shape[1:] or v.shape != k.shape:
        raise ValueError(f"q [Hq, T, D], k, v [Hkv, T, D], got {list(q.shape)}, {list(k.shape)}, {list(v.shape)}")
    out, at = q.new_empty(q.shape[1], q.shape[0] * q.shape[2]), 0
    for n in lens:
        o = ref.attention(*(x[None, :, at:at + n].transpose(1, 2) for x in (q, k, v)))
        out[at:at + n] = o.flatten(2)[0]
        at += n
    return out


def read(pages: Pages, slots: torch.Tensor | None, starts: torch.Tensor, ends: torch.Tensor, n: int):
    """(k, v) bf16 [B, Hkv, n, D] of positions starts[b] + i, i < n, of slot slots[b] (int32 [B]; None: the rows' numbers); zero from
    ends[b] on, ahead of position 0, behind the block table and of a slot that is none.
    Exact: bf16 holds every value of the cache (under exponent bytes of 3 and more, up to the end of f32)."""
    if use_native(pages.k):
        return native().kv8_read(*pages, slots, starts, ends, n)
    B = starts.shape[0]
    _check_ints(starts, (B,), "starts")
    _check_ints(ends, (B,), "ends")
    _check_pages(pages)
    where = _slots(slots, B)
    out = [torch.zeros(B, pages.k.shape[1], n, pages.k.shape[3], dtype=torch.bfloat16, device=pages.k.device) for _ in range(2)]
    for b, (s, a, e) in enumerate(zip(where, starts.tolist(), ends.tolist())):
        lo, hi = max(a, 0), min(a + n, e, pages.table.shape[1] * pages.k.shape[2])
        if 0 <= s < pages.table.shape[0] and lo < hi:
            for o, x in zip(out, _rows(pages, s, lo, hi)):
                o[b, :, lo - a:hi - a] = x.to(torch.bfloat16)
    return tuple(out)


def decode_attention(q: torch.Tensor, pages: Pages, pos: torch.Tensor, slots: torch.Tensor | None, max_len: int,
                     scale: float | None = None) -> torch.Tensor:
    """One token of each sequence: q [B, Hq, D] over positions 0 .. pos[b] of slot slots[b] (int32 [B]; None: the rows'
    numbers) -> [B, Hq * D].  ``max_len`` >= 1 bounds the positions that any row looks at (a host number, for the launch;
    positions at it and behind are not seen), ``scale`` > 0.  A row without keys (pos < 0, or a slot that is none) gives zeros."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    if use_native(q):
        return native().kv8_decode_attn(q, *pages, pos, slots, max_len, scale)
    _check_pages(pages)
    B, Hq, D = q.shape
    Hkv = pages.k.shape[1]
    if D != pages.k.shape[3] or Hq % Hkv or max_len < 1 or not 0 < scale < math.inf:
        raise ValueError(f"q {tuple(q.shape)} over a cache of {Hkv} heads of {pages.k.shape[3]}, max_len {max_len}, scale {scale}")
    _check_ints(pos, (B,), "pos")
    cap = min(max_len, pages.table.shape[1] * pages.k.shape[2])
    out = torch.zeros(B, Hq, D, device=q.device)
    for b, (p, s) in enumerate(zip(pos.tolist(), _slots(slots, B))):
        n = min(p + 1, cap)
        if n > 0 and 0 <= s < pages.table.shape[0]:
            k, v = _rows(pages, s, 0, n)
            w = torch.softmax(torch.matmul(q[b].float().view(Hkv, -1, D), k.transpose(1, 2)) * scale, -1)
            out[b] = torch.matmul(w, v).reshape(Hq, D)
    return out.reshape(B, Hq * D).to(q.dtype)


# ---------------------------------------------------------------------------------------------------- CPU
def _check_ints(t: torch.Tensor, shape: tuple, name: str) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: int32 {list(shape)}, got {t.dtype} {list(t.shape)}")


def _slots(slots: torch.Tensor | None, n: int) -> list[int]:
    if slots is None:
        return list(range(n))
    _check_ints(slots, (n,), "slots")
    return slots.tolist()


def _check_pages(pages: Pages) -> None:
    k, v, ke, ve, table = pages
    want = (*k.shape[:2], k.shape[2] // GROUP) if k.dim() == 4 else None
    if (any(t.dtype != torch.uint8 for t in (k, v, ke, ve)) or k.dim() != 4 or v.shape != k.shape or k.shape[2] % GROUP
            or 0 in k.shape or tuple(ke.shape) != want or tuple(ve.shape) != want):
        raise ValueError("8-bit cache: uint8 codes [pages, Hkv, block, D] (block a multiple of 16), exponents [pages, Hkv, block / 16]")
    if table.dtype != torch.int32 or table.dim() != 2 or 0 in table.shape:
        raise ValueError("block table: int32 [slots, max_pages]")


def _check_rows(qkv, cos, sin, pages: Pages, Hq: int, q_norm, k_norm) -> tuple[int, int, int]:
    _check_pages(pages)
    Hkv, D = pages.k.shape[1], pages.k.shape[3]
    if Hq < Hkv or Hq % Hkv:
        raise ValueError(f"query heads in whole groups of a key head, got {Hq} of {Hkv}")
    if qkv.dim() != 2 or qkv.shape[1] != (Hq + 2 * Hkv) * D:
        raise ValueError(f"qkv [T, (Hq + 2 Hkv) D] = [.., {(Hq + 2 * Hkv) * D}], got {list(qkv.shape)}")
    if cos.dim() != 2 or cos.shape[0] == 0 or cos.shape[1] != D // 2 or cos.shape != sin.shape:
        raise ValueError("cos, sin: [positions, D / 2]")
    if (q_norm is None) != (k_norm is None) or any(w is not None and tuple(w.shape) != (D,) for w in (q_norm, k_norm)):
        raise ValueError("weights [D] of both norms, or of none")
    return qkv.shape[0], Hkv, D


def _odd_f32(x: torch.Tensor) -> torch.Tensor:
    """f64 as the f32 that is rounded to fewer bits as ``x`` is: an odd last bit where f32 does not hold it."""
    f = x.float()
    b = f.view(torch.int32)
    up = torch.where(f.double().abs() < x.abs(), 1, -1).to(torch.int32)
    return torch.where((f.double() != x) & (b % 2 == 0), b + up, b).view(torch.float32)


def _heads(qkv, cos, sin, pos, Hq, Hkv, D, q_norm, k_norm, eps):
    """f32 [T, heads, D] of queries and keys, normed and rotated, and of values; a key is the f32 that rounds as its value does."""
    q, k, v = qkv.view(-1, Hq + 2 * Hkv, D).float().split([Hq, Hkv, Hkv], 1)
    k = k.double()
    if q_norm is not None:
        q = ref.rms_norm(q, q_norm, eps)
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + eps) * k_norm.double()
    c, s = cos[pos].float()[:, None], sin[pos].float()[:, None]

    def turn(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    return turn(q), _odd_f32(turn(k)), v


def _store(pages: Pages, slot: int, group: int, rows: dict[int, int], k: torch.Tensor, v: torch.Tensor) -> None:
    """``rows``: the group's rows that are new, and which row of k, v [T, Hkv, D] each gets."""
    block = pages.k.shape[2]
    page = int(pages.table[slot, group * GROUP // block])
    if not 0 <= page < pages.k.shape[0]:
        return
    at = group * GROUP % block
    new, src, held = (torch.tensor(r, dtype=torch.long, device=k.device) for r in (
        sorted(rows), [rows[r] for r in sorted(rows)], [r for r in range(max(rows)) if r not in rows]))
    for x, codes, exps in ((k, pages.k, pages.k_exp), (v, pages.v, pages.v_exp)):
        x = x[src].transpose(0, 1)  # [Hkv, rows, D]
        e = exponents(torch.where(torch.isfinite(x), x.abs(), 0.0).amax((1, 2)))
        tile = codes[page, :, at:at + GROUP]
        if len(held):
            old = exps[page, :, at // GROUP].to(torch.int32)
            e = torch.maximum(e, old)
            again = encode(decode(tile[:, held], old[:, None, None]), e[:, None, None])
            tile[:, held] = torch.where((e > old)[:, None, None], again, tile[:, held])
        tile[:, new] = encode(x, e[:, None, None])
        exps[page, :, at // GROUP] = e.to(torch.uint8)


def _rows(pages: Pages, slot: int, lo: int, hi: int):
    """f32 [Hkv, hi - lo, D] of keys and values of positions lo .. hi - 1; NaN where the table names no page of the pool."""
    p = torch.arange(lo, hi, device=pages.k.device)
    block = pages.k.shape[2]
    page = pages.table[slot][p // block].long()
    ok = (page >= 0) & (page < pages.k.shape[0])
    page = torch.where(ok, page, 0)
    out = []
    for codes, exps in ((pages.k, pages.k_exp), (pages.v, pages.v_exp)):
        x = decode(codes[page, :, p % block], exps[page, :, p % block // GROUP][..., None])  # [n, Hkv, D]
        out.append(torch.where(ok[:, None, None], x, math.nan).transpose(0, 1))
    return out
