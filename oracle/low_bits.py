"""CPU definition of the operators that hold less in memory, in 64 bits -- TEST
INFRASTRUCTURE ONLY: the 8-bit KV cache, products with 4-bit weights, and the
controls on logits. Written from their formulas (the reference has none of
them); the bounds are what a correct kernel with fp32 sums and one rounding at
its store may be off, element by element.

Codes are held as the numbers they stand for, so that a cache is three float64
arrays: values of the codes, and scales (fp32 numbers).
"""
from __future__ import annotations

import math

import torch

from .long_context import U32, bound_attention, store, u

INT8, E4M3 = torch.int8, torch.float8_e4m3fn
FLOOR = 2.0 ** -80


def top(code):
    return 127.0 if code == INT8 else 448.0


def grid(code):
    """The values of the codes at and above 0, ascending; the index is the code."""
    if code == INT8:
        return torch.arange(128, dtype=torch.float64)
    return torch.arange(127, dtype=torch.uint8).view(E4M3).to(torch.float64)


def nearest(q, code):
    """The code value nearest to q, the even code where two are as near."""
    g = grid(code)
    a = q.abs().contiguous()
    hi = torch.searchsorted(g, a).clamp(max=len(g) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = g[hi] - a, a - g[lo]
    even = torch.where(hi % 2 == 0, hi, lo)
    return g[torch.where(up < down, hi, torch.where(up > down, lo, even))] * torch.sign(q)


def kv8_store(x, slots, codes, scale, block, code):
    """x [T, heads, D] into codes [slots, heads, D] (float64 values) and scale
    [blocks, heads], in place; run by run
    (padded tokens among a run are skipped)."""
    x = x.cpu().to(torch.float64)
    slots = [int(s) for s in slots]
    t = 0
    while t < len(slots):
        if not 0 <= slots[t] < codes.shape[0]:
            t += 1
            continue
        blk, first = slots[t] // block, slots[t] % block
        run, end = [t], t + 1
        while end < len(slots) and (not 0 <= slots[end] < codes.shape[0]
                                    or slots[end] // block == blk):
            if 0 <= slots[end] < codes.shape[0]:
                run.append(end)
            end += 1
        part = x[run]
        for h in range(x.shape[1]):
            if bool(torch.isfinite(part[:, h]).all()):
                s = (part[:, h].abs().max() / top(code)).to(torch.float32).to(torch.float64)
                s = max(float(s), FLOOR)
            else:
                s = math.nan
            if first > 0:
                old = float(scale[blk, h])
                s = math.nan if math.isnan(s) or math.isnan(old) else max(old, s)
                if s > old:
                    kept = slice(blk * block, blk * block + first)
                    codes[kept, h] = nearest(codes[kept, h] * old / s, code)
            for i in run:
                codes[slots[i], h] = nearest(x[i, h] / s, code) if s == s else 0.0
            scale[blk, h] = s
        t = end


def kv8_values(codes, scale, block):
    """[slots, heads, D]: what the cache stands for."""
    n = codes.shape[0]
    return codes * scale.repeat_interleave(block, 0)[:n, :, None]


def bound_value(want, dtype):
    """A product of a code and a scale rounded to fp32, then to dtype."""
    off = want.abs() * U32
    return off + (store(dtype, want.abs() + off) if dtype != torch.float32 else 0.0)


def kv8_decode(q, k, v, table, rids, lens, slots_n, sm_scale=None):
    """Attention over values k, v [slots, KVH, D]: float64 (out [B, H, D], weight
    [B, H, D], keys [B], mags [B, H]) as in long_context.window_decode. Slots
    outside [0, slots_n) are no tokens."""
    B, H, D = q.shape
    kvh = k.shape[1]
    scale = sm_scale if sm_scale is not None else 1.0 / math.sqrt(D)
    q = q.cpu().to(torch.float64)
    out, wgt = (torch.zeros(B, H, D, dtype=torch.float64) for _ in range(2))
    keys, mags = torch.zeros(B, dtype=torch.int64), torch.zeros(B, H, dtype=torch.float64)
    for b, (rid, n) in enumerate(zip(rids, lens)):
        slots = table[rid, :max(n, 0)].long()
        slots = slots[(slots >= 0) & (slots < slots_n)]
        keys[b] = len(slots)
        if len(slots) == 0:
            continue
        for h in range(H):
            kk, vv = k[slots, h // (H // kvh)], v[slots, h // (H // kvh)]
            s = (kk @ q[b, h]) * scale
            e = torch.exp(s - s.max())
            p = e / e.sum()
            out[b, h], wgt[b, h] = p @ vv, p @ vv.abs()
            mags[b, h] = float((kk.abs() @ q[b, h].abs()).max() * abs(scale))
    return out, wgt, keys, mags


def bound_kv8_decode(out, wgt, keys, mags, dtype, head_dim):
    """long_context.bound_attention with a probability (times its token's V scale,
    one more rounding) held as two bf16 numbers or more: 2^-16 of itself. A
    score has one more product, K's scale, within that bound's d."""
    return bound_attention(out, wgt, keys, mags, dtype, head_dim,
                           (2.0 ** -16 if dtype != torch.float32 else 0.0) + 4 * U32)


def w4_weight(codes, scale, zero=None):
    """[N, K] of float64 from codes [N, K / 2] uint8, scale and zero [N, K / group]."""
    n, half = codes.shape
    group = 2 * half // scale.shape[1]
    c = torch.stack([codes % 16, codes // 16], -1).reshape(n, 2 * half).to(torch.float64)
    z = torch.full(scale.shape, 8.0, dtype=torch.float64) if zero is None else zero.to(torch.float64)
    return (c - z.repeat_interleave(group, 1)) * scale.to(torch.float64).repeat_interleave(group, 1)


def linear_w4(x, codes, scale, zero=None, bias=None):
    """(y, what its terms may add up to): the second counts every term of a group
    as one of the largest code with 128 added, the form of the bf16 products."""
    x = x.to(torch.float64)
    w = w4_weight(codes, scale, zero)
    y = x @ w.t()
    group = w.shape[1] // scale.shape[1]
    s = scale.to(torch.float64).abs().repeat_interleave(group, 1)
    mag = x.abs() @ (s * (128 + 15)).t() * 2
    if bias is not None:
        y = y + bias.to(torch.float64)
        mag = mag + bias.to(torch.float64).abs()
    return y, mag


def bound_linear_w4(y, mag, dtype, k):
    """fp32 sums of K terms in any tree of partial sums: no term passes more than
    log2(K) + a chain of 64 additions (an instruction's 32 terms, a group's four
    instructions, the groups of a wave, the waves), each rounded; then the store."""
    off = mag * (64 + math.log2(max(k, 2)) + k / 128) * U32
    return off + store(dtype, y.abs() + off)


def adjust_logits(logits, tokens=None, rids=None, prompt=None, lens=None, repetition=None,
                  frequency=None, presence=None, bias_ids=None, bias_values=None, mask=None):
    """(out, magnitude of what was added up) in float64, token by token."""
    x = logits.to(torch.float64).clone()
    mag = x.abs()
    B, V = x.shape
    for b in range(B):
        if tokens is not None and 0 <= rids[b] < tokens.shape[0]:
            n = min(max(int(lens[b]), 0), tokens.shape[1])
            row = [int(t) for t in tokens[rids[b], :n]]
            said = {}
            for t in row[max(0, int(prompt[b])):]:
                said[t] = said.get(t, 0) + 1
            for t in set(row):
                if not 0 <= t < V:
                    continue
                if repetition is not None:
                    r = float(repetition[b])
                    x[b, t] = x[b, t] / r if x[b, t] > 0 else x[b, t] * r
                    mag[b, t] = mag[b, t] + x[b, t].abs()
                if t in said and frequency is not None:
                    x[b, t] -= float(frequency[b]) * said[t]
                    mag[b, t] += abs(float(frequency[b])) * said[t]
                if t in said and presence is not None:
                    x[b, t] -= float(presence[b])
                    mag[b, t] += abs(float(presence[b]))
        if bias_ids is not None:
            for t, v in zip(bias_ids[b].tolist(), bias_values[b].tolist()):
                if 0 <= t < V:
                    x[b, t] += v
                    mag[b, t] += abs(v)
        if mask is not None:
            for t in range(V):
                if not (int(mask[b, t // 32]) >> (t % 32)) & 1:
                    x[b, t] = -math.inf
    return x, mag


def bound_logits(out, mag, dtype, additions=6):
    """An fp32 rounding of at most the magnitude so far per operation; the store."""
    off = mag * additions * U32
    fin = torch.nan_to_num(out.abs(), posinf=0.0, nan=0.0)
    return off + (store(dtype, fin + off) if dtype != torch.float32 else 0.0)


__all__ = ["U32", "u", "store"]
