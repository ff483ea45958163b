"""CPU restatement of the long-context operators (test infrastructure only):
rotary positions from frequencies, per-head norms with rotation, attention over
a window with sinks, slot maps. float64 (angles: long double), from the
formulas, one request and one row at a time.

The attention and rotation functions also return what a bound on a kernel's
rounding needs (see bound_attention, bound_rotary).
"""
from __future__ import annotations

import math

import numpy as np
import torch


def u(dtype: torch.dtype) -> float:
    """Half a step of a rounding to dtype, relative to the value."""
    return torch.finfo(dtype).eps / 2


U32 = 2.0 ** -24


def store(dtype: torch.dtype, y: torch.Tensor) -> torch.Tensor:
    """The largest error of rounding values of up to |y| to dtype: half a step,
    u |y| for normal numbers; below the smallest normal one (fp16: 2^-14) the
    steps stay at the smallest subnormal (fp16: 2^-24), so half of that."""
    fi = torch.finfo(dtype)
    return (y.abs() * u(dtype)).clamp_min(fi.smallest_normal * fi.eps / 2)


# ---------------------------------------------------------------- rotation
def cos_sin(positions, inv_freq, factor):
    """factor * cos, sin of positions x frequencies, [T, R/2]; the product is
    exact in long double (31 + 24 bits), and so is its reduction to 2^-30."""
    p = np.asarray(positions.cpu().numpy(), dtype=np.longdouble)
    f = np.asarray(inv_freq.cpu().numpy(), dtype=np.longdouble)
    ang = np.remainder(p[:, None] * f[None, :], 2 * np.arctan2(np.longdouble(0), np.longdouble(-1)))
    c = (np.cos(ang) * factor).astype(np.float64)
    s = (np.sin(ang) * factor).astype(np.float64)
    return torch.from_numpy(c), torch.from_numpy(s)


def rotate(x, positions, inv_freq, factor=1.0, interleaved=False):
    """x [T, heads, D] -> (rotated float64, |x0| + |x1| of each element's pair
    times factor, 0 behind the rotated part)."""
    x = x.cpu().to(torch.float64)
    c, s = cos_sin(positions, inv_freq, factor)
    n = inv_freq.numel()
    y, mag = x.clone(), torch.zeros_like(x)
    for i in range(n):
        i0, i1 = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        a, b = x[..., i0], x[..., i1]
        ci, si = c[:, i, None], s[:, i, None]
        y[..., i0] = a * ci - b * si
        y[..., i1] = a * si + b * ci
        mag[..., i0] = mag[..., i1] = (a.abs() + b.abs()) * abs(factor)
    return y, mag


def head_norm(x, gamma, eps):
    x = x.cpu().to(torch.float64)
    if gamma is None:
        return x
    var = (x * x).mean(-1, keepdim=True)
    return x / torch.sqrt(var + eps) * gamma.cpu().to(torch.float64)


def bound_rotary(y, mag, dtype, positions, inv_freq, head_dim=0):
    """How far a correct fp32 kernel's output may be from y: the store's
    rounding; the cosine's and sine's own error (4 ulp of 2^-23 at most 1, and
    the product's and sum's three roundings); the angle, taken in turns in fp64
    (two roundings of the turns, 2^-53 each, then 2^-25 of a turn in fp32); and
    with norms (head_dim > 0) the sum of head_dim squares, the root and three
    products."""
    turns = float(positions.abs().max() if positions.numel() else 0) * float(
        inv_freq.max() if inv_freq.numel() else 0) / (2 * math.pi)
    angle = 2 * math.pi * (2.0 ** -25 + 3 * 2.0 ** -53 * turns)
    rel = angle + 4 * 2.0 ** -23 + 4 * U32
    out = mag * rel
    if head_dim:
        out = out + torch.maximum(mag, y.abs()) * (head_dim / 2 + 8) * U32
    return out + store(dtype, y.abs() + out)


# ---------------------------------------------------------------- attention
def visible(p, length, window, sinks):
    """Keys that the query at position p sees, ascending."""
    low = max(0, p - window + 1)
    return [n for n in range(0, min(sinks, low, length))] + list(range(low, min(p + 1, length)))


def _row(q, k, v, scale):
    """One query head over its visible keys: (out, sum p |v| / l, n keys,
    largest sum |q| |k| scale)."""
    s = (k @ q) * scale
    e = torch.exp(s - s.max())
    p = e / e.sum()
    return p @ v, p @ v.abs(), float((k.abs() @ q.abs()).max() * abs(scale))


def p_rounding(dtype, split):
    """Relative rounding of a probability in P.V: to dtype, or as the sum of two
    numbers of dtype (split), where the second rounds what the first left."""
    return u(dtype) ** 2 if split and dtype != torch.float32 else u(dtype)


def window_prefill(q, k_pool, v_pool, table, rids, starts, lens, shared, window, sinks,
                   sm_scale=None):
    """Returns float64 (out [T, H, D], weight [T, H, D], keys [T], mags [T, H]);
    rows of no request are NaN in out."""
    T, H, D = q.shape
    kvh = k_pool.shape[1]
    scale = sm_scale if sm_scale is not None else 1.0 / math.sqrt(D)
    out = torch.full((T, H, D), float("nan"), dtype=torch.float64)
    wgt = torch.zeros(T, H, D, dtype=torch.float64)
    keys, mags = torch.zeros(T, dtype=torch.int64), torch.zeros(T, H, dtype=torch.float64)
    q, kp, vp = (x.cpu().to(torch.float64) for x in (q, k_pool, v_pool))
    for rid, st, n, c in zip(rids, starts, lens, shared):
        for r in range(n - c):
            see = visible(c + r, n, window, sinks)
            slots = table[rid, see].long()
            keys[st + r] = len(see)
            for h in range(H):
                g = h // (H // kvh)
                out[st + r, h], wgt[st + r, h], mags[st + r, h] = _row(
                    q[st + r, h], kp[slots, g], vp[slots, g], scale)
    return out, wgt, keys, mags


def window_decode(q, k_pool, v_pool, table, rids, lens, window, sinks, sm_scale=None):
    """window_prefill with one row per sequence (length 0: a zero row)."""
    starts = list(range(len(lens)))
    live = [i for i, n in enumerate(lens) if n > 0]
    out, wgt, keys, mags = window_prefill(
        q, k_pool, v_pool, table, [rids[i] for i in live], [starts[i] for i in live],
        [lens[i] for i in live], [lens[i] - 1 for i in live], window, sinks, sm_scale)
    out[[i for i, n in enumerate(lens) if n == 0]] = 0.0
    return out, wgt, keys, mags


def bound_attention(out, wgt, keys, mags, dtype, head_dim, p_round, vmax=0.0):
    """How far a correct kernel's output may be from out. With d the error of a
    score in units of its exponent (head_dim products summed in fp32, the scale
    and the exponential, 2^-21) every p is off by 2 d of itself at most, so are
    they after the division, and each p is rounded by p_round before P.V; sums
    over n keys in fp32, twice (outputs and the denominator); then the store.
    fp16 probabilities below 2^-14 (of a largest one of at least 1) are rounded
    to steps of 2^-24 (vmax: the largest |v|)."""
    d = (head_dim + 8) * U32 * mags[..., None] + 2.0 ** -21
    rel = 2.1 * d + p_round + 2 * (keys[:, None, None] + 16) * U32
    off = wgt * rel
    if dtype == torch.float16:
        off = off + keys[:, None, None] * vmax * 2.0 ** -25
    return off + store(dtype, out.abs() + off)


# ---------------------------------------------------------------- slot maps
def slot_maps(rids, lens, cached, free, table, page, blocks):
    """(slots, positions, start, last, counts, table, blocks) as int lists /
    numpy arrays; table and blocks are copies with the new entries."""
    table = table.copy()
    blocks = None if blocks is None else blocks.copy()
    slots, positions, start, last, used = [], [], [], [], 0
    for rid, n, c in zip(rids, lens, cached):
        start.append(len(slots))
        for at in range(-(-c // page), -(-n // page)):
            if page > 1:
                blocks[rid, at] = free[used]
            else:
                table[rid, at] = free[used]
            used += 1
        for p in range(c, n):
            slot = int(blocks[rid, p // page]) * page + p % page if page > 1 else int(table[rid, p])
            table[rid, p] = slot
            slots.append(slot)
            positions.append(p)
        last.append(len(slots) - 1 if n > c else -1)
    return slots, positions, start, last, [len(slots), used, 0], table, blocks
