"""Operators of long-context serving, as cases to be timed.

A server whose contexts outgrow what a model was trained on, or what it wants
to keep in the cache, needs the token loop's attention path in another form:

* rope: rotary positions from the frequencies themselves (no table over the
  context length), with both layouts of the pairs, a rotated part of the head,
  and the scaled frequencies of long contexts;
* qk_norm: the same rotation after an RMSNorm of every query and key head,
  K and V going to their cache slots in the same pass;
* window_prefill, window_decode: attention over the slot table that sees the
  last `window` tokens and the first `sinks` ones;
* slots: positions, cache slots, start offsets and the slot table's entries of
  a batch, built from its lengths and the free list.

Sizes are those of this repository's configurations and tests: 16/2 and 12/2
heads of 128 (the Qwen2.5-3B and Qwen2-1.5B layers), its 28/4 head group, 32/8
and 8/2 heads of 64, batches up to 128 requests, prompts of up to 24,000 tokens
in one call and contexts of up to 131,072.

`run` computes the plain form (elementary operations, 32 bits; angles 64) or,
with `own` set, calls the framework. `exact` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# query heads, KV heads, head dim
_HEADS = {"3b": (16, 2, 128), "1.5b": (12, 2, 128), "28/4": (28, 4, 128), "32/8x64": (32, 8, 64),
          "8/2x64": (8, 2, 64)}
_THETA, _EPS = 1e6, 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one step of the benchmark's batch, contexts anywhere in the model's range
        {"name": "rope_decode", "kind": "rope", "heads": "3b", "rows": 40, "rotary": 128,
         "interleaved": False, "scaled": False, "far": 32768, "dtype": "bf16"},
        # a full prefill of a model that rotates half of each head in adjacent
        # pairs, its frequencies scaled for contexts of a million tokens
        {"name": "rope_prefill_scaled", "kind": "rope", "heads": "28/4", "rows": 24000,
         "rotary": 64, "interleaved": True, "scaled": True, "far": 1048576, "dtype": "fp16"},
        # one step of a batch: norms, rotation and the new tokens' cache rows
        {"name": "qk_norm_decode", "kind": "qk_norm", "heads": "1.5b", "rows": 40, "rotary": 128,
         "interleaved": False, "scaled": True, "far": 131072, "dtype": "bf16"},
        # the same for a whole prefill of the benchmark's prompts
        {"name": "qk_norm_prefill", "kind": "qk_norm", "heads": "3b", "rows": 24000,
         "rotary": 128, "interleaved": False, "scaled": False, "far": 600, "dtype": "bf16"},
        # the benchmark's prompts under a short window
        {"name": "window_prefill_batch", "kind": "window_prefill", "heads": "3b", "batch": 40,
         "len": 600, "shared": 0.0, "ragged": False, "window": 256, "sinks": 4, "dtype": "bf16"},
        # follow-up turns behind their cached prefixes, an odd window, no sinks
        {"name": "window_prefill_cached", "kind": "window_prefill", "heads": "28/4", "batch": 5,
         "len": 4111, "shared": 0.6, "ragged": True, "window": 1000, "sinks": 0,
         "dtype": "fp16"},
        # one long document: the largest call
        {"name": "window_prefill_long", "kind": "window_prefill", "heads": "3b", "batch": 1,
         "len": 32768, "shared": 0.0, "ragged": False, "window": 4096, "sinks": 4,
         "dtype": "bf16"},
        # a lone user deep into a conversation
        {"name": "window_decode_one", "kind": "window_decode", "heads": "1.5b", "batch": 1,
         "len": 131072, "ragged": False, "window": 4096, "sinks": 4, "dtype": "bf16"},
        # a full batch with long contexts
        {"name": "window_decode_batch", "kind": "window_decode", "heads": "3b", "batch": 40,
         "len": 16384, "ragged": True, "window": 4096, "sinks": 4, "dtype": "bf16"},
        # a server at a high load with short contexts, some below the window
        {"name": "window_decode_wide", "kind": "window_decode", "heads": "32/8x64", "batch": 96,
         "len": 1500, "ragged": True, "window": 1000, "sinks": 1, "dtype": "fp16"},
        # the maps of one decode step
        {"name": "slots_decode", "kind": "slots", "batch": 40, "len": 600, "ragged": True,
         "cached": 1.0, "page": 1},
        # the maps of a large admission, pages of 16 tokens, behind cached prefixes
        {"name": "slots_prefill", "kind": "slots", "batch": 128, "len": 4096, "ragged": True,
         "cached": 0.3, "page": 16},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "qk_norm", "window_prefill", "window_prefill", "window_decode",
                       "window_decode", "slots"])
    dtype = rng.choice(["bf16", "fp16"])
    heads = rng.choice(sorted(_HEADS))
    if kind in ("rope", "qk_norm"):
        d = _HEADS[heads][2]
        return {"kind": kind, "heads": heads, "rows": _log(rng, 1, 24000),
                "rotary": rng.choice([d, d, d // 2, d // 4]), "interleaved": rng.random() < 0.4,
                "scaled": rng.random() < 0.5, "far": _log(rng, 64, 1048576), "dtype": dtype}
    if kind == "window_prefill":
        batch = _log(rng, 1, 48)
        return {"kind": kind, "heads": heads, "batch": batch,
                "len": _log(rng, 1, min(16384, 24000 // batch)),
                "shared": rng.choice([0.0, 0.0, round(rng.uniform(0.1, 0.9), 2)]),
                "ragged": rng.random() < 0.6, "window": _log(rng, 32, 2048),
                "sinks": rng.choice([0, 1, 4, 4, 16, 100]), "dtype": dtype}
    if kind == "window_decode":
        batch = _log(rng, 1, 128)
        return {"kind": kind, "heads": heads, "batch": batch,
                "len": _log(rng, 1, min(131072, 1048576 // batch)), "ragged": rng.random() < 0.6,
                "window": min(_log(rng, 32, 8192), 262144 // batch),
                "sinks": rng.choice([0, 1, 4, 4, 16, 100]), "dtype": dtype}
    batch = _log(rng, 1, 512)
    return {"kind": kind, "batch": batch, "len": _log(rng, 1, min(16384, 262144 // batch)),
            "ragged": rng.random() < 0.6, "cached": rng.choice([0.0, 0.5, 1.0]),
            "page": rng.choice([1, 1, 16, 64])}


# ------------------------------------------------------------------ lengths
def _lens(case):
    """Tokens of each request, this call's included: the longest first."""
    n, b = case["len"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [max(1, n - (i * 7919) % max(1, (2 * n) // 3 + 1)) for i in range(b)]


def _before(case):
    """Tokens of each request that are in the cache before the call; at least
    one of each request is new."""
    part = {"window_prefill": case.get("shared", 0.0), "slots": case.get("cached", 0.0),
            "window_decode": 1.0}[case["kind"]]
    return [min(n - 1, int(n * part)) for n in _lens(case)]


def _visible(first, last, window, sinks):
    """Keys that any query at positions first .. last sees: (sinks, low), the
    tokens [0, sinks) and [low, last]."""
    low = max(0, first - window + 1)
    return (0, 0) if low <= sinks else (sinks, low)


# ------------------------------------------------------------------ inputs
def _inv_freq(rotary, scaled):
    """Frequencies of the rotated pairs; scaled: the interpolation by parts for
    32 times a trained context of 32,768 tokens, and its attention factor."""
    i = torch.arange(0, rotary, 2, dtype=torch.float64) / rotary
    f = _THETA ** -i
    if not scaled:
        return f.float(), 1.0
    turns = 32768 * f / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)  # 1: many turns, kept; 0: stretched
    return (f * keep + f / 32.0 * (1 - keep)).float(), 0.1 * math.log(32.0) + 1.0


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    gc = torch.Generator()
    gc.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s = {"case": case, "kind": case["kind"]}
    if case["kind"] in ("rope", "qk_norm"):
        h, kvh, d = _HEADS[case["heads"]]
        t, dt = case["rows"], _DT[case["dtype"]]
        f, s["factor"] = _inv_freq(case["rotary"], case["scaled"])
        s["inv_freq"] = f.to(dev)
        s["positions"] = torch.randint(0, case["far"], (t,), generator=g, device=dev,
                                       dtype=torch.int32)
        s["interleaved"], s["heads"] = case["interleaved"], (h, kvh, d)
        if case["kind"] == "rope":
            s["q"], s["k"] = randn(t, h, d).to(dt), randn(t, kvh, d).to(dt)
            s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
            return s
        s["qkv"] = (randn(t, (h + 2 * kvh) * d) * 1.7).to(dt)
        s["q_gamma"] = (1 + 0.2 * randn(d)).to(dt)
        s["k_gamma"] = (1 + 0.2 * randn(d)).to(dt)
        slots = t + t // 8 + 16  # rows of the cache that this call leaves alone among them
        s["pool"] = randn(slots, 2 * kvh, d).to(dt)
        s["slots"] = torch.randperm(slots, generator=gc)[:t].to(torch.int32).to(dev)
        s["q_out"] = torch.empty(t, h, d, dtype=dt, device=dev)
        return s

    lens, before, b = _lens(case), _before(case), case["batch"]
    rows = torch.randperm(b + 3, generator=gc)[:b].tolist()
    s["lens"], s["before"], s["max_len"] = lens, before, max(lens)
    s["rows"], s["seq_len"], s["cached"] = ints(rows), ints(lens), ints(before)
    if case["kind"] == "slots":
        page = case["page"]
        pages = [-(-n // page) for n in lens]
        have = [-(-n // page) for n in before]
        total = sum(pages) + 8
        perm = torch.randperm(total, generator=gc).to(torch.int32)
        s["page"], s["t"] = page, sum(n - c for n, c in zip(lens, before))
        width = max(pages) * page
        table = torch.randint(0, total, (b + 3, width // page), generator=gc, dtype=torch.int32)
        at = 0
        for r, n in zip(rows, have):
            table[r, :n] = perm[at:at + n]
            at += n
        s["free"] = perm[at:].to(dev)
        s["tokens"] = (table.long().repeat_interleave(page, 1) * page
                       + torch.arange(page).repeat(width // page)).to(torch.int32).to(dev)
        s["blocks"] = table.to(dev) if page > 1 else None
        new = torch.full((s["t"],), -1, dtype=torch.int32, device=dev)
        s["out"] = [new, new.clone(), torch.empty(b, dtype=torch.int32, device=dev),
                    torch.empty(b, dtype=torch.int32, device=dev),
                    torch.empty(3, dtype=torch.int32, device=dev)]
        return s

    h, kvh, d = _HEADS[case["heads"]]
    dt, w, k = _DT[case["dtype"]], case["window"], case["sinks"]
    s["heads"], s["window"], s["sinks"] = (h, kvh, d), w, k
    # tokens that no query of this call sees have left the cache: their table
    # entries are stale and point at slots of other tokens
    seen = [_visible(c, n - 1, w, k) for n, c in zip(lens, before)]
    live = [(a + n - low) for n, (a, low) in zip(lens, seen)]
    total = sum(live) + 64
    perm = torch.randperm(total, generator=gc).to(torch.int32)
    table = torch.randint(0, total, (b + 3, max(lens)), generator=gc, dtype=torch.int32)
    at = 0
    for r, n, (a, low), m in zip(rows, lens, seen, live):
        table[r, :a] = perm[at:at + a]
        table[r, low:n] = perm[at + a:at + m]
        at += m
    s["tokens"] = table.to(dev)
    pool = randn(total, 2 * kvh, d).to(dt)
    s["k"], s["v"] = pool[:, :kvh], pool[:, kvh:]
    new = [n - c for n, c in zip(lens, before)] if case["kind"] == "window_prefill" else [1] * b
    s["new"], s["start"] = new, ints([sum(new[:i]) for i in range(b)])
    s["q"] = randn(sum(new), h, d).to(dt)
    s["out"] = torch.empty_like(s["q"])
    return s


# ------------------------------------------------------------------ plain forms
def _rotate(x, positions, inv_freq, factor, interleaved):
    """x [T, heads, D] in 32 bits, rotated; the angles in 64."""
    half = inv_freq.numel()
    ang = positions.double()[:, None] * inv_freq.double()
    cos = (torch.cos(ang) * factor).float()[:, None]
    sin = (torch.sin(ang) * factor).float()[:, None]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return y if 2 * half == x.shape[-1] else torch.cat([y, x[..., 2 * half:]], -1)


def _head_norm(x, gamma):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * gamma.float()


def _softmax(x):
    """Over the last axis, in place; a row of -inf gives zeros."""
    m = x.amax(-1, keepdim=True)
    x.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    return x.div_(x.sum(-1, keepdim=True).clamp_min(1e-38))


def _plain_prefill(s):
    """Blocks of c query rows against the span of keys that they can see."""
    (h, kvh, d), w, k = s["heads"], s["window"], s["sinks"]
    dev, dt, t = s["q"].device, s["q"].dtype, s["q"].shape[0]
    c = max(64, min(1024, w // 4))
    blocks = [(b, r) for b, n in enumerate(s["new"]) if n for r in range(0, n, c)]
    req, r0 = torch.tensor(blocks, device=dev).t()
    lens, before, start = s["seq_len"].long()[req], s["cached"].long()[req], s["start"].long()[req]
    row = r0[:, None] + torch.arange(c, device=dev)
    pos = before[:, None] + row                                            # [blocks, c]
    at = torch.where(pos < lens[:, None], start[:, None] + row, t)
    low = (before + r0 - w + 1).clamp_min(0)
    span = min(c + w - 1, s["max_len"])
    first = torch.arange(k, device=dev).expand(len(blocks), k)
    key = torch.cat([first, low[:, None] + torch.arange(span, device=dev)], 1)
    own_place = torch.cat([first < low[:, None], key[:, k:] < lens[:, None]], 1)
    key, p = key[:, None], pos[..., None]
    see = own_place[:, None] & (key <= p) & ((key > p - w) | (key < k))    # [blocks, c, keys]
    slot = s["tokens"][s["rows"].long()[req][:, None], key[:, 0].clamp_max(s["max_len"] - 1)].long()
    slot = torch.where(own_place, slot, 0)
    q = torch.cat([s["q"], s["q"].new_zeros(1, h, d)])[at].float()
    q = q.view(len(blocks), c, kvh, h // kvh, d).permute(0, 2, 3, 1, 4).reshape(
        len(blocks), kvh, -1, d)
    kt = s["k"][slot].float().permute(0, 2, 3, 1).contiguous()
    x = torch.matmul(q, kt).mul_(1 / math.sqrt(d)).view(len(blocks), kvh, h // kvh, c, -1)
    x = _softmax(x.masked_fill_(~see[:, None, None], -math.inf)).view(len(blocks), kvh, -1,
                                                                      key.shape[-1])
    v = s["v"][slot].float().masked_fill_(~own_place[..., None, None], 0.0)
    y = torch.matmul(x, v.permute(0, 2, 1, 3).contiguous())
    y = y.view(len(blocks), kvh, h // kvh, c, d).permute(0, 3, 1, 2, 4).reshape(-1, h, d)
    out = torch.empty(t + 1, h, d, dtype=dt, device=dev)
    out[at.flatten()] = y.to(dt)
    return out[:t]


def _plain_decode(s):
    (h, kvh, d), w, k = s["heads"], s["window"], s["sinks"]
    dev, b = s["q"].device, s["q"].shape[0]
    lens = s["seq_len"].long()[:, None]
    low = (lens - w).clamp_min(0)
    first = torch.arange(k, device=dev).expand(b, k)
    key = torch.cat([first, low + torch.arange(min(w, s["max_len"]), device=dev)], 1)
    see = torch.cat([first < low, key[:, k:] < lens], 1)
    slot = s["tokens"][s["rows"].long()[:, None], key.clamp_max(s["max_len"] - 1)].long()
    slot = torch.where(see, slot, 0)
    q = s["q"].float().view(b, kvh, h // kvh, d)
    kt = s["k"][slot].float().permute(0, 2, 3, 1).contiguous()
    x = torch.matmul(q, kt).mul_(1 / math.sqrt(d))
    x = _softmax(x.masked_fill_(~see[:, None, None], -math.inf))
    v = s["v"][slot].float().masked_fill_(~see[..., None, None], 0.0)
    y = torch.matmul(x, v.permute(0, 2, 1, 3).contiguous())
    return y.reshape(b, h, d).to(s["q"].dtype)


def _plain_slots(s):
    rows, lens, before, page = s["rows"].long(), s["seq_len"].long(), s["cached"].long(), s["page"]
    slots, positions, start, last, counts = s["out"]
    new = lens - before
    ends = new.cumsum(0)
    req = torch.arange(rows.numel(), device=rows.device).repeat_interleave(new, output_size=s["t"])
    pos = torch.arange(s["t"], device=rows.device) - (ends - new)[req] + before[req]
    have, need = (before + page - 1) // page, (lens + page - 1) // page
    taken = (need - have).cumsum(0)
    at = pos // page
    fresh = at >= have[req]
    src = torch.where(fresh, (taken - (need - have))[req] + at - have[req], 0)
    old = s["tokens"] if page == 1 else s["blocks"]
    page_id = torch.where(fresh, s["free"][src], old[rows[req], at])
    slot = page_id * page + (pos % page).to(torch.int32)
    if page > 1:
        s["blocks"][rows[req], at] = page_id
    s["tokens"][rows[req], pos] = slot
    slots.copy_(slot)
    positions.copy_(pos)
    start.copy_(ends - new)
    last.copy_(torch.where(new > 0, ends - 1, -1))
    counts.copy_(torch.stack([ends[-1], taken[-1], torch.zeros_like(ends[-1])]))
    return [*s["out"], s["tokens"]] + ([s["blocks"]] if page > 1 else [])


def run(s):
    if own:
        return _own(s)
    if s["kind"] == "rope":
        return [_rotate(x.float(), s["positions"], s["inv_freq"], s["factor"],
                        s["interleaved"]).to(x.dtype) for x in (s["q"], s["k"])]
    if s["kind"] == "qk_norm":
        h, kvh, d = s["heads"]
        q, k, v = s["qkv"].view(-1, h + 2 * kvh, d).split([h, kvh, kvh], 1)
        q, k = (_rotate(_head_norm(x, gamma), s["positions"], s["inv_freq"], s["factor"],
                        s["interleaved"]).to(v.dtype)
                for x, gamma in ((q, s["q_gamma"]), (k, s["k_gamma"])))
        s["pool"][s["slots"].long()] = torch.cat([k, v], 1)
        return [q, s["pool"]]
    return {"window_prefill": _plain_prefill, "window_decode": _plain_decode,
            "slots": _plain_slots}[s["kind"]](s)


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    from lite_lang_amd import ops
    kind = s["kind"]
    if kind == "rope":
        return list(ops.rope_positions(s["q"], s["k"], s["positions"], s["inv_freq"],
                                       interleaved=s["interleaved"], factor=s["factor"],
                                       q_out=s["q_out"], k_out=s["k_out"]))
    if kind == "qk_norm":
        h, kvh, d = s["heads"]
        q = ops.qk_norm_rope_kv_scatter(s["qkv"], h, kvh, d, s["q_gamma"], s["k_gamma"], _EPS,
                                        s["positions"], s["inv_freq"], s["slots"], s["pool"],
                                        interleaved=s["interleaved"], factor=s["factor"],
                                        q_out=s["q_out"])
        return [q, s["pool"]]
    if kind == "window_prefill":
        return ops.window_prefill_attention(s["q"], s["k"], s["v"], s["out"], s["rows"],
                                            s["start"], s["seq_len"], s["max_len"], s["tokens"],
                                            s["window"], sinks=s["sinks"],
                                            b_shared_seq_len=s["cached"])
    if kind == "window_decode":
        return ops.window_decode_attention(s["q"], s["tokens"], s["rows"], s["seq_len"],
                                           s["max_len"], s["k"], s["v"], s["out"], s["window"],
                                           sinks=s["sinks"])
    ops.build_slot_maps(s["rows"], s["seq_len"], s["cached"], s["free"], s["tokens"], *s["out"],
                        page_size=s["page"], block_table=s["blocks"])
    return [*s["out"], s["tokens"]] + ([s["blocks"]] if s["page"] > 1 else [])


# ------------------------------------------------------------------ its size
def work(case):
    """Each input read once, each output written once; a multiply-add is 2."""
    kind = case["kind"]
    if kind in ("rope", "qk_norm"):
        h, kvh, d = _HEADS[case["heads"]]
        n = case["rows"] * (h + (2 if kind == "qk_norm" else 1) * kvh) * d
        extra = case["rows"] * (8 if kind == "qk_norm" else 4) + case["rotary"] * 2
        return {"bytes": 2 * n * 2 + extra, "flops": n * (7 if kind == "qk_norm" else 3)}
    lens, before = _lens(case), _before(case)
    if kind == "slots":
        t, page = sum(n - c for n, c in zip(lens, before)), case["page"]
        pages = sum(-(-n // page) - -(-c // page) for n, c in zip(lens, before))
        return {"bytes": 12 * t + (4 if page == 1 else 8) * pages + 20 * case["batch"] + 12,
                "flops": 0}
    h, kvh, d = _HEADS[case["heads"]]
    w, k = case["window"], case["sinks"]
    keys = rows = pairs = 0
    for n, c in zip(lens, before):
        c = c if kind == "window_prefill" else n - 1
        a, low = _visible(c, n - 1, w, k)
        keys += a + n - low
        rows += n - c
        # a query at p sees its last min(p + 1, w) tokens and the sinks before them
        p = np.arange(c, n, dtype=np.int64)
        pairs += int((np.minimum(p + 1, w) + np.minimum(np.maximum(p + 1 - w, 0), k)).sum())
    return {"bytes": keys * (2 * kvh * d * 2 + 4) + 2 * rows * h * d * 2,
            "flops": 4 * pairs * h * d}


# ------------------------------------------------------------------ 64 bits
def _x_turn(x, positions, inv_freq, factor, interleaved):
    """Each pair as a complex number times factor * exp(i * position * frequency)."""
    n = inv_freq.numel()
    y = x.clone()
    part = x[..., :2 * n]
    z = (part.unflatten(-1, (n, 2)) if interleaved
         else part.unflatten(-1, (2, n)).transpose(-1, -2)).contiguous()
    ang = positions.double().view(-1, 1, 1) * inv_freq.double()
    z = torch.view_as_complex(z) * torch.polar(torch.full_like(ang, factor), ang)
    z = torch.view_as_real(z)
    y[..., :2 * n] = (z if interleaved else z.transpose(-1, -2)).flatten(-2)
    return y


def _x_attend(q, k, v, first, window, sinks):
    """q [n, H, D] at positions first .., keys at their own positions 0 .. L-1
    (those that no query sees hold anything)."""
    n, h, d = q.shape
    kvh = k.shape[1]
    out = torch.empty(n, h, d, dtype=torch.float64, device=q.device)
    step = 512
    for r in range(0, n, step):
        m = min(step, n - r)
        low = max(0, first + r - window + 1)
        at = torch.arange(low, first + r + m, device=q.device)
        if low > 0 and sinks > 0:
            at = torch.cat([torch.arange(0, min(sinks, low), device=q.device), at])
        gap = torch.arange(first + r, first + r + m, device=q.device)[:, None] - at
        see = (gap >= 0) & ((gap < window) | (at < sinks))
        for c in range(h):
            kk, vv = k[at, c // (h // kvh)], v[at, c // (h // kvh)]
            e = q[r:r + m, c].contiguous().double() @ kk.double().t().contiguous() / math.sqrt(d)
            p = torch.softmax(e.masked_fill(~see, -math.inf), -1)
            out[r:r + m, c] = p @ vv.double()
    return out


def _x_slots(s):
    rows, page = s["rows"].tolist(), s["page"]
    free = s["free"].cpu().numpy()
    tokens = s["tokens"].cpu().numpy().copy()
    blocks = s["blocks"].cpu().numpy().copy() if page > 1 else None
    slots, positions, start, last, taken = [], [], [], [], 0
    for r, n, c in zip(rows, s["lens"], s["before"]):
        start.append(sum(map(len, slots)))
        have, need = -(-c // page), -(-n // page)
        mine = free[taken:taken + need - have]
        taken += need - have
        if page > 1:
            blocks[r, have:need] = mine
            ids = blocks[r, :need]
        else:
            ids = tokens[r, :need].copy()
            ids[have:] = mine
        p = np.arange(c, n)
        tokens[r, c:n] = ids[p // page] * page + p % page
        slots.append(tokens[r, c:n].copy())
        positions.append(p)
        last.append(start[-1] + n - c - 1 if n > c else -1)
    t = sum(map(len, slots))
    got = [np.concatenate(slots), np.concatenate(positions), start, last, [t, taken, 0], tokens]
    got += [blocks] if page > 1 else []
    return [torch.as_tensor(np.asarray(x, dtype=np.int32)) for x in got]


def exact(case, seed):
    if case["kind"] in ("window_prefill", "window_decode"):
        w = work(case)
        if w["flops"] > 2.5e12:
            return None
    s = prepare(case, seed)
    if case["kind"] == "slots":
        return _x_slots(s)
    if case["kind"] == "rope":
        return [_x_turn(x.double(), s["positions"], s["inv_freq"], s["factor"], s["interleaved"])
                for x in (s["q"], s["k"])]
    if case["kind"] == "qk_norm":
        h, kvh, d = s["heads"]
        x = s["qkv"].double().view(-1, h + 2 * kvh, d)
        pool = s["pool"].double()

        def side(y, gamma):
            y = y / (y.square().sum(-1, keepdim=True) / d + _EPS).sqrt() * gamma.double()
            return _x_turn(y, s["positions"], s["inv_freq"], s["factor"], s["interleaved"])

        pool.index_copy_(0, s["slots"].long(),
                         torch.cat([side(x[:, h:h + kvh], s["k_gamma"]), x[:, h + kvh:]], 1))
        return [side(x[:, :h], s["q_gamma"]), pool]
    outs, at = [], 0
    for i, (r, n) in enumerate(zip(s["rows"].tolist(), s["lens"])):
        slot = s["tokens"][r, :n].long()
        outs.append(_x_attend(s["q"][at:at + s["new"][i]], s["k"][slot], s["v"][slot],
                              n - s["new"][i], s["window"], s["sinks"]))
        at += s["new"][i]
    return torch.cat(outs)
