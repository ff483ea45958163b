"""GPU parity of the 8-bit cache, 4-bit products and logit controls against
oracle/low_bits.py.

Codes and scales are compared exactly, other floating outputs are held to the
oracle's bounds. Memory that a call must not read holds NaN (scales, floating
codes), memory that it must not write holds a pattern that is compared.
"""
import threading

import numpy as np
import pytest
import torch

from oracle import low_bits as O

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INT8, E4M3 = O.INT8, O.E4M3


def _ops():
    from lite_lang_amd import ops
    return ops


def _i32(v, dev="cuda", dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=dev)


def _inside(got, want, bound, what=""):
    """got within bound of want, element by element; NaN and infinities where want has them."""
    got = got.detach().cpu().to(torch.float64)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN"
    fin = torch.isfinite(want)
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]), f"{what}: infinities"
    excess = (got - want).abs()[fin] - bound[fin]
    if excess.numel():
        worst = float(((got - want).abs()[fin] / bound[fin].clamp_min(1e-300)).max())
        print(f"  {what}: worst {worst:.3f} of the bound", flush=True)
        assert float(excess.max()) <= 0.0, f"{what}: {worst:.3f} of the bound"


class Cache:
    """An 8-bit cache on the device beside the oracle's: K and V heads of one
    pool (or with rows of other strides), unused codes and scales NaN."""

    def __init__(self, slots, kvh, d, code, block, pad=0, extra=3):
        self.P, self.kvh, self.d, self.code, self.block = slots, kvh, d, code, block
        blocks = -(-slots // block)
        self.raw = torch.full((slots, 2 * kvh, d + pad), 0x7f, dtype=torch.uint8, device="cuda")
        pool = self.raw.view(code)[..., :d]
        self.k, self.v = pool[:, :kvh], pool[:, kvh:]
        self.scale = torch.full((blocks, 2 * kvh + extra), float("nan"), device="cuda")
        self.ks, self.vs = self.scale[:, :kvh], self.scale[:, kvh:2 * kvh]
        self.codes = pool.cpu().float().to(torch.float64)
        self.want = self.scale[:, :2 * kvh].cpu().to(torch.float64)

    @property
    def args(self):
        return self.k, self.v, self.ks, self.vs, self.block

    def store(self, k, v, slots):
        _ops().kv8_store(k.cuda() if not k.is_cuda else k, v.cuda() if not v.is_cuda else v,
                         _i32(slots), *self.args)
        O.kv8_store(torch.cat([k.cpu(), v.cpu()], 1), slots, self.codes, self.want, self.block,
                    self.code)

    def check(self):
        pool = self.raw.view(self.code)
        got = pool[..., :self.d].cpu().float().to(torch.float64)
        assert torch.equal(torch.nan_to_num(self.scale[:, :2 * self.kvh].cpu().double(), nan=-1.0),
                           torch.nan_to_num(self.want, nan=-1.0)), "scales"
        assert torch.equal(torch.nan_to_num(got, nan=999.0),
                           torch.nan_to_num(self.codes, nan=999.0)), "codes"
        assert bool((self.raw[..., self.d:] == 0x7f).all()), "beside the rows"
        assert bool(torch.isnan(self.scale[:, 2 * self.kvh:]).all()), "beside the scales"

    def values(self):
        y = O.kv8_values(self.codes, self.want, self.block)
        return y[:, :self.kvh], y[:, self.kvh:]


FORMS = [(2, 128, BF16, INT8, 16), (4, 128, F16, E4M3, 64), (8, 64, BF16, E4M3, 1),
         (1, 96, F32, INT8, 4), (3, 80, BF16, INT8, 32), (1, 10, F16, E4M3, 2),
         (2, 256, F32, E4M3, 8), (1, 128, BF16, INT8, 1), (5, 64, F16, INT8, 128),
         (2, 520, BF16, INT8, 16)]


def _pages(g, lens, block, spare=2):
    """(slot table rows, pages in no order) of requests with whole pages of a block."""
    need = [-(-n // block) for n in lens]
    perm = torch.randperm(sum(need) + spare, generator=g)
    table = torch.full((len(lens) + 1, max(need + [1]) * block), -1, dtype=torch.int32)
    at = 0
    for i, m in enumerate(need):
        ids = perm[at:at + m]
        table[i, :m * block] = (ids[:, None] * block + torch.arange(block)).flatten().int()
        at += m
    return table, (sum(need) + spare) * block


@pytest.mark.parametrize("kvh,d,dtype,code,block", FORMS)
def test_kv8_store(cuda, kvh, d, dtype, code, block):
    """Prompts, then single tokens and chunks that continue blocks, with ever
    larger values (scales grow, codes are rounded again) and smaller ones."""
    print(f"case: store {kvh}x{d} {dtype} {code} block {block}", flush=True)
    g = torch.Generator().manual_seed(d + block)
    final = [3 * block + 5, 40, block, 1, 70]
    table, slots = _pages(g, final, block)
    c = Cache(slots, kvh, d, code, block)
    done = [0] * len(final)
    for step in range(9):
        new = [min(n - a, (n * 2 // 3 if step == 0 else 1 if step < 5 else 7) if i != 4 or step else 0)
               for i, (n, a) in enumerate(zip(final, done))]
        sl = [int(s) for i, m in enumerate(new) for s in table[i, done[i]:done[i] + m]]
        sl = sl[:3] + [-1] + sl[3:] + [slots, -5, 2 ** 31 - 1]  # padded tokens among them
        mag = (1.0, 0.5, 2.0, 2.1, 0.01, 8.0, 1.0, 30.0, 1.0)[step]
        k = (torch.randn(len(sl), kvh, d, generator=g) * mag).to(dtype)
        v = (torch.randn(len(sl), kvh, d, generator=g) * mag * 3).to(dtype)
        c.store(k, v, sl)
        c.check()
        done = [a + m for a, m in zip(done, new)]


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_kv8_store_ties_and_borders(cuda, code, dtype):
    """Quotients half-way between two codes, and fp32 values one step beside
    those, for scales of 1 and of 24 bits."""
    gr = O.grid(code)
    mids = (gr[1:] + gr[:-1]) / 2
    for scale in ((1.0, 0.25) if dtype == BF16 else (1.0, 1.7182818, 0.0333333, 3.1e-7, 5.5e20)):
        s = float(np.float32(O.top(code) * np.float32(scale)) / np.float32(O.top(code)))
        x = torch.cat([mids, gr[:-1]]) * s
        x = torch.cat([x, torch.nextafter(x.float(), torch.tensor(3e38)).double(),
                       torch.nextafter(x.float(), torch.tensor(0.0)).double(), -x])
        x = x[x.abs() < O.top(code) * scale]
        d = 128
        x = torch.nn.functional.pad(x, (0, -len(x) % (d - 1))).view(-1, 1, d - 1)
        x = torch.cat([x, torch.full((x.shape[0], 1, 1), O.top(code) * scale)], -1).to(dtype)
        print(f"case: ties {code} {dtype} scale {scale} x {tuple(x.shape)}", flush=True)
        c = Cache(x.shape[0], 1, d, code, 1)
        c.store(x, -x, list(range(x.shape[0])))
        c.check()


@pytest.mark.parametrize("code", [INT8, E4M3])
def test_kv8_store_extremes(cuda, code):
    """Zeros, the smallest and the largest numbers, infinities and NaN: the scale's
    floor, a NaN scale for that head alone, and a block that begins anew."""
    d, block = 64, 4
    rows = {"zero": 0.0, "tiny": 1e-44, "small": 1e-30, "huge": 3.4e38, "inf": float("inf"),
            "-inf": -float("inf"), "nan": float("nan")}
    for name, val in rows.items():
        print(f"case: extremes {code} {name}", flush=True)
        c = Cache(8 * block, 2, d, code, block)
        x = torch.randn(3, 2, d, generator=torch.Generator().manual_seed(1))
        x[1, 1] = 0.0
        x[1, 1, 3] = val
        x[0, 1] = x[2, 1] = 0.0
        c.store(x, torch.randn(3, 2, d), [4, 5, 6])
        c.check()
        c.store(torch.ones(1, 2, d), torch.ones(1, 2, d), [7])  # continues the block
        c.check()
        bad = not np.isfinite(val)
        assert bool(torch.isnan(c.ks[1]).any()) == bad
        c.store(torch.ones(2, 2, d), torch.ones(2, 2, d), [4, 5])  # begins it anew
        c.check()
        assert bool(torch.isfinite(c.ks[1]).all())


def test_kv8_store_strides(cuda):
    """Heads inside a projection's rows, rows of odd strides, pools whose rows are
    not aligned, K and V in pools of their own."""
    g = torch.Generator().manual_seed(3)
    for d, pad, width in ((64, 3, 0), (128, 8, 5), (96, 1, 8), (64, 0, 3)):
        print(f"case: strides {d} {pad} {width}", flush=True)
        kvh, T, block = 2, 21, 8
        c = Cache(48, kvh, d, INT8, block, pad=pad)
        row = torch.randn(T, (4 + 2 * kvh) * d + width, generator=g).to(BF16).cuda()
        k = row[:, 4 * d:(4 + kvh) * d].unflatten(1, (kvh, d))
        v = row[:, (4 + kvh) * d:(4 + 2 * kvh) * d].unflatten(1, (kvh, d))
        c.store(k, v, list(range(16, 16 + T)))
        c.check()
        one = k[:, :1].expand(T, kvh, d)  # one head for all
        c.store(one, v, list(range(16, 16 + T)))
        c.check()


def test_kv8_store_of_a_long_prompt(cuda):
    """More runs than a wave takes, runs across the waves' borders."""
    g = torch.Generator().manual_seed(8)
    for block in (1, 16, 64):
        final = [1500, 777, 1024, 33]
        table, slots = _pages(g, final, block)
        c = Cache(slots, 2, 64, INT8, block)
        for lo, hi in ((0.0, 0.37), (0.37, 1.0)):
            sl = [int(s) for i, n in enumerate(final) for s in table[i, int(n * lo):int(n * hi)]]
            x = torch.randn(len(sl), 2, 64, generator=g).to(BF16)
            c.store(x, x.flip(0) * 2, sl)
            c.check()


@pytest.mark.parametrize("code", [INT8, E4M3])
def test_kv8_store_on_a_cache_of_single_slots(cuda, code):
    """PageCache's slots, freed and handed out again in another order, with a scale for
    each: prompts, steps and new requests on the slots of former ones."""
    from types import SimpleNamespace

    from lite_lang_amd.models.cache import PageCache
    g = torch.Generator().manual_seed(4)
    pc = PageCache(6, 64, 0.0, 1, 64, 2, torch_dtype=BF16, kv_max_size=120, device=cuda)
    c = Cache(120, 2, 64, code, 1)
    live, lens = [], {}

    def add(rids, new):
        slots = pc.alloc_token_idxs(rids, [lens[r] for r in rids], new)
        x = torch.randn(len(slots), 2, 64, generator=g).to(BF16)
        c.store(x, x.flip(0) * 3, slots.tolist())
        for r, n in zip(rids, new):
            lens[r] += n

    for step in range(12):
        fresh = [pc.alloc_req() for _ in range((3, 0, 1, 2)[step % 4])]
        lens.update({r: 0 for r in fresh})
        if fresh:
            add(fresh, [5 + 3 * i + step % 3 for i in range(len(fresh))])
        live += fresh
        add(live, [1] * len(live))
        c.check()
        while len(live) > 3:  # the oldest go, its slots to the next
            r = live.pop(step % 2)
            pc.free_req(SimpleNamespace(rid=r, length=lens.pop(r) + 1))
    q = torch.randn(len(live), 4, 64, generator=g).to(BF16)
    out, n = torch.empty_like(q, device="cuda"), [lens[r] for r in live]
    _ops().kv8_decode_attention(q.cuda(), pc.req_to_tokens_, _i32(live), _i32(n), max(n), *c.args, out)
    want = O.kv8_decode(q, *c.values(), pc.req_to_tokens_.cpu(), live, n, c.P)
    _inside(out, want[0], O.bound_kv8_decode(*want, BF16, 64), "out")


def test_kv8_far_slots(cuda):
    """Slots whose rows lie beyond 2^31 and 2^32 bytes."""
    kvh, d, block = 8, 128, 16
    P = ((1 << 32) // (2 * kvh * d) + 4096) // block * block
    pool = torch.empty(P, 2 * kvh, d, dtype=INT8, device="cuda")
    scale = torch.empty(P // block, 2 * kvh, device="cuda")
    cache = (pool[:, :kvh], pool[:, kvh:], scale[:, :kvh], scale[:, kvh:], block)
    g = torch.Generator().manual_seed(2)
    n = 40
    for first in ((1 << 31) // (2 * kvh * d) - 32, P - 48):
        print(f"case: far slots from {first}", flush=True)
        sl = torch.arange(first, first + n, dtype=torch.int32)
        x = torch.randn(n, kvh, d, generator=g).to(BF16)
        small = Cache(n, kvh, d, INT8, block)
        small.store(x, x * 2, list(range(n)))
        small.check()
        _ops().kv8_store(x.cuda(), (x * 2).cuda(), sl.cuda(), *cache)
        blocks = slice(first // block, first // block + 3)
        assert torch.equal(pool[first:first + n], small.raw.view(INT8))
        assert torch.equal(scale[blocks], small.scale[:, :2 * kvh])
        q = torch.randn(1, 16, d, generator=g).to(BF16).cuda()
        a, b = torch.empty_like(q), torch.empty_like(q)
        req, ln, st = _i32([0]), _i32([n]), _i32([0])
        ko = [torch.empty(n, kvh, d, dtype=BF16, device="cuda") for _ in range(4)]
        for cc, t, o, kk in ((cache, sl.view(1, n).cuda(), a, ko[:2]),
                             (small.args, torch.arange(n, dtype=torch.int32).view(1, n).cuda(), b,
                              ko[2:])):
            _ops().kv8_decode_attention(q, t, req, ln, n, *cc, o)
            _ops().kv8_load(*cc, t, req, st, ln, n, *kk)
        assert torch.equal(a, b) and torch.equal(ko[0], ko[2]) and torch.equal(ko[1], ko[3])


# ---------------------------------------------------------------- reading back
def _filled(g, lens, kvh, d, code, block, dtype, pad=0, mag=1.0):
    """A cache that holds contexts of these lengths, its table (garbage behind
    them) and the request rows."""
    table, slots = _pages(g, lens, block)
    c = Cache(slots, kvh, d, code, block, pad=pad)
    sl = [int(s) for i, n in enumerate(lens) for s in table[i, :n]]
    if sl:
        x = (torch.randn(len(sl), kvh, d, generator=g) * mag).to(dtype)
        y = torch.randn(len(sl), kvh, d, generator=g).to(dtype)
        c.store(x, y, sl)
    order = torch.randperm(len(lens) + 1, generator=g)
    rids = torch.argsort(order)[:len(lens)].tolist()
    return c, table[order], rids


@pytest.mark.parametrize("kvh,d,dtype,code,block", FORMS)
def test_kv8_load(cuda, kvh, d, dtype, code, block):
    g = torch.Generator().manual_seed(d)
    lens = [37, 0, 1, 2 * block + 3, 90]
    c, table, rids = _filled(g, lens, kvh, d, code, block, dtype)
    table[rids[4], 5], table[rids[4], 7] = -1, c.P  # no tokens: zeros
    start = [3, 40, 41, 45, 50 + 2 * block]
    rows = start[4] + 90 - 4  # the last request's last rows do not fit
    for idx in (torch.int32, torch.int64):
        print(f"case: load {kvh}x{d} {dtype} {code} block {block} {idx}", flush=True)
        out = [torch.full((rows, kvh, d), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        _ops().kv8_load(*c.args, table.cuda(), _i32(rids, dtype=idx), _i32(start, dtype=idx),
                        _i32(lens, dtype=idx), max(lens), *out)
        for got, val in zip(out, c.values()):
            want = torch.full((rows, kvh, d), 7.0, dtype=torch.float64)
            for r, s, n in zip(rids, start, lens):
                for i in range(min(n, rows - s)):
                    slot = int(table[r, i])
                    want[s + i] = val[slot] if 0 <= slot < c.P else 0.0
            _inside(got, want, O.bound_value(want, dtype), "values")


def test_kv8_load_bounds_and_strides(cuda):
    """Lengths beyond the bound, requests outside the table, outputs of other
    strides, rows of pools that are not aligned."""
    g = torch.Generator().manual_seed(4)
    for d, pad in ((64, 0), (64, 3), (96, 8)):
        print(f"case: load strides {d} {pad}", flush=True)
        c, table, rids = _filled(g, [30, 20, 9], 2, d, INT8, 8, BF16, pad=pad)
        wide = torch.full((70, 5, d + pad), 7.0, dtype=BF16, device="cuda")
        k, v = wide[:, 1:3, :d], wide[:, 3:5, :d]
        req = rids[:1] + [-1] + rids[1:] + [table.shape[0]]
        _ops().kv8_load(*c.args, table.cuda(), _i32(req), _i32([0, 12, 15, 40, 50]),
                        _i32([30, 4, 20, -3, 9]), 12, k, v)
        for got, val in zip((k, v), c.values()):
            want = torch.full((70, 2, d), 7.0, dtype=torch.float64)
            want[:12] = val[table[rids[0], :12].long()]
            want[15:27] = val[table[rids[1], :12].long()]
            _inside(got, want, O.bound_value(want, BF16), "values")
        assert bool((wide[:, 0] == 7.0).all()) and bool((wide[..., d:] == 7.0).all())


def test_kv8_lengths_below_zero(cuda):
    """Lengths below 0 are of empty requests, in 64 bits too: those whose low 32
    bits are a small, and the largest, positive number."""
    g = torch.Generator().manual_seed(5)
    c, table, rids = _filled(g, [20, 30], 2, 64, INT8, 8, BF16)
    rids = rids[:1] * 5 + rids[1:]
    lens = [-1, -2 ** 31, -2 ** 33 + 5, -2 ** 32 + 2 ** 31 - 1, -2 ** 63, 30]
    i64 = lambda v: _i32(v, dtype=torch.int64)  # noqa: E731
    out = [torch.full((40, 2, 64), 7.0, dtype=BF16, device="cuda") for _ in range(2)]
    _ops().kv8_load(*c.args, table.cuda(), i64(rids), i64([0, 1, 2, 3, 4, 5]), i64(lens), 30, *out)
    for got, val in zip(out, c.values()):
        want = torch.full((40, 2, 64), 7.0, dtype=torch.float64)
        want[5:35] = val[table[rids[5], :30].long()]
        _inside(got, want, O.bound_value(want, BF16), "values")
    q = torch.randn(6, 4, 64, generator=g).to(BF16).cuda()
    o = torch.full_like(q, 7.0)
    _ops().kv8_decode_attention(q, table.cuda(), i64(rids), i64(lens), 30, *c.args, o)
    assert bool((o[:5] == 0).all()) and bool((o[5] != 0).any())


# ---------------------------------------------------------------- attention
ATT = [(16, 2, 128, BF16, INT8, 16), (12, 2, 128, BF16, E4M3, 64), (28, 4, 128, F16, INT8, 1),
       (32, 8, 64, F16, E4M3, 16), (8, 2, 64, BF16, INT8, 32), (4, 4, 128, F32, INT8, 16),
       (40, 2, 64, BF16, INT8, 8), (17, 1, 128, F32, E4M3, 2), (4, 1, 256, BF16, INT8, 16),
       (6, 3, 96, BF16, INT8, 4), (2, 1, 10, F16, E4M3, 16), (2, 2, 512, BF16, INT8, 128)]


def _decode_case(H, kvh, d, dtype, code, block, lens, seed=0, idx=torch.int32, bound=None,
                 scale=None, mag=1.0, pad=0, spoil=False):
    print(f"case: kv8 decode H={H}/{kvh} D={d} {dtype} {code} block {block} lens={lens[:6]} "
          f"x{len(lens)}", flush=True)
    g = torch.Generator().manual_seed(seed)
    c, table, rids = _filled(g, lens, kvh, d, code, block, BF16 if dtype == F32 else dtype, pad=pad)
    if spoil:  # slots that are none, whole requests of them
        for i, (r, n) in enumerate(zip(rids, lens)):
            at = torch.randperm(max(n, 1), generator=g)[:n // 3 if i else n]
            table[r, at] = torch.where(torch.rand(len(at), generator=g) < 0.5, -1, c.P).int()
    cap = [min(max(n, 0), bound) if bound is not None else n for n in lens]
    B = len(lens)
    q = (torch.randn(B, H, d, generator=g) * mag).to(dtype)
    wide = torch.full((B, H, d + pad), 7.0, dtype=dtype, device="cuda")
    qd = wide.clone()
    qd[..., :d] = q.cuda()
    out = wide[..., :d]
    _ops().kv8_decode_attention(qd[..., :d], table.cuda(), _i32(rids, dtype=idx),
                                _i32(lens, dtype=idx), bound if bound is not None else max(lens),
                                *c.args, out, sm_scale=scale)
    torch.cuda.synchronize()
    want = O.kv8_decode(q, *c.values(), table, rids, cap, c.P, scale)
    _inside(out, want[0], O.bound_kv8_decode(*want, dtype, d), "out")
    assert bool((wide[..., d:] == 7.0).all())
    return out


@pytest.mark.parametrize("H,kvh,d,dtype,code,block", ATT)
def test_kv8_decode_attention(cuda, H, kvh, d, dtype, code, block):
    _decode_case(H, kvh, d, dtype, code, block, [1, 2, 0, 333, 16, 17, 129], seed=d,
                 idx=torch.int64 if block == 16 else torch.int32)


@pytest.mark.parametrize("H,kvh,d,dtype,code,block", ATT)
def test_kv8_decode_attention_of_slots_that_are_none(cuda, H, kvh, d, dtype, code, block):
    """Table entries outside the cache are not attended to; a request of them
    alone is an empty one."""
    out = _decode_case(H, kvh, d, dtype, code, block, [40, 100, 33, 260], seed=d, spoil=True)
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("B,n", [(1, 9000), (3, 5000), (8, 3000), (40, 700), (130, 90)])
def test_kv8_decode_attention_splits(cuda, B, n):
    """Few long sequences and many short ones, a workspace that held NaN."""
    lens = [max(1, n - 131 * i) if i % 5 else n for i in range(B)]
    for H, kvh, d, dtype, code in ((4, 2, 128, BF16, INT8), (2, 1, 64, F16, E4M3)):
        need = _ops()._kv8_decode_bytes(B, H, kvh, d, n)
        if need:
            _ops().workspace(cuda, "kv8_decode", need).fill_(255)
        _decode_case(H, kvh, d, dtype, code, 16, lens, seed=B, mag=3.0)


def test_captured_kv8_decodes_share_no_workspace(cuda):
    """Two captured decodes in parts, replayed on two streams at the same time after
    their lengths changed, equal to eager calls."""
    servers, graphs, streams = [], [], []
    for seed, (H, kvh, d, dtype, code) in enumerate([(8, 2, 128, BF16, INT8), (4, 1, 64, F16, E4M3)]):
        g = torch.Generator().manual_seed(seed)
        c, table, rids = _filled(g, [2500, 900, 1800], kvh, d, code, 16, BF16)
        q = torch.randn(3, H, d, generator=g).to(dtype).cuda()
        lens, out = _i32([2500, 900, 1800]), torch.empty(3, H, d, dtype=dtype, device="cuda")
        assert _ops()._kv8_decode_bytes(3, H, kvh, d, 2500) > 0, "a case in parts"
        args = (q, table.cuda(), _i32(rids), lens, 2500, *c.args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _ops().kv8_decode_attention(*args, out)
        servers.append((args, lens, out))
        graphs.append(graph)
        streams.append(torch.cuda.Stream())
    for new in ([2500, 900, 1800], [1, 0, 1700], [2049, 2, 128], [2500, 900, 1800]):
        for _, lens, out in servers:
            lens.copy_(_i32(new))
            out.fill_(7.0)
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for args, _, out in servers:
            ref = torch.empty_like(out)
            _ops().kv8_decode_attention(*args, ref)
            assert torch.equal(out, ref), f"lengths {new}"


@pytest.mark.parametrize("B,most", [(1, 768), (1, 769), (70, 2000), (33, 2049)])
def test_kv8_decode_attention_around_the_plans_border(cuda, B, most):
    """Contexts in one workgroup and in parts, lengths below the call's bound."""
    g = np.random.RandomState(most)
    lens = [most] + [0 if i % 9 == 4 else int(n) for i, n in enumerate(g.randint(1, 400, size=B - 1))]
    _decode_case(4, 1, 64, BF16, INT8, 16, lens, seed=B)
    _decode_case(2, 1, 128, F16, E4M3, 32, lens[:3], seed=B, bound=most)


@pytest.mark.parametrize("B,H,kvh", [(1, 520, 520), (3, 513, 513), (2, 8200, 1)])
def test_kv8_decode_attention_of_more_head_blocks_than_places(cuda, B, H, kvh):
    """More head blocks than workgroups run at a time: one workgroup to each. Some
    heads against the oracle, the others against calls of those heads alone."""
    d, n = 64, 2100
    print(f"case: {B} requests of {H}/{kvh} heads", flush=True)
    need = _ops()._kv8_decode_bytes(B, H, kvh, d, n)
    assert need == (1 + B) * H * (d * 4 + 8) + B * 8, "one workgroup to a head block"
    _ops().workspace(cuda, "kv8_decode", need).fill_(255)
    g = torch.Generator().manual_seed(B)
    lens = [n, 1, 700][:B]
    pool = torch.randint(-127, 128, (n, 2 * kvh, d), generator=g, dtype=torch.int8)
    scale = torch.rand(-(-n // 16), 2 * kvh, generator=g) * 0.01 + 0.001
    q = torch.randn(B, H, d, generator=g).to(BF16)
    table = torch.stack([torch.randperm(n, generator=g) for _ in range(B)]).int()
    pd, sd, qd, td, rows, ln = pool.cuda(), scale.cuda(), q.cuda(), table.cuda(), _i32(range(B)), _i32(lens)
    out = torch.full_like(qd, 7.0)
    _ops().kv8_decode_attention(qd, td, rows, ln, n, pd[:, :kvh], pd[:, kvh:], sd[:, :kvh],
                                sd[:, kvh:], 16, out)
    torch.cuda.synchronize()
    G = H // kvh
    few = [0, kvh // 2, kvh - 1] if kvh > 1 else [0]
    for kh in few:
        heads = list(range(kh * G, kh * G + min(G, 16)))
        vals = O.kv8_values(pool.double(), scale.double(), 16)
        want = O.kv8_decode(q[:, heads], vals[:, [kh]], vals[:, [kvh + kh]], table, range(B), lens, n)
        _inside(out[:, heads], want[0], O.bound_kv8_decode(*want, BF16, d), f"head {kh}")
    # 64 KV heads (or 1,024 query heads) at a time, dealt out over more workgroups.
    # Each output is off by half a bf16 step; the sums before it by 2^-16 of the
    # values' mean magnitude (0.35) each, and fp32's roundings.
    step = 64 if kvh > 1 else 1
    for k0 in range(0, kvh, step):
        k1, h0, h1 = min(k0 + step, kvh), k0 * G, min(k0 + step, kvh) * G
        for a in range(h0, h1, 1024 if kvh == 1 else h1):
            b = min(a + 1024, h1) if kvh == 1 else h1
            ref = torch.empty(B, b - a, d, dtype=BF16, device="cuda")
            _ops().kv8_decode_attention(qd[:, a:b], td, rows, ln, n, pd[:, k0:k1],
                                        pd[:, kvh + k0:kvh + k1], sd[:, k0:k1],
                                        sd[:, kvh + k0:kvh + k1], 16, ref)
            off = (out[:, a:b].float() - ref.float()).abs()
            top = torch.maximum(out[:, a:b].float().abs(), ref.float().abs())
            assert bool((off <= 2.0 ** -7 * top + 2e-5).all()), (a, float(off.max()))


def test_kv8_decode_attention_bounds_and_scales(cuda):
    _decode_case(8, 2, 128, BF16, INT8, 16, [500, 90, 3], bound=100)
    _decode_case(4, 2, 64, BF16, INT8, 16, [0, 0], bound=16)
    _decode_case(4, 2, 64, BF16, INT8, 16, [30, 2], bound=0)
    _decode_case(4, 2, 128, BF16, INT8, 16, [200, 31], scale=0.5)
    _decode_case(4, 2, 128, F16, INT8, 16, [200, 31], mag=6.0)
    for pad in (3, 8):
        _decode_case(4, 2, 128, BF16, INT8, 16, [200, 31], pad=pad)
        _decode_case(4, 2, 64, F32, E4M3, 16, [200, 31], pad=pad)


def test_kv8_decode_attention_rows_outside_the_table(cuda):
    g = torch.Generator().manual_seed(1)
    c, table, rids = _filled(g, [20, 30], 2, 64, INT8, 16, BF16)
    q = torch.randn(4, 4, 64, generator=g).to(BF16).cuda()
    out, ref = torch.full_like(q, 7.0), torch.full_like(q[1:3], 7.0)
    req = [-1] + rids + [table.shape[0]]
    _ops().kv8_decode_attention(q, table.cuda(), _i32(req), _i32([5, 20, 30, 9]), 30, *c.args, out)
    _ops().kv8_decode_attention(q[1:3], table.cuda(), _i32(rids), _i32([20, 30]), 30, *c.args, ref)
    assert torch.equal(out[1:3], ref)
    assert bool((out[0] == 0).all()) and bool((out[3] == 0).all())


def test_kv8_nan_scales_stay_in_their_head(cuda):
    """A NaN among one head's tokens reaches that head's outputs and no others."""
    g = torch.Generator().manual_seed(1)
    for d, kind in ((128, 0), (64, 1)):
        c, table, rids = _filled(g, [70, 40], 2, d, INT8, 16, BF16)
        (c.ks, c.vs)[kind][int(table[rids[0], 50]) // 16, 1] = float("nan")
        q = torch.randn(2, 8, d, generator=g).to(BF16).cuda()
        out = torch.empty_like(q)
        _ops().kv8_decode_attention(q, table.cuda(), _i32(rids), _i32([70, 40]), 70, *c.args, out)
        nan = torch.isnan(out).cpu()
        assert bool(nan[0, 4:].all()) and not bool(nan[0, :4].any()) and not bool(nan[1].any())


@pytest.mark.parametrize("B,most", [(300, 700), (700, 260), (257, 1300)])
def test_kv8_decode_attention_of_many_requests(cuda, B, most):
    """More requests than a workgroup has threads, empty ones among them, shares
    that begin and end inside requests."""
    g = np.random.RandomState(B)
    lens = [0 if i % 7 == 3 else int(n) for i, n in enumerate(g.randint(1, most, size=B))]
    lens[0], lens[-1], lens[5] = 0, 0, most
    _decode_case(2, 1, 64, BF16, INT8, 16, lens, seed=B)
    lens[7] = 2300  # more than a workgroup takes: in parts
    _decode_case(2, 1, 64, BF16, INT8, 16, lens, seed=B)


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_kv8_decode_attention_of_scales_far_apart(cuda, code, dtype):
    """V (and K) whose scales grow by 2^50 and fall by 2^80 along the context, and
    queries of any size: no sum leaves fp32's range where the outputs do not."""
    g = torch.Generator().manual_seed(9)
    for mags in ((1e-12, 1.0, 1e4), (1e4, 1e-20, 1.0), (1e-22, 1e-22, 1e-22), (1e20, 1e20, 1e18)):
        for qmag in (1e-6, 1.0):
            print(f"case: scales {code} {dtype} {mags} {qmag}", flush=True)
            n, d = 3 * 160, 64
            c = Cache(n, 1, d, code, 16)
            for i, m in enumerate(mags):
                sl = list(range(160 * i, 160 * i + 160))
                k = torch.randn(160, 1, d, generator=g) * min(m, 1.0)
                c.store(k.to(BF16), (torch.randn(160, 1, d, generator=g) * m).to(BF16), sl)
            q = (torch.randn(2, 4, d, generator=g) * qmag).to(dtype)
            table = torch.arange(n, dtype=torch.int32).view(1, n)
            out = torch.empty(2, 4, d, dtype=dtype, device="cuda")
            _ops().kv8_decode_attention(q.cuda(), table.cuda(), _i32([0, 0]), _i32([n, 200]), n,
                                        *c.args, out)
            want = O.kv8_decode(q, *c.values(), table, [0, 0], [n, 200], n)
            _inside(out, want[0], O.bound_kv8_decode(*want, dtype, d), "out")


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("first", [False, True])
def test_kv8_decode_attention_of_tokens_beside_far_larger_ones(cuda, code, first):
    """Tokens of V scales 2^-50 of others' that no query looks at (their scores are 200
    below): the outputs are the small ones' to the usual bound."""
    g = torch.Generator().manual_seed(12)
    n, d = 480, 64
    for big in (160, 16):
        c = Cache(n, 1, d, code, 16)
        far = torch.zeros(n, dtype=torch.bool)
        far[:big if first else 0] = True
        if not first:
            far[n - big:] = True
        k = torch.where(far[:, None, None], -5.0, 0.5) * torch.ones(n, 1, d)
        v = torch.randn(n, 1, d, generator=g) * torch.where(far, 2.0 ** 50, 1.0)[:, None, None]
        c.store(k.to(BF16), v.to(BF16), list(range(n)))
        q = (torch.rand(1, 4, d, generator=g) * 0.2 + 4.5).to(BF16)
        out = torch.empty(1, 4, d, dtype=BF16, device="cuda")
        table = torch.arange(n, dtype=torch.int32).view(1, n)
        _ops().kv8_decode_attention(q.cuda(), table.cuda(), _i32([0]), _i32([n]), n, *c.args, out)
        want = O.kv8_decode(q, *c.values(), table, [0], [n], n)
        assert float(want[1].max()) < 4.0, "the far ones do not count"
        _inside(out, want[0], O.bound_kv8_decode(*want, BF16, d), "out")


@pytest.mark.parametrize("code", [INT8, E4M3])
@pytest.mark.parametrize("d", [64, 128, 256, 96])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_kv8_decode_attention_of_the_largest_queries(cuda, code, d, dtype):
    """Queries up to the type's largest, over keys that keep the scores small; heads
    of ordinary queries, of zeros and of the smallest beside them."""
    g = torch.Generator().manual_seed(d)
    n = 300
    for mag in (2.0 ** 49, 2.0 ** 52, 2.0 ** 100, 2.0 ** 117, 2.0 ** 118, 2.0 ** 124, 3e38):
        # (of 2^-80 and more in the scale: the smallest that a block has)
        size = max(1.0 / mag, 2.0 ** -70)
        print(f"case: queries of {mag:.3g}, keys of {size:.3g} {code} {dtype} D={d}", flush=True)
        c = Cache(n, 1, d, code, 16)
        k = (torch.randn(n, 1, d, generator=g) * size).to(BF16)
        c.store(k, torch.randn(n, 1, d, generator=g).to(BF16), list(range(n)))
        q = ((0.5 + torch.rand(2, 4, d, generator=g) * 0.49) * mag).to(dtype)
        q[:, 1] = torch.randn(2, d, generator=g)
        q[:, 2] = 0.0
        q[:, 3] = 1e-37
        assert bool(torch.isfinite(q).all())
        table = torch.arange(n, dtype=torch.int32).view(1, n)
        out = torch.empty(2, 4, d, dtype=dtype, device="cuda")
        scale = 1.0 / max(mag * size, 1.0) / d ** 0.5
        _ops().kv8_decode_attention(q.cuda(), table.cuda(), _i32([0, 0]), _i32([n, 129]), n,
                                    *c.args, out, sm_scale=scale)
        want = O.kv8_decode(q, *c.values(), table, [0, 0], [n, 129], n, scale)
        _inside(out, want[0], O.bound_kv8_decode(*want, dtype, d), "out")


# ---------------------------------------------------------------- 4-bit products
def _weight(g, N, K, group, dtype, zero):
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scale = ((torch.rand(N, K // group, generator=g) + 0.5) * 0.05).to(dtype)
    z = torch.randint(0, 16, scale.shape, generator=g, dtype=torch.uint8) if zero else None
    return codes, scale, z, _ops().W4Weight(codes.cuda(), scale.cuda(), None if z is None else z.cuda())


@pytest.mark.parametrize("N,K,group", [(16, 32, 32), (1, 128, 128), (17, 64, 64), (100, 96, 32),
                                       (100, 192, 64), (256, 128, 128), (333, 1536, 128),
                                       (2053, 640, 128), (70, 8960, 64), (48, 11008, 128)])
@pytest.mark.parametrize("dtype,zero", [(BF16, False), (BF16, True), (F16, False), (F16, True)])
def test_linear_w4(cuda, N, K, group, dtype, zero):
    g = torch.Generator().manual_seed(N + K)
    codes, scale, z, w = _weight(g, N, K, group, dtype, zero)
    assert w.shape == (N, K) and w.group == group
    for M in (1, 2, 7, 16, 17, 33, 40, 64, 65, 150):
        print(f"case: w4 {M}x{N}x{K} group {group} {dtype} zero={zero}", flush=True)
        x = torch.randn(M, K, generator=g).to(dtype)
        if M == 7:
            x = x + 2  # sums that do not cancel
        bias = torch.randn(N, generator=g).to(dtype) if M % 2 else None
        out = torch.full((M + 1, N), 7.0, dtype=dtype, device="cuda")
        r = _ops().linear_w4(x.cuda(), w, None if bias is None else bias.cuda(), out=out[:M])
        assert r.data_ptr() == out.data_ptr() and bool((out[M] == 7.0).all())
        y, mag = O.linear_w4(x, codes, scale, z, bias)
        _inside(out[:M], y, O.bound_linear_w4(y, mag, dtype, K), "y")


@pytest.mark.parametrize("N,K,group,dtype,zero", [(32800, 256, 128, BF16, False),
                                                  (65553, 128, 64, F16, True),
                                                  (65600, 160, 32, BF16, True),
                                                  (9000, 384, 128, F16, False)])
def test_linear_w4_of_many_outputs(cuda, N, K, group, dtype, zero):
    """Weights wide enough for several tiles to a wave, and the plans between."""
    g = torch.Generator().manual_seed(N)
    codes, scale, z, w = _weight(g, N, K, group, dtype, zero)
    for M in (1, 5, 20, 40, 64, 130):
        print(f"case: w4 {M}x{N}x{K} group {group} {dtype} zero={zero}", flush=True)
        x = torch.randn(M, K, generator=g).to(dtype)
        y, mag = O.linear_w4(x, codes, scale, z)
        _inside(_ops().linear_w4(x.cuda(), w), y, O.bound_linear_w4(y, mag, dtype, K), "y")


def test_linear_w4_splits_are_added_in_order(cuda):
    """Few outputs and long sums: the same bits from a workspace that held NaN and
    from one of a captured graph, replayed beside other work."""
    g = torch.Generator().manual_seed(11)
    codes, scale, z, w = _weight(g, 130, 11008, 128, BF16, True)
    for M in (17, 40, 100):
        x = torch.randn(M, 11008, generator=g).to(BF16).cuda()
        need = _ops()._linear_w4_bytes(M, 130, 11008)
        assert need > M * 130 * 4
        first = _ops().linear_w4(x, w).clone()
        _ops().workspace(cuda, "linear_w4", need).fill_(255)
        assert torch.equal(_ops().linear_w4(x, w), first)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = _ops().linear_w4(x, w)
        for _ in range(3):
            y.zero_()
            graph.replay()
            other = _ops().linear_w4(x * 2, w)
            torch.cuda.synchronize()
            assert torch.equal(y, first) and not torch.equal(other, first)


def test_linear_w4_strides(cuda):
    """Rows of x and y inside wider ones, aligned and not; the row order; M = 0."""
    g = torch.Generator().manual_seed(5)
    N, K = 130, 256
    codes, scale, z, w = _weight(g, N, K, 64, BF16, True)
    for M in (3, 20, 70):
        for pad, at in ((8, 8), (3, 1), (1, 0)):
            print(f"case: w4 strides M={M} pad={pad} at={at}", flush=True)
            wide = torch.randn(M, K + pad, generator=g).to(BF16).cuda()
            x = wide[:, at:at + K]
            out = torch.full((M, N + pad), 7.0, dtype=BF16, device="cuda")
            _ops().linear_w4(x, w, out=out[:, at:at + N])
            y, mag = O.linear_w4(x.cpu(), codes, scale, z)
            _inside(out[:, at:at + N], y, O.bound_linear_w4(y, mag, BF16, K), "y")
            out[:, at:at + N] = 7.0
            assert bool((out == 7.0).all())
    assert _ops().linear_w4(torch.empty(0, K, dtype=BF16, device="cuda"), w).shape == (0, N)
    one = torch.randn(1, K, generator=g).to(BF16).cuda()
    same = _ops().linear_w4(one.expand(5, K), w)
    assert torch.equal(same, same[:1].expand(5, N))


def test_linear_w4_zero_bytes_count_by_four_bits(cuda):
    g = torch.Generator().manual_seed(6)
    codes, scale, z, w = _weight(g, 32, 128, 32, BF16, True)
    w2 = _ops().W4Weight(codes.cuda(), scale.cuda(), (z | 0xa0).cuda())
    x = torch.randn(4, 128, generator=g).to(BF16).cuda()
    assert torch.equal(_ops().linear_w4(x, w), _ops().linear_w4(x, w2))


@pytest.mark.parametrize("N,K,group,zero", [(100, 160, 32, False), (333, 256, 128, True),
                                            (48, 11008, 128, False), (32800, 256, 64, True),
                                            (9000, 192, 64, False)])
def test_linear_w4_of_the_largest_and_smallest_inputs(cuda, N, K, group, zero):
    """bf16 inputs up to the type's largest, with scales that keep the results finite,
    and down to its smallest: no sum leaves fp32's range where the result does not."""
    g = torch.Generator().manual_seed(N + K)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    z = torch.randint(0, 16, (N, K // group), generator=g, dtype=torch.uint8) if zero else None
    unit = torch.rand(N, K // group, generator=g) + 0.5
    # the largest: 3.39e38 in every input; of one sign and of both
    for mag, size, sign in ((3.38e38, 1e-7, False), (3.38e38, 1e-7, True), (1e34, 1e-3, False),
                            (2e36, 1e-3, True), (1e-30, 0.05, True), (1e-36, 0.05, True),
                            (3e-38, 0.05, True)):
        scale = (unit * size).to(BF16)
        w = _ops().W4Weight(codes.cuda(), scale.cuda(), None if z is None else z.cuda())
        for M in (1, 16, 20, 40, 70):
            print(f"case: w4 {M}x{N}x{K} group {group} zero={zero} of {mag}", flush=True)
            x = (1 - torch.rand(M, K, generator=g) * 0.2) * mag
            x = (x * (torch.randint(0, 2, (M, K), generator=g) * 2 - 1) if sign else x).to(BF16)
            assert bool(torch.isfinite(x).all())
            y, m = O.linear_w4(x, codes, scale, z)
            bound = O.bound_linear_w4(y, m, BF16, K)
            assert float(y.abs().max()) < 3e38
            _inside(_ops().linear_w4(x.cuda(), w), y, bound, "y")
            wide = torch.zeros(M, K + 1, dtype=BF16, device="cuda")
            wide[:, 1:] = x.cuda()
            _inside(_ops().linear_w4(wide[:, 1:], w), y, bound, "y, rows of any address")


W4_EXACT = [(48, 11008, 128, (1, 16, 17, 40, 64, 65, 150)), (130, 8960, 64, (2, 16, 33, 100)),
            (17, 160, 32, (1, 3, 16, 20, 70)), (333, 1536, 128, (5, 48, 600)),
            (9000, 384, 64, (1, 16, 20, 64)), (33000, 192, 32, (5, 16, 40, 130)),
            (70, 1152, 128, (2000,))]


@pytest.mark.parametrize("N,K,group,rows", W4_EXACT)
@pytest.mark.parametrize("dtype,zero", [(BF16, False), (BF16, True), (F16, False), (F16, True)])
def test_linear_w4_counts_every_input_once(cuda, N, K, group, rows, dtype, zero):
    """Rows of x of seven entries of 1 and -1, each input of the weight in one of them,
    and scales of 1 and 2: sums below 7 * 15 * 2 + 1, which every type holds exactly,
    so that an input that is lost, taken twice or met with another group's scale or
    zero point shows in the bits."""
    g = torch.Generator().manual_seed(N + K)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scale = torch.randint(1, 3, (N, K // group), generator=g).to(dtype)
    z = torch.randint(0, 16, scale.shape, generator=g, dtype=torch.uint8) if zero else None
    w = _ops().W4Weight(codes.cuda(), scale.cuda(), None if z is None else z.cuda())
    full = O.w4_weight(codes, scale, z).to(torch.float32).cuda()
    bias = torch.randint(-1, 2, (N,), generator=g).to(dtype).cuda()
    for M in rows:
        print(f"case: w4 exact {M}x{N}x{K} group {group} {dtype} zero={zero}", flush=True)
        order = torch.cat([torch.randperm(K, generator=g) for _ in range(-(-7 * M // K))])
        for at in range(0, len(order) if 7 * M <= K else 1, 7 * M):
            pos = order[at:at + 7 * M]
            pos = torch.cat([pos, order[:7 * M - len(pos)]]).view(M, 7).cuda()
            sign = (torch.randint(0, 2, (M, 7), generator=g) * 2 - 1).float().cuda()
            x = torch.zeros(M, K, device="cuda").scatter_add_(1, pos, sign)
            want = torch.zeros(M, N, device="cuda")
            for i in range(7):
                want += full[:, pos[:, i]].t() * sign[:, i, None]
            want = (want + bias).to(dtype)
            got = _ops().linear_w4(x.to(dtype), w, bias)
            assert torch.equal(got, want), f"inputs from {at} on"
            if at == 0:
                wide = torch.zeros(M, K + 1, dtype=dtype, device="cuda")
                wide[:, 1:] = x
                assert torch.equal(_ops().linear_w4(wide[:, 1:], w, bias), want), "rows of any address"


@pytest.mark.parametrize("dtype,zero", [(BF16, False), (BF16, True), (F16, False), (F16, True)])
def test_linear_w4_of_small_whole_numbers_is_exact(cuda, dtype, zero):
    """Full rows of -1, 0 and 1: every sum, of x (128 + c) too, is a whole number below
    2^24 (11,008 * 143), so the result is the exact one, rounded once."""
    g = torch.Generator().manual_seed(3)
    for N, K, group in ((130, 11008, 128), (48, 8960, 64), (9000, 1536, 32), (33000, 512, 128)):
        codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
        scale = torch.full((N, K // group), 0.125).to(dtype)
        z = torch.randint(0, 16, scale.shape, generator=g, dtype=torch.uint8) if zero else None
        w = _ops().W4Weight(codes.cuda(), scale.cuda(), None if z is None else z.cuda())
        full = O.w4_weight(codes, scale, z).cuda()
        for M in (1, 16, 17, 40, 70):
            print(f"case: w4 whole {M}x{N}x{K} group {group} {dtype} zero={zero}", flush=True)
            x = torch.randint(-1, 2, (M, K), generator=g).cuda()
            want = (x.double() @ full.t()).to(dtype)
            assert torch.equal(_ops().linear_w4(x.to(dtype), w), want)


def test_linear_w4_rows_do_not_mix(cuda):
    """Infinities and NaN in one row of x leave the other rows' bits."""
    g = torch.Generator().manual_seed(6)
    for dtype in (BF16, F16):
        _, _, _, w = _weight(g, 80, 256, 128, dtype, False)
        for M in (2, 20, 70):
            x = torch.randn(M, 256, generator=g).to(dtype).cuda()
            good = _ops().linear_w4(x, w)
            x[M // 2, 9], x[M // 2, 200] = float("inf"), float("nan")
            bad = _ops().linear_w4(x, w)
            assert not bool(torch.isfinite(bad[M // 2]).any())
            keep = torch.arange(M) != M // 2
            assert torch.equal(bad[keep], good[keep])


# ---------------------------------------------------------------- logits
def _logit_case(B, V, n, nb, masked, dtype, seed=0, which=(1, 1, 1), idx=torch.int32, pad=0,
                inplace=False):
    print(f"case: logits {B}x{V} tokens {n} biases {nb} mask {masked} {dtype} {which}", flush=True)
    g = torch.Generator().manual_seed(seed)
    wide = (torch.randn(B, V + pad, generator=g) * 4).to(dtype).cuda()
    x = wide[:, :V]
    toks = rids = prompt = lens = None
    pen = [None, None, None]
    if n is not None:
        toks = torch.randint(-2, V + 3, (B + 2, max(n, 1)), generator=g, dtype=torch.int32)
        toks[:, ::3] = toks[:, :1].clone()  # one token over and over
        rids = torch.randperm(B + 2, generator=g)[:B].tolist()
        lens = [n, 0, n // 2, 1, n + 9][:B] + [n] * max(0, B - 5)
        prompt = [n // 2, 0, n, 0, 1][:B] + [n // 3] * max(0, B - 5)
        rep = 0.5 + torch.rand(B, generator=g)
        pen = [t if on else None for t, on in
               zip((rep, torch.randn(B, generator=g), torch.randn(B, generator=g)), which)]
    ids = vals = mask = None
    if nb is not None:
        ids = torch.randint(-1, V + 2, (B, nb), generator=g, dtype=torch.int32)
        vals = torch.randn(B, nb, generator=g) * 10
    if masked:
        mask = torch.randint(-2 ** 31, 2 ** 31, (B, -(-V // 32) + 1), generator=g).to(torch.int32)
        mask[0] = 0  # nothing is left
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    ii = lambda v: None if v is None else _i32(v, dtype=idx)  # noqa: E731
    out = x if inplace else torch.full_like(wide, 7.0)[:, :V]
    xc = x.cpu()
    r = _ops().adjust_logits(x, dev(toks), ii(rids), ii(prompt), ii(lens), repetition=dev(pen[0]),
                             frequency=dev(pen[1]), presence=dev(pen[2]), bias_ids=dev(ids),
                             bias_values=dev(vals), mask=dev(mask), out=out)
    assert r is out
    want, mag = O.adjust_logits(xc, toks, rids, prompt, lens, *pen, ids, vals, mask)
    _inside(out, want, O.bound_logits(want, mag, dtype, 6 + (nb or 0)), "logits")
    if not inplace:
        assert torch.equal(x.cpu(), xc)
        if pad:
            assert bool((out.as_strided((B, V + pad), (V + pad, 1))[:, V:] == 7.0).all())
    return out


@pytest.mark.parametrize("V", [1, 31, 33, 1000, 4096, 4097, 10001])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_adjust_logits(cuda, V, dtype):
    """Ids outside the vocabulary, tokens over and over, empty and over-long
    histories, several biases for one token, rows that the mask leaves empty."""
    for seed, (n, nb, masked) in enumerate([(50, 7, True), (1, None, False), (300, 40, False),
                                            (None, 3, True), (700, 0, True)]):
        _logit_case(5, V, n, nb, masked, dtype, seed=seed, idx=torch.int64 if seed else torch.int32)


def test_adjust_logits_parts(cuda):
    """Each control alone; odd row strides; in place."""
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 0, 0)):
        _logit_case(3, 5000, 200, None, False, F32, which=which)
    _logit_case(3, 5000, None, None, False, BF16)
    _logit_case(3, 5000, None, None, True, BF16)
    for pad in (1, 3, 8):
        _logit_case(4, 4999, 60, 5, True, F32, pad=pad)
        _logit_case(4, 4999, 60, 5, True, BF16, pad=pad, inplace=True)
    _logit_case(2, 300, 9000, 1, False, F32)


def test_adjust_logits_counts_many(cuda):
    """One token 100,000 times; every token of a long prompt; argmax of a row that
    nothing is left of."""
    V, n = 5003, 100000
    t = torch.full((1, n), 4097, dtype=torch.int32, device="cuda")
    x = torch.ones(1, V, device="cuda")
    args = (t, _i32([0]), _i32([0]), _i32([n]))
    y = _ops().adjust_logits(x, *args, frequency=torch.ones(1, device="cuda"))
    assert float(y[0, 4097]) == 1.0 - n and float(y.sum()) == V - n
    y = _ops().adjust_logits(x, t, _i32([0]), _i32([n]), _i32([n]),
                             repetition=torch.full((1,), 2.0, device="cuda"),
                             frequency=torch.ones(1, device="cuda"))
    assert float(y[0, 4097]) == 0.5  # of the prompt: no frequency
    y = _ops().adjust_logits(x, mask=torch.zeros(1, 157, dtype=torch.int32, device="cuda"))
    assert bool(torch.isneginf(y).all()) and int(_ops().argmax(y)[0]) == 0


def test_adjust_logits_of_no_history(cuda):
    """A table without columns counts nothing."""
    x = torch.randn(2, 50, device="cuda")
    none = torch.empty(3, 0, dtype=torch.int32, device="cuda")
    y = _ops().adjust_logits(x, none, _i32([0, 1]), _i32([0, 0]), _i32([0, 0]),
                             repetition=torch.full((2,), 2.0, device="cuda"))
    assert torch.equal(x, y)


@pytest.mark.parametrize("V,nb,kind", [(151936, 1 << 20, "random"), (5000, 1 << 20, "one"),
                                       (3000, 1000, "random"), (3000, 257, "two"),
                                       (70000, 40000, "random"), (2048, 64, "one")])
def test_adjust_logits_many_biases_of_a_token(cuda, V, nb, kind):
    """Lists that name tokens again and again, up to the longest: each token's sum
    is added up in the list's order, bit for bit."""
    print(f"case: {nb} biases ({kind}) of {V} tokens", flush=True)
    g = np.random.RandomState(nb % 1000)
    B = 2
    ids = {"random": g.randint(-3, V + 3, size=(B, nb)), "one": np.full((B, nb), V - 1),
           "two": g.randint(0, 2, size=(B, nb)) * (V - 1)}[kind].astype(np.int32)
    vals = (g.randn(B, nb) * 10.0 ** g.randint(-3, 4, size=(B, nb))).astype(np.float32)
    x = g.randn(B, V).astype(np.float32)
    want = x.copy()
    for b in range(B):
        total = np.full(V, -0.0, np.float32)
        ok = (ids[b] >= 0) & (ids[b] < V)
        np.add.at(total, ids[b][ok], vals[b][ok])  # entry after entry, each addition rounded
        hit = np.zeros(V, bool)
        hit[ids[b][ok]] = True
        want[b] = np.where(hit, x[b] + total, x[b])
    for pieces in (1, 2):  # rows of biases next to each other, and apart
        di = torch.from_numpy(np.tile(ids, (1, pieces))).cuda()[:, :nb]
        dv = torch.from_numpy(np.tile(vals, (1, pieces))).cuda()[:, :nb]
        y = _ops().adjust_logits(torch.from_numpy(x).cuda(), bias_ids=di, bias_values=dv)
        assert torch.equal(y.cpu(), torch.from_numpy(want)), f"rows of {pieces}"


def test_adjust_logits_sums_biases_first(cuda):
    """Two biases of 4 on 1e8, whose neighbours are 8 apart: their sum is added, not
    one after the other (which would leave 1e8)."""
    x = torch.full((1, 70), 1e8, device="cuda")
    y = _ops().adjust_logits(x, bias_ids=_i32([[3, 5, 3, -1]]),
                             bias_values=torch.tensor([[4.0, 4.0, 4.0, 9.0]], device="cuda"))
    want = torch.full((1, 70), 1e8)
    want[0, 3] = 1e8 + 8
    assert torch.equal(y.cpu(), want)


def test_adjust_logits_of_an_empty_table(cuda):
    """Tables of no row or no column count nothing, other controls go on."""
    x = torch.randn(2, 50, device="cuda")
    two, bias = torch.full((2,), 2.0, device="cuda"), torch.ones(2, 1, device="cuda")
    for rows, cols in ((3, 0), (0, 5), (0, 0)):
        t = torch.empty(rows, cols, dtype=torch.int32, device="cuda")
        y = _ops().adjust_logits(x, t, _i32([0, 1]), _i32([0, 0]), _i32([3, 3]), repetition=two,
                                 frequency=two, presence=two, bias_ids=_i32([[7], [-1]]),
                                 bias_values=bias)
        want = x.clone()
        want[0, 7] += 1.0
        assert torch.equal(y, want)
        with pytest.raises(ValueError, match="CPU"):
            _ops().adjust_logits(x, t, _i32([0, 1]), _i32([0, 0]), _i32([3, 3]), repetition=two.cpu())


def test_adjust_logits_infinities(cuda):
    """-inf stays -inf under a penalty and a bias, a mask rules NaN out."""
    inf = float("inf")
    x = torch.tensor([[-inf, inf, float("nan"), 1.0, float("nan")]], device="cuda")
    t = torch.arange(5, dtype=torch.int32, device="cuda").view(1, 5)
    y = _ops().adjust_logits(x, t, _i32([0]), _i32([0]), _i32([5]),
                             repetition=torch.full((1,), 2.0, device="cuda"),
                             presence=torch.ones(1, device="cuda"), bias_ids=t,
                             bias_values=torch.ones(1, 5, device="cuda"), mask=_i32([[0b01111]]))
    y = y.cpu()[0]
    assert y[0] == -inf and y[1] == inf and torch.isnan(y[2]) and y[3] == 0.5 and y[4] == -inf


# ---------------------------------------------------------------- a run of them
class Server:
    """A decode step of one layer and an lm head on 4-bit weights and an 8-bit
    cache: the calls of one step, each on what the one before left."""

    def __init__(self, B, seed, block=16, code=INT8):
        ops, g = _ops(), torch.Generator().manual_seed(seed)
        self.B, self.H, self.kvh, self.d, self.hid, self.V = B, 4, 2, 64, 256, 1000
        self.cap = 128
        H, kvh, d, hid = self.H, self.kvh, self.d, self.hid
        mk = lambda n, k: _weight(g, n, k, 64, BF16, True)[3]  # noqa: E731
        self.wqkv, self.wo, self.wl = mk((H + 2 * kvh) * d, hid), mk(hid, H * d), mk(self.V, hid)
        self.emb = torch.randn(self.V, hid, generator=g).to(BF16).cuda()
        self.f = ops.rope_frequencies(d)[0].cuda()
        pages = B * self.cap // block
        perm = torch.randperm(pages, generator=g)
        self.table = (perm[:, None] * block + torch.arange(block)).view(B, self.cap).int().cuda()
        pool = torch.zeros(pages * block, 2 * kvh, d, dtype=torch.uint8, device="cuda").view(code)
        self.pool, self.block = pool, block
        self.scale = torch.zeros(pages, 2 * kvh, device="cuda")
        self.cache = (pool[:, :kvh], pool[:, kvh:], self.scale[:, :kvh], self.scale[:, kvh:], block)
        self.rows = torch.arange(B, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor([3 + i for i in range(B)], dtype=torch.int32, device="cuda")
        self.prompt = self.lens.clone()
        self.history = torch.randint(0, self.V, (B, self.cap), generator=g, dtype=torch.int32).cuda()
        self.rep = torch.full((B,), 1.3, device="cuda")
        self.freq = torch.full((B,), 0.2, device="cuda")
        self.mask = torch.randint(-2 ** 31, 2 ** 31, (B, 32), generator=g).to(torch.int32).cuda()
        self.tok = torch.zeros(B, dtype=torch.int64, device="cuda")
        self.out = torch.empty(B, H, d, dtype=BF16, device="cuda")
        # the prompts' tokens
        T = int(self.lens.sum())
        x = torch.randn(T, (H + 2 * kvh) * d, generator=g).to(BF16).cuda()
        k, v = (x[:, a * d:b * d].unflatten(1, (kvh, d)) for a, b in ((H, H + kvh), (H + kvh, H + 2 * kvh)))
        slots = torch.cat([self.table[i, :n] for i, n in enumerate(self.lens.tolist())])
        ops.kv8_store(k, v, slots, *self.cache)

    def step(self):
        ops, H, kvh, d = _ops(), self.H, self.kvh, self.d
        pos = self.lens
        slots = self.table.gather(1, pos[:, None].long())[:, 0].contiguous()
        self.history.scatter_(1, pos[:, None].long(), self.tok[:, None].int())
        self.lens.add_(1)
        qkv = ops.linear_w4(self.emb[self.tok], self.wqkv)
        q = qkv[:, :H * d].unflatten(1, (H, d))
        k = qkv[:, H * d:(H + kvh) * d].unflatten(1, (kvh, d))
        v = qkv[:, (H + kvh) * d:].unflatten(1, (kvh, d))
        ops.rope_positions(q, k, self.lens - 1, self.f)
        ops.kv8_store(k, v, slots, *self.cache)
        ops.kv8_decode_attention(q, self.table, self.rows, self.lens, self.cap, *self.cache, self.out)
        y = ops.linear_w4(ops.linear_w4(self.out.flatten(1), self.wo), self.wl)
        y = ops.adjust_logits(y, self.history, self.rows, self.prompt, self.lens,
                              repetition=self.rep, frequency=self.freq, mask=self.mask)
        self.tok.copy_(ops.argmax(y))
        return y


def test_a_run_of_steps_stays_in_the_mask(cuda):
    s = Server(5, 1)
    for _ in range(30):
        y = s.step()
        assert bool(torch.isfinite(y[torch.arange(5), s.tok]).all())
        bit = (s.mask[torch.arange(5), s.tok // 32] >> (s.tok % 32)) & 1
        assert bool((bit == 1).all())
    # the cache that the steps left gives what prefill attention gives of its values
    n = s.lens.tolist()
    start = [sum(n[:i]) for i in range(5)]
    k, v = (torch.empty(sum(n), s.kvh, s.d, dtype=BF16, device="cuda") for _ in range(2))
    _ops().kv8_load(*s.cache, s.table, s.rows, _i32(start), s.lens, s.cap, k, v)
    q = torch.randn(5, s.H, s.d, device="cuda").to(BF16)
    a, b = torch.empty_like(q), torch.empty_like(q)
    _ops().kv8_decode_attention(q, s.table, s.rows, s.lens, s.cap, *s.cache, a)
    table = torch.zeros(5, s.cap, dtype=torch.int32, device="cuda")
    for i in range(5):
        table[i, :n[i]] = torch.arange(start[i], start[i] + n[i], device="cuda")
    _ops().prefill_attention(q, k, v, b, s.rows, s.rows, s.lens, 1, table, s.lens - 1)
    # values rounded to bf16 and probabilities once more: a few of their roundings
    assert float((a.float() - b.float()).abs().max()) <= 6 * O.u(BF16) * float(b.float().abs().max())


def test_captured_steps_replay(cuda):
    """Two servers' steps in two graphs, replayed in turn and at the same time on
    two streams, equal to eager ones."""
    servers = [Server(4, 7), Server(3, 8, code=E4M3)]
    eager = [Server(4, 7), Server(3, 8, code=E4M3)]
    graphs = []
    for s, e in zip(servers, eager):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.step()
        torch.cuda.current_stream().wait_stream(side)
        e.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.y = s.step()
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in servers]
    for it in range(8):
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
            if it % 2:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        for s, e in zip(servers, eager):
            want = e.step()
            assert torch.equal(s.y, want) and torch.equal(s.tok, e.tok), f"replay {it}"
            assert torch.equal(s.pool.view(torch.uint8), e.pool.view(torch.uint8))
            assert torch.equal(s.scale, e.scale)


def test_threads_with_streams_of_their_own(cuda):
    """Four threads' servers, each on its stream, give what they give alone."""
    alone = []
    for i in range(4):
        s = Server(3, 20 + i)
        alone.append([s.step().clone() for _ in range(6)])
    bad = []

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            s = Server(3, 20 + i)
            for y in alone[i]:
                if not torch.equal(s.step(), y):
                    bad.append(i)
            st.synchronize()

    torch.cuda.synchronize()
    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


@pytest.mark.parametrize("shared", [False, True])
def test_threads_whose_calls_hand_on_parts(cuda, shared):
    """Four threads' decodes and products in parts, which a second launch adds up from
    the stream's workspace: on streams of their own, and on one that all share."""
    ops, work = _ops(), []
    for i in range(4):
        g = torch.Generator().manual_seed(30 + i)
        lens = [2500 + 100 * i, 900, 2100]
        c, table, rids = _filled(g, lens, 2, 64, INT8, 16, BF16)
        q = torch.randn(3, 4, 64, generator=g).to(BF16).cuda()
        w = _weight(g, 130, 11008, 128, BF16, True)[3]
        x = torch.randn(40, 11008, generator=g).to(BF16).cuda()
        assert ops._kv8_decode_bytes(3, 4, 2, 64, max(lens)) > 0
        assert ops._linear_w4_bytes(40, 130, 11008) > 0
        work.append((c, q, table.cuda(), _i32(rids), _i32(lens), max(lens), x, w))

    def call(i):
        c, q, table, rids, lens, most, x, w = work[i]
        out = torch.empty_like(q)
        ops.kv8_decode_attention(q, table, rids, lens, most, *c.args, out)
        return out, ops.linear_w4(x, w)

    alone = [call(i) for i in range(4)]
    torch.cuda.synchronize()
    one, bad = torch.cuda.Stream(), []

    def run(i):
        st = one if shared else torch.cuda.Stream()
        with torch.cuda.stream(st):
            outs = [call(i) for _ in range(50)]
            st.synchronize()
            for o, y in outs:
                if not (torch.equal(o, alone[i][0]) and torch.equal(y, alone[i][1])):
                    bad.append(i)

    ts = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad


def test_calls_of_nothing(cuda):
    ops = _ops()
    c = Cache(32, 2, 64, INT8, 16)
    none = torch.empty(0, 2, 64, dtype=BF16, device="cuda")
    ops.kv8_store(none, none, _i32([]), *c.args)
    ops.kv8_load(*c.args, _i32([[0] * 8]), _i32([]), _i32([]), _i32([]), 8, none, none)
    q = torch.empty(0, 4, 64, dtype=BF16, device="cuda")
    assert ops.kv8_decode_attention(q, _i32([[0] * 8]), _i32([]), _i32([]), 8, *c.args, q) is q
    ops.adjust_logits(torch.empty(0, 9, device="cuda"))
    torch.cuda.synchronize()
    c.check()
