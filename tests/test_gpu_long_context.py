"""GPU parity of the long-context operators against oracle/long_context.py.

Floating outputs are held to the oracle's bounds (bound_rotary,
bound_attention: what a correct fp32 kernel with one rounding at its store may
be off, element by element); integers and copied values are compared exactly.
Memory that a call must not read (stale table entries' slots, unused rows)
holds NaN, memory that it must not write holds a pattern that is compared.
"""
import numpy as np
import pytest
import torch

from oracle import long_context as O

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _ops():
    from lite_lang_amd import ops
    return ops


def _i32(v, dev, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=dev)


def _inside(got, want, bound, what=""):
    """got within bound of want, element by element; NaN only where want is."""
    got = got.detach().cpu().to(torch.float64)
    ok = ~torch.isnan(want)
    assert not torch.isnan(got[ok]).any(), f"{what}: NaN"
    excess = (got - want).abs()[ok] - bound[ok]
    if excess.numel():
        worst = float(((got - want).abs()[ok] / bound[ok]).max())
        print(f"  {what}: worst {worst:.3f} of the bound", flush=True)
        assert float(excess.max()) <= 0.0, f"{what}: {worst:.3f} of the bound"


# ---------------------------------------------------------------- rotation
# (q heads, k heads, head dim, rotated, interleaved): the model's, partial and
# interleaved, a head of 96, odd sizes, the smallest pair, the widest head
ROT = [(16, 2, 128, 128, False), (28, 4, 128, 64, True), (8, 2, 64, 64, True),
       (32, 8, 64, 16, False), (3, 1, 96, 32, False), (2, 2, 80, 80, True), (1, 1, 10, 6, False),
       (1, 1, 2, 2, True), (4, 2, 256, 256, False), (2, 1, 128, 0, False), (5, 3, 128, 24, False)]


def _rot_inputs(cuda, T, H, K, D, R, dtype, seed, pos64=False, far=2 ** 31 - 1):
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn(T, H, D, generator=g).to(dtype), torch.randn(T, K, D, generator=g).to(dtype)
    pos = torch.randint(0, far, (T,), generator=g)
    if T > 2:
        pos[0], pos[1] = 0, far  # the first and the farthest position
    f = (1e6 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))).float()
    pos = pos.to(torch.int64 if pos64 else torch.int32)
    return q, k, pos, f


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("H,K,D,R,inter", ROT)
def test_rope_positions(cuda, H, K, D, R, inter, dtype):
    for T, far, factor in ((1, 40, 1.0), (7, 2 ** 31 - 1, 1.25), (45, 1 << 20, 1.0)):
        print(f"case: rope T={T} H={H}/{K} D={D} R={R} inter={inter} {dtype} far={far}", flush=True)
        q, k, pos, f = _rot_inputs(cuda, T, H, K, D, R, dtype, T + D, pos64=T == 7, far=far)
        qd, kd = q.to(cuda), k.to(cuda)
        qo, ko = torch.full_like(qd, 7.0), torch.full_like(kd, 7.0)
        r = _ops().rope_positions(qd, kd, pos.to(cuda), f.to(cuda), interleaved=inter,
                                  factor=factor, q_out=qo, k_out=ko)
        assert r[0] is qo and r[1] is ko
        for x, y, name in ((q, qo, "q"), (k, ko, "k")):
            want, mag = O.rotate(x, pos, f, factor, inter)
            _inside(y, want, O.bound_rotary(want, mag, dtype, pos, f), name)
            assert torch.equal(y.cpu()[..., R:], x[..., R:]), "elements behind the rotated part"
        assert torch.equal(qd.cpu(), q) and torch.equal(kd.cpu(), k)
        # in place: the same bits
        _ops().rope_positions(qd, kd, pos.to(cuda), f.to(cuda), interleaved=inter, factor=factor)
        assert torch.equal(qd, qo) and torch.equal(kd, ko)


@pytest.mark.parametrize("pad", [0, 3, 8])
def test_rope_positions_strided_rows(cuda, pad):
    """Heads inside a wider row (the projection's output, with rows padded to
    odd and even strides), outputs of other strides, k None."""
    T, H, K, D = 37, 4, 2, 64
    for dtype in (BF16, F32):
        q, k, pos, f = _rot_inputs(cuda, T, H, K, D, D, dtype, 5, far=9000)
        row = torch.full((T, (H + K) * D + pad), 3.0, dtype=dtype, device=cuda)
        qd = row[:, :H * D].unflatten(1, (H, D))
        kd = row[:, H * D:(H + K) * D].unflatten(1, (K, D))
        qd.copy_(q), kd.copy_(k)
        print(f"case: strided rope pad={pad} {dtype}", flush=True)
        wide = torch.zeros(T, 2 * H, D, dtype=dtype, device=cuda)
        _ops().rope_positions(qd, None, pos.to(cuda), f.to(cuda), q_out=wide[:, ::2])
        want, mag = O.rotate(q, pos, f)
        _inside(wide[:, ::2], want, O.bound_rotary(want, mag, dtype, pos, f), "q")
        assert not wide[:, 1::2].any()
        _ops().rope_positions(qd, kd, pos.to(cuda), f.to(cuda))
        _inside(qd, want, O.bound_rotary(want, mag, dtype, pos, f), "q in place")
        want, mag = O.rotate(k, pos, f)
        _inside(kd, want, O.bound_rotary(want, mag, dtype, pos, f), "k in place")
        if pad:
            assert bool((row[:, -pad:] == 3.0).all()), "padding of the rows"


@pytest.mark.parametrize("row", [(1 << 27) - 8, 1 << 27])
def test_rope_of_rows_far_apart(cuda, row):
    """Rows 2^24 units of 16 bytes apart, and one less."""
    H, D = 2, 64
    q, _, pos, f = _rot_inputs(cuda, 3, H, 1, D, D, BF16, 7, far=9000)
    wide = torch.empty(3, row, dtype=BF16, device=cuda)
    qd = wide[:, 64:64 + H * D].unflatten(1, (H, D))
    qd.copy_(q)
    wide[:, :64], wide[:, 64 + H * D:64 + 2 * H * D] = 5.0, 6.0
    print(f"case: rope rows of {row}", flush=True)
    _ops().rope_positions(qd, None, pos.to(cuda), f.to(cuda))
    want, mag = O.rotate(q, pos, f)
    _inside(qd, want, O.bound_rotary(want, mag, BF16, pos, f), "q")
    assert bool((wide[:, :64] == 5.0).all())
    assert bool((wide[:, 64 + H * D:64 + 2 * H * D] == 6.0).all())


def test_qk_norm_to_far_slots(cuda):
    """Cache rows behind 2^32 bytes of the pool; padded tokens among them."""
    H, K, D, T = 4, 8, 128, 40
    P = (1 << 31) // (2 * K * D) + 5000
    g = torch.Generator().manual_seed(8)
    x = torch.randn(T, (H + 2 * K) * D, generator=g).to(BF16)
    gk = (1 + 0.2 * torch.randn(D, generator=g)).to(BF16)
    pos = torch.randint(0, 9000, (T,), generator=g).to(torch.int32)
    f, _ = _ops().rope_frequencies(D)
    slots = (P - 1 - torch.randperm(4000, generator=g)[:T]).to(torch.int32)
    slots[3], slots[7], slots[11] = -1, P, -(1 << 31)
    pool = torch.empty(P, 2 * K, D, dtype=BF16, device=cuda)
    pool[-5000:] = 7.0
    print("case: qk norm far slots", flush=True)
    _ops().qk_norm_rope_kv_scatter(x.to(cuda), H, K, D, None, gk.to(cuda), 1e-6, pos.to(cuda),
                                   f.to(cuda), slots.to(cuda), pool)
    tail = pool[-5000:].cpu()
    rows = x.view(T, H + 2 * K, D)
    normed = O.head_norm(rows[:, H:H + K], gk, 1e-6)
    want, mag = O.rotate(normed, pos, f)
    stored = [t for t in range(T) if t not in (3, 7, 11)]
    at = [int(slots[t]) - (P - 5000) for t in stored]
    b = O.bound_rotary(want, mag, BF16, pos, f, D)
    _inside(tail[at, :K], want[stored], b[stored], "k")
    assert torch.equal(tail[at, K:], rows[stored, H + K:])
    rest = torch.ones(5000, dtype=torch.bool)
    rest[at] = False
    assert bool((tail[rest] == 7.0).all())


@pytest.mark.parametrize("D", [64, 20])
def test_rope_of_nothing_rotated_needs_no_positions(cuda, D):
    """The C entry point takes null positions and frequencies with rotary_dim 0
    (16-byte rows and others): a copy."""
    import ctypes

    from lite_lang_amd import _lib
    x = torch.randn(5, 3, D, device=cuda).bfloat16()
    y = torch.zeros_like(x)
    rc = _lib.load().ll_rope_positions(x.data_ptr(), 3 * D, D, y.data_ptr(), 3 * D, D, 3, None, 0,
                                       0, None, 0, 0, 0, None, 0, None, 0, 0, ctypes.c_float(1.0),
                                       5, D, _ops().dtype_code(x), _ops()._stream(x))
    assert rc == 0 and torch.equal(x, y)


def test_calls_of_no_tokens(cuda):
    q, none, f = torch.zeros(0, 4, 64, device=cuda), _i32([], cuda), torch.ones(32, device=cuda)
    pool = torch.zeros(5, 4, 64, device=cuda)
    out, _ = _ops().rope_positions(q, None, none, f)
    assert out.shape == (0, 4, 64)
    out = _ops().qk_norm_rope_kv_scatter(torch.zeros(0, 8 * 64, device=cuda), 4, 2, 64, None, None,
                                         1e-6, none, f, none, pool)
    assert out.shape == (0, 4, 64)
    table = torch.zeros(2, 8, dtype=torch.int32, device=cuda)
    _ops().window_prefill_attention(q, pool[:, :2], pool[:, 2:], q, none, none, none, 8, table, 4)
    _ops().window_decode_attention(q, table, none, none, 8, pool[:, :2], pool[:, 2:], q, 4)
    torch.cuda.synchronize()


def test_rope_positions_agrees_with_the_table_form(cuda):
    """With an exact fp32 cos/sin table in hand the framework's rotary_emb gives
    the same rotation, to the table's fp32 rounding."""
    T, H, K, D = 64, 4, 2, 128
    q, k, pos, f = _rot_inputs(cuda, T, H, K, D, D, F32, 8, far=5000)
    c, s = O.cos_sin(pos, f, 1.0)
    a, b = q.to(cuda), k.to(cuda)
    _ops().rotary_emb(a, b, c.float().to(cuda), s.float().to(cuda))
    x, y = _ops().rope_positions(q.to(cuda), k.to(cuda), pos.to(cuda), f.to(cuda))
    want, mag = O.rotate(q, pos, f)
    bound = O.bound_rotary(want, mag, F32, pos, f)
    _inside(a, x.cpu().double(), 2 * bound, "q")
    want, mag = O.rotate(k, pos, f)
    _inside(b, y.cpu().double(), 2 * O.bound_rotary(want, mag, F32, pos, f), "k")


# ---------------------------------------------------------------- norm + rotation
def _qk_case(cuda, T, H, K, D, R, inter, dtype, seed, gammas=(True, True), inplace=False, pad=0,
             scale=1.7):
    g = torch.Generator().manual_seed(seed)
    n = (H + 2 * K) * D
    qkv = (torch.randn(T, n, generator=g) * scale).to(dtype)
    if T > 2:
        qkv[1] = 0  # a zero row: the norm's eps alone
    gam = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype) if x else None for x in gammas]
    f = (1e6 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))).float()
    pos = torch.randint(0, 100000, (T,), generator=g).to(torch.int32)
    P = T + 9
    slots = torch.randperm(P, generator=g)[:T].to(torch.int32)
    keep = torch.ones(T, dtype=torch.bool)
    if T > 5:  # padded tokens
        slots[3], slots[5] = -1, P
        keep[3] = keep[5] = False
    pool = torch.randn(P, 2 * K, D, generator=g).to(dtype)
    eps = 1e-6
    buf = torch.full((T, n + pad), 3.0, dtype=dtype, device=cuda)
    qkvd = buf[:, :n]
    qkvd.copy_(qkv)
    pd = pool.to(cuda)
    qo = None if inplace else torch.full((T, H, D), 7.0, dtype=dtype, device=cuda)
    q = _ops().qk_norm_rope_kv_scatter(
        qkvd, H, K, D, *(None if x is None else x.to(cuda) for x in gam), eps, pos.to(cuda),
        f.to(cuda), slots.to(cuda), pd, interleaved=inter, factor=1.1, q_out=qo)
    x = qkv.view(T, H + 2 * K, D)
    for part, gm, got, name in ((x[:, :H], gam[0], q, "q"),
                                (x[:, H:H + K], gam[1], pd[slots[keep].long(), :K], "k")):
        want, mag = O.rotate(O.head_norm(part, gm, eps), pos, f, 1.1, inter)
        b = O.bound_rotary(want, mag, dtype, pos, f, head_dim=D if gm is not None else 0)
        if name == "k":
            want, b = want[keep], b[keep]
        _inside(got, want, b, name)
    pc = pd.cpu()
    assert torch.equal(pc[slots[keep].long(), K:], x[keep][:, H + K:]), "v"
    rest = torch.ones(P, dtype=torch.bool)
    rest[slots[keep].long()] = False
    assert torch.equal(pc[rest], pool[rest]), "slots of no token"
    tail = qkvd.cpu()[:, H * D if inplace else 0:]
    assert torch.equal(tail, qkv[:, H * D if inplace else 0:]), "qkv outside q"
    if pad:
        assert bool((buf[:, n:] == 3.0).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("H,K,D,R,inter", ROT)
def test_qk_norm_rope_kv_scatter(cuda, H, K, D, R, inter, dtype):
    for T, kw in ((1, {}), (40, {"inplace": True}), (77, {"gammas": (True, False)}),
                  (9, {"gammas": (False, False)})):
        print(f"case: qk norm T={T} H={H}/{K} D={D} R={R} inter={inter} {dtype} {kw}", flush=True)
        _qk_case(cuda, T, H, K, D, R, inter, dtype, T + D + R, **kw)


@pytest.mark.parametrize("pad", [1, 8])
def test_qk_norm_rope_kv_scatter_padded_rows(cuda, pad):
    print(f"case: qk norm rows padded by {pad}", flush=True)
    _qk_case(cuda, 50, 12, 2, 128, 128, False, BF16, 2, pad=pad)
    _qk_case(cuda, 50, 4, 2, 64, 32, True, F32, 3, pad=pad, inplace=True)


def test_qk_norm_of_a_long_prefill(cuda):
    """More tokens than one pass of the grid, and the head group of 7."""
    _qk_case(cuda, 3001, 7, 1, 128, 128, False, BF16, 4)
    _qk_case(cuda, 2050, 8, 2, 64, 64, True, F16, 5, scale=30.0)
    # two to eight tokens per workgroup
    _qk_case(cuda, 4099, 28, 4, 64, 64, False, BF16, 6)
    _qk_case(cuda, 8197, 6, 1, 80, 48, True, F16, 7, inplace=True)
    _qk_case(cuda, 16391, 1, 1, 64, 32, False, F32, 8)


# ---------------------------------------------------------------- attention
def _cache(g, lens, before, window, sinks, KVH, D, dtype):
    """A pool and a slot table whose stale entries (keys that no query sees) and
    whose unused rows lead to NaN."""
    live = []
    for n, c in zip(lens, before):
        low = max(0, c - window + 1)
        live.append([p for p in range(n) if p < sinks or p >= low])
    total = sum(map(len, live))
    P = total + 7
    pool = torch.randn(P, 2 * KVH, D, generator=g).to(dtype)
    perm = torch.randperm(P, generator=g)
    pool[perm[total:]] = float("nan")
    B, width = len(lens), max(max(lens), 1) + 5
    table = perm[total + torch.randint(0, P - total, (B + 2, width), generator=g)].to(torch.int32)
    rids = torch.randperm(B + 2, generator=g)[:B].tolist()
    at = 0
    for r, ps in zip(rids, live):
        table[r, ps] = perm[at:at + len(ps)].to(torch.int32)
        at += len(ps)
    return pool, table, rids


def _prefill_case(cuda, H, KVH, D, dtype, lens, before, window, sinks, seed=0, idx=torch.int32,
                  pad=0, scale=None, mag=1.0, most=None):
    print(f"case: window prefill H={H}/{KVH} D={D} {dtype} lens={lens} before={before} "
          f"window={window} sinks={sinks} pad={pad}", flush=True)
    g = torch.Generator().manual_seed(seed)
    pool, table, rids = _cache(g, lens, before, window, sinks, KVH, D, dtype)
    new = [max(0, n - c) for n, c in zip(lens, before)]
    starts = [2 + sum(new[:i]) for i in range(len(lens))]  # rows 0, 1 and the last belong to nobody
    T = sum(new) + 3
    q = (torch.randn(T, H, D, generator=g) * mag).to(dtype)
    qd = torch.zeros(T, H, D + pad, dtype=dtype, device=cuda)[..., :D]
    qd.copy_(q)
    out = torch.full((T, H, D + pad), 7.0, dtype=dtype, device=cuda)[..., :D]
    pd = pool.to(cuda)
    shared = None if not any(before) else _i32(before, cuda, idx)
    _ops().window_prefill_attention(qd, pd[:, :KVH], pd[:, KVH:], out, _i32(rids, cuda, idx),
                                    _i32(starts, cuda, idx), _i32(lens, cuda, idx),
                                    max(lens) if most is None else most, table.to(cuda), window, sinks=sinks, b_shared_seq_len=shared,
                                    sm_scale=scale)
    torch.cuda.synchronize()
    want, wgt, keys, mags = O.window_prefill(q, pool[:, :KVH], pool[:, KVH:], table, rids, starts,
                                             lens, before, window, sinks, scale)
    b = O.bound_attention(want, wgt, keys, mags, dtype, D, O.p_rounding(dtype, False),
                          float(pool[:, KVH:].float().nan_to_num().abs().max()))
    if most is not None:  # rows behind the bound may hold anything
        for at, n in zip(starts, new):
            want[at + most:at + max(n, most)] = float("nan")
    _inside(out, want, b, "out")
    nobody = torch.ones(T, dtype=torch.bool)
    nobody[2:2 + sum(new)] = False
    assert bool((out.cpu()[nobody] == 7.0).all()), "rows of no request"
    return out


HEADS = [(16, 2, 128, BF16), (7, 1, 128, F16), (8, 2, 64, BF16), (4, 4, 64, F16), (2, 1, 96, BF16),
         (4, 2, 128, F32), (2, 1, 48, F32)]


@pytest.mark.parametrize("H,KVH,D,dtype", HEADS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 0), (64, 4), (100, 70), (33, 1), (1000, 4),
                                          (2 ** 40, 2 ** 40)])
def test_window_prefill_attention(cuda, H, KVH, D, dtype, window, sinks):
    """Windows of one token, below, at and above a tile; sinks of a whole tile
    and more; windows and sinks beyond any length; ragged lengths from one."""
    _prefill_case(cuda, H, KVH, D, dtype, [1, 150, 67, 2], [0, 0, 0, 0], window, sinks, seed=window)


@pytest.mark.parametrize("H,KVH,D,dtype", HEADS[:4])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 0), (40, 3), (130, 65), (600, 2)])
def test_window_prefill_attention_behind_a_prefix(cuda, H, KVH, D, dtype, window, sinks):
    """Chunks behind cached prefixes, parts of which have left the cache; one
    request of the batch has no new token, one has its first prefix token."""
    _prefill_case(cuda, H, KVH, D, dtype, [300, 65, 30, 129, 2], [211, 64, 30, 0, 1], window, sinks,
                  seed=window + 1, idx=torch.int64)


def test_window_prefill_attention_of_many_row_blocks(cuda):
    """More row blocks than a workgroup takes at once; the window's low end
    moves through several tiles; windows one off a tile boundary."""
    for window, sinks in ((63, 0), (64, 1), (65, 64), (191, 5), (192, 0), (193, 130)):
        _prefill_case(cuda, 4, 1, 64, BF16, [700, 1], [0, 0], window, sinks, seed=window)
    _prefill_case(cuda, 3, 1, 128, F16, [900], [333], 257, 4, seed=9)


def test_window_prefill_attention_of_many_requests(cuda):
    """More (row block, request, head) items than workgroups."""
    g = np.random.RandomState(5)
    lens = g.randint(1, 60, size=300).tolist()
    before = [int(n * g.rand()) for n in lens]
    _prefill_case(cuda, 4, 2, 64, BF16, lens, before, 20, 2, seed=5)


def test_window_prefill_attention_odd_strides_and_scales(cuda):
    """Rows that no 16-byte load may read, a scale of the caller's, sharp and
    flat scores."""
    _prefill_case(cuda, 4, 2, 64, BF16, [90, 33], [0, 0], 50, 2, pad=3)
    _prefill_case(cuda, 4, 2, 64, BF16, [90, 33], [0, 0], 50, 2, pad=8)
    _prefill_case(cuda, 4, 2, 128, BF16, [200], [0], 50, 2, scale=0.5)
    _prefill_case(cuda, 4, 2, 128, F16, [200], [0], 50, 2, mag=6.0)
    _prefill_case(cuda, 4, 2, 128, BF16, [200], [0], 50, 0, mag=1e-3)


def test_window_prefill_of_a_window_beyond_the_context_is_causal(cuda):
    """A window that covers everything gives the framework's causal attention:
    both are within the same bound of the oracle, so twice it apart."""
    g = torch.Generator().manual_seed(12)
    H, KVH, D, lens = 16, 2, 128, [333, 70]
    pool = torch.randn(sum(lens), 2 * KVH, D, generator=g).to(BF16).to(cuda)
    table = torch.zeros(2, 333, dtype=torch.int32)
    table[0], table[1, :70] = torch.arange(333), torch.arange(333, 403)
    table, q = table.to(cuda), torch.randn(403, H, D, generator=g).to(BF16).to(cuda)
    a, b = torch.empty_like(q), torch.empty_like(q)
    args = (_i32([0, 1], cuda), _i32([0, 333], cuda), _i32(lens, cuda), 333, table)
    _ops().prefill_attention(q, pool[:, :KVH], pool[:, KVH:], a, *args)
    _ops().window_prefill_attention(q, pool[:, :KVH], pool[:, KVH:], b, *args, 333)
    scale = a.float().abs().max()
    assert float((a.float() - b.float()).abs().max()) <= 4 * float(scale) * O.u(BF16)


def _decode_case(cuda, H, KVH, D, dtype, lens, window, sinks, seed=0, idx=torch.int32, bound=None,
                 scale=None, mag=1.0):
    print(f"case: window decode H={H}/{KVH} D={D} {dtype} lens={lens[:6]} x{len(lens)} "
          f"window={window} sinks={sinks}", flush=True)
    g = torch.Generator().manual_seed(seed)
    cap = [min(n, bound) if bound is not None else n for n in lens]
    pool, table, rids = _cache(g, cap, [n - 1 for n in cap], window, sinks, KVH, D, dtype)
    B = len(lens)
    q = (torch.randn(B, H, D, generator=g) * mag).to(dtype)
    pd = pool.to(cuda)
    out = torch.full((B, H, D), 7.0, dtype=dtype, device=cuda)
    _ops().window_decode_attention(q.to(cuda), table.to(cuda), _i32(rids, cuda, idx),
                                   _i32(lens, cuda, idx), bound if bound is not None else max(lens),
                                   pd[:, :KVH], pd[:, KVH:], out, window, sinks=sinks,
                                   sm_scale=scale)
    torch.cuda.synchronize()
    want, wgt, keys, mags = O.window_decode(q, pool[:, :KVH], pool[:, KVH:], table, rids, cap,
                                            window, sinks, scale)
    b = O.bound_attention(want, wgt, keys, mags, dtype, D, O.p_rounding(dtype, True),
                          float(pool[:, KVH:].float().nan_to_num().abs().max()))
    _inside(out, want, b, "out")
    return out


@pytest.mark.parametrize("H,KVH,D,dtype", HEADS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (16, 4), (100, 70), (300, 3),
                                          (2 ** 40, 2 ** 40)])
def test_window_decode_attention(cuda, H, KVH, D, dtype, window, sinks):
    _decode_case(cuda, H, KVH, D, dtype, [1, 2, 0, 333, 16, 17, 129], window, sinks, seed=window,
                 idx=torch.int64 if sinks == 4 else torch.int32)


@pytest.mark.parametrize("B,n,window,sinks", [(1, 9000, 4096, 4), (3, 5000, 1500, 0),
                                              (8, 3000, 1024, 100), (40, 700, 600, 4),
                                              (70, 300, 128, 1)])
def test_window_decode_attention_splits(cuda, B, n, window, sinks):
    """Few sequences with long windows and many with short ones: every split
    count, lengths below and above the window."""
    lens = [max(1, n - 131 * i) if i % 5 else n for i in range(B)]
    _decode_case(cuda, 4, 2, 128, BF16, lens, window, sinks, seed=B)
    _decode_case(cuda, 2, 1, 64, F16, lens, window, sinks, seed=B + 1)


def test_window_decode_attention_takes_the_bound(cuda):
    """Tokens past max_len_in_batch are ignored; all sequences may be empty."""
    _decode_case(cuda, 8, 2, 128, BF16, [500, 90, 3], 64, 2, bound=100)
    _decode_case(cuda, 4, 2, 64, BF16, [0, 0], 64, 2, bound=16)


def test_window_decode_attention_scales(cuda):
    _decode_case(cuda, 4, 2, 128, BF16, [200, 31], 50, 2, scale=0.5)
    _decode_case(cuda, 4, 2, 128, F16, [200, 31], 50, 2, mag=6.0)


def test_window_attention_far_slots(cuda):
    """Rows of a pool beyond 2^31 elements (and 2^32 bytes)."""
    KVH, D, H = 8, 128, 8
    P = (1 << 31) // (2 * KVH * D) + 5000
    pool = torch.empty(P, 2 * KVH, D, dtype=BF16, device=cuda)
    g = torch.Generator().manual_seed(6)
    n, window, sinks = 300, 100, 4
    rows = torch.randn(n, 2 * KVH, D, generator=g).to(BF16)
    slots = (P - 1 - torch.randperm(4000, generator=g)[:n]).to(torch.int32)
    pool[slots.long().to(cuda)] = rows.to(cuda)
    table = slots.view(1, n)
    q = torch.randn(n, H, D, generator=g).to(BF16)
    small, ident = rows, torch.arange(n, dtype=torch.int32).view(1, n)
    vmax = float(rows.float().abs().max())
    for prefill in (True, False):
        print(f"case: far slots prefill={prefill}", flush=True)
        qq = q if prefill else q[:1]
        out = torch.empty_like(qq, device=cuda)
        a = (_i32([0], cuda), _i32([0], cuda), _i32([n], cuda))
        if prefill:
            _ops().window_prefill_attention(qq.to(cuda), pool[:, :KVH], pool[:, KVH:], out, *a, n,
                                            table.to(cuda), window, sinks=sinks)
            want = O.window_prefill(qq, small[:, :KVH], small[:, KVH:], ident, [0], [0], [n], [0],
                                    window, sinks)
        else:
            _ops().window_decode_attention(qq.to(cuda), table.to(cuda), a[0], a[2], n,
                                           pool[:, :KVH], pool[:, KVH:], out, window, sinks=sinks)
            want = O.window_decode(qq, small[:, :KVH], small[:, KVH:], ident, [0], [n], window,
                                   sinks)
        _inside(out, want[0], O.bound_attention(*want, BF16, D, O.p_rounding(BF16, not prefill),
                                                vmax), "out")
    del pool
    torch.cuda.empty_cache()


# ---------------------------------------------------------------- slot maps
def _maps_case(cuda, lens, before, page, seed=0, idx=torch.int32, spare=0, cap_extra=0, width=None,
               rids=None, expect=0):
    print(f"case: slot maps B={len(lens)} new={sum(lens) - sum(before)} page={page} "
          f"expect={expect}", flush=True)
    g = np.random.RandomState(seed)
    B = len(lens)
    cols = width if width is not None else (-(-max(lens + [1]) // page) + 1) * page
    R = B + 3
    rids = rids if rids is not None else g.permutation(R)[:B].tolist()
    need = sum(-(-n // page) - -(-c // page) for n, c in zip(lens, before))
    have = [-(-c // page) for c in before]
    ids = g.permutation(need + max(spare, 0) + sum(have) + 5).astype(np.int32)
    blocks = g.randint(0, 1000, size=(R, -(-cols // page))).astype(np.int32)
    table = g.randint(0, 1000, size=(R, cols)).astype(np.int32)
    at = need + max(spare, 0)
    free = ids[:need + spare]
    for r, c, h in zip(rids, before, have):
        if 0 <= r < R:
            own = ids[at:at + h]
            at += h
            if page > 1:
                blocks[r, :h] = own
            m = min(c, cols)
            p = np.arange(m)
            table[r, :m] = (own[p // page] * page + p % page) if page > 1 else own[:m]
    T = max(0, sum(lens) - sum(before))
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(cuda)  # noqa: E731
    wide = torch.full((R, cols + 3), -9, dtype=torch.int32, device=cuda)  # rows with a tail
    wide[:, :cols] = dev(table)
    td, bd = wide[:, :cols], dev(blocks) if page > 1 else None
    slots = torch.full((max(0, T + cap_extra),), -5, dtype=torch.int32, device=cuda)
    pos, counts = slots.clone(), _i32([9, 9, 9], cuda)
    start, last = _i32([-5] * B, cuda), _i32([-5] * B, cuda)
    _ops().build_slot_maps(_i32(rids, cuda, idx), _i32(lens, cuda, idx), _i32(before, cuda, idx),
                           dev(free), td, slots, pos, start, last, counts, page_size=page,
                           block_table=bd)
    torch.cuda.synchronize()
    assert bool((wide[:, cols:] == -9).all())
    if expect:
        assert counts[2].item() == expect, counts.tolist()
        assert np.array_equal(td.cpu().numpy(), table)
        assert bd is None or np.array_equal(bd.cpu().numpy(), blocks)
        for t in (slots, pos, start, last):
            assert bool((t == -5).all())
        return
    want = O.slot_maps(rids, lens, before, free, table, page, blocks if page > 1 else None)
    assert counts.tolist() == want[4]
    assert slots[:T].tolist() == want[0] and pos[:T].tolist() == want[1]
    assert start.tolist() == want[2] and last.tolist() == want[3]
    assert bool((slots[T:] == -5).all()) and bool((pos[T:] == -5).all())
    assert np.array_equal(td.cpu().numpy(), want[5])
    assert bd is None or np.array_equal(bd.cpu().numpy(), want[6])


@pytest.mark.parametrize("page", [1, 2, 16, 100])
def test_slot_maps(cuda, page):
    """Pages that cached and new tokens share, requests without new tokens
    (first, last, in a row), prefixes that end on a page's border."""
    _maps_case(cuda, [5], [0], page)
    _maps_case(cuda, [1], [0], page, cap_extra=3)
    _maps_case(cuda, [7, 7, 40, 16, 33, 200, 9], [7, 0, 39, 16, 16, 100, 9], page, seed=1, spare=4,
               cap_extra=700, idx=torch.int64)
    _maps_case(cuda, [3, 3], [3, 3], page)  # nothing new
    _maps_case(cuda, [0, 12, 0], [0, 0, 0], page)
    lens = np.random.RandomState(2).randint(1, 900, size=40).tolist()
    _maps_case(cuda, lens, [n - 1 for n in lens], page, seed=2)  # a decode step
    _maps_case(cuda, lens, [n // 3 for n in lens], page, seed=3)
    _maps_case(cuda, [5000, 1], [0, 0], page, seed=4)


@pytest.mark.parametrize("B", [255, 256, 257, 1000, 8192])
def test_slot_maps_of_large_batches(cuda, B):
    lens = np.random.RandomState(B).randint(0, 9, size=B).tolist()
    before = [int(n * f) for n, f in zip(lens, np.random.RandomState(B + 1).rand(B))]
    _maps_case(cuda, lens, before, 1, seed=B)
    _maps_case(cuda, lens, before, 4, seed=B)


@pytest.mark.parametrize("page", [1, 16])
def test_slot_maps_of_many_tokens(cuda, page):
    """Room for more tokens than a thread each: none, few and all of it used."""
    _maps_case(cuda, [3, 3], [3, 3], page, cap_extra=1300001)
    _maps_case(cuda, [700, 30, 1], [11, 0, 0], page, seed=1, cap_extra=400000)
    _maps_case(cuda, [70001, 0, 130000, 150003, 17], [33, 0, 1000, 0, 16], page, seed=2)


def test_slot_maps_report_what_does_not_fit(cuda):
    """Nothing but counts is written where something is wrong."""
    _maps_case(cuda, [5, 9], [2, 0], 1, spare=-1, expect=8)
    _maps_case(cuda, [33, 40], [16, 0], 16, spare=-1, expect=8)
    _maps_case(cuda, [5, 9], [2, 0], 1, cap_extra=-1, expect=4)
    _maps_case(cuda, [5, 9], [2, 0], 1, rids=[1, 5], expect=2)
    _maps_case(cuda, [5, 9], [2, 0], 1, rids=[-1, 0], expect=2)
    _maps_case(cuda, [5, 9], [2, 0], 1, rids=[2, 2], expect=2)
    _maps_case(cuda, [5, 9], [2, 0], 1, width=8, expect=1)
    _maps_case(cuda, [5, 9], [2, 0], 4, width=8, expect=1)
    # a prefix longer than its request, and the other one's 9 pages against the
    # 9 + 5 - 6 = 8 that are free: both are told
    _maps_case(cuda, [5, 9], [6, 0], 1, cap_extra=2, expect=1 + 8)
    # a padded entry without new tokens may sit on any row
    _maps_case(cuda, [5, 0, 0], [2, 0, 0], 1, rids=[2, 2, -1])


def test_slot_maps_of_no_requests(cuda):
    e, c = _i32([], cuda), _i32([9, 9, 9], cuda)
    table = torch.zeros(2, 4, dtype=torch.int32, device=cuda)
    _ops().build_slot_maps(e, e, e, _i32([1], cuda), table, _i32([-5], cuda), _i32([-5], cuda),
                           e.clone(), e.clone(), c)
    assert c.tolist() == [0, 0, 0]


# ---------------------------------------------------------------- a run of them
class _Server:
    """A layer's attention as a server with a bounded cache runs it: maps, norms
    + rotation + cache rows, windowed attention; prompts, then single tokens."""

    H, KVH, D, WINDOW, SINKS, PAGE, EPS = 8, 2, 64, 24, 3, 4, 1e-6

    def __init__(self, cuda, seed, B=3, width=96):
        g = torch.Generator().manual_seed(seed)
        self.g, self.dev, self.B = g, cuda, B
        pages = B * width // self.PAGE
        self.free = torch.randperm(pages, generator=g).to(torch.int32).to(cuda)
        self.taken = 0
        self.pool = torch.full((pages * self.PAGE, 2 * self.KVH, self.D), float("nan"), dtype=BF16,
                               device=cuda)
        self.table = torch.zeros(B + 1, width, dtype=torch.int32, device=cuda)
        self.blocks = torch.zeros(B + 1, width // self.PAGE, dtype=torch.int32, device=cuda)
        self.rows = _i32([2, 0, 3][:B], cuda)
        self.gq, self.gk = ((1 + 0.2 * torch.randn(self.D, generator=g)).to(BF16) for _ in "qk")
        self.f, self.factor = _ops().rope_frequencies(
            self.D, scaling={"type": "yarn", "factor": 8.0}, max_position=64)
        # what the calls read; a captured graph keeps these addresses
        self.on_dev = [x.to(cuda) for x in (self.gq, self.gk, self.f)]
        self.hist = [[] for _ in range(B)]  # qkv rows of each request, on the CPU

    def qkv(self, new):
        rows = torch.randn(sum(new), (self.H + 2 * self.KVH) * self.D, generator=self.g).to(BF16)
        for h, part in zip(self.hist, rows.split(new)):
            h.extend(part)
        return rows

    def call(self, qkv, lens, cached, max_len, decode, free, out):
        """The four calls on device tensors; nothing is read by the host."""
        ops, dev, T = _ops(), self.dev, qkv.shape[0]
        i = lambda n: torch.empty(n, dtype=torch.int32, device=dev)  # noqa: E731
        slots, pos, start, last, counts = i(T), i(T), i(self.B), i(self.B), i(3)
        ops.build_slot_maps(self.rows, lens, cached, free, self.table, slots, pos, start, last,
                            counts, page_size=self.PAGE, block_table=self.blocks)
        q = torch.empty(T, self.H, self.D, dtype=BF16, device=dev)
        gq, gk, f = self.on_dev
        ops.qk_norm_rope_kv_scatter(qkv, self.H, self.KVH, self.D, gq, gk, self.EPS, pos, f, slots,
                                    self.pool, factor=self.factor, q_out=q)
        k, v = self.pool[:, :self.KVH], self.pool[:, self.KVH:]
        if decode:
            ops.window_decode_attention(q, self.table, self.rows, lens, max_len, k, v, out,
                                        self.WINDOW, sinks=self.SINKS)
        else:
            ops.window_prefill_attention(q, k, v, out, self.rows, start, lens, max_len, self.table,
                                         self.WINDOW, sinks=self.SINKS, b_shared_seq_len=cached)
        return counts

    def want(self, new):
        """(out, bound) of the new rows from the whole history, in 64 bits. q, k
        and v are rounded to bf16 where the kernels store them; a store may land
        one step off the oracle's, which is u(bf16) of every |q| |k| twice in a
        score, and of |v|."""
        outs, bounds = [], []
        for h, n in zip(self.hist, new):
            x = torch.stack(h).view(len(h), self.H + 2 * self.KVH, self.D)
            pos = torch.arange(len(h))
            rot = lambda y, gm: O.rotate(O.head_norm(y, gm, self.EPS), pos, self.f,  # noqa: E731
                                         self.factor)[0].to(BF16).double()
            q, k = rot(x[:, :self.H], self.gq), rot(x[:, self.H:self.H + self.KVH], self.gk)
            v = x[:, self.H + self.KVH:].double()
            ident = torch.arange(len(h)).view(1, -1)
            o, w, keys, mags = O.window_prefill(q[len(h) - n:], k, v, ident, [0], [0], [len(h)],
                                                [len(h) - n], self.WINDOW, self.SINKS)
            b = O.bound_attention(o, w, keys, mags, BF16, self.D, O.u(BF16))
            flips = 2 * 2 * 2 * O.u(BF16) * mags[..., None] * w
            outs.append(o)
            bounds.append(b + flips)
        return torch.cat(outs), torch.cat(bounds)


def test_a_run_of_prompts_and_single_tokens(cuda):
    s = _Server(cuda, 11)
    lens, used = [0, 0, 0], 0
    for step, new in enumerate(([30, 1, 13], [9, 40, 1], [1, 1, 1], [1, 1, 1], [5, 1, 20])):
        cached, lens = lens, [a + b for a, b in zip(lens, new)]
        print(f"case: run step {step} new={new}", flush=True)
        qkv = s.qkv(new).to(cuda)
        out = torch.empty(sum(new), s.H, s.D, dtype=BF16, device=cuda)
        counts = s.call(qkv, _i32(lens, cuda), _i32(cached, cuda), max(lens), max(new) == 1,
                        s.free[used:].contiguous(), out)
        tokens, pages, err = counts.tolist()
        assert (tokens, err) == (sum(new), 0)
        used += pages
        want, bound = s.want(new)
        _inside(out, want, bound, f"step {step}")


def test_a_captured_run_replays(cuda):
    """Two servers' decode steps, captured into two graphs, replayed in turn and
    on two streams at once, each against its eager result."""
    servers, graphs = [], []
    for seed in (21, 22):
        s = _Server(cuda, seed)
        new = [40, 25, 60]
        out = torch.empty(sum(new), s.H, s.D, dtype=BF16, device=cuda)
        used = s.call(s.qkv(new).to(cuda), _i32(new, cuda), _i32([0, 0, 0], cuda), 60, False,
                      s.free, out).tolist()[1]
        s.lens, s.cached = _i32([n + 1 for n in new], cuda), _i32(new, cuda)
        s.x = s.qkv([1, 1, 1]).to(cuda)
        s.out = torch.empty(3, s.H, s.D, dtype=BF16, device=cuda)
        s.now = s.free[used:].contiguous()
        s.call(s.x, s.lens, s.cached, 96, True, s.now, s.out)
        torch.cuda.synchronize()
        s.eager = s.out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.call(s.x, s.lens, s.cached, 96, True, s.now, s.out)
        servers.append(s)
        graphs.append(graph)
        want, bound = s.want([1, 1, 1])
        _inside(s.eager, want, bound, "eager")
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for s, graph in zip(servers, graphs):
            s.out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert bool((s.out == s.eager).all()), "replay"
        for s in servers:
            s.out.zero_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for s in servers:
            assert bool((s.out == s.eager).all()), "replay on two streams"


def test_other_streams_and_threads(cuda):
    """Calls on a stream of the caller's, and from several threads at once."""
    import threading
    s = _Server(cuda, 31)
    new = [50, 30, 10]
    x = s.qkv(new).to(cuda)
    out = torch.empty(90, s.H, s.D, dtype=BF16, device=cuda)
    s.call(x, _i32(new, cuda), _i32([0, 0, 0], cuda), 50, False, s.free, out)
    torch.cuda.synchronize()
    lens, q = _i32(new, cuda), torch.randn(3, s.H, s.D, device=cuda).to(BF16)
    k, v = s.pool[:, :s.KVH], s.pool[:, s.KVH:]
    want = torch.empty_like(q)
    _ops().window_decode_attention(q, s.table, s.rows, lens, 4000, k, v, want, 4000)
    torch.cuda.synchronize()
    outs = [torch.zeros_like(q) for _ in range(4)]

    def work(i):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                _ops().window_decode_attention(q, s.table, s.rows, lens, 4000, k, v, outs[i], 4000)
        st.synchronize()

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for o in outs:
        assert bool((o == want).all())


# ---------------------------------------------------------------- the less usual calls
@pytest.mark.parametrize("H,KVH,D,dtype", [(32, 1, 64, BF16), (20, 1, 128, F16), (10, 2, 128, BF16),
                                           (6, 1, 64, F16)])
def test_window_attention_of_other_head_groups(cuda, H, KVH, D, dtype):
    """More query heads per KV head than a matrix tile's columns, groups that
    leave a workgroup's head slots empty."""
    _prefill_case(cuda, H, KVH, D, dtype, [70, 1, 140], [0, 0, 75], 50, 3, seed=H)
    _decode_case(cuda, H, KVH, D, dtype, [70, 1, 900], 600, 3, seed=H)


def test_window_prefill_attention_of_far_apart_prefixes(cuda):
    """Requests hundreds of row blocks apart in their contexts, under a window
    that is whole for none of them, and for some."""
    for window, sinks in ((20000, 0), (3000, 5)):
        _prefill_case(cuda, 4, 1, 64, BF16, [130, 9000, 1, 4500], [0, 8900, 0, 4444], window, sinks,
                      seed=window)


@pytest.mark.parametrize("H,KVH,D,dtype", HEADS[:5])
def test_window_prefill_attention_takes_the_bound(cuda, H, KVH, D, dtype):
    """A bound of the query rows alone, and requests with more rows than it."""
    for lens, before, most in (([500, 40, 333], [430, 0, 333], 70), ([130, 900], [0, 890], 130),
                               ([700, 5, 64], [0, 0, 0], 200), ([90] * 70, [0, 80] * 35, 32)):
        _prefill_case(cuda, H, KVH, D, dtype, lens, before, 50, 3, seed=most, most=most)


@pytest.mark.parametrize("H,KVH,D,dtype", HEADS[:4])
def test_window_prefill_attention_of_short_prompts(cuda, H, KVH, D, dtype):
    """Prompts of up to 128 tokens, few and many, alone and behind prefixes."""
    for window, sinks in ((9, 2), (200, 0)):
        _prefill_case(cuda, H, KVH, D, dtype, [1], [0], window, sinks, seed=1)
        _prefill_case(cuda, H, KVH, D, dtype, [128, 1, 33], [0, 0, 0], window, sinks, seed=2)
        _prefill_case(cuda, H, KVH, D, dtype, [128, 64, 70], [100, 64, 1], window, sinks, seed=3)
        _prefill_case(cuda, H, KVH, D, dtype, [100 - 2 * i for i in range(40)], [0] * 40, window,
                      sinks, seed=4)


@pytest.mark.parametrize("H,KVH", [(7, 1), (14, 2), (2, 2)])
def test_window_prefill_attention_of_one_head_or_all_per_item(cuda, H, KVH):
    """Row blocks of 32 and of 256 rows: ragged ends, prefixes, whole windows
    and not, several blocks and requests per workgroup."""
    for window, sinks in ((31, 0), (32, 3), (257, 70)):
        _prefill_case(cuda, H, KVH, 64, BF16, [600, 33, 257, 32], [0, 1, 256, 0], window, sinks,
                      seed=window)
    _prefill_case(cuda, H, KVH, 128, F16, [1500, 300], [1100, 0], 500, 1, seed=7)
    lens = [1 + 13 * i % 190 for i in range(90)]
    _prefill_case(cuda, H, KVH, 64, F16, lens, [n // 2 if i % 2 else 0 for i, n in enumerate(lens)],
                  60, 4, seed=8)


def test_window_prefill_attention_of_more_than_64_passes(cuda):
    """More items than 64 for each of the card's workgroups."""
    lens = [1 + i % 7 for i in range(300)]
    _prefill_case(cuda, 64, 64, 64, BF16, lens, [0] * 300, 3, 1, seed=64)


def test_window_prefill_attention_of_many_mixed_requests(cuda):
    """More requests than a wave has lanes, with whole windows and without."""
    g = np.random.RandomState(15)
    lens = g.randint(1, 400, size=140).tolist()
    before = [int(n * g.rand()) if i % 3 else 0 for i, n in enumerate(lens)]
    _prefill_case(cuda, 2, 1, 64, BF16, lens, before, 150, 2, seed=15)


def test_prefill_attention_into_rows_of_8_byte_alignment(cuda):
    """The causal form takes output rows that start anywhere: the same bits as
    into aligned ones."""
    g = torch.Generator().manual_seed(17)
    H, KVH, D, n = 8, 2, 64, 150
    pool = torch.randn(n, 2 * KVH, D, generator=g).to(BF16).to(cuda)
    table = torch.arange(n, dtype=torch.int32, device=cuda).view(1, n)
    q = torch.randn(n, H, D, generator=g).to(BF16).to(cuda)
    a = torch.empty_like(q)
    wide = torch.full((n, H, D + 4), 7.0, dtype=BF16, device=cuda)
    b = wide[..., 4:]
    for o in (a, b):
        _ops().prefill_attention(q, pool[:, :KVH], pool[:, KVH:], o, _i32([0], cuda),
                                 _i32([0], cuda), _i32([n], cuda), n, table)
    assert torch.equal(a, b) and bool((wide[..., :4] == 7.0).all())


def test_captured_split_decodes_share_no_workspace(cuda):
    """Two captured decodes whose lists are split, replayed on two streams at
    once with eager ones of the same shape in between."""
    g = torch.Generator().manual_seed(18)
    H, KVH, D, n, window = 8, 2, 128, 3000, 2500
    pool = torch.randn(2 * n, 2 * KVH, D, generator=g).to(BF16).to(cuda)
    table = torch.randperm(2 * n, generator=g).to(torch.int32).view(2, n).to(cuda)
    need = _ops()._window_decode_bytes(1, H, KVH, D, n, window, 0)
    assert need > 0
    k, v, lens = pool[:, :KVH], pool[:, KVH:], _i32([n], cuda)
    qs = [torch.randn(1, H, D, generator=g).to(BF16).to(cuda) for _ in range(3)]
    rows = [_i32([r], cuda) for r in (0, 1, 0)]
    outs = [torch.empty_like(q) for q in qs]

    def call(i):
        _ops().window_decode_attention(qs[i], table, rows[i], lens, n, k, v, outs[i], window)

    for i in range(3):
        call(i)
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                call(i)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            for _ in range(20):
                call(2)
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_captured_window_prefill_follows_its_lengths(cuda):
    """A captured prefill replayed after its lengths, offsets and prefixes
    changed in place: the items follow the lengths on the device."""
    g = torch.Generator().manual_seed(19)
    H, KVH, D, window, sinks, most = 8, 2, 64, 70, 3, 300
    pool = torch.randn(600, 2 * KVH, D, generator=g).to(BF16)
    table = torch.randperm(600, generator=g).to(torch.int32).view(2, 300)
    q = torch.randn(most, H, D, generator=g).to(BF16)
    pd, td, qd = pool.to(cuda), table.to(cuda), q.to(cuda)
    out = torch.empty_like(qd)
    rows, start, lens, before = (_i32(x, cuda) for x in ([0, 1], [0, 100], [100, 200], [0, 0]))

    def call():
        _ops().window_prefill_attention(qd, pd[:, :KVH], pd[:, KVH:], out, rows, start, lens, most,
                                        td, window, sinks=sinks, b_shared_seq_len=before)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for ls, bs in (([100, 200], [0, 0]), ([300, 1], [170, 0]), ([130, 130], [130, 0]),
                   ([299, 300], [298, 100])):
        new = [n - c for n, c in zip(ls, bs)]
        for dst, val in ((start, [0, new[0]]), (lens, ls), (before, bs)):
            dst.copy_(_i32(val, cuda))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        want, wgt, keys, mags = O.window_prefill(q, pool[:, :KVH], pool[:, KVH:], table, [0, 1],
                                                 [0, new[0]], ls, bs, window, sinks)
        b = O.bound_attention(want, wgt, keys, mags, BF16, D, O.p_rounding(BF16, False),
                              float(pool[:, KVH:].float().abs().max()))
        _inside(out, want, b, f"replay {ls}")
        assert bool((out[sum(new):] == 7.0).all())


@pytest.mark.parametrize("H,KVH,D,dtype", HEADS)
@pytest.mark.parametrize("n,window", [(90, 40), (3000, 2500)])
def test_window_attention_padded_entries_may_sit_on_any_row(cuda, H, KVH, D, dtype, n, window):
    """Entries of length 0 beside live ones, of one split and several, on rows
    before and behind the table: they give zero rows, and the live ones what
    they give alone. A prefill's requests without query rows may sit there too.
    (The table is the middle of a larger buffer, whose other entries lead to NaN:
    a use of such a row would show, and read no other memory.)"""
    g = torch.Generator().manual_seed(n)
    pool = torch.randn(n + 5, 2 * KVH, D, generator=g).to(dtype).to(cuda)
    pool[n:] = float("nan")
    wide = torch.full((5, n), n, dtype=torch.int32, device=cuda)
    wide[2] = torch.randperm(n, generator=g).to(torch.int32)
    table = wide[2:3]
    q = torch.randn(4, H, D, generator=g).to(dtype).to(cuda)
    k, v = pool[:, :KVH], pool[:, KVH:]
    for idx in (torch.int32, torch.int64):
        print(f"case: padded decode H={H}/{KVH} D={D} {dtype} n={n} {idx}", flush=True)
        rows, lens = _i32([-1, 0, 1, -2], cuda, idx), _i32([0, n, 0, 0], cuda, idx)
        out = torch.full_like(q, 7.0)
        _ops().window_decode_attention(q, table, rows, lens, n, k, v, out, window, sinks=3)
        alone = torch.empty_like(q)
        _ops().window_decode_attention(q, table, _i32([0] * 4, cuda), _i32([n] * 4, cuda), n, k, v,
                                       alone, window, sinks=3)
        assert torch.equal(out[1], alone[1])
        assert not out[[0, 2, 3]].any()
        # all of them empty, under a bound of no tokens and of some
        for most in (0, 5):
            out.fill_(7.0)
            _ops().window_decode_attention(q, table, rows, _i32([0] * 4, cuda, idx), most, k, v,
                                           out, window, sinks=3)
            assert not out.any()
        print(f"case: padded prefill H={H}/{KVH} D={D} {dtype} n={n} {idx}", flush=True)
        start, before = _i32([0, 0, 9, 4], cuda, idx), _i32([0, n - 4, 9, 8], cuda, idx)
        out.fill_(7.0)
        _ops().window_prefill_attention(q, k, v, out, rows, start, _i32([0, n, 9, 5], cuda, idx), 4,
                                        table, window, sinks=3, b_shared_seq_len=before)
        _ops().window_prefill_attention(q, k, v, alone, _i32([0], cuda), _i32([0], cuda),
                                        _i32([n], cuda), 4, table, window, sinks=3,
                                        b_shared_seq_len=_i32([n - 4], cuda))
        assert torch.equal(out, alone)


def test_rope_of_the_most_tokens(cuda):
    """2^24 tokens whose heads fill a workgroup each (a grid of 2^32 threads has
    no room for one token per workgroup): the bits of smaller calls."""
    T, H, D, part = 1 << 24, 64, 16, 1 << 21
    g = torch.Generator().manual_seed(24)
    q = torch.randn(1, H, D, generator=g).to(BF16).to(cuda).expand(T, H, D)
    pos = torch.arange(T, dtype=torch.int32, device=cuda)
    f, _ = _ops().rope_frequencies(D)
    f = f.to(cuda)
    print("case: rope of 2^24 tokens", flush=True)
    out, small = (torch.zeros(n, H, D, dtype=BF16, device=cuda) for n in (T, part))
    _ops().rope_positions(q, None, pos, f, q_out=out)
    for at in range(0, T, part):
        _ops().rope_positions(q[:part], None, pos[at:at + part], f, q_out=small)
        assert torch.equal(out[at:at + part], small), f"tokens from {at}"
    del out, small
    torch.cuda.empty_cache()


@pytest.mark.parametrize("B", [2, 40, 64, 65, 130])
def test_window_prefill_attention_of_levels_beside_none(cuda, B):
    """Requests whose row blocks lie at many levels of their context's start
    beside requests that have none of those (whole windows behind long prefixes,
    no new tokens): the lanes of a wave that list the levels without adding any."""
    g = np.random.RandomState(B)
    lens, before = [], []
    for i in range(B):
        kind = i % 3
        at = int(g.randint(300, 900)) if kind == 1 else 0
        new = 0 if kind == 2 else int(g.randint(1, 260))
        lens.append(max(1, at + new))
        before.append(lens[-1] if kind == 2 else at)
    for H, KVH, window in ((8, 2, 290), (7, 1, 200)):
        _prefill_case(cuda, H, KVH, 64, BF16, lens, before, window, 2, seed=B)


def test_window_prefill_of_cached_requests_alone(cuda):
    """A step whose requests are all in the cache has no query row."""
    pool = torch.full((20, 4, 64), float("nan"), device=cuda)
    table = torch.zeros(3, 8, dtype=torch.int32, device=cuda)
    a = [_i32(x, cuda) for x in ([2, 0, 1], [0, 0, 0], [8, 3, 0])]
    none, wide = torch.zeros(0, 4, 64, device=cuda), torch.full((4, 4, 64), 7.0, device=cuda)
    for q, o in ((none, none.clone()), (none, wide[:0]), (wide[4:], none), (wide[:0], wide[1:1])):
        r = _ops().window_prefill_attention(q, pool[:, :2], pool[:, 2:], o, *a, 8, table, 4,
                                            b_shared_seq_len=a[2])
        assert r is o
    torch.cuda.synchronize()
    assert bool((wide == 7.0).all())
    with pytest.raises(ValueError, match="device"):  # still checked
        _ops().window_prefill_attention(none.cpu(), pool[:, :2], pool[:, 2:], none, *a, 8, table, 4)


@pytest.mark.parametrize("B,H,KVH,D,n,sinks,splits", [(3, 8, 2, 128, 131072, 4, 42),
                                                      (3, 4, 2, 64, 70000, 4, 85),
                                                      (2, 2, 1, 128, 131072, 0, 128),
                                                      (1, 2, 1, 64, 131072, 0, 336)])
def test_window_decode_attention_of_more_splits_than_a_chunk(cuda, B, H, KVH, D, n, sinks, splits):
    """Windows so long that the merge takes its splits 16 at a time, a last chunk
    that is not full, sequences too short for most of the splits, and a workspace
    that held NaN before the call. (Sharp scores, so that a split's keys show: the
    outputs are a few dozen keys' mean.)"""
    window = n - 5
    need = _ops()._window_decode_bytes(B, H, KVH, D, n, window, sinks)
    rows = B * H * splits
    assert need == (rows * D * 4 + 255) // 256 * 256 + rows * 8, "the split count of this case"
    lens = [n, 100, 5000][:B]
    for seed in (1, 2):
        _ops().workspace(cuda, "window_decode", need).fill_(255)  # NaN as fp32
        out = _decode_case(cuda, H, KVH, D, BF16, lens, window, sinks, seed=seed, mag=3.0)
        assert float(out.float().abs().mean()) > 0.05


@pytest.mark.parametrize("H,KVH,D,dtype", HEADS[:4])
def test_prefill_into_rows_that_start_anywhere(cuda, H, KVH, D, dtype):
    """Outputs whose rows start at 8-byte, 4-byte and 2-byte addresses, windowed
    and causal: the bits of aligned rows, and nothing beside them. (The kernel of
    other shapes sums in another order: its bits would differ.)"""
    g = torch.Generator().manual_seed(D + H)
    lens, before = [150, 40, 33], [0, 7, 0]
    new = [n - c for n, c in zip(lens, before)]
    T, n = sum(new), max(lens)
    pool = torch.randn(3 * n, 2 * KVH, D, generator=g).to(dtype).to(cuda)
    table = torch.randperm(3 * n, generator=g).to(torch.int32).view(3, n).to(cuda)
    q = torch.randn(T, H, D, generator=g).to(dtype).to(cuda)
    k, v, start = pool[:, :KVH], pool[:, KVH:], [0, new[0], new[0] + new[1]]
    a = [_i32(x, cuda) for x in ([0, 1, 2], start, lens)]
    for window in (None, 60):
        for pad, at in ((4, 4), (2, 2), (3, 1), (1, 1)):
            print(f"case: rows of {D + pad} from {at}, window {window} {dtype}", flush=True)
            wide = torch.full((T, H, D + pad), 7.0, dtype=dtype, device=cuda)
            outs = [torch.empty_like(q), wide[..., at:at + D]]
            for o in outs:
                if window is None:
                    _ops().prefill_attention(q, k, v, o, *a, n, table,
                                             b_shared_seq_len=_i32(before, cuda))
                else:
                    _ops().window_prefill_attention(q, k, v, o, *a, n, table, window, sinks=2,
                                                    b_shared_seq_len=_i32(before, cuda))
            assert torch.equal(*outs)
            wide[..., at:at + D] = 7.0
            assert bool((wide == 7.0).all())
