"""Long-context operators on the CPU: frequencies, the oracle itself, refusals.

No kernel runs here: refused calls return before anything is launched.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import long_context as O


def _ops():
    from lite_lang_amd import ops
    return ops


# ---------------------------------------------------------------- frequencies
def test_plain_frequencies_are_powers_of_theta():
    f, factor = _ops().rope_frequencies(64, theta=1e6)
    want = [1e6 ** (-2 * i / 64) for i in range(32)]
    assert factor == 1.0 and f.dtype == torch.float32
    assert np.allclose(f.double().numpy(), want, rtol=2.0 ** -24, atol=0)
    f4, _ = _ops().rope_frequencies(64, theta=1e6, scaling={"rope_type": "linear", "factor": 4.0})
    assert np.allclose(f4.double().numpy() * 4, want, rtol=2.0 ** -23, atol=0)


def test_yarn_keeps_fast_pairs_and_stretches_slow_ones():
    orig, s, dim, theta = 32768, 4.0, 128, 1e6
    plain, _ = _ops().rope_frequencies(dim, theta=theta)
    f, factor = _ops().rope_frequencies(
        dim, theta=theta, scaling={"type": "yarn", "factor": s,
                                   "original_max_position_embeddings": orig})
    assert factor == pytest.approx(0.1 * math.log(s) + 1.0)
    turns = orig * plain.double() / (2 * math.pi)
    ratio = (f / plain).double()
    # one pair of slack on either side: the ends of the ramp are whole pairs
    assert torch.allclose(ratio[:-1][turns[1:] > 32], torch.tensor(1.0, dtype=torch.float64))
    assert torch.allclose(ratio[1:][turns[:-1] < 1], torch.tensor(1 / s, dtype=torch.float64))
    assert bool((ratio[1:] <= ratio[:-1] + 1e-6).all())


@pytest.mark.parametrize("scaling", [
    {"rope_type": "linear", "factor": 8.0},
    {"rope_type": "dynamic", "factor": 4.0},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096},
    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096,
     "beta_fast": 24, "beta_slow": 2, "attention_factor": 1.25},
    {"rope_type": "longrope", "long_factor": [1 + 0.25 * i for i in range(32)],
     "short_factor": [1 + 0.01 * i for i in range(32)], "factor": 8.0,
     "original_max_position_embeddings": 4096},
])
@pytest.mark.parametrize("length", [None, 1000, 30000])
def test_scaled_frequencies_match_transformers(scaling, length):
    """Against transformers' own initialisers, for the configs it writes; fp32
    there, so to a few of its roundings (its power and quotients: 2^-20)."""
    mod = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import Qwen2Config
    cfg = Qwen2Config(hidden_size=256, num_attention_heads=4, num_key_value_heads=2,
                      max_position_embeddings=4096, rope_theta=10000.0,
                      rope_scaling=dict(scaling, rope_theta=10000.0))
    kind = scaling["rope_type"]
    try:
        want, want_factor = mod.ROPE_INIT_FUNCTIONS[kind](cfg, "cpu", seq_len=length)
    except (AttributeError, KeyError, TypeError) as e:
        pytest.skip(f"this transformers reads such a config otherwise: {e!r}")
    if kind == "longrope" and length is None:
        length = 30000  # without a length theirs takes the short factors, ours the long ones
        want, want_factor = mod.ROPE_INIT_FUNCTIONS[kind](cfg, "cpu", seq_len=length)
    got, factor = _ops().rope_frequencies(64, theta=10000.0, scaling=scaling, max_position=4096,
                                          length=length)
    assert factor == pytest.approx(want_factor, rel=1e-6)
    assert torch.allclose(got.double(), want.double(), rtol=2.0 ** -18, atol=0)


@pytest.mark.parametrize("extra", [{"mscale": 1.0, "mscale_all_dim": 0.8}, {"mscale": 0.7},
                                   {"mscale": 1.0, "mscale_all_dim": 1.0}])
@pytest.mark.parametrize("s", [1.0, 40.0])
def test_yarn_factor_from_two_magnitudes(extra, s):
    """m(mscale) / m(mscale_all_dim) where both are given, m(1) else."""
    sc = {"rope_type": "yarn", "factor": s, "original_max_position_embeddings": 4096, **extra}
    f, factor = _ops().rope_frequencies(64, theta=10000.0, scaling=sc)
    m = lambda k: 0.1 * k * math.log(s) + 1.0  # noqa: E731
    want = m(extra["mscale"]) / m(extra["mscale_all_dim"]) if len(extra) == 2 else m(1.0)
    assert factor == pytest.approx(want, rel=1e-12)
    mod = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import Qwen2Config
    cfg = Qwen2Config(hidden_size=256, num_attention_heads=4, num_key_value_heads=2,
                      max_position_embeddings=int(4096 * s), rope_theta=10000.0,
                      rope_scaling=dict(sc, rope_theta=10000.0))
    theirs, theirs_factor = mod.ROPE_INIT_FUNCTIONS["yarn"](cfg, "cpu")
    assert factor == pytest.approx(theirs_factor, rel=1e-6)
    assert torch.allclose(f.double(), theirs.double(), rtol=2.0 ** -18, atol=0)


def test_bad_frequencies_are_refused():
    ops = _ops()
    for bad in (0, -2, 7):
        with pytest.raises(ValueError):
            ops.rope_frequencies(bad)
    with pytest.raises(ValueError, match="unknown"):
        ops.rope_frequencies(64, scaling={"rope_type": "spiral"})
    with pytest.raises(ValueError, match="max_position"):
        ops.rope_frequencies(64, scaling={"rope_type": "yarn", "factor": 4.0})
    with pytest.raises(ValueError, match="factors"):
        ops.rope_frequencies(64, scaling={"rope_type": "longrope", "long_factor": [1.0],
                                          "original_max_position_embeddings": 4096})


# ---------------------------------------------------------------- the oracle
def test_oracle_rotation_is_a_rotation():
    """Lengths are kept, and rotated q . rotated k depends on the difference of
    their positions alone."""
    g = torch.Generator().manual_seed(3)
    f = (10000.0 ** (-torch.arange(0, 16, 2) / 16)).float()
    q, k = torch.randn(1, 1, 16, generator=g), torch.randn(1, 1, 16, generator=g)
    for inter in (False, True):
        dots = []
        for p in (0, 5, 1 << 30):
            a, _ = O.rotate(q, torch.tensor([p + 3]), f, 1.0, inter)
            b, _ = O.rotate(k, torch.tensor([p]), f, 1.0, inter)
            assert float(a.square().sum()) == pytest.approx(float(q.double().square().sum()))
            dots.append(float((a * b).sum()))
        assert dots[0] == pytest.approx(dots[1], abs=1e-9)
        assert dots[0] == pytest.approx(dots[2], abs=1e-7)


def test_oracle_window_covers_the_context_when_it_is_long():
    from oracle import ops as full
    g = torch.Generator().manual_seed(4)
    lens, H, KVH, D = [9, 1, 6], 4, 2, 8
    table = torch.randperm(30, generator=g).int().view(3, 10)
    pool = torch.randn(30, 2 * KVH, D, generator=g)
    q = torch.randn(3, H, D, generator=g)
    want = full.decode_attention(q, table, [0, 1, 2], lens, pool[:, :KVH], pool[:, KVH:])
    for w, s in ((9, 0), (100, 3), (4, 5), (8, 1)):
        got, *_ = O.window_decode(q, pool[:, :KVH], pool[:, KVH:], table, [0, 1, 2], lens, w, s)
        assert torch.allclose(got, want.double(), atol=1e-12)
    assert O.visible(9, 20, 3, 2) == [0, 1, 7, 8, 9]
    assert O.visible(3, 20, 3, 2) == [0, 1, 2, 3]
    assert O.visible(0, 20, 1, 0) == [0]


# ---------------------------------------------------------------- refusals
def _attention_args(T=4, H=4, KVH=2, D=64, dtype=torch.bfloat16, B=2):
    q = torch.zeros(T, H, D, dtype=dtype)
    pool = torch.zeros(16, 2 * KVH, D, dtype=dtype)
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    return dict(q=q, k=pool[:, :KVH], v=pool[:, KVH:], o=torch.empty_like(q), rid=i32(B),
                start=i32(B), n=i32(B), table=torch.zeros(2, 8, dtype=torch.int32))


def _prefill(a, window=4, sinks=0, **kw):
    return _ops().window_prefill_attention(a["q"], a["k"], a["v"], a["o"], a["rid"], a["start"],
                                           a["n"], 8, a["table"], window, sinks=sinks, **kw)


def _decode(a, window=4, sinks=0):
    return _ops().window_decode_attention(a["q"], a["table"], a["rid"], a["n"], 8, a["k"], a["v"],
                                          a["o"], window, sinks=sinks)


@pytest.mark.parametrize("call", [_prefill, _decode])
def test_window_attention_refuses_bad_arguments(call):
    B = 2 if call is _prefill else 4
    good = _attention_args(B=B)
    with pytest.raises(ValueError, match="device tensors"):
        call(good)  # CPU tensors
    with pytest.raises(ValueError, match="window"):
        call(good, window=0)
    with pytest.raises(ValueError, match="window"):
        call(good, sinks=-1)
    for name, bad in (("q", torch.zeros(4, 3, 64, dtype=torch.bfloat16)),
                      ("q", torch.zeros(4, 4, 64)),
                      ("o", torch.zeros(4, 4, 32, dtype=torch.bfloat16)),
                      ("table", torch.zeros(2, 8, dtype=torch.int64)),
                      ("table", torch.zeros(8, 2, dtype=torch.int32).t()),
                      ("rid", torch.zeros(B + 1, dtype=torch.int32)),
                      ("n", torch.zeros(2 * B, dtype=torch.int32)[::2])):
        with pytest.raises(AssertionError):
            call(dict(good, **{name: bad}))


def test_rope_refuses_bad_arguments():
    ops = _ops()
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    pos, f = torch.zeros(3, dtype=torch.int32), torch.ones(32)
    with pytest.raises(ValueError, match="device tensors"):
        ops.rope_positions(q, k, pos, f)
    for args in ((q, k[:2], pos, f), (q, k.half(), pos, f), (q, k, pos[:2], f),
                 (q, k, pos, torch.ones(33)), (q, k, pos, f.double()),
                 (q.transpose(1, 2), k, pos, f)):
        with pytest.raises(AssertionError):
            ops.rope_positions(*args)
    with pytest.raises(AssertionError):
        ops.rope_positions(q, k, pos, f, q_out=torch.zeros(3, 4, 32))


def test_qk_norm_refuses_bad_arguments():
    ops = _ops()
    base = dict(qkv=torch.zeros(3, 8 * 64), g=torch.ones(64), pos=torch.zeros(3, dtype=torch.int32),
                f=torch.ones(32), slots=torch.zeros(3, dtype=torch.int32),
                pool=torch.zeros(9, 4, 64))

    def call(**kw):
        a = dict(base, **kw)
        return ops.qk_norm_rope_kv_scatter(a["qkv"], 4, 2, 64, a["g"], a["g"], 1e-6, a["pos"],
                                           a["f"], a["slots"], a["pool"])

    with pytest.raises(ValueError, match="device tensors"):
        call()
    for kw in ({"qkv": torch.zeros(3, 7 * 64)}, {"g": torch.ones(32)}, {"g": torch.ones(64).half()},
               {"pos": torch.zeros(4, dtype=torch.int32)}, {"slots": torch.zeros(3).long()},
               {"pool": torch.zeros(9, 3, 64)}, {"pool": torch.zeros(9, 4, 64).half()}):
        with pytest.raises(AssertionError):
            call(**kw)


def test_slot_maps_refuse_bad_arguments():
    ops = _ops()
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    base = dict(rid=i32(2), n=i32(2), c=i32(2), free=i32(4), table=i32(3, 8), slots=i32(6),
                pos=i32(6), start=i32(2), last=i32(2), counts=i32(3))

    def call(page=1, blocks=None, **kw):
        return ops.build_slot_maps(*dict(base, **kw).values(), page_size=page, block_table=blocks)

    with pytest.raises(ValueError, match="device tensors"):
        call()
    with pytest.raises(ValueError, match="block table"):
        call(page=16)
    with pytest.raises(ValueError, match="page_size"):
        call(page=0)
    for kw in ({"c": i32(3)}, {"slots": i32(5)}, {"counts": i32(2)}, {"table": i32(3, 8).long()},
               {"free": i32(2, 2)}):
        with pytest.raises(AssertionError):
            call(**kw)
    with pytest.raises(AssertionError):
        call(page=4, blocks=i32(2, 2))


def test_c_entry_points_refuse_before_any_launch():
    """Codes and messages of the C entry points; the pointers are never
    dereferenced, since every call returns before a launch."""
    from lite_lang_amd import _lib
    L = _lib.load()
    p, f = 256, ctypes.c_float

    def err():
        return L.ll_last_error().decode()

    def prefill(H=4, KVH=2, D=64, window=8, sinks=0, q=p, scale=1.0, most=8, B=2):
        return L.ll_window_prefill_attention(q, H * D, D, p, 2 * KVH * D, D, p, 2 * KVH * D, D, p,
                                             H * D, D, p, 8, p, 0, p, 0, p, 0, None, 0, B, H, KVH,
                                             D, most, window, sinks, f(scale), 2, None)

    def decode(H=4, KVH=2, D=64, window=8, sinks=0, q=p, scale=1.0, most=8, B=2):
        return L.ll_window_decode_attention(q, H * D, D, p, 2 * KVH * D, D, p, 2 * KVH * D, D, p, 8,
                                            p, 0, p, 0, p, H * D, D, B, H, KVH, D, most, window,
                                            sinks, f(scale), 2, None, 0, None)

    for call in (prefill, decode):
        assert call(q=None) == -1 and "null pointer" in err()
        assert call(H=3) == -1 and "multiple" in err()
        assert call(window=0) == -1 and "window" in err()
        assert call(sinks=-1) == -1 and "sinks" in err()
        for scale in (0.0, -1.0, float("nan"), float("inf")):
            assert call(scale=scale) == -1 and "sm_scale" in err()
        assert call(D=512) == -1 and "head_dim" in err()
        assert call(B=-1) == -1 and "requests" in err()
        assert call(B=1 << 25) == -1 and "requests" in err()
        assert call(H=0) == -1 and "heads" in err()
        assert call(most=(1 << 30) + 1) == -1 and "out of range" in err()

    def rope(R=64, D=64, ntok=2, out=p, pos=p):
        return L.ll_rope_positions(p, 4 * D, D, out, 4 * D, D, 4, None, 0, 0, None, 0, 0, 0, pos, 0,
                                   p, R, 0, f(1.0), ntok, D, 2, None)

    assert rope(out=None) == -1 and "null" in err()
    assert rope(pos=None) == -1 and "null" in err()
    assert rope(R=66) == -1 and rope(R=63) == -1 and rope(ntok=-1) == -1 and rope(D=2048) == -1
    assert rope(ntok=0) == 0  # nothing to do

    assert rope(ntok=(1 << 24) + 1) == -1 and "tokens" in err()

    def wide(st, sh, heads=4, ntok=2):  # into rows or heads that share an address
        return L.ll_rope_positions(p, 256, 64, p, st, sh, heads, None, 0, 0, None, 0, 0, 0, p, 0, p,
                                   64, 0, f(1.0), ntok, 64, 2, None)

    assert wide(0, 64) == -1 and "stride 0" in err()
    assert wide(256, 0) == -1 and "stride 0" in err()

    def norm(q_st=512, q_sh=64, pool_st=256, pool_sh=64):
        return L.ll_qk_norm_rope_kv_scatter(p, 512, 2, 4, 2, 64, p, q_st, q_sh, p, p, f(1e-6), p, 0,
                                            p, 64, 0, f(1.0), p, p, pool_st, pool_sh, 9, 2, None)

    for kw in ({"q_st": 0}, {"q_sh": 0}, {"pool_st": 0}, {"pool_sh": 0}):
        assert norm(**kw) == -1 and "stride 0" in err()

    def maps(page=1, blocks=None, batch=2, rows=4, counts=p, free=p, nfree=3):
        return L.ll_build_slot_maps(p, 0, p, 0, p, 0, batch, free, nfree, page, blocks, 8, 8, p, 8,
                                    rows, 8, p, p, 6, p, p, counts, None)

    assert maps(counts=None) == -1 and "null" in err()
    assert maps(free=None) == -1 and "null" in err()
    assert maps(page=0) == -1 and maps(page=16) == -1 and "block table" in err()
    assert maps(batch=8193) == -1 and maps(rows=1 << 19) == -1 and maps(nfree=-1) == -1


# ---------------------------------------------------------------- counts beyond 32 bits
_QUERIES = """
import ctypes, json, sys
L = ctypes.CDLL(sys.argv[1])
out = []
for name, args in json.load(sys.stdin):
    fn = getattr(L, name)
    fn.restype = ctypes.c_int64
    out.append(fn(*[ctypes.c_int64(a) for a in args]))
print(json.dumps(out))
"""


def test_decode_size_queries_take_any_counts():
    """Counts whose product wraps to 0 in 32 bits, and none at all: no bytes, for
    the entry points refuse them. (In a process of its own: a division by such a
    product ends it.)"""
    import json
    import subprocess
    import sys

    from lite_lang_amd import build
    name = "ll_window_decode_attention_workspace_size"
    calls = [(name, [1 << 24, 256, 256, 128, 4096, 1024, 0]),
             (name, [1 << 32, 256, 256, 128, 4096, 1024, 0]),
             (name, [1 << 22, 4, 2, 128, 4096, 1024, 0]),
             (name, [1 << 40, 16, 2, 64, 1 << 30, 1 << 30, 0]),
             (name, [4, 16, 1 << 40, 64, 1 << 20, 1 << 20, 0]),
             (name, [4, 16, 2, 64, 1 << 40, 1 << 40, 0]),
             (name, [1 << 16, 8, 1, 128, 1 << 30, 1 << 30, 0]),
             (name, [0, 16, 2, 64, 1 << 20, 1 << 20, 0])]
    plain = "ll_decode_attention_workspace_size"
    calls += [(plain, [1 << 24, 256, 256, 128, 4096]), (plain, [1 << 32, 16, 2, 128, 4096]),
              (plain, [1 << 16, 8, 1, 128, 1 << 30]), (plain, [0, 16, 2, 128, 4096]), (plain, [4, 16, 0, 128, 4096])]
    live = [(name, [1, 16, 2, 128, 4096, 4096, 0]), (plain, [1, 16, 2, 128, 4096])]
    r = subprocess.run([sys.executable, "-c", _QUERIES, build.LIB_PATH], capture_output=True,
                       input=json.dumps(calls + live), text=True)
    assert r.returncode == 0, f"ended with {r.returncode}: {r.stderr}"
    sizes = json.loads(r.stdout)
    assert sizes[:len(calls)] == [0] * len(calls) and min(sizes[len(calls):]) > 0


def test_decode_refuses_more_workgroups_than_a_launch_holds():
    from lite_lang_amd import _lib
    L, p = _lib.load(), 256

    def window(B, H, KVH, D=128, most=4096, win=1024):
        return L.ll_window_decode_attention(p, H * D, D, p, 2 * KVH * D, D, p, 2 * KVH * D, D, p, 8,
                                            p, 0, p, 0, p, H * D, D, B, H, KVH, D, most, win, 0,
                                            ctypes.c_float(1.0), 2, None, 0, None)

    def plain(B, H, KVH, D=128, most=4096):
        return L.ll_decode_attention(p, H * D, D, p, 2 * KVH * D, D, p, 2 * KVH * D, D, p, 8, p, 0,
                                     p, 0, p, H * D, D, B, H, KVH, D, most, ctypes.c_float(1.0), 2,
                                     None, 0, None)

    for B, H, KVH in ((1 << 24, 256, 256), (1 << 23, 1, 1), (1 << 22, 4, 2), (1 << 24, 16, 2)):
        for call in (window, plain):
            assert call(B, H, KVH) == -1 and "workgroups" in L.ll_last_error().decode()
    # fewer units, each of many splits (4096 tokens at most in one)
    assert window(1 << 16, 8, 1, most=1 << 30, win=1 << 30) == -1
    assert "workgroups" in L.ll_last_error().decode()
    assert plain(1 << 16, 8, 1, most=1 << 30) == -1
    assert "workgroups" in L.ll_last_error().decode()
    # a product that wraps to 0, off the 16-bit paths
    assert window(1 << 24, 256, 256, D=96) == -1 and "65535" in L.ll_last_error().decode()


def test_window_prefill_without_query_rows_does_nothing():
    """Requests that are all in the cache: the tensors of their 0 rows have no
    address. One address without the other is still an error."""
    from lite_lang_amd import _lib
    L, p = _lib.load(), 256

    def call(q, out):
        return L.ll_window_prefill_attention(q, 256, 64, p, 256, 64, p, 256, 64, out, 256, 64, p, 8,
                                             p, 0, p, 0, p, 0, p, 0, 2, 4, 2, 64, 8, 8, 0,
                                             ctypes.c_float(1.0), 2, None)

    assert call(None, None) == 0
    for q, out in ((None, p), (p, None)):
        assert call(q, out) == -1 and "null pointer" in L.ll_last_error().decode()


def test_prefill_refuses_more_work_items_than_a_launch_holds():
    """Counts of row blocks, requests and heads whose product wraps in 32 bits
    (to none, and to fewer items than there are) and ones just above what a grid
    of 2^32 threads takes."""
    from lite_lang_amd import _lib
    L, p = _lib.load(), 256

    def args(H, KVH, D, B, most):
        return [p, H * D, D, p, 2 * KVH * D, D, p, 2 * KVH * D, D, p, H * D, D, p, 8, p, 0, p, 0, p,
                0, None, 0, B, H, KVH, D, most]

    def window(H, KVH, B, most, win=100, D=128, dtype=2):
        return L.ll_window_prefill_attention(*args(H, KVH, D, B, most), win, 0, ctypes.c_float(1.0),
                                             dtype, None)

    def plain(H, KVH, B, most, D=128, dtype=2):
        return L.ll_prefill_attention(*args(H, KVH, D, B, most), ctypes.c_float(1.0), dtype, None)

    # 2^24 blocks of 64 rows x 2^11 (request, KV head)s: 2^35; the same and one block
    for call in (window, plain):
        for most in (1 << 30, (1 << 30) - 63, (1 << 30) - (1 << 20)):
            for H, KVH, B in ((8, 2, 1 << 10), (16, 2, 1 << 10), (7, 1, 1 << 11), (2, 2, 1 << 20),
                              (4, 4, 1 << 24)):
                assert call(H, KVH, B, most) == -1 and "work items" in L.ll_last_error().decode()
    # 2^22 blocks of 256 rows, 2^23 of 64 and of 128, one head group each: 2^29 items
    for H, KVH, B, most in ((2, 2, 64, 1 << 30), (8, 2, 32, 1 << 29), (4, 2, 32, 1 << 30)):
        assert window(H, KVH, B, most) == -1 and "work items" in L.ll_last_error().decode()
    assert plain(4, 1, 1 << 24, 1 << 30) == -1 and "work items" in L.ll_last_error().decode()
    # off the 16-bit paths: a grid of one wave per row
    for call in (window, plain):
        assert call(4, 2, 2, 1 << 26, D=96) == -1 and "rows" in L.ll_last_error().decode()
        assert call(4, 2, 2, 1 << 26, dtype=0) == -1 and "rows" in L.ll_last_error().decode()
    assert plain(4, 2, 2, 1 << 31) == -1 and "out of range" in L.ll_last_error().decode()
    assert plain(4, 2, 2, (1 << 38) + 5) == -1 and "out of range" in L.ll_last_error().decode()
