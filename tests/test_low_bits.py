"""8-bit cache, 4-bit products and logit controls on the CPU: the oracle itself,
refusals of the C ABI and of the Python calls. No kernel runs here: refused
calls return before anything is launched.
"""
import ctypes
import math
import re

import pytest
import torch

from oracle import low_bits as O

INT8, E4M3 = O.INT8, O.E4M3


def _ops():
    from lite_lang_amd import ops
    return ops


# ---------------------------------------------------------------- the oracle
def test_oracle_codes_are_the_nearest():
    """int8 as round() gives them; e4m3 as torch's conversion of fp32 numbers that
    hold the quotient exactly."""
    g = torch.Generator().manual_seed(1)
    q = torch.randn(4000, generator=g).double() * 40
    q = torch.cat([q, torch.arange(-126.5, 127.0, 1.0).double(), torch.zeros(1)]).clamp(-127, 127)
    assert torch.equal(O.nearest(q, INT8), q.round())
    x = torch.cat([torch.randn(4000, generator=g) * 100, torch.randn(4000, generator=g) * 2.0 ** -7,
                   (O.grid(E4M3)[1:].float() + O.grid(E4M3)[:-1].float()) / 2]).clamp(-448, 448)
    assert torch.equal(O.nearest(x.double(), E4M3), x.to(E4M3).double())


@pytest.mark.parametrize("code", [INT8, E4M3])
def test_oracle_store_continues_and_begins_blocks(code):
    """A scale never shrinks within a block, codes follow it, a run from a block's
    first slot forgets what was there."""
    codes, scale = torch.zeros(16, 1, 4).double(), torch.full((2, 1), 9.0).double()
    x = torch.tensor([[[1.0, -2.0, 0.5, 4.0]]])
    O.kv8_store(x, [8], codes, scale, 8, code)
    s = float(torch.tensor(4.0 / O.top(code), dtype=torch.float32))
    assert float(scale[1, 0]) == s and float(scale[0, 0]) == 9.0
    first = codes[8].clone()
    O.kv8_store(x * 0.25, [9], codes, scale, 8, code)
    assert float(scale[1, 0]) == s and torch.equal(codes[8], first)
    O.kv8_store(x * 3, [10, -1, 99, 11][:2], codes, scale, 8, code)
    s3 = float(torch.tensor(12.0 / O.top(code), dtype=torch.float32))
    assert float(scale[1, 0]) == s3
    assert torch.equal(codes[8], O.nearest(first * s / s3, code))
    O.kv8_store(x * 0.01, [8], codes, scale, 8, code)
    assert float(scale[1, 0]) < s
    assert torch.equal(O.kv8_values(codes, scale, 8)[9], codes[9] * scale[1])
    O.kv8_store(torch.tensor([[[1.0, math.nan, 0.0, 0.0]]]), [9], codes, scale, 8, code)
    assert math.isnan(float(scale[1, 0])) and float(codes[9].abs().max()) == 0.0


def test_oracle_decode_of_a_plain_cache_is_softmax():
    g = torch.Generator().manual_seed(2)
    k, v = torch.randn(9, 2, 8, generator=g).double(), torch.randn(9, 2, 8, generator=g).double()
    q = torch.randn(1, 4, 8, generator=g)
    t = torch.tensor([[3, 1, 40, 8, 0]])
    out = O.kv8_decode(q, k, v, t, [0], [4], 9)[0]
    for h in range(4):
        kk, vv = k[[3, 1, 8], h // 2], v[[3, 1, 8], h // 2]
        p = torch.softmax(kk @ q[0, h].double() / math.sqrt(8), 0)
        assert torch.allclose(out[0, h], p @ vv, atol=1e-12)


def test_oracle_w4_weight():
    codes = torch.tensor([[0x21, 0xf8] + [0x88] * 14], dtype=torch.uint8)
    scale = torch.tensor([[0.5]], dtype=torch.bfloat16)
    w = O.w4_weight(codes, scale)
    assert w.shape == (1, 32) and w[0, :4].tolist() == [-3.5, -3.0, 0.0, 3.5]
    assert O.w4_weight(codes, scale, torch.tensor([[1]]))[0, 0] == 0.0


def test_oracle_logits_by_hand():
    x = torch.tensor([[2.0, -2.0, 1.0, 0.5, 3.0]])
    t = torch.tensor([[0, 1, 2, 2, 9]], dtype=torch.int32)
    y, _ = O.adjust_logits(x, t, [0], [2], [5], torch.tensor([2.0]), torch.tensor([0.25]),
                           torch.tensor([1.0]), torch.tensor([[3, 3, -1]]),
                           torch.tensor([[1.0, 2.0, 7.0]]), torch.tensor([[0b01111]]))
    assert y[0].tolist() == [1.0, -4.0, 0.5 - 0.5 - 1.0, 3.5, -math.inf]


# ---------------------------------------------------------------- the C ABI
def _err(L):
    return L.ll_last_error().decode()


def test_records_match_their_entry_points():
    from lite_lang_amd import _lib
    text = open(_lib.HEADER_PATH).read()
    for name, rec, fn in (("LLKv8StoreCall", _lib.KV8_STORE_CALL, "ll_kv8_store"),
                          ("LLKv8LoadCall", _lib.KV8_LOAD_CALL, "ll_kv8_load"),
                          ("LLKv8DecodeAttentionCall", _lib.KV8_DECODE_ATTENTION_CALL,
                           "ll_kv8_decode_attention"),
                          ("LLLinearW4Call", _lib.LINEAR_W4_CALL, "ll_linear_w4"),
                          ("LLAdjustLogitsCall", _lib.ADJUST_LOGITS_CALL, "ll_adjust_logits")):
        body = re.search(r"typedef struct \{([^}]*)\} %s;" % name, text).group(1)
        names = re.findall(r"(\w+)(?=[,;])", body)
        args = re.search(r"^int %s\(([^;]*)\);" % fn, text, re.M).group(1)
        assert names == [a.split()[-1].lstrip("*") for a in args.split(",")]
        assert rec.size == 8 * len(names) == 8 * len(_lib.SIGNATURES[fn][1])


def _store(L, p=256, k=256, T=3, KVH=2, D=64, block=16, code=0, dtype=2, n=64, kc=128, kch=64,
           ks=2, ksh=1):
    return L.ll_kv8_store(k, KVH * D, D, p, KVH * D, D, p, T, KVH, D, p, kc, kch, p, KVH * D, D, p,
                          ks, ksh, p, KVH, 1, n, block, code, dtype, None)


def _load(L, p=256, k=256, KVH=2, D=64, block=16, code=0, dtype=2, n=64, B=2, most=8, rows=9,
          ko=128, koh=64):
    return L.ll_kv8_load(k, KVH * D, D, p, KVH * D, D, p, KVH, 1, p, KVH, 1, n, block, code, p, 8, 4,
                         p, 0, p, 0, p, 0, B, most, p, ko, koh, p, KVH * D, D, rows, KVH, D, dtype,
                         None)


def _decode(L, p=256, q=256, H=4, KVH=2, D=64, block=16, code=0, dtype=2, n=64, B=2, most=8,
            scale=1.0, ob=256, oh=64, ws=None, wsn=0):
    return L.ll_kv8_decode_attention(q, H * D, D, p, KVH * D, D, p, KVH * D, D, p, KVH, 1, p, KVH, 1,
                                     n, block, code, p, 8, 4, p, 0, p, 0, p, ob, oh, B, H, KVH, D,
                                     most, ctypes.c_float(scale), dtype, ws, wsn, None)


def test_kv8_entry_points_refuse_bad_arguments():
    from lite_lang_amd import _lib
    L = _lib.load()
    for call in (_store, _load, _decode):
        assert call(L, p=None) == -1 and "null pointer" in _err(L)
        assert call(L, code=2) == -1 and "code kind" in _err(L)
        assert call(L, code=-1) == -1 and "code kind" in _err(L)
        for block in (0, -16, 3, 24, 256):
            assert call(L, block=block) == -1 and "power of two" in _err(L)
        for n in (-1, 1 << 31):
            assert call(L, n=n) == -1 and "slots" in _err(L)
        assert call(L, KVH=0) == -1 and call(L, KVH=1 << 16) == -1
        assert call(L, D=0) == -1 and "head_dim" in _err(L)
        assert call(L, D=2048) == -1 and "head_dim" in _err(L)
        assert call(L, dtype=7) == -2 and "dtype" in _err(L)
    assert _store(L, k=None) == -1 and _load(L, k=None) == -1 and _decode(L, q=None) == -1
    assert _store(L, T=0) == 0 and _store(L, T=-1) == -1
    assert _store(L, T=(1 << 24) + 1) == -1 and "tokens" in _err(L)
    assert _store(L, T=1 << 24, KVH=60000, D=8, kc=480000, kch=8) == -1 and "heads" in _err(L)
    for kw in ({"kc": 0}, {"kch": 0}, {"ks": 0}, {"ksh": 0}):
        assert _store(L, **kw) == -1 and "stride 0" in _err(L)
    assert _load(L, B=0) == 0 and _load(L, rows=0) == 0 and _load(L, most=0) == 0
    assert _load(L, B=65536) == -1 and "requests" in _err(L)
    assert _load(L, most=(1 << 30) + 1) == -1 and _load(L, rows=-1) == -1
    for kw in ({"ko": 0}, {"koh": 0}):
        assert _load(L, **kw) == -1 and "stride 0" in _err(L)
    assert _decode(L, B=0) == 0 and _decode(L, B=-1) == -1 and _decode(L, B=1 << 25) == -1
    assert _decode(L, H=3) == -1 and _decode(L, H=0) == -1 and _decode(L, H=1 << 17) == -1
    assert _decode(L, most=(1 << 30) + 1) == -1 and _decode(L, most=-1) == -1
    for scale in (0.0, -1.0, math.nan, math.inf):
        assert _decode(L, scale=scale) == -1 and "sm_scale" in _err(L)
    for kw in ({"ob": 0}, {"oh": 0}):
        assert _decode(L, **kw) == -1 and "stride 0" in _err(L)
    assert _decode(L, most=4096) == -1 and "workspace needs" in _err(L)
    assert _decode(L, most=4096, ws=256, wsn=64) == -1 and "workspace needs" in _err(L)
    assert _decode(L, most=4096, ws=264, wsn=1 << 30) == -1 and "aligned" in _err(L)
    for B, H, KVH in ((1 << 24, 256, 256), (1 << 24, 16, 2), (1 << 24, 65535, 1)):
        for D in (64, 80, 128):
            assert _decode(L, B=B, H=H, KVH=KVH, D=D, most=1 << 30) == -1, _err(L)


def test_kv8_workspace_query_takes_any_counts():
    from lite_lang_amd import _lib
    fn = _lib.load().ll_kv8_decode_attention_workspace_size
    for a in ((0, 16, 2, 128, 4096), (-1, 16, 2, 128, 4096), (4, 0, 0, 128, 4096),
              (4, 16, 0, 128, 4096), (1 << 40, 16, 2, 64, 1 << 30), (4, 16, 1 << 40, 64, 1 << 20),
              (4, 16, 2, 64, 1 << 40), (4, 16, 2, 64, 0), (4, 16, 2, 64, -5), (4, 16, 3, 64, 4096),
              (1 << 24, 65535, 1, 128, 1 << 30), (4, 16, 2, 96, 4096)):
        assert fn(*a) == 0, a


def test_kv8_workspace_holds_a_part_of_every_workgroup():
    """Head blocks below and above the 512 workgroups that run at a time: each has
    one at least, so that W + batch parts of W >= 1 fit (fp32 sums, a maximum and a
    sum for each query head, two words for each request)."""
    from lite_lang_amd import _lib
    fn = _lib.load().ll_kv8_decode_attention_workspace_size
    for D in (64, 128, 256):
        for B in (1, 2, 3, 4, 5, 9):
            for H, KVH in ((511, 511), (512, 512), (513, 513), (520, 520), (1024, 1024), (8192, 1),
                           (8200, 1), (16400, 2), (65535, 65535), (65535, 1)):
                for most in (2049, 4096, 1 << 20):
                    need = fn(B, H, KVH, D, most)
                    w = max(512 // (KVH * -(-H // KVH // 16)), B // 4, 1)
                    assert need == (w + B) * H * (D * 4 + 8) + B * 8, (B, H, KVH, D, most)


def test_w4_entry_points_refuse_bad_arguments():
    from lite_lang_amd import _lib
    L, p = _lib.load(), 256

    def pack(codes=p, N=16, K=128, group=64, n=1 << 20, out=p, zero=p):
        return L.ll_w4_pack(codes, K // 2, p, 2, zero, 2, N, K, group, out, n, None)

    def lin(x=p, N=16, K=128, group=64, M=2, dtype=2, ldy=16, ldx=128, w=p):
        return L.ll_linear_w4(x, ldx, w, 1, group, None, p, ldy, M, N, K, dtype, None, 0, None)

    assert pack(codes=None) == -1 and "null" in _err(L)
    assert lin(x=None) == -1 and "null" in _err(L)
    for kw in ({"N": 0}, {"K": 0}, {"K": 96}, {"group": 16}, {"group": 0}, {"N": 1 << 40},
               {"K": 1 << 40}):
        assert pack(**kw) == -1 and "group" in _err(L)
        assert lin(**kw) == -1 and "group" in _err(L)
        a = {"N": 16, "K": 128, "group": 64, **kw}
        assert L.ll_w4_packed_bytes(a["N"], a["K"], a["group"], 1) == 0
    want = L.ll_w4_packed_bytes(16, 128, 64, 1)
    assert want > L.ll_w4_packed_bytes(16, 128, 64, 0) > 16 * 64
    assert pack(n=want - 1) == -1 and "bytes" in _err(L)
    assert pack(out=264) == -1 and "aligned" in _err(L)
    assert pack(N=1 << 26, K=1 << 26, n=1 << 60) == -1 and "too large" in _err(L)
    assert lin(M=0) == 0 and lin(M=-1) == -1 and lin(M=(1 << 19) + 1) == -1
    assert lin(dtype=0) == -1 and "bf16" in _err(L)
    assert lin(w=264) == -1 and "aligned" in _err(L)
    long = {"N": 32, "K": 11008, "M": 40, "ldx": 11008, "ldy": 32, "group": 128}
    assert lin(**long) == -1 and "workspace needs" in _err(L)
    assert lin(ldy=15) == -1 and "strides" in _err(L)
    assert lin(ldx=-8) == -1 and "strides" in _err(L)


def test_adjust_logits_refuses_bad_arguments():
    from lite_lang_amd import _lib
    L, p = _lib.load(), 256

    def call(x=p, out=p, B=2, V=8, tok=p, req=p, rep=p, ids=p, vals=p, nb=1, ldo=8, cols=4, dtype=0):
        return L.ll_adjust_logits(x, 8, out, ldo, B, V, tok, 4, 2, cols, req, 0, p, 0, p, 0, rep,
                                  None, None, ids, 1, vals, 1, nb, p, 1, dtype, None)

    assert call(x=None) == -1 and "null" in _err(L)
    assert call(out=None) == -1 and "null" in _err(L)
    assert call(req=None) == -1 and "rows and lengths" in _err(L)
    assert call(tok=None) == -1 and "penalties need" in _err(L)
    assert call(ids=None) == -1 and call(vals=None) == -1 and call(nb=-1) == -1
    assert call(nb=(1 << 20) + 1) == -1 and "biases" in _err(L)
    assert call(B=0) == 0 and call(V=0) == 0
    assert call(B=65536) == -1 and call(V=(1 << 31) - 1) == -1 and call(B=-1) == -1
    assert call(ldo=7) == -1 and "overlap" in _err(L)
    assert call(cols=1 << 31) == -1 and "tokens" in _err(L)
    assert call(dtype=5) == -2 and "dtype" in _err(L)


# ---------------------------------------------------------------- the Python calls
def test_python_calls_refuse_cpu_tensors_and_bad_shapes():
    ops = _ops()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    pool = torch.zeros(32, 4, 64, dtype=INT8)
    sc = torch.zeros(2, 4)
    cache = (pool[:, :2], pool[:, 2:], sc[:, :2], sc[:, 2:])
    x = torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="CPU"):
        ops.kv8_store(x, x, i(3), *cache, 16)
    with pytest.raises(ValueError, match="do not cover"):
        ops.kv8_store(x, x, i(3), *cache, 8)
    with pytest.raises(ValueError, match="do not cover"):
        ops.kv8_store(x, x, i(3), *cache, 0)
    with pytest.raises(TypeError, match="int8 or"):
        ops.kv8_store(x, x, i(3), cache[0].float(), cache[1].float(), *cache[2:], 16)
    for bad in ((x[:, :1], x, i(3)), (x, x[:2], i(3)), (x, x.half(), i(3)), (x, x, i(2)),
                (x, x, i(3).long()), (x, x, i(3, 1)), (x.transpose(1, 2), x, i(3)),
                (x[..., ::2], x, i(3))):
        with pytest.raises(AssertionError):
            ops.kv8_store(*bad, *cache, 16)
    with pytest.raises(AssertionError):
        ops.kv8_store(x, x, i(3), cache[0], cache[1].view(E4M3), *cache[2:], 16)
    with pytest.raises(AssertionError):
        ops.kv8_store(x, x, i(3), cache[0], cache[1], sc[:, :2].half(), sc[:, 2:], 16)
    out = torch.zeros(9, 2, 64)
    with pytest.raises(ValueError, match="CPU"):
        ops.kv8_load(*cache, 16, i(2, 8), i(2), i(2), i(2), 8, out, out)
    for kw in ({"most": 9}, {"most": -1}, {"req": i(3)}, {"out": out[:, :1]}, {"t": i(2, 8).long()}):
        a = {"most": 8, "req": i(2), "out": out, "t": i(2, 8), **kw}
        with pytest.raises(AssertionError):
            ops.kv8_load(*cache, 16, a["t"], a["req"], i(2), i(2), a["most"], a["out"], out)
    q = torch.zeros(2, 4, 64)
    with pytest.raises(ValueError, match="CPU"):
        ops.kv8_decode_attention(q, i(2, 8), i(2), i(2), 8, *cache, 16, q)
    for kw in ({"most": 9}, {"q": q[:, :3]}, {"q": q[..., :32]}, {"req": i(3)}, {"out": q.half()},
               {"t": i(2, 8).long()}):
        a = {"most": 8, "q": q, "req": i(2), "t": i(2, 8), **kw}
        with pytest.raises(AssertionError):
            ops.kv8_decode_attention(a["q"], a["t"], a["req"], i(2), a["most"], *cache, 16,
                                     a.get("out", a["q"]))


def test_python_w4_and_logits_refuse_bad_arguments():
    ops = _ops()
    codes, scale = torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 2, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CPU"):
        ops.W4Weight(codes, scale)
    for bad in (torch.zeros(16, 8), torch.zeros(16, 3), torch.zeros(16, 0), torch.zeros(16, 128)):
        with pytest.raises(ValueError, match="groups are of"):
            ops.W4Weight(codes, bad.bfloat16())
    for bad in ((codes.int(), scale), (codes, scale.float()), (codes, scale[:8]),
                (codes, scale, torch.zeros(16, 2)), (codes, scale, torch.zeros(8, 2, dtype=torch.uint8))):
        with pytest.raises(AssertionError):
            ops.W4Weight(*bad)
    x = torch.zeros(2, 9)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="CPU"):
        ops.adjust_logits(x)
    with pytest.raises(ValueError, match="need the tokens"):
        ops.adjust_logits(x, repetition=torch.ones(2))
    with pytest.raises(ValueError, match="bias_ids"):
        ops.adjust_logits(x, bias_values=torch.ones(2, 3))
    hist = (i(4, 5), i(2), i(2), i(2))
    for a, kw in ((hist[:3], {}), ((i(4, 5), i(3), i(2), i(2)), {}), ((i(4, 5).long(), *hist[1:]), {}),
                  (hist, {"repetition": torch.ones(3)}), (hist, {"presence": torch.ones(2).half()}),
                  ((), {"bias_ids": i(2, 3), "bias_values": torch.ones(2, 4)}),
                  ((), {"bias_ids": i(2, 3).long(), "bias_values": torch.ones(2, 3)}),
                  ((), {"mask": i(2, 0)}), ((), {"mask": i(3, 1)}), ((), {"mask": i(2, 1).long()}),
                  ((), {"out": x[:1]}), ((), {"out": x.half()})):
        with pytest.raises(AssertionError):
            ops.adjust_logits(x, *a, **kw)


def test_a_history_of_no_columns_is_checked_like_any_other():
    """The arguments that a table of five columns would have refused, with none."""
    ops = _ops()
    x = torch.zeros(2, 9)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    for cols in (0, 5):
        hist = (i(4, cols), i(2), i(2), i(2))
        with pytest.raises(ValueError, match="CPU"):
            ops.adjust_logits(x, *hist, repetition=torch.ones(2))
        with pytest.raises(TypeError, match="int32 or int64"):
            ops.adjust_logits(x, hist[0], i(2).float(), i(2), i(2))
        for a, kw in ((hist[:1], {}), (hist[:3], {}), ((hist[0], i(3), i(2), i(2)), {}),
                      ((hist[0].long(), *hist[1:]), {}), ((hist[0].float(), *hist[1:]), {}),
                      (hist, {"repetition": torch.ones(3)}), (hist, {"frequency": torch.ones(2, 1)}),
                      (hist, {"presence": torch.ones(2).half()})):
            with pytest.raises(AssertionError):
                ops.adjust_logits(x, *a, **kw)
