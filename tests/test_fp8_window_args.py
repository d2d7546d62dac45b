"""What the e4m3 linears and the windowed attention refuse, without a GPU: arguments are
checked before any device call, so the pointers here are only numbers."""
import ctypes

import pytest

P = 1 << 20          # an aligned address that is never read
I3 = ctypes.c_int64 * 3


def test_scale_bytes(lib):
    assert lib.da3b_fp8_scale_bytes(1, 1) == 512
    assert lib.da3b_fp8_scale_bytes(128, 512) == 512
    assert lib.da3b_fp8_scale_bytes(129, 512) == 1024
    assert lib.da3b_fp8_scale_bytes(129, 513) == 2048
    assert lib.da3b_fp8_scale_bytes(0, 64) == 0 and lib.da3b_fp8_scale_bytes(5, -1) == 0
    assert lib.da3b_fp8_scale_bytes(2_000_000_000, 4096) == 8 * 15_625_000 * 512   # above 32 bits


QUANT = dict(x=P, dtype=0, rows=4, K=100, ldx=100, q=P, ldq=112, scales=P)


@pytest.mark.parametrize("change,rc", [
    (dict(x=None), -100), (dict(q=None), -100), (dict(scales=None), -100), (dict(rows=-1), -100),
    (dict(K=0), -1), (dict(K=-5), -1), (dict(ldx=99), -1), (dict(ldq=100), -1), (dict(ldq=96), -1),
    (dict(q=P + 8), -1), (dict(scales=P + 4), -1), (dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(x=P + 1), -1),
    (dict(rows=0), 0), (dict(rows=(1 << 31) - 1), -1), (dict(K=(1 << 31) - 1, ldx=(1 << 31) - 1, ldq=(1 << 31) - 16), -1),
])
def test_quantize_refusals(lib, change, rc):
    a = {**QUANT, **change}
    assert lib.da3b_quantize_fp8(*a.values(), None) == rc


LN = dict(x=P, rows=4, K=100, ldx=100, g=P, b=None, eps=1e-6, q=P, ldq=112, scales=P)


@pytest.mark.parametrize("change,rc", [
    (dict(x=None), -100), (dict(g=None), -100), (dict(q=None), -100), (dict(scales=None), -100), (dict(rows=-1), -100),
    (dict(K=0), -1), (dict(K=16385, ldx=16385, ldq=16400), -1), (dict(ldx=99), -1), (dict(ldq=104), -1),
    (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(x=P + 2), -1), (dict(b=P + 2), -1), (dict(rows=0), 0),
])
def test_layernorm_refusals(lib, change, rc):
    a = {**LN, **change}
    assert lib.da3b_layernorm_fp8(*a.values(), None) == rc


LIN = dict(x=P, M=4, K=100, ldx=112, xs=P, w=P, N=30, ldw=112, ws=P, bias=None, act=0, out=P, dt=0, ldo=30)
COMMON = [
    (dict(x=None), -100), (dict(xs=None), -100), (dict(w=None), -100), (dict(ws=None), -100), (dict(out=None), -100),
    (dict(M=-1), -100), (dict(K=0), -1), (dict(N=0), -1), (dict(ldx=96), -1),
    (dict(ldx=100), -1), (dict(ldw=104), -1), (dict(x=P + 8), -1), (dict(w=P + 1), -1), (dict(xs=P + 4), -1),
    (dict(ws=P + 8), -1), (dict(bias=P + 2), -1), (dict(ldo=29), -1), (dict(M=0), 0), (dict(M=(1 << 31) - 1), -1),
    (dict(N=(1 << 31) - 1, ldo=(1 << 31) - 1), -1),
]


@pytest.mark.parametrize("change,rc", COMMON + [
    (dict(act=4), -100), (dict(act=-1), -100), (dict(dt=3), -100), (dict(dt=-1), -100), (dict(out=P + 1), -1),
    (dict(dt=2, out=P + 2), -1)])
def test_linear_refusals(lib, change, rc):
    a = {**LIN, **change}
    assert lib.da3b_linear_fp8(*a.values(), None) == rc


@pytest.mark.parametrize("change,rc", COMMON + [
    (dict(act=4), -100), (dict(os=None), -100), (dict(ldo=40), -1), (dict(out=P + 8), -1), (dict(os=P + 8), -1)])
def test_linear_q_refusals(lib, change, rc):
    a = {**{k: v for k, v in LIN.items() if k != "dt"}, "ldo": 32, "os": P, **change}
    assert lib.da3b_linear_fp8_q(*a.values(), None) == rc


@pytest.mark.parametrize("change,rc", COMMON + [(dict(scale=P + 2), -1), (dict(out=P + 2), -1)])
def test_linear_resid_refusals(lib, change, rc):
    a = {**LIN, **change}
    assert lib.da3b_linear_fp8_resid_f32(a["x"], a["M"], a["K"], a["ldx"], a["xs"], a["w"], a["N"], a["ldw"], a["ws"],
                                         a["bias"], a.get("scale"), a["out"], a["ldo"], None) == rc


# q, k, v, out [2][5][4][64] / [2][9][2][64]
ATT = dict(q=P, qs=(1280, 256, 64), k=P, ks=(1152, 128, 64), v=P, vs=(1152, 128, 64), out=P, os=(1280, 256, 64), dt=0,
           nseq=2, q_len=5, k_len=9, heads=4, kv_heads=2, D=64, ql=None, kl=None, left=3, right=0, sinks=1, scale=0.125)


@pytest.mark.parametrize("change,rc", [
    (dict(q=None), -100), (dict(k=None), -100), (dict(v=None), -100), (dict(out=None), -100), (dict(qs=None), -100),
    (dict(ks=None), -100), (dict(vs=None), -100), (dict(os=None), -100), (dict(dt=2), -100), (dict(dt=-1), -100),
    (dict(nseq=-1), -100), (dict(q_len=-1), -100), (dict(k_len=-1), -100), (dict(heads=0), -100), (dict(kv_heads=0), -100),
    (dict(kv_heads=3), -100), (dict(kv_heads=8), -100), (dict(D=96), -100), (dict(D=32), -100), (dict(sinks=-1), -100),
    (dict(scale=-1.0), -100), (dict(scale=float("nan")), -100), (dict(scale=float("inf")), -100),
    (dict(q_len=(1 << 30) + 1), -1), (dict(k_len=(1 << 30) + 1), -1),
    (dict(qs=(1280, 256, 60)), -1), (dict(ks=(1152, 130, 64)), -1), (dict(vs=(0, 128, 64)), -1),
    (dict(os=(-1280, 256, 64)), -1), (dict(ks=(1152, 128, 32)), -1), (dict(ks=(1 << 40, 128, 64)), -1),
    (dict(q=P + 8), -1), (dict(k=P + 2), -1), (dict(v=P + 8), -1), (dict(out=P + 8), -1),
    (dict(nseq=0), 0), (dict(q_len=0), 0),
])
def test_attention_window_refusals(lib, change, rc):
    a = {**ATT, **change}
    args = [I3(*v) if isinstance(v, tuple) else v for v in a.values()]
    assert lib.da3b_attention_window(*args, None) == rc


def test_buffers_without_rows_may_be_null(lib):
    """As the tensors of an empty batch are: nothing is launched, and nothing is refused."""
    a = {**QUANT, "rows": 0, "x": None, "q": None, "scales": None}
    assert lib.da3b_quantize_fp8(*a.values(), None) == 0
    a = {**LN, "rows": 0, "x": None, "q": None, "scales": None}
    assert lib.da3b_layernorm_fp8(*a.values(), None) == 0
    e = {**LIN, "M": 0, "x": None, "xs": None, "out": None}
    assert lib.da3b_linear_fp8(*e.values(), None) == 0
    assert lib.da3b_linear_fp8(*{**e, "w": None}.values(), None) == -100
    a = {**{k: v for k, v in e.items() if k != "dt"}, "ldo": 32, "os": None}
    assert lib.da3b_linear_fp8_q(*a.values(), None) == 0
    assert lib.da3b_linear_fp8_resid_f32(None, 0, 100, 112, None, P, 30, 112, P, None, None, None, 30, None) == 0
    for change in (dict(nseq=0), dict(q_len=0)):
        a = {**ATT, **change, "q": None, "out": None}
        assert lib.da3b_attention_window(*[I3(*v) if isinstance(v, tuple) else v for v in a.values()], None) == 0
