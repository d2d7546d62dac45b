"""The e4m3 linears with block scales against plain torch.

The quantiser is exact arithmetic, so its codes and scale bytes are compared bit for bit
with torch's conversion to float8_e4m3fn. Linears are compared in 64 bits with the values
that codes and scales stand for. Their tolerance: products of two e4m3 values are exact,
and each of the K additions of an f32 sum is off by at most 2^-23 of the largest partial sum
(a tensor core may cut, not round, when it aligns its terms), itself at most
S = sum |x||w|; the scale, bias and activation add a few roundings of 2^-24; then the output
type rounds by half a step (f16 2^-11, bf16 2^-8, e4m3 2^-4 of the value, and 2^-10 of the
block's scale for its subnormals). GELU's erf is good to 1.5e-7 (3e-7 for the other form)
absolutely, half of that times |y| for the value."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
DT = [torch.float16, torch.bfloat16, torch.float32]
HALF_STEP = [2.0 ** -11, 2.0 ** -8, 2.0 ** -24]


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


def st():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def up(v, m):
    return -(-v // m) * m


def plain_quant(x):
    """Codes (uint8 [R][K]) and scale bytes (uint8 [R][ceil(K/128)]) of x, by the rule of
    the header: NaN and infinities are NaN, the scale is that of the finite values."""
    R, K = x.shape
    nb = up(K, 128) // 128
    b = torch.nn.functional.pad(x.float(), (0, nb * 128 - K)).view(R, nb, 128)
    fin = torch.isfinite(b)
    amax = torch.where(fin, b.abs(), torch.zeros_like(b)).amax(2)
    m, k = torch.frexp(amax)
    e = torch.where(m <= 0.875, k - 9, k - 8).clamp(min=-127)
    e = torch.where(amax > 0, e, torch.zeros_like(e))
    v = torch.ldexp(b.double(), -e[:, :, None].double()).float()
    v = torch.where(fin, v, torch.full_like(v, float("nan")))
    return v.to(F8).view(torch.uint8).reshape(R, nb * 128)[:, :K], (e + 127).to(torch.uint8)


def tiles_of(bytes_, K, fill=0):
    R, nb = bytes_.shape
    t, g = up(R, 128) // 128, up(K, 512) // 512
    full = torch.full((t * 128, g * 4), fill, dtype=torch.uint8, device=bytes_.device)
    full[:R, :nb] = bytes_
    return full.view(t, 4, 32, g, 4).permute(3, 0, 2, 1, 4).contiguous()


def bytes_of(tiles, R, K):
    t, g, nb = up(R, 128) // 128, up(K, 512) // 512, up(K, 128) // 128
    return tiles.view(g, t, 32, 4, 4).permute(1, 3, 2, 0, 4).reshape(t * 128, g * 4)[:R, :nb]


def values(codes, bytes_, K):
    c = codes[:, :K].contiguous().view(F8).double()
    s = torch.exp2(bytes_.double() - 127).repeat_interleave(128, 1)[:, :K]
    return c * s


def gpu_quant(lib, x, fill=0xAA):
    R, K = x.shape
    q = torch.full((R, up(K, 16)), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((lib.da3b_fp8_scale_bytes(R, K),), fill, dtype=torch.uint8, device="cuda")
    assert lib.da3b_quantize_fp8(x.data_ptr(), DT.index(x.dtype), R, K, x.stride(0), q.data_ptr(), q.stride(0),
                                 s.data_ptr(), st()) == 0
    return q, s


def spread_rows(R, K, dtype, seed):
    """Rows and blocks over many magnitudes, zeros, blocks of zeros and border values."""
    g = gen(seed)
    x = torch.randn(R, K, device="cuda", generator=g)
    lim = 14 if dtype == torch.float16 else 100
    x = x * torch.exp2(torch.randint(-lim, lim - 2, (R, 1), device="cuda", generator=g).float())
    x = x * torch.exp2(torch.randint(-4, 1, (1, K), device="cuda", generator=g).float())
    x[0, : min(K, 128)] = 0.0
    if R > 1:
        x[1] = 448.0 / 1024
    if R > 2:
        x[2] = 449.0 if dtype != torch.bfloat16 else 450.0
    if R > 3:
        x[3, ::3] = 0.0
    return x.clamp(-6e4, 6e4).to(dtype) if dtype == torch.float16 else x.to(dtype)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("R,K", [(1, 1), (1, 128), (3, 129), (130, 512), (257, 1000), (64, 4096), (5, 2064), (1370, 1024)])
def test_quantize_bit_exact(lib, dtype, R, K):
    x = spread_rows(R, K, dtype, R + K)
    q, s = gpu_quant(lib, x)
    codes, b = plain_quant(x)
    assert torch.equal(q[:, :K], codes)
    assert (q[:, K:] == 0).all()
    assert torch.equal(bytes_of(s, R, K), b)


@pytest.mark.parametrize("dtype", DT)
def test_quantize_strided_and_unaligned(lib, dtype):
    R, K = 70, 300
    buf = spread_rows(R, 1021, dtype, 3)
    x = buf[:, 5:5 + K]
    q, s = gpu_quant(lib, x)
    codes, b = plain_quant(x)
    assert torch.equal(q[:, :K], codes) and torch.equal(bytes_of(s, R, K), b)


def test_quantize_nonfinite_and_extremes(lib):
    x = torch.randn(6, 256, device="cuda", generator=gen(4))
    x[0, 3], x[1, 200], x[2, 5] = float("inf"), float("-inf"), float("nan")
    x[3, :128] = float("nan")
    x[4] = 3.4028234e38
    x[5] = 1e-45                                   # subnormal f32
    x[5, 7] = -3e-39
    q, s = gpu_quant(lib, x)
    codes, b = plain_quant(x)
    nan = (codes & 0x7F) == 0x7F
    assert torch.equal((q & 0x7F) == 0x7F, nan)
    assert torch.equal(q[~nan], codes[~nan]) and torch.equal(bytes_of(s, 6, 256), b)


@pytest.mark.parametrize("R,K,beta", [(1, 1, True), (1, 17, True), (9, 384, False), (300, 768, True), (33, 1024, True),
                                      (5, 1500, True), (129, 2048, False), (3, 2500, True), (17, 5000, True),
                                      (2, 16384, True)])
def test_layernorm(lib, R, K, beta):
    g = gen(R + K)
    x = torch.randn(R, K, device="cuda", generator=g) * 3 + 5
    gm = 1 + 0.2 * torch.randn(K, device="cuda", generator=g)
    bt = 0.1 * torch.randn(K, device="cuda", generator=g) if beta else None
    q = torch.empty(R, up(K, 16), dtype=torch.uint8, device="cuda")
    s = torch.empty(lib.da3b_fp8_scale_bytes(R, K), dtype=torch.uint8, device="cuda")
    assert lib.da3b_layernorm_fp8(x.data_ptr(), R, K, K, gm.data_ptr(), bt.data_ptr() if beta else None, 1e-6,
                                  q.data_ptr(), up(K, 16), s.data_ptr(), st()) == 0
    xd = x.double()
    d = xd - xd.mean(1, keepdim=True)
    y = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-6) * gm.double()
    if beta:
        y = y + bt.double()
    check_quantised(q, bytes_of(s, R, K), y, 3e-6 * y.abs() + 3e-6 * 10, K)


@pytest.mark.parametrize("R,K,pad,beta", [(5001, 1024, 0, True), (4000, 528, 8, False), (9001, 384, 16, True), (7003, 16, 0, True)])
def test_layernorm_many_rows(lib, R, K, pad, beta):
    """More rows than the device holds warps: each row as if it were normalised alone."""
    g = gen(R + K)
    x = torch.randn(R, K + pad, device="cuda", generator=g)[:, :K] * torch.rand(R, 1, device="cuda", generator=g) + 0.5
    x = torch.nn.functional.pad(x, (0, pad), value=float("nan"))
    gm = 1 + 0.2 * torch.randn(K, device="cuda", generator=g)
    bt = 0.1 * torch.randn(K, device="cuda", generator=g)

    def run(first, n):
        q = torch.empty(n, K, dtype=torch.uint8, device="cuda")
        s = torch.empty(lib.da3b_fp8_scale_bytes(n, K), dtype=torch.uint8, device="cuda")
        assert lib.da3b_layernorm_fp8(x[first].data_ptr(), n, K, K + pad, gm.data_ptr(), bt.data_ptr() if beta else None,
                                      1e-6, q.data_ptr(), K, s.data_ptr(), st()) == 0
        return q, bytes_of(s, n, K)

    q, b = run(0, R)
    xd = x[:, :K].double()
    d = xd - xd.mean(1, keepdim=True)
    y = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-6) * gm.double()
    if beta:
        y = y + bt.double()
    # the mean is off by 2^-23 of the largest |x|, divided by the row's spread
    err = 3e-6 * y.abs() + 3e-5 + 2.0 ** -22 * xd.abs().amax(1, keepdim=True) / d.pow(2).mean(1, keepdim=True).add(1e-6).sqrt() * gm.double().abs()
    check_quantised(q, b, y, err, K)
    for first, n in ((0, 128), (R // 2, 77), (R - 1, 1)):
        q1, b1 = run(first, n)
        assert torch.equal(q1, q[first:first + n]) and torch.equal(b1, b[first:first + n])


def check_quantised(q, b, y, err, N):
    """Codes and scale bytes against y (64 bits) known to within err: the scale belongs to a
    block maximum inside the error, and each value is off by at most half a step."""
    R = y.shape[0]
    nb = b.shape[1]
    pad = nb * 128 - N
    top = torch.nn.functional.pad(y.abs(), (0, pad)).view(R, nb, 128).amax(2)
    slack = torch.nn.functional.pad(err, (0, pad)).view(R, nb, 128).amax(2)
    e = b.double() - 127
    empty = top - slack <= 0
    assert ((top - slack <= 448 * torch.exp2(e)) | empty).all()
    assert ((top + slack > 448 * torch.exp2(e - 1)) | empty | (b == 0)).all()
    got = values(q, b, N)
    sc = torch.exp2(e).repeat_interleave(128, 1)[:, :N]
    lim = 2.0 ** -4 * (y.abs() + err) + 2.0 ** -10 * sc + err
    assert ((got - y).abs() <= lim).all(), float(((got - y).abs() - lim).max())


def make_linear(lib, M, K, N, seed, pad=0):
    g = gen(seed)
    x = torch.randn(M, K, device="cuda", generator=g) * torch.exp2(torch.randint(-3, 4, (M, 1), device="cuda", generator=g).float())
    w = torch.randn(N, K, device="cuda", generator=g) / math.sqrt(K)
    w[:, ::7] *= 8
    out = []
    for t in (x, w):
        c, b = plain_quant(t)
        ld = up(K, 16) + pad
        q = torch.full((t.shape[0], ld), 0x7F, dtype=torch.uint8, device="cuda")   # NaN codes past K
        q[:, :K] = c
        out += [q, tiles_of(b, K, fill=255), values(c, b, K)]
    bias = torch.randn(N, device="cuda", generator=g)
    return out, bias


def act64(y, act):
    if act == 1:
        return torch.relu(y)
    return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5))) if act else y


def reference(xv, wv, bias, act, K):
    y = xv @ wv.t()
    S = xv.abs() @ wv.abs().t()
    err = (K + 8) * 2.0 ** -23 * S
    if bias is not None:
        y = y + bias.double()
        err = err + 2.0 ** -23 * (y.abs() + bias.double().abs())
    z = act64(y, act)
    # |GELU'| <= 1.13; erf within 3e-7
    return z, 1.13 * err + (2e-7 * y.abs() + 2.0 ** -22 * y.abs() if act >= 2 else 0)


SHAPES = [(1, 1, 1), (1, 1024, 256), (3, 100, 5), (17, 128, 16), (128, 512, 128), (129, 640, 130), (300, 384, 1152),
          (64, 4096, 1024), (1370, 768, 200), (333, 1000, 771), (2500, 256, 260), (6, 16, 1000), (1, 4097, 33),
          (16, 1536, 384), (33, 2048, 1024), (5000, 128, 384)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_f32(lib, M, K, N):
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, M + K + N)
    y = torch.full((M + 1, N), 7.0, device="cuda")
    assert lib.da3b_linear_fp8(xq.data_ptr(), M, K, xq.stride(0), xs.data_ptr(), wq.data_ptr(), N, wq.stride(0),
                               ws.data_ptr(), bias.data_ptr(), 0, y.data_ptr(), 2, N, st()) == 0
    ref, err = reference(xv, wv, bias, 0, K)
    bad = (y[:M].double() - ref).abs() - err - 2.0 ** -24 * ref.abs()
    assert (bad <= 0).all(), float(bad.max())
    assert (y[M:] == 7.0).all()
    assert lib.da3b_device_status() == 0


@pytest.mark.parametrize("M,K,N", SHAPES[::2])
@pytest.mark.parametrize("dt,act,with_bias", [(0, 0, False), (0, 2, True), (1, 1, True), (1, 3, True), (2, 2, True)])
def test_linear_types_and_activations(lib, M, K, N, dt, act, with_bias):
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, M + K + N + act, pad=32)
    ldo = N + 3
    y = torch.full((M, ldo), 7.0, dtype=DT[dt], device="cuda")
    b = bias if with_bias else None
    assert lib.da3b_linear_fp8(xq.data_ptr(), M, K, xq.stride(0), xs.data_ptr(), wq.data_ptr(), N, wq.stride(0),
                               ws.data_ptr(), b.data_ptr() if with_bias else None, act, y.data_ptr(), dt, ldo, st()) == 0
    ref, err = reference(xv, wv, b, act, K)
    tiny = 2.0 ** -25 if dt == 0 else 0.0          # f16 subnormals
    bad = (y[:, :N].double() - ref).abs() - (1 + 2 * HALF_STEP[dt]) * err - HALF_STEP[dt] * ref.abs() - tiny
    assert (bad <= 0).all(), float(bad.max())
    assert (y[:, N:] == 7.0).all()


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("with_scale", [False, True])
def test_linear_resid(lib, M, K, N, with_scale):
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, M + K + N + 9)
    g = gen(M)
    r0 = torch.randn(M, N + 4, device="cuda", generator=g)
    sc = torch.randn(N, device="cuda", generator=g) if with_scale else None
    r = r0.clone()
    assert lib.da3b_linear_fp8_resid_f32(xq.data_ptr(), M, K, xq.stride(0), xs.data_ptr(), wq.data_ptr(), N,
                                         wq.stride(0), ws.data_ptr(), bias.data_ptr(),
                                         sc.data_ptr() if with_scale else None, r.data_ptr(), N + 4, st()) == 0
    y, err = reference(xv, wv, bias, 0, K)
    if with_scale:
        y, err = y * sc.double(), (err + 2.0 ** -24 * y.abs()) * sc.double().abs()
    ref = r0[:, :N].double() + y
    bad = (r[:, :N].double() - ref).abs() - err - 2.0 ** -23 * (ref.abs() + y.abs())
    assert (bad <= 0).all(), float(bad.max())
    assert torch.equal(r[:, N:], r0[:, N:])


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("act", [0, 2])
def test_linear_quantised_output(lib, M, K, N, act):
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, M + K + N + 5)
    ldo = up(N, 16) + 16
    q = torch.full((M, ldo), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((lib.da3b_fp8_scale_bytes(M, N),), 0xAA, dtype=torch.uint8, device="cuda")
    assert lib.da3b_linear_fp8_q(xq.data_ptr(), M, K, xq.stride(0), xs.data_ptr(), wq.data_ptr(), N, wq.stride(0),
                                 ws.data_ptr(), bias.data_ptr(), act, q.data_ptr(), ldo, s.data_ptr(), st()) == 0
    ref, err = reference(xv, wv, bias, act, K)
    check_quantised(q, bytes_of(s, M, N), ref, err, N)
    assert (q[:, N:] == 0x55).all()


def test_host_outputs_are_refused(lib):
    """An output in pageable host memory is refused before anything is launched."""
    M, K, N = 4, 128, 32
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, 1)
    x = torch.randn(M, K, device="cuda")
    host = torch.zeros(4096, dtype=torch.uint8)
    h = (host.data_ptr() + 63) // 64 * 64
    args = (xq.data_ptr(), M, K, xq.stride(0), xs.data_ptr(), wq.data_ptr(), N, wq.stride(0), ws.data_ptr(), None)
    assert lib.da3b_quantize_fp8(x.data_ptr(), 2, M, K, K, h, K, xs.data_ptr(), st()) == -104
    assert lib.da3b_quantize_fp8(x.data_ptr(), 2, M, K, K, xq.data_ptr(), K, h, st()) == -104
    assert lib.da3b_layernorm_fp8(x.data_ptr(), M, K, K, bias.data_ptr(), None, 1e-6, h, K, xs.data_ptr(), st()) == -104
    assert lib.da3b_linear_fp8(*args, 0, h, 0, N, st()) == -104
    assert lib.da3b_linear_fp8_q(*args, 0, xq.data_ptr(), N, h, st()) == -104
    assert lib.da3b_linear_fp8_resid_f32(*args, None, h, N, st()) == -104
    assert (host == 0).all()


def test_host_inputs_are_refused(lib):
    """So is an input there, the optional ones among them."""
    M, K, N = 4, 128, 32
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, 1)
    x, y = torch.randn(M, K, device="cuda"), torch.full((M, N), 7.0, device="cuda")
    host = torch.zeros(1 << 16, dtype=torch.uint8)
    h = (host.data_ptr() + 63) // 64 * 64
    q, s = xq.data_ptr(), xs.data_ptr()
    assert lib.da3b_quantize_fp8(h, 2, M, K, K, q, K, s, st()) == -104
    ln = [x.data_ptr(), M, K, K, bias.data_ptr(), bias.data_ptr(), 1e-6, q, K, s, st()]
    for i in (0, 4, 5):
        assert lib.da3b_layernorm_fp8(*ln[:i], h, *ln[i + 1:]) == -104
    lin = [q, M, K, xq.stride(0), s, wq.data_ptr(), N, wq.stride(0), ws.data_ptr(), bias.data_ptr()]
    for i in (0, 4, 5, 8, 9):
        a = lin[:i] + [h] + lin[i + 1:]
        assert lib.da3b_linear_fp8(*a, 0, y.data_ptr(), 2, N, st()) == -104
        assert lib.da3b_linear_fp8_resid_f32(*a, None, y.data_ptr(), N, st()) == -104
    assert lib.da3b_linear_fp8_resid_f32(*lin, h, y.data_ptr(), N, st()) == -104
    assert (y == 7.0).all()


def test_linear_into_pinned_memory(lib):
    M, K, N = 40, 256, 96
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, 1)
    y = torch.zeros(M, N).pin_memory()
    d = torch.zeros(M, N, device="cuda")
    for o in (y, d):
        assert lib.da3b_linear_fp8(xq.data_ptr(), M, K, xq.stride(0), xs.data_ptr(), wq.data_ptr(), N, wq.stride(0),
                                   ws.data_ptr(), bias.data_ptr(), 0, o.data_ptr(), 2, N, st()) == 0
    torch.cuda.synchronize()
    assert torch.equal(y, d.cpu())


def test_quantised_output_with_infinities(lib):
    """A product that overflows (a scale of 2^120 against one of 2^20) gives infinities and NaN:
    NaN codes, and the scale of the block's finite values; other rows are as ever."""
    M, K, N = 150, 256, 300
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, 6)
    b, wb = bytes_of(xs, M, K).clone(), bytes_of(ws, N, K).clone()
    b[9], wb[200:] = 247, 160
    xs2, ws2 = tiles_of(b, K), tiles_of(wb, K)
    q = torch.empty(M, up(N, 16), dtype=torch.uint8, device="cuda")
    s = torch.empty(lib.da3b_fp8_scale_bytes(M, N), dtype=torch.uint8, device="cuda")
    y = torch.empty(M, N, device="cuda")
    args = (xq.data_ptr(), M, K, xq.stride(0), xs2.data_ptr(), wq.data_ptr(), N, wq.stride(0), ws2.data_ptr(), bias.data_ptr(), 0)
    assert lib.da3b_linear_fp8_q(*args, q.data_ptr(), up(N, 16), s.data_ptr(), st()) == 0
    assert lib.da3b_linear_fp8(*args, y.data_ptr(), 2, N, st()) == 0
    assert not torch.isfinite(y[9, 200:]).all() and torch.isfinite(y[:9]).all()
    codes, want = plain_quant(y)
    nan = (codes & 0x7F) == 0x7F
    assert nan.any() and torch.equal((q[:, :N] & 0x7F) == 0x7F, nan)
    assert torch.equal(q[:, :N][~nan], codes[~nan]) and torch.equal(bytes_of(s, M, N), want)


def test_linear_nan_stays_in_its_row(lib):
    """A NaN activation makes its row NaN and no other; rows past M and columns past K hold
    NaN codes and NaN scales already (make_linear)."""
    M, K, N = 150, 300, 140
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, 1)
    xq[7, 299] = 0x7F
    for act in (0, 1, 2):
        y = torch.zeros(M, N, device="cuda")
        assert lib.da3b_linear_fp8(xq.data_ptr(), M, K, xq.stride(0), xs.data_ptr(), wq.data_ptr(), N, wq.stride(0),
                                   ws.data_ptr(), bias.data_ptr(), act, y.data_ptr(), 2, N, st()) == 0
        nan = torch.isnan(y)
        assert nan[7].all() and not nan[:7].any() and not nan[8:].any()


def test_linear_is_deterministic_and_row_independent(lib):
    """The same call twice gives the same bits, on any stream and from a replayed graph."""
    M, K, N = 70, 4096, 300
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, 2)

    def call(y):
        assert lib.da3b_linear_fp8(xq.data_ptr(), M, K, xq.stride(0), xs.data_ptr(), wq.data_ptr(), N, wq.stride(0),
                                   ws.data_ptr(), bias.data_ptr(), 2, y.data_ptr(), 2, N, st()) == 0

    a, b, c = (torch.zeros(M, N, device="cuda") for _ in range(3))
    call(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            call(b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(c)
    for _ in range(2):
        c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, c)
    assert torch.equal(a, b)


def test_mlp_chain(lib):
    """LayerNorm -> fc1 with GELU and a quantised output -> fc2 onto the residual stream,
    captured as one graph, against 64 bits with the same roundings: values next to a border
    of e4m3 may fall either way, which moves an output by at most a step of one term; the
    2-norm of the difference is held to 1e-3 of the result's (a hundred times what sums in
    f32 would leave if one value in a thousand fell the other way: 2^-3 * sqrt(1e-3) of a
    term, averaged over the 1536 terms of an output)."""
    M, D, H = 300, 384, 1536
    g = gen(11)
    x = torch.randn(M, D, device="cuda", generator=g) * 2
    gm, bt = 1 + 0.1 * torch.randn(D, device="cuda", generator=g), 0.1 * torch.randn(D, device="cuda", generator=g)
    ls = 0.1 * (1 + 0.1 * torch.randn(D, device="cuda", generator=g))
    w1, w2 = torch.randn(H, D, device="cuda", generator=g) / 20, torch.randn(D, H, device="cuda", generator=g) / 40
    b1, b2 = torch.randn(H, device="cuda", generator=g) * 0.1, torch.randn(D, device="cuda", generator=g) * 0.1
    q1, s1 = gpu_quant(lib, w1)
    q2, s2 = gpu_quant(lib, w2)
    xq, hq = torch.empty(M, D, dtype=torch.uint8, device="cuda"), torch.empty(M, H, dtype=torch.uint8, device="cuda")
    xs = torch.empty(lib.da3b_fp8_scale_bytes(M, D), dtype=torch.uint8, device="cuda")
    hs = torch.empty(lib.da3b_fp8_scale_bytes(M, H), dtype=torch.uint8, device="cuda")
    r = x.clone()

    def chain():
        assert lib.da3b_layernorm_fp8(r.data_ptr(), M, D, D, gm.data_ptr(), bt.data_ptr(), 1e-6, xq.data_ptr(), D,
                                      xs.data_ptr(), st()) == 0
        assert lib.da3b_linear_fp8_q(xq.data_ptr(), M, D, D, xs.data_ptr(), q1.data_ptr(), H, D, s1.data_ptr(),
                                     b1.data_ptr(), 2, hq.data_ptr(), H, hs.data_ptr(), st()) == 0
        assert lib.da3b_linear_fp8_resid_f32(hq.data_ptr(), M, H, H, hs.data_ptr(), q2.data_ptr(), D, H, s2.data_ptr(),
                                             b2.data_ptr(), ls.data_ptr(), r.data_ptr(), D, st()) == 0

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    r.copy_(x)
    graph.replay()
    torch.cuda.synchronize()

    xd = x.double()
    d = xd - xd.mean(1, keepdim=True)
    n = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-6) * gm.double() + bt.double()
    nv = values(*plain_quant(n.float()), D)
    h = act64(nv @ values(q1, bytes_of(s1, H, D), D).t() + b1.double(), 2)
    hv = values(*plain_quant(h.float()), H)
    y = ls.double() * (hv @ values(q2, bytes_of(s2, D, H), H).t() + b2.double())
    assert ((r.double() - xd) - y).norm() <= 1e-3 * y.norm()


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.mem_get_info()[0] < 30 << 30, reason="needs 30 GB")
def test_linear_offsets_past_32_bits(lib):
    """Rows whose byte offsets pass 2^32, codes and outputs both."""
    M, K, N = 1_100_000, 4096, 16
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, 128, K, N, 3)
    big = xq.repeat(M // 128 + 1, 1)[:M]
    g, nb = up(K, 512) // 512, up(M, 128) // 128
    tiles = xs.view(g, 1, 512).expand(g, nb, 512).contiguous()
    ldo = 2100
    y = torch.empty(M, ldo, dtype=torch.float16, device="cuda")
    assert lib.da3b_linear_fp8(big.data_ptr(), M, K, K, tiles.data_ptr(), wq.data_ptr(), N, wq.stride(0), ws.data_ptr(),
                               bias.data_ptr(), 0, y.data_ptr(), 0, ldo, st()) == 0
    first = y[:128, :N].clone()
    ref, err = reference(xv, wv, bias, 0, K)
    assert ((first.double() - ref).abs() <= err + 2.0 ** -11 * (ref.abs() + err) + 2.0 ** -25).all()
    assert torch.equal(y[M // 128 * 128 - 128: M // 128 * 128, :N], first)
    assert torch.equal(y[M // 128 * 128:, :N], first[: M % 128])
