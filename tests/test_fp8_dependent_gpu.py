"""The e4m3 producers and linears start while the kernel ahead of them in the stream may
still be running: whatever that kernel writes, inputs and parameters alike, is what they
read. Everything is rewritten by the launch just before each call, over and over, with no
wait of the host in between, and each call's result is kept and compared at the end."""
import pytest

torch = pytest.importorskip("torch")

from test_fp8_gpu import DT, bytes_of, check_quantised, gen, make_linear, plain_quant, reference, st, up

pytestmark = pytest.mark.gpu

ROUNDS = 12


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("R,K", [(1, 256), (300, 1000), (5000, 1024)])
def test_quantiser_reads_what_the_kernel_ahead_wrote(lib, dtype, R, K):
    g = gen(R + K)
    new = [(torch.randn(R, K, device="cuda", generator=g) * 2.0 ** i).to(dtype) for i in range(ROUNDS)]
    x = torch.zeros(R, K, dtype=dtype, device="cuda")
    q = torch.zeros(ROUNDS, R, up(K, 16), dtype=torch.uint8, device="cuda")
    s = torch.zeros(ROUNDS, lib.da3b_fp8_scale_bytes(R, K), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for i in range(ROUNDS):
        x.copy_(new[i])
        assert lib.da3b_quantize_fp8(x.data_ptr(), DT.index(dtype), R, K, K, q[i].data_ptr(), up(K, 16), s[i].data_ptr(),
                                     st()) == 0
    for i in range(ROUNDS):
        codes, b = plain_quant(new[i])
        assert torch.equal(q[i, :, :K], codes) and torch.equal(bytes_of(s[i], R, K), b)


@pytest.mark.parametrize("R,K", [(1, 256), (300, 1000), (5000, 1024), (2000, 768), (700, 1536), (40, 5008)])
def test_layernorm_reads_what_the_kernels_ahead_wrote(lib, R, K):
    g = gen(R + K)
    new = [torch.randn(R + 2, K, device="cuda", generator=g) * (i + 1) for i in range(ROUNDS)]
    buf = torch.zeros(R + 2, K, device="cuda")           # rows, then gamma and beta
    q = torch.zeros(ROUNDS, R, up(K, 16), dtype=torch.uint8, device="cuda")
    s = torch.zeros(ROUNDS, lib.da3b_fp8_scale_bytes(R, K), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for i in range(ROUNDS):
        buf.copy_(new[i])
        assert lib.da3b_layernorm_fp8(buf.data_ptr(), R, K, K, buf[R].data_ptr(), buf[R + 1].data_ptr(), 1e-6,
                                      q[i].data_ptr(), up(K, 16), s[i].data_ptr(), st()) == 0
    for i in range(ROUNDS):
        x, gm, bt = new[i][:R].double(), new[i][R].double(), new[i][R + 1].double()
        d = x - x.mean(1, keepdim=True)
        n = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-6)
        y = n * gm + bt
        # n is off by 3e-6 of itself and, through the mean, by 3e-6; products and sum round once each
        check_quantised(q[i], bytes_of(s[i], R, K), y, 3e-6 * (n.abs() + 1) * gm.abs() + 2.0 ** -22 * (y.abs() + bt.abs()), K)


@pytest.mark.parametrize("M,K,N", [(1, 256, 128), (130, 512, 300), (1370, 256, 512)])
def test_linear_reads_what_the_kernels_ahead_wrote(lib, M, K, N):
    """Rows quantised by the launch ahead, bias and scale written by the one before that."""
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, M + K + N)
    g = gen(M)
    rows = [(torch.randn(M, K, device="cuda", generator=g) * (i + 1)).half() for i in range(ROUNDS)]
    par = [torch.randn(2, N, device="cuda", generator=g) for _ in range(ROUNDS)]
    x, p = torch.zeros_like(rows[0]), torch.zeros(2, N, device="cuda")
    q, s = torch.zeros(M, K, dtype=torch.uint8, device="cuda"), torch.zeros_like(xs)
    y = torch.zeros(ROUNDS, M, N, device="cuda")
    torch.cuda.synchronize()
    for i in range(ROUNDS):
        x.copy_(rows[i])
        p.copy_(par[i])
        assert lib.da3b_quantize_fp8(x.data_ptr(), 0, M, K, K, q.data_ptr(), K, s.data_ptr(), st()) == 0
        assert lib.da3b_linear_fp8_resid_f32(q.data_ptr(), M, K, K, s.data_ptr(), wq.data_ptr(), N, wq.stride(0),
                                             ws.data_ptr(), p[0].data_ptr(), p[1].data_ptr(), y[i].data_ptr(), N, st()) == 0
    for i in range(ROUNDS):
        c, b = plain_quant(rows[i])
        v = c.view(torch.float8_e4m3fn).double() * torch.exp2(b.double() - 127).repeat_interleave(128, 1)[:, :K]
        ref, err = reference(v, wv, par[i][0], 0, K)
        sc = par[i][1].double()
        lim = (err + 2.0 ** -24 * ref.abs()) * sc.abs() + 2.0 ** -23 * 2 * (ref * sc).abs()
        assert ((y[i].double() - ref * sc).abs() <= lim).all()
    assert lib.da3b_device_status() == 0
