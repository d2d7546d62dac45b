"""How exact the e4m3 linear's sums are, as a whole: the bounds of test_fp8_gpu hold each
element to the worst case of its own terms, which at long reductions would let sums in far
fewer bits pass. Here the 2-norm of the difference over that of the result is bounded.

The terms are of either sign and independent, so a partial sum's 2-norm over the outputs is
at most the whole sum's. An accumulator in f32 takes K / 32 additions (one for each product
instruction), each off by at most 2^-23 of its partial sum (cut, not rounded), and the 32
products of one addition are aligned with each other, 32 times at most 2^-23 of a block's sum
once more; bias and the output's own rounding add less than 8 of these. So the quotient is at
most (K / 32 + 40) 2^-23: 2.0e-5 at K = 4096, where sums in 16 bits are off by 2^-11 and
sums cut at 14 bits by 2^-14, 6e-5, a step."""
import pytest

torch = pytest.importorskip("torch")

from test_fp8_gpu import make_linear, st

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K,N", [(1, 4096, 1024), (130, 1024, 300), (700, 4096, 512), (1370, 1000, 771), (2500, 2048, 1024)])
def test_two_norm_of_the_sums(lib, M, K, N):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    (xq, xs, xv, wq, ws, wv), bias = make_linear(lib, M, K, N, M + K + N)
    y = torch.empty(M, N, device="cuda")
    assert lib.da3b_linear_fp8(xq.data_ptr(), M, K, xq.stride(0), xs.data_ptr(), wq.data_ptr(), N, wq.stride(0),
                               ws.data_ptr(), None, 0, y.data_ptr(), 2, N, st()) == 0
    ref = xv @ wv.t()
    assert (y.double() - ref).norm() <= (K / 32 + 40) * 2.0 ** -23 * ref.norm()
    assert lib.da3b_device_status() == 0
