"""Windowed attention at the smallest scales: 0 is a plain mean of what a query sees, and a
scale below 1e-30 is that scale, also where the scores are far above its inverse's order."""
import pytest

torch = pytest.importorskip("torch")

from test_attention_window_gpu import call, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,Tk,left,sinks", [(1, 300, -1, 0), (4, 300, 99, 2), (260, 260, -1, 0), (260, 700, 99, 2)])
@pytest.mark.parametrize("scale,power", [(0.0, 57), (1e-36, 57), (1e-33, 52), (0.0, 0)])
def test_large_scores_times_small_scales(lib, D, Tq, Tk, left, sinks, scale, power):
    """bf16 queries and keys of the order 2^power: scores of the order 2^(2 power + 3)."""
    q, k, v = make(1, Tq, Tk, 2, 1, D, torch.bfloat16, Tk + D)
    q, k = q * 2.0 ** power, k * 2.0 ** power
    o = torch.full_like(q, float("nan"))
    call(lib, q, k, v, o, left, 0, sinks, scale=scale)
    check(q, k, v, o, left, 0, sinks, scale=scale)
    assert lib.da3b_device_status() == 0
