"""Windowed attention launched while the device's status word records a wait that ran out:
every wait then gives up early, so a call may stop anywhere. What it stores is right all the
same: a row is either left as it was or holds the result, never a sum of shares that some CTA
did not finish. The word keeps its code until it is read, and calls are as ever after that."""
import pytest

torch = pytest.importorskip("torch")

from test_attention_window_gpu import call, make, st

pytestmark = pytest.mark.gpu

TIMEOUT_FULL = 1  # the probe's code


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


def whole_rows_or_none(lib, B, Tq, Tk, h, kvh, D, left, right, sinks):
    q, k, v = make(B, Tq, Tk, h, kvh, D, torch.float16, Tk + D)
    want = torch.full_like(q, 7.0)
    call(lib, q, k, v, want, left, right, sinks)
    assert lib.da3b_device_status() == 0
    for _ in range(5):
        o = torch.full_like(q, 7.0)
        assert lib.da3b_debug_wait_timeout(1_000_000, 0, None, None, st()) == 0
        call(lib, q, k, v, o, left, right, sinks)
        assert lib.da3b_device_status() == TIMEOUT_FULL
        right_row = (o == want).all(-1)
        untouched = (o == 7.0).all(-1)
        assert (right_row | untouched).all()
    o = torch.full_like(q, 7.0)
    call(lib, q, k, v, o, left, right, sinks)
    assert lib.da3b_device_status() == 0
    assert torch.equal(o, want)


@pytest.mark.parametrize("B,Tq,Tk,h,kvh,D,left,right,sinks", [
    (1, 300, 6000, 4, 2, 64, -1, -1, 0),
    (1, 300, 6000, 4, 2, 128, -1, -1, 0),
    (1, 256, 3392, 6, 2, 128, 2878, 17, 300),
])
def test_split_items(lib, B, Tq, Tk, h, kvh, D, left, right, sinks):
    whole_rows_or_none(lib, B, Tq, Tk, h, kvh, D, left, right, sinks)


@pytest.mark.parametrize("B,Tq,Tk,h,kvh,D", [(1, 1, 20000, 4, 4, 64), (2, 2, 20000, 8, 2, 128)])
def test_few_queries(lib, B, Tq, Tk, h, kvh, D):
    whole_rows_or_none(lib, B, Tq, Tk, h, kvh, D, -1, 0, 3)
