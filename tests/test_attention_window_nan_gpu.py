"""Windowed attention: NaN scores make a row NaN wherever they stand among the keys (part of
the exponentials are computed another way than the rest, by the key's place)."""
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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,Tk", [(1, 9), (203, 203), (150, 2000)])
def test_nan_query_that_sees_one_key(lib, D, dtype, Tq, Tk):
    """Every query sees its own key alone, so that each place holds the only score of a row."""
    q, k, v = make(1, Tq, Tk, 2, 2, D, dtype, Tk + D)
    q[:, ::2] = float("nan")
    o = torch.zeros_like(q)
    call(lib, q, k, v, o, 0, 0, 0)
    assert torch.isnan(o[:, ::2]).all()
    assert torch.equal(o[:, 1::2], v[:, Tk - Tq:][:, 1::2])   # a weight of one


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_nan_key_at_every_place_of_eight(lib, D, dtype):
    """The rows that see the NaN key are NaN, whatever else they see; the others hold."""
    T, left = 170, 3
    for at in range(80, 88):
        q, k, v = make(1, T, T, 1, 1, D, dtype, at + D)
        clean = torch.zeros_like(q)
        call(lib, q, k, v, clean, left, 0, 0)
        check(q, k, v, clean, left, 0, 0)
        k[0, at] = float("nan")
        o = torch.zeros_like(q)
        call(lib, q, k, v, o, left, 0, 0)
        assert torch.isnan(o[0, at:at + left + 1]).all()
        o[0, at:at + left + 1] = clean[0, at:at + left + 1]
        assert torch.equal(o, clean)
