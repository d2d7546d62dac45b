"""Windowed attention: a masked key has no weight, not a small one. Values next to the type's
largest, which only the rows that see them may feel, leave the other rows as they are."""
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


@pytest.mark.parametrize("dtype,big", [(torch.float16, 6e4), (torch.bfloat16, 3e38)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq,Tk,left,right,sinks", [(5, 203, -1, 0, 0), (203, 203, -1, 0, 0), (203, 203, 60, 0, 2),
                                                    (120, 900, 70, 9, 3)])
def test_large_values_of_later_keys(lib, D, dtype, big, Tq, Tk, left, right, sinks):
    """The last two keys' values are huge; only the last rows see them. Bit for bit the rows
    before are those of a call without them."""
    q, k, v = make(1, Tq, Tk, 2, 1, D, dtype, Tk + D)
    want, got = torch.zeros_like(q), torch.zeros_like(q)
    call(lib, q, k, v, want, left, right, sinks)
    check(q, k, v, want, left, right, sinks)
    v[:, Tk - 2:] = big
    call(lib, q, k, v, got, left, right, sinks)
    n = Tq - 2 - right
    assert torch.equal(got[:, :n], want[:, :n])
    assert (got[:, n:].float() != want[:, n:].float()).any()


@pytest.mark.parametrize("dtype,big", [(torch.float16, 6e4), (torch.bfloat16, 3e38)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("at", range(96, 104))
def test_large_values_behind_the_window(lib, D, dtype, big, at):
    """A huge value at each place of eight; rows whose window has passed it are as without it."""
    T, left = 203, 20
    q, k, v = make(1, T, T, 2, 1, D, dtype, at + D)
    want, got = torch.zeros_like(q), torch.zeros_like(q)
    call(lib, q, k, v, want, left, 0, 0)
    check(q, k, v, want, left, 0, 0)
    v[:, at] = big
    call(lib, q, k, v, got, left, 0, 0)
    assert torch.equal(got[:, :at], want[:, :at]) and torch.equal(got[:, at + left + 1:], want[:, at + left + 1:])
