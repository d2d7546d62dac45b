"""Windowed attention with the key tiles of an item split over a cluster: shares that hold,
or end on, key tiles that no query sees. Such tiles lie between the sinks and the oldest
window where that gap is shorter than 128 keys. The formula, the tolerances and the calls are
those of test_attention_window_gpu."""
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


def unseen_keys_are_nan(k, v, ql, kl, left, sinks):
    """NaN and infinities in every key that no query of its sequence sees."""
    for b in range(k.shape[0]):
        k[b, kl[b]:], v[b, kl[b]:] = float("nan"), float("inf")
        lo = max(kl[b] - ql[b] - left, 0)
        if lo > sinks:
            k[b, sinks:lo], v[b, sinks:lo] = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,Tq,Tk,h,kvh,left,right,sinks", [
    # a share's last tile is one of the gap that some items have
    (128, 256, 3392, 6, 2, 2878, 17, 300),
    (64, 3209, 3209, 6, 2, 1307, 0, 1369),
    # shares with one or two gap tiles at other places
    (128, 300, 2048, 2, 2, 1500, 0, 140),
    (64, 300, 2048, 2, 2, 1500, 0, 140),
    (64, 129, 1500, 3, 1, 1200, -1, 64),
    (128, 129, 1500, 3, 1, 1200, -1, 64),
])
def test_share_ends_on_a_tile_no_query_sees(lib, D, Tq, Tk, h, kvh, left, right, sinks, dtype):
    q, k, v = make(1, Tq, Tk, h, kvh, D, dtype, Tk + D)
    unseen_keys_are_nan(k, v, [Tq], [Tk], left, sinks)
    for _ in range(20):
        o = torch.full_like(q, 7.0)
        call(lib, q, k, v, o, left, right, sinks)
    check(q, k, v, o, left, right, sinks)
    assert lib.da3b_device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,sinks,kl", [(128, 64, 140), (128, 64, 192), (64, 48, 145), (64, 48, 170), (64, 96, 200)])
def test_share_of_nothing_but_a_tile_no_query_sees(lib, D, sinks, kl, dtype):
    """The split is chosen for the longest sequence; a short one gives a CTA a single tile, and
    that is one of the gap."""
    T, left = 1000, 1
    q, k, v = make(3, T, T, 1, 1, D, dtype, kl + D)
    ql, kls = [T, 1, 2], [T, kl, kl]
    unseen_keys_are_nan(k, v, ql, kls, left, sinks)
    qd, kd = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (ql, kls))
    for _ in range(20):
        o = torch.full_like(q, 7.0)
        call(lib, q, k, v, o, left, -1, sinks, qd, kd)
    check(q, k, v, o, left, -1, sinks, ql, kls, fill=7.0)
    assert lib.da3b_device_status() == 0
