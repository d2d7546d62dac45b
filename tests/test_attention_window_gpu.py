"""Windowed attention with sinks against the formula in 64 bits.

Tolerance of an output element, with A = sum_j p_j |v_j| of its row: the probabilities are
rounded to the 16-bit type before the product with V (half a step: f16 2^-11, bf16 2^-8),
their exponentials are good to 1e-4 (a cubic on part of them), scores are f32 sums (D + 2
roundings of 2^-24 of scale * |q||k|, then the exponent's own rounding, 2^-23 of its size),
f16 probabilities below 2^-14 of the row's reference maximum are off by up to 2^-25, and the
output rounds by half a step."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

I3 = ctypes.c_int64 * 3
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


def st():
    return torch.cuda.current_stream().cuda_stream


def s3(t):
    return I3(t.stride(0), t.stride(1), t.stride(2))


def call(lib, q, k, v, o, left, right, sinks, ql=None, kl=None, scale=None):
    B, Tq, h, D = q.shape
    rc = lib.da3b_attention_window(q.data_ptr(), s3(q), k.data_ptr(), s3(k), v.data_ptr(), s3(v), o.data_ptr(), s3(o),
                                   0 if q.dtype == torch.float16 else 1, B, Tq, k.shape[1], h, k.shape[2], D,
                                   ql.data_ptr() if ql is not None else None, kl.data_ptr() if kl is not None else None,
                                   left, right, sinks, scale if scale is not None else 1 / math.sqrt(D), st())
    assert rc == 0


def sees(ql, kl, left, right, sinks):
    i = torch.arange(ql, device="cuda")[:, None] + (kl - ql)
    j = torch.arange(kl, device="cuda")[None]
    m = torch.ones(ql, kl, dtype=torch.bool, device="cuda")
    if right >= 0:
        m &= j <= i + right
    if left >= 0:
        m &= (j >= i - left) | (j < sinks)
    return m


def check(q, k, v, o, left, right, sinks, ql=None, kl=None, scale=None, fill=None):
    B, Tq, h, D = q.shape
    scale = scale if scale is not None else 1 / math.sqrt(D)
    half = HALF[q.dtype]
    r = h // k.shape[2]
    for b in range(B):
        nq = min(max(int(ql[b]), 0), Tq) if ql is not None else Tq
        nk = min(max(int(kl[b]), 0), k.shape[1]) if kl is not None else k.shape[1]
        if fill is not None:
            assert (o[b, nq:] == fill).all(), "rows past the length were written"
        if nq == 0:
            continue
        m = sees(nq, nk, left, right, sinks)
        for i in range(h):
            qq = q[b, :nq, i].double()
            kk, vv = k[b, :nk, i // r].double(), v[b, :nk, i // r].double()
            dead = ~m.any(0)
            kk, vv = kk.masked_fill(dead[:, None], 0.0), vv.masked_fill(dead[:, None], 0.0)
            s = (qq @ kk.t() * scale).masked_fill(~m, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) if nk else s
            ref = p @ vv
            got = o[b, :nq, i].double()
            none = ~m.any(1)
            assert (got[none] == 0).all(), "a query that sees nothing"
            A = p @ vv.abs()
            mag = qq.norm(dim=1, keepdim=True) * (kk.norm(dim=1).max() if nk else 0.0) * scale
            rel = half + 1e-4 + 2 * ((D + 2) * 2.0 ** -24 * mag + 2.0 ** -23 * mag * 1.45)
            tiny = 2.0 ** -25 * (m.double() @ vv.abs()) if q.dtype == torch.float16 else 0.0
            lim = 1.01 * (rel * (A + ref.abs()) + half * ref.abs()) + tiny + 2.0 ** -25
            bad = (got - ref).abs() - lim
            assert (bad <= 0).all(), (b, i, float(bad.max()), int(bad.argmax()))


def make(B, Tq, Tk, h, kvh, D, dtype, seed, qmul=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(B, Tq, h, D, device="cuda", generator=g) * qmul).to(dtype)
    k = torch.randn(B, Tk, kvh, D, device="cuda", generator=g).to(dtype)
    v = torch.randn(B, Tk, kvh, D, device="cuda", generator=g).to(dtype)
    return q, k, v


CASES = [
    # B, Tq, Tk, heads, kv_heads, left, right, sinks
    (1, 1, 1, 1, 1, 0, 0, 0),
    (2, 1, 1, 3, 3, -1, -1, 5),
    (1, 1, 500, 4, 4, 100, 0, 3),
    (3, 1, 2000, 8, 2, 511, 0, 4),
    (2, 5, 777, 6, 2, 63, 0, 1),
    (1, 16, 16, 2, 2, -1, 0, 0),
    (2, 64, 64, 2, 1, 5, 0, 2),
    (1, 127, 127, 2, 2, -1, -1, 0),
    (1, 129, 129, 1, 1, 0, 0, 0),          # each query sees itself only
    (1, 200, 200, 4, 2, 31, 0, 40),        # sinks reach into the window
    (2, 300, 300, 2, 2, 64, 17, 3),
    (1, 257, 1000, 3, 3, 200, -1, 130),    # a new chunk over a cache
    (1, 700, 700, 2, 1, -1, 0, 0),
    (1, 1000, 300, 2, 2, 50, 0, 4),        # more queries than keys: the first see nothing
    (1, 390, 1500, 2, 2, 128, 128, 1000),  # sinks beyond most of the keys
    (1, 513, 513, 2, 2, 383, 0, 64),
    (4, 130, 640, 4, 1, 255, 0, 0),
    (1, 100, 100, 2, 2, 1 << 30, 1 << 30, 1 << 30),
    (1, 3, 5000, 2, 2, -1, 0, 0),
    (1, 40, 3000, 12, 1, 1000, 0, 7),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("c", CASES)
def test_window(lib, c, D, dtype):
    B, Tq, Tk, h, kvh, left, right, sinks = c
    q, k, v = make(B, Tq, Tk, h, kvh, D, dtype, sum(c[:5]) + D)
    o = torch.full_like(q, float("nan"))
    call(lib, q, k, v, o, left, right, sinks)
    check(q, k, v, o, left, right, sinks)
    assert lib.da3b_device_status() == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Tq", [1, 4, 150, 400])
def test_lengths_and_unseen_keys(lib, D, Tq):
    """Lengths 0, 1, odd, full and out of range; everything that no query sees is NaN or
    infinite: keys from kl on, and the gap between the sinks and the oldest window."""
    dtype = torch.float16
    B, Tk, h, kvh, left, right, sinks = 7, 400, 4, 2, 37, 0, 5
    q, k, v = make(B, Tq, Tk, h, kvh, D, dtype, Tq + D)
    kl = [0, 1, 63, 64, 129, 400, 999]
    ql = [min(Tq, max(1, n)) for n in kl]
    ql[5] = 0
    ql[6] = Tq + 50
    for b in range(B):
        nk, nq = min(kl[b], Tk), min(ql[b], Tq)
        k[b, nk:], v[b, nk:] = float("nan"), float("inf")
        lo = max(nk - nq - left, 0)
        if lo > sinks:
            k[b, sinks:lo], v[b, sinks:lo] = float("inf"), float("nan")
        q[b, nq:] = float("nan")
    o = torch.full_like(q, 7.0)
    qd, kd = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (ql, kl))
    call(lib, q, k, v, o, left, right, sinks, qd, kd)
    check(q, k, v, o, left, right, sinks, ql, kl, fill=7.0)
    assert lib.da3b_device_status() == 0


def test_negative_lengths_are_empty(lib):
    q, k, v = make(2, 70, 70, 2, 2, 64, torch.float16, 5)
    o = torch.full_like(q, 7.0)
    ql = torch.tensor([-3, 70], dtype=torch.int32, device="cuda")
    kl = torch.tensor([70, -9], dtype=torch.int32, device="cuda")
    call(lib, q, k, v, o, -1, 0, 0, ql, kl)
    assert (o[0] == 7.0).all() and (o[1] == 0).all()


def test_host_output_is_refused(lib):
    q, k, v = make(1, 5, 9, 2, 2, 64, torch.float16, 6)
    o = torch.zeros(q.numel() + 64, dtype=torch.float16)
    h = (o.data_ptr() + 63) // 64 * 64
    assert lib.da3b_attention_window(q.data_ptr(), s3(q), k.data_ptr(), s3(k), v.data_ptr(), s3(v), h, s3(q), 0, 1, 5, 9,
                                     2, 2, 64, None, None, 3, 0, 1, 0.125, st()) == -104
    assert (o == 0).all()


def test_host_inputs_are_refused(lib):
    """Lengths in host memory, the likeliest of these mistakes, among them."""
    q, k, v = make(1, 5, 9, 2, 2, 64, torch.float16, 6)
    o = torch.full_like(q, 7.0)
    host = torch.zeros(1 << 14, dtype=torch.uint8)
    h = (host.data_ptr() + 63) // 64 * 64
    n = torch.tensor([5], dtype=torch.int32)
    a = [q.data_ptr(), s3(q), k.data_ptr(), s3(k), v.data_ptr(), s3(v), o.data_ptr(), s3(q), 0, 1, 5, 9, 2, 2, 64, None, None,
         3, 0, 1, 0.125, st()]
    for i, p in ((0, h), (2, h), (4, h), (15, n.data_ptr()), (16, n.data_ptr())):
        assert lib.da3b_attention_window(*a[:i], p, *a[i + 1:]) == -104
    assert lib.da3b_attention_window(*a) == 0 and (o != 7.0).any()


def test_no_keys_at_all(lib):
    q, k, v = make(2, 33, 1, 2, 2, 64, torch.float16, 6)
    o = torch.full_like(q, 7.0)
    B, Tq, h, D = q.shape
    assert lib.da3b_attention_window(q.data_ptr(), s3(q), k.data_ptr(), s3(k), v.data_ptr(), s3(v), o.data_ptr(), s3(o),
                                     0, B, Tq, 0, h, 2, D, None, None, 3, 0, 1, 0.125, st()) == 0
    assert (o == 0).all()


@pytest.mark.parametrize("Tq", [1, 300])
@pytest.mark.parametrize("layout", ["packed", "heads_first", "padded"])
def test_strides(lib, layout, Tq):
    B, Tk, h, D, dtype = 2, 300, 4, 64, torch.float16
    g = torch.Generator(device="cuda").manual_seed(8)
    if layout == "packed":
        x = torch.randn(B, Tk, 3, h, D, device="cuda", generator=g).half()
        q, k, v = x[:, Tk - Tq:, 0], x[:, :, 1], x[:, :, 2]
        buf = torch.full((B, Tq, h, D), 7.0, dtype=dtype, device="cuda")
        o = buf
    elif layout == "heads_first":
        q, k, v = (torch.randn(B, h, t, D, device="cuda", generator=g).half().transpose(1, 2) for t in (Tq, Tk, Tk))
        buf = torch.full((B, h, Tq, D), 7.0, dtype=dtype, device="cuda")
        o = buf.transpose(1, 2)
    else:
        q, k, v = (torch.randn(B, t + 3, h + 2, D + 8, device="cuda", generator=g).half()[:, :t, 1:h + 1, :D]
                   for t in (Tq, Tk, Tk))
        buf = torch.full((B, Tq + 5, h + 1, D + 16), 7.0, dtype=dtype, device="cuda")
        o = buf[:, :Tq, :h, :D]
    call(lib, q, k, v, o, 99, 0, 2)
    check(q, k, v, o, 99, 0, 2)
    if layout == "padded":
        assert (buf[:, Tq:] == 7.0).all() and (buf[:, :, h:] == 7.0).all() and (buf[..., D:] == 7.0).all()


@pytest.mark.parametrize("Tq", [1, 260])
def test_large_and_rising_scores(lib, Tq):
    """Scores that rise along the keys by far more than 16-bit probabilities could hold
    without moving the maximum, large scales, and scale 0 (a plain mean)."""
    dtype = torch.float16
    q, k, v = make(1, Tq, 700, 2, 2, 64, dtype, 12)
    k = (k * torch.linspace(0.05, 6.0, 700, device="cuda")[None, :, None, None]).half()
    o = torch.empty_like(q)
    for scale in (0.125, 1.0, 0.0):
        call(lib, q, k, v, o, -1, 0, 0, scale=scale)
        check(q, k, v, o, -1, 0, 0, scale=scale)
    q2, k2 = q.abs(), -k.abs()                     # all scores far below zero
    call(lib, q2, k2, v, o, -1, 0, 0)
    check(q2, k2, v, o, -1, 0, 0)


@pytest.mark.parametrize("Tq", [1, 200])
def test_nan_query_and_key_reach_their_rows_only(lib, Tq):
    """A NaN query makes its own row NaN. A NaN key that some queries see makes those rows
    not finite."""
    q, k, v = make(1, Tq, 400, 2, 1, 64, torch.float16, 13)
    q[0, Tq - 1, 1] = float("nan")
    o = torch.zeros_like(q)
    call(lib, q, k, v, o, 100, 0, 3)
    nan = torch.isnan(o)
    assert nan[0, Tq - 1, 1].all() and int(nan.sum()) == 64
    k[0, 399] = float("nan")
    call(lib, q, k, v, o, 100, 0, 3)
    assert not torch.isfinite(o[0, Tq - 1]).any()


def test_streams_graph_and_repeat(lib):
    """Two streams at once, and a replayed graph whose lengths change between replays, give
    the same bits as a plain call."""
    for Tq, Tk, kls in ((1, 9000, (9000, 4000)), (300, 900, (900, 350))):
        q, k, v = make(2, Tq, Tk, 4, 2, 128, torch.bfloat16, Tk)
        kl = torch.tensor([kls[0], kls[1]], dtype=torch.int32, device="cuda")
        want = []
        for a in ((kls[0], kls[1]), (kls[1], kls[0])):
            kl.copy_(torch.tensor(a, dtype=torch.int32))
            o = torch.zeros_like(q)
            call(lib, q, k, v, o, 2000, 0, 4, None, kl)
            want.append(o)
        torch.cuda.synchronize()
        outs = [torch.zeros_like(q) for _ in range(2)]
        streams = [torch.cuda.Stream() for _ in range(2)]
        for _ in range(5):
            for o, s in zip(outs, streams):
                with torch.cuda.stream(s):
                    call(lib, q, k, v, o, 2000, 0, 4, None, kl)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[1]) and torch.equal(outs[1], want[1])
        o = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(lib, q, k, v, o, 2000, 0, 4, None, kl)
        for a, w in (((kls[0], kls[1]), want[0]), ((kls[1], kls[0]), want[1])):
            kl.copy_(torch.tensor(a, dtype=torch.int32))
            o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, w)


def test_same_as_full_attention(lib):
    """Without limits it is da3b_attention on the same packed buffer, to 16 bits."""
    B, T, h = 2, 1370, 6
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(B, T, 3, h, 64, device="cuda", generator=g).half()
    a, b = (torch.empty(B, T, h, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    assert lib.da3b_attention(x.data_ptr(), B, T, h, a.data_ptr(), st()) == 0
    call(lib, x[:, :, 0], x[:, :, 1], x[:, :, 2], b, -1, -1, 0)
    check(x[:, :, 0], x[:, :, 1], x[:, :, 2], b, -1, -1, 0)
    assert (a.float() - b.float()).abs().max() <= 2e-3


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.mem_get_info()[0] < 40 << 30, reason="needs 40 GB")
@pytest.mark.parametrize("Tq", [1, 130])
def test_offsets_past_32_bits(lib, Tq):
    """A cache whose element offsets pass 2^32: the window lies at its end."""
    Tk, D = 4_500_000, 128
    k = torch.zeros(1, Tk, 8, D, dtype=torch.float16, device="cuda")
    v = torch.full_like(k, 0.0)
    g = torch.Generator(device="cuda").manual_seed(2)
    for t in (k, v):
        t[:, -600:] = torch.randn(1, 600, 8, D, device="cuda", generator=g).half()
        t[:, :3] = torch.randn(1, 3, 8, D, device="cuda", generator=g).half()
    q = torch.randn(1, Tq, 8, D, device="cuda", generator=g).half()
    o = torch.empty_like(q)
    call(lib, q, k, v, o, 400, 0, 3)
    kk, vv = torch.cat([k[:, :3], k[:, -600:]], 1), torch.cat([v[:, :3], v[:, -600:]], 1)
    want = torch.empty_like(q)
    call(lib, q, kk, vv, want, 400, 0, 3)
    check(q, kk, vv, want, 400, 0, 3)
    assert (o.float() - want.float()).abs().max() <= 4e-3


def test_no_keys(lib):
    """k_len 0 (k and v may be null): zeros in the rows that count, the others as they were."""
    B, Tq, h, D = 3, 5, 4, 128
    q = torch.randn(B, Tq, h, D, device="cuda").half()
    o = torch.full_like(q, 7.0)
    ql = torch.tensor([5, 0, 2], dtype=torch.int32, device="cuda")
    kv = I3(1, 1, 1)                                       # an empty tensor's strides mean nothing
    assert lib.da3b_attention_window(q.data_ptr(), s3(q), None, kv, None, kv, o.data_ptr(), s3(o), 0, B, Tq, 0, h, 2, D,
                                     ql.data_ptr(), None, 3, 0, 1, 0.1, st()) == 0
    for b, n in enumerate((5, 0, 2)):
        assert (o[b, :n] == 0).all() and (o[b, n:] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Tq,Tk,h,kvh,left,right,sinks", [
    (50, 300, 420, 8, 4, 100, 0, 3),          # several items for each multiprocessor, of unlike lengths
    (40, 131, 131, 12, 12, -1, -1, 0),
    (30, 900, 900, 4, 1, 17, 5, 40),
    (300, 33, 70, 2, 1, -1, 0, 0),
])
def test_more_items_than_multiprocessors(lib, B, Tq, Tk, h, kvh, left, right, sinks, D, dtype):
    """Sequences of all lengths, 0 and 1 among them, with more queries than keys or fewer, and
    NaN in every key past a length: what one item leaves behind must not reach the next."""
    q, k, v = make(B, Tq, Tk, h, kvh, D, dtype, B + D)
    g = torch.Generator().manual_seed(B)
    kl = torch.randint(0, Tk + 1, (B,), generator=g, dtype=torch.int32)
    ql = torch.minimum(torch.randint(0, Tq + 1, (B,), generator=g, dtype=torch.int32), kl + 3)
    kl[:4], ql[:4] = torch.tensor([0, 1, Tk, Tk]), torch.tensor([2, 1, Tq, 0])
    for b in range(B):
        k[b, kl[b]:], v[b, kl[b]:] = float("nan"), float("inf")
    kl, ql = kl.cuda(), ql.cuda()
    o = torch.full_like(q, 7.0)
    call(lib, q, k, v, o, left, right, sinks, ql, kl)
    check(q, k, v, o, left, right, sinks, ql, kl, fill=7.0)
    again = torch.full_like(q, 7.0)
    call(lib, q, k, v, again, left, right, sinks, ql, kl)
    assert torch.equal(o, again)              # whichever multiprocessor takes an item
    assert lib.da3b_device_status() == 0
