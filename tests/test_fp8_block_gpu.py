"""A transformer block made of the e4m3 linears, their LayerNorm and quantiser and the
windowed attention, as one CUDA graph for the prompt and one for a single token a sequence:
keys and values go from their linear straight into a cache. Each stage is held against 64
bits from the buffers that the stage before it left, with that operator's own tolerance."""
import math
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

from conftest import ROOT
from test_attention_window_gpu import call, check
from test_fp8_gpu import DT, HALF_STEP, bytes_of, check_quantised, gen, gpu_quant, plain_quant, reference, st, values

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.synchronize()


class Block:
    """The weights of a block, and one pass of it over M rows."""

    def __init__(self, lib, dtype, heads, kv, D, seed):
        g = gen(seed)
        self.lib, self.dt, self.heads, self.kv, self.D = lib, DT.index(dtype), heads, kv, D
        W, H = heads * D, 4 * heads * D
        self.W, self.H = W, H

        def weight(n, k):
            q, s = gpu_quant(lib, torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k))
            return q, s, 0.1 * torch.randn(n, device="cuda", generator=g), values(q, bytes_of(s, n, k), k)

        self.q, self.k, self.v = weight(W, W), weight(kv * D, W), weight(kv * D, W)
        self.proj, self.fc1, self.fc2 = weight(W, W), weight(H, W), weight(W, H)
        self.g1, self.g2 = (1 + 0.1 * torch.randn(W, device="cuda", generator=g) for _ in range(2))
        self.b1, self.b2 = (0.1 * torch.randn(W, device="cuda", generator=g) for _ in range(2))
        self.s1, self.s2 = (0.5 + 0.1 * torch.randn(W, device="cuda", generator=g) for _ in range(2))

    def buffers(self, M, dtype):
        e = lambda *s, t=torch.uint8: torch.empty(*s, dtype=t, device="cuda")
        n = self.lib.da3b_fp8_scale_bytes
        return {"r": e(M, self.W, t=torch.float32), "mid": e(M, self.W, t=torch.float32),
                "x": (e(M, self.W), e(n(M, self.W))), "a": (e(M, self.W), e(n(M, self.W))),
                "y": (e(M, self.W), e(n(M, self.W))), "h": (e(M, self.H), e(n(M, self.H))),
                "q": e(M, self.W, t=dtype), "o": e(M, self.W, t=dtype)}

    def linear(self, x, M, w, y, ldo):
        N, K = w[0].shape[0], w[3].shape[1]
        assert self.lib.da3b_linear_fp8(x[0].data_ptr(), M, K, K, x[1].data_ptr(), w[0].data_ptr(), N, w[0].stride(0),
                                        w[1].data_ptr(), w[2].data_ptr(), 0, y.data_ptr(), self.dt, ldo, st()) == 0

    def resid(self, x, M, w, scale, r):
        N, K = w[0].shape[0], w[3].shape[1]
        assert self.lib.da3b_linear_fp8_resid_f32(x[0].data_ptr(), M, K, K, x[1].data_ptr(), w[0].data_ptr(), N,
                                                  w[0].stride(0), w[1].data_ptr(), w[2].data_ptr(), scale.data_ptr(),
                                                  r.data_ptr(), N, st()) == 0

    def norm(self, r, M, g, b, x):
        assert self.lib.da3b_layernorm_fp8(r.data_ptr(), M, self.W, self.W, g.data_ptr(), b.data_ptr(), 1e-6,
                                           x[0].data_ptr(), self.W, x[1].data_ptr(), st()) == 0

    def run(self, f, M, kc, vc, ldkv, q4, k4, v4, o4, win, ql, kl):
        lib, W = self.lib, self.W
        self.norm(f["r"], M, self.g1, self.b1, f["x"])
        self.linear(f["x"], M, self.q, f["q"], W)
        self.linear(f["x"], M, self.k, kc, ldkv)
        self.linear(f["x"], M, self.v, vc, ldkv)
        call(lib, q4, k4, v4, o4, *win, ql=ql, kl=kl)
        assert lib.da3b_quantize_fp8(f["o"].data_ptr(), self.dt, M, W, W, f["a"][0].data_ptr(), W, f["a"][1].data_ptr(),
                                     st()) == 0
        self.resid(f["a"], M, self.proj, self.s1, f["r"])
        f["mid"].copy_(f["r"])
        self.norm(f["r"], M, self.g2, self.b2, f["y"])
        w = self.fc1
        assert lib.da3b_linear_fp8_q(f["y"][0].data_ptr(), M, W, W, f["y"][1].data_ptr(), w[0].data_ptr(), self.H,
                                     w[0].stride(0), w[1].data_ptr(), w[2].data_ptr(), 2, f["h"][0].data_ptr(), self.H,
                                     f["h"][1].data_ptr(), st()) == 0
        self.resid(f["h"], M, self.fc2, self.s2, f["r"])

    def verify(self, f, r0, M, k, v):
        """k, v: the rows that the pass wrote into the cache, [M][kv * D]."""
        W, H = self.W, self.H
        self.verify_norm(r0, self.g1, self.b1, f["x"], M)
        xv = values(f["x"][0], bytes_of(f["x"][1], M, W), W)
        for w, y in ((self.q, f["q"]), (self.k, k), (self.v, v)):
            ref, err = reference(xv, w[3], w[2], 0, W)
            half = HALF_STEP[self.dt]
            lim = (1 + 2 * half) * err + half * ref.abs() + (2.0 ** -25 if self.dt == 0 else 0.0)
            assert ((y.double() - ref).abs() <= lim).all()
        codes, b = plain_quant(f["o"])
        assert torch.equal(f["a"][0], codes) and torch.equal(bytes_of(f["a"][1], M, W), b)
        self.verify_resid(values(codes, b, W), self.proj, self.s1, r0, f["mid"])
        self.verify_norm(f["mid"], self.g2, self.b2, f["y"], M)
        ref, err = reference(values(f["y"][0], bytes_of(f["y"][1], M, W), W), self.fc1[3], self.fc1[2], 2, W)
        check_quantised(f["h"][0], bytes_of(f["h"][1], M, H), ref, err, H)
        self.verify_resid(values(f["h"][0], bytes_of(f["h"][1], M, H), H), self.fc2, self.s2, f["mid"], f["r"])

    def verify_norm(self, r, g, b, x, M):
        d = r.double() - r.double().mean(1, keepdim=True)
        y = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-6) * g.double() + b.double()
        check_quantised(x[0], bytes_of(x[1], M, self.W), y, 3e-6 * y.abs() + 3e-5, self.W)

    def verify_resid(self, xv, w, scale, before, after):
        y, err = reference(xv, w[3], w[2], 0, xv.shape[1])
        y, err = y * scale.double(), (err + 2.0 ** -24 * y.abs()) * scale.double().abs()
        ref = before.double() + y
        assert ((after.double() - ref).abs() <= err + 2.0 ** -23 * (ref.abs() + y.abs())).all()


@pytest.mark.parametrize("dtype,heads,kv,D,T,win", [
    (torch.float16, 6, 6, 64, 333, (100, 100, 1)),      # both ways, the first token seen by all
    (torch.bfloat16, 4, 2, 128, 200, (63, 0, 4)),       # causal, shared key heads
])
def test_block(lib, dtype, heads, kv, D, T, win):
    B, cap, steps = 3, T + 4, 3
    blk = Block(lib, dtype, heads, kv, D, T)
    W, G = heads * D, kv * D
    kc, vc = (torch.full((B, cap, kv, D), 9.0, dtype=dtype, device="cuda") for _ in range(2))
    ql = torch.tensor([T, T - 37, 1], dtype=torch.int32, device="cuda")
    kl = ql.clone()

    # The prompt: the same rows of all sequences side by side, padded to T.
    full = blk.buffers(B * T, dtype)
    kn, vn = (torch.empty(B, T, kv, D, dtype=dtype, device="cuda") for _ in range(2))
    four = lambda t, n, h: t.view(B, n, h, D)
    x0 = torch.randn(B * T, W, device="cuda", generator=gen(1)) * 2

    def prompt():
        blk.run(full, B * T, kn, vn, G, four(full["q"], T, heads), kn, vn, four(full["o"], T, heads), win, ql, kl)
        kc[:, :T].copy_(kn)
        vc[:, :T].copy_(vn)

    full["o"].zero_()                                    # rows past the lengths keep this
    graph = torch.cuda.CUDAGraph()
    full["r"].copy_(x0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        prompt()
    full["r"].copy_(x0)
    graph.replay()
    torch.cuda.synchronize()
    assert lib.da3b_device_status() == 0
    blk.verify(full, x0, B * T, kn.view(B * T, G), vn.view(B * T, G))
    check(four(full["q"], T, heads), kn, vn, four(full["o"], T, heads), *win, ql=ql, kl=kl, fill=0.0)

    # One token a sequence: row p of the cache is written by the linears themselves, at a
    # row stride of a whole sequence's cache.
    one = blk.buffers(B, dtype)
    for s in range(steps):
        p = T + s                                        # the slot; ragged lengths count up to it
        klen = torch.tensor([p + 1, p + 1, s + 1], dtype=torch.int32, device="cuda")
        x1 = torch.randn(B, W, device="cuda", generator=gen(50 + s))
        keep_k, keep_v = kc.clone(), vc.clone()
        step = torch.cuda.CUDAGraph()
        with torch.cuda.graph(step):
            blk.run(one, B, kc[:, p], vc[:, p], cap * G, four(one["q"], 1, heads), kc, vc, four(one["o"], 1, heads),
                    win, None, klen)
        one["r"].copy_(x1)
        step.replay()
        torch.cuda.synchronize()
        assert lib.da3b_device_status() == 0
        blk.verify(one, x1, B, kc[:, p].reshape(B, G), vc[:, p].reshape(B, G))
        keep_k[:, p], keep_v[:, p] = kc[:, p], vc[:, p]
        assert torch.equal(kc, keep_k) and torch.equal(vc, keep_v)   # no other row of the cache
        check(four(one["q"], 1, heads), kc, vc, four(one["o"], 1, heads), *win, kl=klen)


FIRST = """
import ctypes, torch
from da3cpplib_b200 import _lib
lib = _lib.load()
I3 = ctypes.c_int64 * 3
e = lambda *s, t=torch.uint8: torch.zeros(*s, dtype=t, device="cuda")
x, b = torch.randn(64, 128, device="cuda").half(), torch.randn(128, device="cuda")
q, s, qw, sw = e(64, 128), e(512), e(128, 128), e(512)
w = torch.randn(128, 128, device="cuda")
y, o, o1 = e(64, 128, t=torch.float16), e(64, 128, t=torch.float16), e(128, t=torch.float16)
kv, o2 = torch.randn(3000, 128, device="cuda").half(), e(64, 128, t=torch.float16)

def run():
    st = torch.cuda.current_stream().cuda_stream
    a = lambda T, o: lib.da3b_attention_window(y.data_ptr(), I3(T * 128, 128, 64), y.data_ptr(), I3(8192, 128, 64),
        y.data_ptr(), I3(8192, 128, 64), o.data_ptr(), I3(T * 128, 128, 64), 0, 1, T, 64, 2, 2, 64, None, None, 9, 0, 1,
        0.125, st)
    return [lib.da3b_quantize_fp8(w.data_ptr(), 2, 128, 128, 128, qw.data_ptr(), 128, sw.data_ptr(), st),
            lib.da3b_quantize_fp8(x.data_ptr(), 0, 64, 128, 128, q.data_ptr(), 128, s.data_ptr(), st),
            lib.da3b_linear_fp8(q.data_ptr(), 64, 128, 128, s.data_ptr(), qw.data_ptr(), 128, 128, sw.data_ptr(),
                                b.data_ptr(), 0, y.data_ptr(), 0, 128, st), a(64, o), a(1, o1),
            lib.da3b_attention_window(y.data_ptr(), I3(8192, 128, 64), kv.data_ptr(), I3(1, 128, 64), kv.data_ptr(),
                I3(1, 128, 64), o2.data_ptr(), I3(8192, 128, 64), 0, 1, 64, 3000, 2, 2, 64, None, None, -1, -1, 0,
                0.125, st)]   # keys split over a cluster

torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    rc = run()
print(rc)
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (y, o, o1, o2)]
print(run())
torch.cuda.synchronize()
assert all(t.abs().max() > 0 for t in got) and all(torch.equal(i, j) for i, j in zip(got, (y, o, o1, o2)))
assert lib.da3b_device_status() == 0
print("same")
"""


def test_first_calls_of_a_process_in_a_capture():
    """Captured before anything else of the library ran: the same results as eager calls."""
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split("\n")[-2] == "same", r.stdout + r.stderr
