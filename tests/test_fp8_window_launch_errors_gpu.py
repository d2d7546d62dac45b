"""A launch that fails is reported by its own call and by no other. The failure is the
host's: the stream's capture has been made invalid, so that nothing can be launched on it."""
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

from conftest import ROOT

pytestmark = pytest.mark.gpu

SCRIPT = """
import ctypes, torch
from da3cpplib_b200 import _lib
lib, rt = _lib.load(), ctypes.CDLL("libcudart.so.12")
V, I3 = ctypes.c_void_p, ctypes.c_int64 * 3
e = lambda *s, t=torch.uint8: torch.zeros(*s, dtype=t, device="cuda")
x, w, b = torch.randn(64, 128, device="cuda"), torch.randn(128, 128, device="cuda"), torch.randn(128, device="cuda")
q, s, qw, sw = e(64, 128), e(512), e(128, 128), e(512)
y, o = e(64, 128, t=torch.float16), e(64, 128, t=torch.float16)
qkv, full = torch.randn(100, 3 * 128, device="cuda").half(), e(100, 128, t=torch.float16)

def att(T, Tk):
    return lambda st: lib.da3b_attention_window(y.data_ptr(), I3(T * 128, 128, 64), y.data_ptr(), I3(8192, 128, 64),
        y.data_ptr(), I3(8192, 128, 64), o.data_ptr(), I3(T * 128, 128, 64), 0, 1, T, Tk, 2, 2, 64, None, None, 9, 0, 1,
        0.125, st)

CALLS = {
    "weights": lambda st: lib.da3b_quantize_fp8(w.data_ptr(), 2, 128, 128, 128, qw.data_ptr(), 128, sw.data_ptr(), st),
    "quantise": lambda st: lib.da3b_quantize_fp8(x.data_ptr(), 2, 64, 128, 128, q.data_ptr(), 128, s.data_ptr(), st),
    "norm": lambda st: lib.da3b_layernorm_fp8(x.data_ptr(), 64, 128, 128, b.data_ptr(), None, 1e-6, q.data_ptr(), 128,
                                              s.data_ptr(), st),
    "linear": lambda st: lib.da3b_linear_fp8(q.data_ptr(), 64, 128, 128, s.data_ptr(), qw.data_ptr(), 128, 128,
                                             sw.data_ptr(), b.data_ptr(), 0, y.data_ptr(), 0, 128, st),
    "many": att(64, 64), "few": att(1, 64), "no keys": att(64, 0),
}

def plain():
    st = torch.cuda.current_stream().cuda_stream
    return [c(st) for c in CALLS.values()] + [lib.da3b_attention(qkv.data_ptr(), 1, 100, 2, full.data_ptr(), st)]

assert not any(plain()), plain()
torch.cuda.synchronize()
for name, call in CALLS.items():
    side = torch.cuda.Stream()
    h = V(side.cuda_stream)
    assert rt.cudaStreamBeginCapture(h, 1) == 0
    assert rt.cudaStreamSynchronize(h) != 0              # not allowed in a capture, and ends it
    assert call(side.cuda_stream) == -4, name
    g = V()
    assert rt.cudaStreamEndCapture(h, ctypes.byref(g)) != 0
    rt.cudaGetLastError()
    assert not any(plain()), (name, plain())
torch.cuda.synchronize()
assert lib.da3b_device_status() == 0
print("ok")
"""


def test_a_failed_launch_is_its_own_calls_error():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    r = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.split("\n")[-2] == "ok", r.stdout + r.stderr
