"""Managed memory is served wherever its pages are, and whichever device was current when it
was allocated."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from test_fp8_gpu import bytes_of, plain_quant, st

pytestmark = pytest.mark.gpu

V = ctypes.c_void_p


@pytest.fixture
def managed():
    """Allocates managed memory while a device is current; frees it at the end."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    rt = ctypes.CDLL("libcudart.so.12")
    rt.cudaMallocManaged.argtypes = [ctypes.POINTER(V), ctypes.c_size_t, ctypes.c_uint]
    rt.cudaMemcpy.argtypes = [V, V, ctypes.c_size_t, ctypes.c_int]
    kept = []

    def alloc(n, device):
        p = V()
        with torch.cuda.device(device):
            assert rt.cudaMallocManaged(ctypes.byref(p), n, 1) == 0
        kept.append(p)
        return p.value

    yield rt, alloc
    torch.cuda.synchronize()
    for p in kept:
        rt.cudaFree(p)


def run(lib, managed, device):
    rt, alloc = managed
    R, K = 70, 256
    x = torch.randn(R, K, device="cuda")
    n = lib.da3b_fp8_scale_bytes(R, K)
    xm, qm, sm = alloc(R * K * 4, device), alloc(R * K, device), alloc(n, device)
    host = x.cpu()
    ctypes.memmove(xm, host.data_ptr(), R * K * 4)             # its pages are the host's now
    assert lib.da3b_quantize_fp8(xm, 2, R, K, K, qm, K, sm, st()) == 0
    q, s = torch.empty(R, K, dtype=torch.uint8, device="cuda"), torch.empty(n, dtype=torch.uint8, device="cuda")
    assert rt.cudaMemcpy(q.data_ptr(), qm, R * K, 4) == 0 and rt.cudaMemcpy(s.data_ptr(), sm, n, 4) == 0
    codes, b = plain_quant(x)
    assert torch.equal(q, codes) and torch.equal(bytes_of(s, R, K), b)


def test_managed_memory(lib, managed):
    run(lib, managed, 0)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_managed_memory_allocated_under_another_device(lib, managed):
    run(lib, managed, 1)
