"""Errors of the calls on sequences are those of the call that reports them."""
import ctypes

import pytest

import fyusenet_amd as fa
from fyusenet_amd import capi
from tests.test_gpu_sequences import close, reference, stream, values

torch = pytest.importorskip("torch")


@pytest.mark.gpu
def test_cache_that_does_not_fit():
    """A cache larger than the memory is refused, and leaves nothing behind that another call reports."""
    q, k, v = values(1, "f16", (1, 8, 4, 64), (1, 8, 2, 64), (1, 8, 2, 64))
    out = torch.empty_like(q)
    for _ in range(2):
        with pytest.raises(fa.FynException) as e:
            fa.SequenceCache(fa.STORAGE_F16, 64, 4, 2, 64, 1024, 1 << 20, 4, 1024)    # (32 TB)
        assert e.value.code == capi.ERR_DEVICE
        fa.attention(q, k, v, out, stream=stream())
        close(out[0], *reference(q[0], k[0], v[0], 0))
        with pytest.raises(fa.FynException):
            fa.SequenceCache(fa.STORAGE_F16, 64, 4, 2, 64, 1024, 1 << 20, 4, 1024)
        c = fa.SequenceCache(fa.STORAGE_F16, 1, 4, 2, 64, 16, 4, 2)
        with pytest.raises(fa.FynException):
            fa.SequenceCache(fa.STORAGE_F16, 64, 4, 2, 64, 1024, 1 << 20, 4, 1024)
        c.extend([0], [8], stream=stream())
        c.write(0, k[0], v[0], stream=stream())
        with pytest.raises(fa.FynException):
            fa.SequenceCache(fa.STORAGE_F16, 64, 4, 2, 64, 1024, 1 << 20, 4, 1024)
        c.attend(0, q[0], out[0], stream=stream())
        close(out[0], *reference(q[0], k[0], v[0], 0))
        assert (torch.zeros(4, device="cuda") + 1).sum().item() == 4   # (nor one of torch's)
        c.close()


@pytest.mark.gpu
def test_an_error_of_somebody_else():
    """The last error that another call has left in the thread is not reported as that of a launch, and is still there afterwards."""
    hip = ctypes.CDLL(capi.lib()._name)   # (the runtime that the library uses)
    hip.hipMalloc.argtypes, hip.hipGetLastError.restype, hip.hipPeekAtLastError.restype = [ctypes.c_void_p, ctypes.c_size_t], ctypes.c_int, ctypes.c_int
    q, k, v = values(1, "f16", (1, 8, 4, 64), (1, 8, 2, 64), (1, 8, 2, 64))
    many, = values(2, "f16", (4, 130, 32, 64))
    out, wide, got = torch.empty_like(q), torch.empty_like(many), torch.empty_like(k[0])
    torch.cuda.synchronize()
    at, s = ctypes.c_void_p(), stream()
    try:
        left = hip.hipMalloc(ctypes.byref(at), 1 << 50)
        assert left != 0 and hip.hipPeekAtLastError() == left
        c = fa.SequenceCache(fa.STORAGE_F16, 1, 4, 2, 64, 16, 4, 2)
        fa.attention(q, k, v, out, stream=s)
        fa.attention(many, many, many, wide, stream=s)
        c.extend([0], [8], stream=s)
        c.write(0, k[0], v[0], stream=s)
        c.attend(0, q[0], out[0], stream=s)
        c.read([0], 0, got, torch.empty_like(got), stream=s)
        c.copy([0], [1], stream=s)
        assert hip.hipPeekAtLastError() == left
    finally:
        hip.hipGetLastError()
    close(out[0], *reference(q[0], k[0], v[0], 0))
    assert torch.equal(got, k[0])
