"""GPU tests (-m gpu) of fills and copies between the host and the device beside streams that do not wait for the default one."""
import ctypes as C

import numpy as np
import pytest

import nvr_import

nvr = nvr_import.load()
pytestmark = pytest.mark.gpu


def test_fills_are_over_when_the_call_returns():
    """A launch on a stream of the library right behind a fill of some milliseconds reads what the fill wrote, at its very end."""
    L = nvr.lib()
    nvr.check(L.nvr_device_set(0))
    nvr.check(L.nvr_ops_set_dtype(b"float16"))
    stream = C.c_void_p()
    nvr.check(L.nvr_stream_create(C.byref(stream)))
    n, rows, cols = 8 << 30, 16, 1024
    big, out, ws = nvr.DeviceBuffer(n), nvr.DeviceBuffer(rows * cols * 2), nvr.DeviceBuffer(L.nvr_lora_workspace_bytes(rows, 64, cols, 8))
    none = nvr.DeviceBuffer.from_numpy(np.full(rows, -1, np.int32))
    tail = big.ptr + n - rows * cols * 2
    for byte in (0x11, 0x22, 0x33):
        nvr.check(L.nvr_device_memset(big.ptr, byte, n))
        nvr.check(L.nvr_lora_add(tail, cols, None, None, None, none.ptr, 0, rows, 64, cols, 8, tail, cols, out.ptr, cols, ws.ptr, stream))      # (rows without an adapter: a copy)
        nvr.check(L.nvr_stream_synchronize(stream))
        assert (out.to_numpy((rows * cols * 2,), np.uint8) == byte).all()
    nvr.check(L.nvr_stream_destroy(stream))


def test_copies_to_the_host_from_inside_an_allocation_and_of_nothing():
    """Pointers into the middle of an allocation are the device's; a copy of nothing from no pointer is nothing, and leaves no error to the launches behind it."""
    L = nvr.lib()
    nvr.check(L.nvr_device_set(0))
    a = np.arange(100000, dtype=np.int32)
    b = nvr.DeviceBuffer.from_numpy(a)
    got = np.zeros(17, np.int32)
    nvr.check(L.nvr_memcpy_d2h(got.ctypes.data, b.ptr + 4 * 70001, got.nbytes))
    assert np.array_equal(got, a[70001:70018])
    nvr.check(L.nvr_memcpy_d2h(got.ctypes.data, None, 0))
    nvr.check(L.nvr_ops_set_dtype(b"float16"))
    nvr.check(L.nvr_fill_const(b.ptr, 64, 0.0, None))
    assert (b.to_numpy((32,), np.int32) == 0).all()
