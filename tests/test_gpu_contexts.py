"""GPU: which context the C entries run in: the caller's current one, or the device's where there is none."""

import ctypes
import threading

import pytest
import torch

from cernels_b200 import _lib
from tests import ffn_reference as R

pytestmark = pytest.mark.gpu


def test_a_context_that_the_caller_made_current_stays():
    cu, lib = ctypes.CDLL("libcuda.so.1"), _lib.load()
    torch.cuda.init()
    torch.zeros(1, device="cuda")
    before, made, now = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    assert cu.cuCtxGetCurrent(ctypes.byref(before)) == 0
    assert cu.cuCtxCreate_v2(ctypes.byref(made), 0, torch.cuda.current_device()) == 0
    try:
        assert made.value != before.value
        s, ok = _lib.FfnShape(4, 64, 64), 1 << 20  # an entry that checks the device and then refuses: nothing is launched
        assert lib.cernels_gated_ffn(ctypes.byref(s), ok, 64, ok, ok, ok, None, ok, 1 << 20, None) == 6
        assert cu.cuCtxGetCurrent(ctypes.byref(now)) == 0 and now.value == made.value
    finally:
        cu.cuCtxPopCurrent_v2(ctypes.byref(now))
        cu.cuCtxDestroy_v2(made)
    assert cu.cuCtxGetCurrent(ctypes.byref(now)) == 0 and now.value == before.value


def test_a_thread_without_a_context_gets_the_devices():
    """The entry is the first CUDA call of its thread (as in autograd's threads), and it encodes TMA maps."""
    lib = _lib.load()
    T, H, F = 130, 64, 48
    x, wg, wu, wd, _ = R.case(T, H, F, seed=1)
    out = torch.empty_like(x)
    s, codes = _lib.FfnShape(T, H, F), []
    ws = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    args = [ctypes.byref(s), x.data_ptr(), H, wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), out.data_ptr(), ws.data_ptr(), 1 << 16,
            torch.cuda.current_stream().cuda_stream]
    torch.cuda.synchronize()
    th = threading.Thread(target=lambda: codes.append(lib.cernels_gated_ffn(*args)))
    th.start()
    th.join()
    torch.cuda.synchronize()
    assert codes == [0]
    R.assert_within("y", out, *R.forward(x, wg, wu, wd)[:2])
