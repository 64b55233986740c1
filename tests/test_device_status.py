"""How a kernel's wait that ran out reaches a Python caller: chpl_b200.check_device()."""
import ctypes

import pytest

import chpl_b200
from chpl_b200 import _lib


def test_linear_wait_rejects_bad_limits():
    L = _lib.load()
    assert L.chpl_diag_linear_wait(None, 0) == _lib.CHPL_ERR_INVALID
    assert L.chpl_diag_linear_wait(None, 3_000_000_000) == _lib.CHPL_ERR_INVALID


@pytest.mark.parametrize("rc,status,code", [(0, 0, None), (0, _lib.CHPL_ERR_TIMEOUT, _lib.CHPL_ERR_TIMEOUT), (_lib.CHPL_ERR_CUDA, 0, _lib.CHPL_ERR_CUDA)])
def test_check_device_raises_what_the_library_reports(monkeypatch, rc, status, code):
    class Fake:
        @staticmethod
        def chpl_device_status(p):
            ctypes.cast(p, ctypes.POINTER(ctypes.c_int))[0] = status
            return rc

        @staticmethod
        def chpl_last_error_string():
            return b"fake"

    monkeypatch.setattr(_lib, "_lib", Fake())
    if code is None:
        return chpl_b200.check_device()
    with pytest.raises(chpl_b200.ChplError) as err:
        chpl_b200.check_device()
    assert err.value.code == code


@pytest.mark.gpu
def test_a_linear_wait_that_runs_out_is_reported_once(cuda):
    """Queued between two layers; the context and the layers stay usable."""
    import torch

    from chpl_b200 import linear
    x, w = torch.randn(64, 256, device="cuda").half(), torch.randn(128, 256, device="cuda").half()
    chpl_b200.check_device()
    want = linear.forward(x, w)
    assert _lib.load().chpl_diag_linear_wait(torch.cuda.current_stream().cuda_stream, 20_000_000) == _lib.CHPL_OK
    got = linear.forward(x, w)
    with pytest.raises(chpl_b200.ChplError) as err:
        chpl_b200.check_device()
    assert err.value.code == _lib.CHPL_ERR_TIMEOUT
    chpl_b200.check_device("cuda:0")
    assert torch.equal(got, want) and torch.equal(linear.forward(x, w), want)
