"""The score operators' C entry points refuse wrong arguments before anything is enqueued, and
say what is wrong.  No GPU: the calls here never get as far as a launch."""
import ctypes as C

import numpy as np
import pytest

import filtervectorcode_refactor_amd as F
from filtervectorcode_refactor_amd import _lib

BUF = np.zeros(4096, np.uint8)
P = (BUF.ctypes.data + 63) // 64 * 64  # never read: every call below is refused
NAN = float("nan")


def _refused(rc, *words):
    assert rc == _lib.UNG_HIP_EINVAL
    for w in words:
        assert w in _lib.last_error(), _lib.last_error()


def test_quantize():
    f = F.load().ung_hip_fp8_quantize
    _refused(f(P, 9, 4, 4, 4, 0, P, P, None, None, None), "type 9")
    _refused(f(None, 0, 4, 4, 4, 0, P, P, None, None, None), "null")
    _refused(f(P, 0, 4, 4, 4, 0, None, None, None, None, None), "null")
    _refused(f(P, 0, 4, 4, 4, 0, P, None, None, None, None), "null")
    _refused(f(P, 0, 4, 4, 4, 1, None, None, P, P, None), "null")
    _refused(f(P, 0, 4, 4, 3, 0, P, P, None, None, None), "row_stride 3")
    _refused(f(P, 0, 4, 4, 4, 0, P + 8, P, None, None, None), "alignment")
    _refused(f(P + 2, 0, 4, 4, 4, 0, P, P, None, None, None), "alignment")
    _refused(f(P, 0, 1 << 40, 4, 4, 0, P, P, None, None, None), "too many")
    assert f(None, 0, 0, 4, 4, 0, None, None, None, None, None) == 0


def test_matmul():
    f = F.load().ung_hip_fp8_matmul
    _refused(f(P, P, P, P, 0, 4, 4, 100, P, 0, 4, None, 0, None), "100")
    _refused(f(P, P, P, P, 0, 4, 4, 128, P, 5, 4, None, 0, None), "type 5")
    _refused(f(P, None, P, P, 0, 4, 4, 128, P, 0, 4, None, 0, None), "null")
    _refused(f(P, P, P, P, 0, 4, 4, 128, None, 0, 4, None, 0, None), "null")
    _refused(f(P, P, P, P, 0, 4, 4, 128, P, 0, 3, None, 0, None), "c_stride 3")
    _refused(f(P + 1, P, P, P, 0, 4, 4, 128, P, 0, 4, None, 0, None), "alignment")
    _refused(f(P, P, P, P, 0, 1 << 33, 4, 128, P, 0, 4, None, 0, None), "too large")
    assert f(None, None, None, None, 0, 0, 4, 128, None, 0, 4, None, 0, None) == 0
    _refused(F.load().ung_hip_fp8_matmul_workspace(4, 4, 128, 0, None), "null")


def test_top_scores():
    f = F.load().ung_hip_top_scores
    _refused(f(P, 7, 4, 4, 4, 2, 1.0, P, P, P, None, 0, None), "type 7")
    _refused(f(P, 0, 4, 4, 4, 0, 1.0, P, P, P, None, 0, None), "k=0")
    _refused(f(P, 0, 4, 4, 4, 129, 1.0, P, P, P, None, 0, None), "k=129")
    for t in (0.0, -1.0, NAN, float("inf")):
        _refused(f(P, 0, 4, 4, 4, 2, t, P, P, P, None, 0, None), "temperature")
    _refused(f(None, 0, 4, 4, 4, 2, 1.0, P, P, P, None, 0, None), "null")
    _refused(f(P, 0, 4, 4, 4, 2, 1.0, None, P, P, None, 0, None), "null")
    _refused(f(P, 0, 4, 4, 2, 2, 1.0, P, P, P, None, 0, None), "row_stride")
    _refused(f(P + 1, 1, 4, 4, 4, 2, 1.0, P, P, P, None, 0, None), "aligned")
    _refused(f(P, 0, 4, 1 << 31, 1 << 31, 2, 1.0, P, P, P, None, 0, None), "too many")
    need = C.c_uint64()
    assert F.load().ung_hip_top_scores_workspace(P, 0, 1, 1_000_000, 1_000_000, 8, C.byref(need)) == 0
    assert need.value > 0  # a long row is cut into pieces
    _refused(f(P, 0, 1, 1_000_000, 1_000_000, 8, 1.0, P, P, P, None, 0, None), "workspace")
    _refused(f(P, 0, 1, 1_000_000, 1_000_000, 8, 1.0, P, P, P, P, need.value - 1, None), "workspace")
    _refused(F.load().ung_hip_top_scores_workspace(P, 0, 1, 9, 9, 8, None), "null")
    assert f(None, 0, 0, 4, 4, 2, 1.0, None, None, None, None, 0, None) == 0


@pytest.mark.parametrize("k", [0, 4])
def test_distill(k):
    lib = F.load()
    fwd, bwd, step = lib.ung_hip_distill_forward, lib.ung_hip_distill_backward, lib.ung_hip_distill_step
    _refused(fwd(P, 3, 4, 4, 4, P, P, k, None, 1.0, P, P, None, 0, None), "type 3")
    _refused(fwd(P, 0, 4, 4, 4, P, P, 200, None, 1.0, P, P, None, 0, None), "k=200")
    _refused(fwd(P, 0, 4, 4, 4, P, P, k, None, NAN, P, P, None, 0, None), "temperature")
    _refused(fwd(P, 0, 4, 4, 4, P, P, k, None, 1.0, None, P, None, 0, None), "null")
    _refused(fwd(P, 0, 4, 4, 4, P, P, k, None, 1.0, P, P + 4, None, 0, None), "16-byte")
    if k:
        _refused(fwd(P, 0, 4, 4, 4, None, P, k, None, 1.0, P, P, None, 0, None), "null")
    _refused(bwd(P, 0, 4, 4, 4, P, P, k, P, None, 1.0, None, 4, None), "null")
    _refused(bwd(P, 0, 4, 4, 4, P, P, k, None, None, 1.0, P, 4, None), "saved")
    _refused(bwd(P, 0, 4, 4, 4, P, P, k, P, None, 1.0, P, 3, None), "grad_stride")
    _refused(step(P, 0, 4, 4, 4, P, P, k, None, None, 1.0, None, P, 4, None, 0, None), "null loss")
    _refused(step(P, 0, 4, 4, 4, P, P, k, None, None, 1.0, P, P + 2, 4, None, 0, None), "aligned")
    need = C.c_uint64()
    assert lib.ung_hip_distill_workspace(P, 0, 1, 1_000_000, 1_000_000, C.byref(need)) == 0 and need.value > 0
    _refused(step(P, 0, 1, 1_000_000, 1_000_000, P, P, k, None, None, 1.0, P, P, 1_000_000, None, 0, None), "workspace")
    assert step(None, 0, 0, 4, 4, None, None, k, None, None, 1.0, None, None, 4, None, 0, None) == 0


def test_more_blocks_than_a_launch_takes():
    """A launch counts its threads in 32 bits: more are refused by name, not by the launch."""
    lib, rows = F.load(), 1 << 25
    _refused(lib.ung_hip_fp8_quantize(P, 0, 1 << 31, 1, 1, 0, P, P, P, P, None), "too many")
    _refused(lib.ung_hip_fp8_quantize(P, 0, 1 << 31, 1, 1, 1, P, P, None, None, None), "too many")
    _refused(lib.ung_hip_fp8_matmul(P, P, P, P, 0, 128, (1 << 31) - 1, 0, P, 0, 1 << 31, None, 0, None), "too large")
    _refused(lib.ung_hip_top_scores(P, 0, rows, 4, 4, 2, 1.0, P, P, P, None, 0, None), "too many")
    _refused(lib.ung_hip_distill_forward(P, 0, rows, 4, 4, P, P, 4, None, 1.0, P, P, None, 0, None), "too many")
    _refused(lib.ung_hip_distill_backward(P, 0, rows, 4, 4, P, P, 4, P, None, 1.0, P, 4, None), "too many")
    _refused(lib.ung_hip_distill_step(P, 0, rows, 4, 4, P, P, 4, None, None, 1.0, P, P, 4, None, 0, None), "too many")
