"""The score operators' C entry points at sizes and values that no launch serves: refused by
name, whatever the sizes, with nothing enqueued.  No GPU."""
import ctypes as C

import numpy as np
import pytest

import filtervectorcode_refactor_amd as F
from filtervectorcode_refactor_amd import _lib

BUF = np.zeros(1 << 16, np.uint8)
P = (BUF.ctypes.data + 63) // 64 * 64  # never read: every call below is refused


def _refused(rc, *words):
    assert rc == _lib.UNG_HIP_EINVAL, rc
    for w in words:
        assert w in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("m,n,kp,word", [
    ((1 << 64) - 1, (1 << 64) - 1, 128, "too large"), (1 << 40, 1 << 40, 128, "too large"),
    (1 << 39, 1 << 39, 1 << 20, "too large"), (1 << 33, 4, 128, "too large"), (4, 1 << 33, 128, "too large"),
    (4, 4, 1 << 40, "too large"), (1 << 20, 1 << 20, 128, "too large"), (4, 4, 100, "100")])
@pytest.mark.parametrize("type", [0, 1, 2])
def test_matmul_workspace_of_what_no_product_takes(m, n, kp, word, type):
    """The workspace's size is refused where the product is, not made from sizes that wrap round."""
    need = C.c_uint64(7)
    _refused(F.load().ung_hip_fp8_matmul_workspace(m, n, kp, type, C.byref(need)), "workspace", word)
    assert need.value == 7
    _refused(F.load().ung_hip_fp8_matmul(P, P, P, P, 0, m, n, kp, P, type, n, None, 0, None), word)
    for empty in ((0, n), (m, 0)):
        if kp % 128 == 0:
            assert F.load().ung_hip_fp8_matmul_workspace(*empty, kp, type, C.byref(need)) == 0 and need.value == 0
            need.value = 7
