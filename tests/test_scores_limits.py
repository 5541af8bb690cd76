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


F32, BF16 = 0, 2


def _grad_calls(lib, scores, type, rows, len_, stride, grad, grad_stride):
    """Messages of the two entry points that write a gradient; a null argument that is looked at
    later refuses what the gradient's place does not."""
    for rc in (lambda: lib.ung_hip_distill_backward(scores, type, rows, len_, stride, P, P, 2, None, None, 1.0, grad,
                                                    grad_stride, None),
               lambda: lib.ung_hip_distill_step(scores, type, rows, len_, stride, P, P, 2, None, None, 1.0, None, grad,
                                                grad_stride, None, 0, None)):
        assert rc() == _lib.UNG_HIP_EINVAL
        yield _lib.last_error()


def _meet(rows, len_, stride, at, grad_stride):
    """Whether an element of the rows at 0 and one of the rows at `at` are the same."""
    if rows == 1:
        return abs(at) < len_
    a = np.arange(rows)[:, None] * stride + np.arange(len_)
    b = at + np.arange(rows)[:, None] * grad_stride + np.arange(len_)
    return bool(np.isin(a, b).any())


@pytest.mark.parametrize("type,size", [(F32, 4), (BF16, 2)])
@pytest.mark.parametrize("rows,len_,stride,grad_stride", [
    (4, 10, 10, 10), (4, 10, 12, 12), (4, 10, 20, 20), (4, 10, 25, 25), (4, 10, 31, 31), (1, 10, 10, 10),
    (4, 10, 20, 40), (4, 10, 40, 20), (5, 3, 7, 11), (5, 3, 11, 7), (7, 2, 5, 2), (3, 1, 4, 6)])
def test_gradients_that_overlap_the_scores_in_part(type, size, rows, len_, stride, grad_stride):
    """A gradient over some of the scores that other blocks still read: refused.  Over all of them
    in place, between their rows or beside them: not refused."""
    lib = F.load()
    middle = P + (1 << 14)
    far = rows * max(stride, grad_stride) + 3
    for at in range(-far, far + 1):
        in_place = at == 0 and (stride == grad_stride or rows == 1)
        refused = not in_place and _meet(rows, len_, stride, at, grad_stride)
        for message in _grad_calls(lib, middle, type, rows, len_, stride, middle + at * size, grad_stride):
            assert ("overlaps" in message) == refused, (at, message)


def test_wide_rows_beside_each_other_are_looked_at_quickly():
    """Halves of one buffer's rows, many of them: decided by the strides, not row by row."""
    lib, rows, len_ = F.load(), 10_000_000, 50
    for at, refused in ((50, False), (49, True), (150, False), (151, True), (-50, False), (-49, True), (-150, False),
                        (-151, True)):
        for message in _grad_calls(lib, 1 << 40, F32, rows, len_, 200, (1 << 40) + at * 4, 200):
            assert ("overlaps" in message) == refused, (at, message)


@pytest.mark.parametrize("t", [1e-45, 1e-40, 1e-39, 2.9e-39, 4.2e-39])
def test_temperatures_whose_reciprocal_overflows(t):
    """log2(e) / T past float32 makes 0 * inf of a row's largest score: refused, not NaN."""
    lib = F.load()
    _refused(lib.ung_hip_top_scores(P, 0, 4, 4, 4, 2, t, None, P, P, None, 0, None), "temperature")
    _refused(lib.ung_hip_distill_forward(P, 0, 4, 4, 4, P, P, 2, None, t, None, P, None, 0, None), "temperature")
    _refused(lib.ung_hip_distill_backward(P, 0, 4, 4, 4, P, P, 2, None, None, t, P, 4, None), "temperature")
    _refused(lib.ung_hip_distill_step(P, 0, 4, 4, 4, P, P, 2, None, None, t, None, P, 4, None, 0, None), "temperature")


@pytest.mark.parametrize("t", [4.3e-39, 1e-38, 1e-3, 1.0, 1e30, 3e38])
def test_temperatures_that_are_served(t):
    _refused(F.load().ung_hip_top_scores(P, 0, 4, 4, 4, 2, t, None, P, P, None, 0, None), "null values")
