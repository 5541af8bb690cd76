"""The C entry points of the table loss, the 8-bit whole numbers and the gradients refuse wrong
arguments before anything is enqueued, and say what is wrong.  No GPU: the calls here never get as
far as a launch."""
import ctypes as C

import numpy as np
import pytest
import torch

import filtervectorcode_refactor_amd as F
from filtervectorcode_refactor_amd import _lib
from filtervectorcode_refactor_amd import scores as S

BUF = np.zeros(4096, np.uint8)
P = (BUF.ctypes.data + 63) // 64 * 64  # never read: every call below is refused
NAN, INF = float("nan"), float("inf")


def _refused(rc, *words):
    assert rc == _lib.UNG_HIP_EINVAL
    for w in words:
        assert w in _lib.last_error(), _lib.last_error()


def test_int8_quantize():
    f = F.load().ung_hip_int8_quantize
    _refused(f(P, 9, 4, 4, 4, P, P, None), "type 9")
    _refused(f(None, 0, 4, 4, 4, P, P, None), "null")
    _refused(f(P, 0, 4, 4, 4, None, P, None), "null")
    _refused(f(P, 0, 4, 4, 4, P, None, None), "null")
    _refused(f(P, 0, 4, 4, 3, P, P, None), "row_stride 3")
    _refused(f(P, 0, 4, 4, 4, P + 8, P, None), "alignment")
    _refused(f(P + 1, 1, 4, 4, 4, P, P, None), "alignment")
    _refused(f(P, 0, 1 << 40, 4, 4, P, P, None), "too many")
    assert f(None, 0, 0, 4, 4, None, None, None) == 0


def test_int8_matmul():
    f = F.load().ung_hip_int8_matmul
    _refused(f(P, P, P, P, 4, 4, 100, P, 0, 4, None, 0, None), "100")
    _refused(f(P, P, P, P, 4, 4, 131072, P, 0, 4, None, 0, None), "131072")
    _refused(f(P, P, P, P, 4, 4, 128, P, 5, 4, None, 0, None), "type 5")
    _refused(f(P, None, P, P, 4, 4, 128, P, 0, 4, None, 0, None), "null")
    _refused(f(P, P, None, P, 4, 4, 128, P, 0, 4, None, 0, None), "null")
    _refused(f(P, P, P, P, 4, 4, 128, None, 0, 4, None, 0, None), "null")
    _refused(f(P, P, P, P, 4, 4, 128, P, 0, 3, None, 0, None), "c_stride 3")
    _refused(f(P + 1, P, P, P, 4, 4, 128, P, 0, 4, None, 0, None), "alignment")
    _refused(f(P, P, P, P, 1 << 33, 4, 128, P, 0, 4, None, 0, None), "too large")
    _refused(f(P, P, P, P, 1 << 30, 1 << 30, 128, P, 0, 1 << 30, None, 0, None), "too large")
    assert f(None, None, None, None, 0, 4, 128, None, 0, 4, None, 0, None) == 0
    _refused(F.load().ung_hip_int8_matmul_workspace(4, 4, 128, 0, None), "null")


def test_int8_linear():
    lib = F.load()
    f = lib.ung_hip_int8_linear
    _refused(f(P, 9, 4, 4, 4, P, P, 4, P, 0, 4, None, 0, None), "type 9")
    _refused(f(P, 0, 4, 4, 4, P, P, 4, P, 9, 4, None, 0, None), "type 9")
    _refused(f(None, 0, 4, 4, 4, P, P, 4, P, 0, 4, None, 0, None), "null")
    _refused(f(P, 0, 4, 4, 4, None, P, 4, P, 0, 4, None, 0, None), "null")
    _refused(f(P, 0, 4, 4, 4, P, None, 4, P, 0, 4, None, 0, None), "null")
    _refused(f(P, 0, 4, 4, 4, P, P, 4, None, 0, 4, None, 0, None), "null")
    _refused(f(P, 0, 4, 4, 3, P, P, 4, P, 0, 4, None, 0, None), "row_stride 3")
    _refused(f(P, 0, 4, 4, 4, P, P, 4, P, 0, 3, None, 0, None), "c_stride 3")
    _refused(f(P + 2, 0, 4, 4, 4, P, P, 4, P, 0, 4, None, 0, None), "aligned")
    _refused(f(P, 0, 4, 4, 4, P + 8, P, 4, P, 0, 4, None, 0, None), "alignment")
    _refused(f(P, 0, 4, 130945, 130945, P, P, 4, P, 0, 4, None, 0, None), "131072")
    _refused(f(P, 0, 1 << 33, 4, 4, P, P, 4, P, 0, 4, None, 0, None), "too large")
    need = C.c_uint64()
    # what scores.linear_int8 counts on: no workspace for few short rows, one past each bound
    for rows, cols, n, none in ((S.FEW_ROWS, S.FEW_LONG, S.FEW_TABLE, True), (S.FEW_ROWS + 1, 4, 4, False),
                                (1, S.FEW_LONG + 1, 4, False), (1, 4, S.FEW_TABLE + 1, False)):
        assert lib.ung_hip_int8_linear_workspace(rows, cols, n, 0, C.byref(need)) == 0 and (need.value == 0) == none
    assert lib.ung_hip_int8_linear_workspace(5, 4, 4, 0, C.byref(need)) == 0
    _refused(f(P, 0, 5, 4, 4, P, P, 4, P, 0, 4, P, need.value - 1, None), "workspace")
    _refused(f(P, 0, 5, 4, 4, P, P, 4, P, 0, 4, None, need.value, None), "workspace")
    _refused(lib.ung_hip_int8_linear_workspace(5, 4, 4, 0, None), "null")
    _refused(lib.ung_hip_int8_linear_workspace(5, 4, 4, 7, C.byref(need)), "type 7")
    assert f(None, 0, 0, 4, 4, None, None, 4, None, 0, 4, None, 0, None) == 0


def _sizes(type=0, n=4, v=8, d=4, xs=4, ts=4, x=P, t=P):
    return x, xs, t, ts, type, n, v, d


def test_table_loss():
    lib = F.load()
    need = C.c_uint64()
    for backward in (0, 1):
        assert lib.ung_hip_table_loss_workspace(*_sizes(), backward, C.byref(need)) == 0 and need.value > 0
        size = need.value

        def f(sizes=_sizes(), ids=P, without=None, temperature=1.0, a=P, b=P, ws=P, bytes_=size, **kw):
            if not backward:
                return lib.ung_hip_table_loss_forward(*sizes, ids, without, temperature, a, b, ws, bytes_, None)
            return lib.ung_hip_table_loss_backward(*sizes, ids, without, kw.get("lse", P), kw.get("weight"), temperature, a,
                                                   kw.get("dxs", 4), b, kw.get("dts", 4), ws, bytes_, None)

        _refused(f(_sizes(type=3)), "type 3")
        _refused(f(_sizes(n=1 << 40)), "too many")
        _refused(f(_sizes(v=1 << 31)), "too many")
        _refused(f(_sizes(d=(1 << 20) + 1, xs=1 << 21, ts=1 << 21)), "too many")
        _refused(f(_sizes(n=(1 << 27) + 1, v=0)), "too many")
        _refused(f(_sizes(n=1 << 24, v=1 << 24)), "too many")
        _refused(f(_sizes(xs=3)), "strides 3")
        _refused(f(_sizes(ts=3)), "and 3")
        _refused(f(_sizes(x=P + 2)), "aligned")
        _refused(f(_sizes(t=P + 1)), "aligned")
        for t in (0.0, -1.0, NAN, INF, 1e-45):
            _refused(f(temperature=t), "temperature")
        _refused(f(ids=None), "null")
        _refused(f(ids=P + 2), "aligned")
        _refused(f(without=P + 2), "aligned")
        _refused(f(_sizes(x=None), bytes_=1 << 20), "null")
        _refused(f(_sizes(t=None), bytes_=1 << 20), "null")
        _refused(f(ws=None), "workspace")
        _refused(f(bytes_=size - 1), "workspace")
        _refused(f(ws=P + 4), "workspace")
        if backward:
            _refused(f(lse=None), "null lse")
            _refused(f(weight=P + 2), "weight")
            _refused(f(a=P + 2), "dx")
            _refused(f(dxs=3), "strides 3")
            _refused(f(dts=3), "and 3")
            assert f(a=None, b=None) == 0
        else:
            _refused(f(a=None), "loss")
            _refused(f(b=P + 1), "lse")
            assert f(_sizes(n=0)) == 0
    _refused(lib.ung_hip_table_loss_workspace(*_sizes(), 0, None), "null")
    _refused(lib.ung_hip_table_loss_workspace(*_sizes(type=-1), 0, C.byref(need)), "type -1")


def _list(*sizes, at=P, types=0):
    n = len(sizes)
    where = at if isinstance(at, list) else [at + 512 * i for i in range(n)]
    kinds = types if isinstance(types, list) else [types] * n
    return (C.c_void_p * n)(*where), (C.c_int * n)(*kinds), (C.c_uint64 * n)(*sizes), n


def test_gradients():
    lib = F.load()
    need = C.c_uint64()
    grads, types, sizes, n = _list(10, 0, 100)
    assert lib.ung_hip_gradient_workspace(sizes, n, C.byref(need)) == 0 and need.value >= 24
    size = need.value
    norm, clip = lib.ung_hip_gradient_norm, lib.ung_hip_clip_gradients
    _refused(lib.ung_hip_gradient_workspace(sizes, n, None), "null")
    _refused(lib.ung_hip_gradient_workspace(None, 2, C.byref(need)), "null")
    _refused(norm(None, types, sizes, n, P, P, size, None), "null")
    _refused(norm(grads, types, sizes, n, None, P, size, None), "norm")
    _refused(norm(grads, types, sizes, n, P + 2, P, size, None), "norm")
    _refused(norm(grads, types, sizes, n, P, None, size, None), "workspace")
    _refused(norm(grads, types, sizes, n, P, P, size - 1, None), "workspace")
    _refused(norm(grads, types, sizes, n, P, P + 8, size, None), "workspace")
    for at, kinds, words in (([P, P, None], 0, "tensor 2 is null"), ([P, P, P + 2], 0, "tensor 2 is null or not aligned"),
                             (P, [0, 0, 7], "type 7 of tensor 2")):
        g, k, s, _ = _list(10, 0, 100, at=at, types=kinds)
        _refused(norm(g, k, s, n, P, P, size, None), words)
        _refused(clip(g, None, k, s, n, 1.0, P, P, size, None), words)
    g, k, s, _ = _list(1 << 41)
    _refused(norm(g, k, s, 1, P, P, 1 << 40, None), "too many")
    for most in (-1.0, NAN, -INF):
        _refused(clip(grads, None, types, sizes, n, most, P, P, size, None), "negative or NaN")


@pytest.mark.parametrize("grads,out", [
    ([P, P], None), ([P, P + 396], None), ([P, P + 1024], [P + 1024, P]), ([P], [P + 4]), ([P + 4], [P]),
    ([P, P + 1024], [P + 2048, P + 2444]), ([P, P + 1024], [P + 2048, P + 100]),
])
def test_gradients_that_overlap(grads, out):
    lib = F.load()
    g, k, s, n = _list(*[100] * len(grads), at=grads)
    to = None if out is None else (C.c_void_p * n)(*out)
    _refused(lib.ung_hip_clip_gradients(g, to, k, s, n, 1.0, P, P, 1 << 16, None), "overlap")


def test_tensors_on_the_cpu_are_refused():
    x, ids = torch.randn(4, 128), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: S.table_loss_forward(x, x, ids), lambda: S.table_loss(x, x, ids),
                 lambda: S.table_loss_backward(None, x, x, ids, x[:, 0]), lambda: S.quantize_int8(x),
                 lambda: S.linear_int8(x, x.to(torch.int8), x[:, 0]), lambda: S.gradient_norm([x]),
                 lambda: S.clip_gradients([x], 1.0)):
        with pytest.raises(ValueError, match="a tensor on the GPU is needed"):
            call()


def test_table_loss_in_autograd(monkeypatch):
    """Plain forms in the kernels' place: which gradients are asked for, and that there is no second
    derivative."""
    asked = []

    def backward(weight, x, table, ids, lse, without=None, temperature=1.0, need=(True, True)):
        asked.append(tuple(need))
        return tuple(t.new_ones(t.shape) * weight.sum() if n else None for t, n in zip((x, table), need))

    monkeypatch.setattr(S, "table_loss_forward", lambda x, t, ids, without, temperature: (x.sum(1), x.sum(1)))
    monkeypatch.setattr(S, "table_loss_backward", backward)
    ids = torch.zeros(5, dtype=torch.int32)
    x, t = torch.randn(5, 8, requires_grad=True), torch.randn(6, 8, requires_grad=True)
    S.table_loss(x, t, ids).sum().backward()
    S.table_loss(x, t.detach(), ids).sum().backward()
    S.table_loss(x.detach(), t, ids).sum().backward()
    assert asked == [(True, True), (True, False), (False, True)]
    assert torch.equal(x.grad, torch.full((5, 8), 10.0)) and torch.equal(t.grad, torch.full((6, 8), 10.0))
    (dx,) = torch.autograd.grad(S.table_loss(x, t, ids).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        dx.square().sum().backward()


def test_the_rule_for_one_launch_is_the_librarys():
    """Where scores.linear_int8 brings no workspace the library needs none, from no columns on."""
    need = C.c_uint64()
    for rows in (0, 1, S.FEW_ROWS, S.FEW_ROWS + 1):
        for cols in (0, 1, 128, S.FEW_LONG, S.FEW_LONG + 1):
            for n in (0, 1, S.FEW_TABLE, S.FEW_TABLE + 1):
                assert F.load().ung_hip_int8_linear_workspace(rows, cols, n, 0, C.byref(need)) == 0
                assert not S._in_one_launch(rows, cols, n) or need.value == 0, (rows, cols, n)
                if rows and n:
                    assert S._in_one_launch(rows, cols, n) == (need.value == 0), (rows, cols, n)


@pytest.mark.parametrize("type,n,v,d,fine", [
    (2, 65_536, 1_000_000, 64, True), (2, 400_000, 1_300_000, 64, True), (2, 1 << 20, 1 << 20, 64, False),
    (0, 100_000, 2_000_000, 64, True), (0, 1 << 19, 1 << 20, 64, False), (1, 1 << 27, 1000, 8, True),
    (2, 1 << 27, 1 << 20, 8, False), (2, 32, (1 << 31) - 1000, 64, True), (2, 1, (1 << 31) - 1000, 64, True), (2, 20_000_000, 100, 2048, True),
])
def test_table_loss_takes_what_its_launches_take(type, n, v, d, fine):
    """Threads of a launch are counted in 32 bits: 2^23 tiles of 256 x 256 scores in 16 bits, 2^24 of 128 x 128
    in 32; the backward pass, which is launched in pieces, refuses what the forward pass does."""
    need = C.c_uint64()
    for backward in (0, 1):
        rc = F.load().ung_hip_table_loss_workspace(*_sizes(type, n, v, d, d, d), backward, C.byref(need))
        if fine:
            assert rc == 0 and need.value > 0, _lib.last_error()
        else:
            _refused(rc, "too many")
