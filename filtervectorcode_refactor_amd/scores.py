"""Score operators on torch tensors: what trains the embedding model behind a base set and
scores queries against its table.  Thin calls of the C ABI's score operators
(include/ung_hip.h); work is enqueued on torch's current stream and nothing waits.

  quantize_fp8       rows to 8 bits with a scale for each block of 128, transposed too
  matmul_fp8         product of such operands; matmul_fp8_grad: its gradients
  linear_fp8         the differentiable layer made of them
  quantize_int8      rows to 8-bit whole numbers with a scale a row; matmul_int8: their product
  linear_int8        rows times a table kept in 8-bit whole numbers
  top_scores         first k scores of each row in (score, id) order, and log-sum-exp
  distill_forward, distill_backward, distill_step, distill_loss
                     the loss against a teacher's top scores: its passes, both passes in one
                     call, and the differentiable function
  entries_of_neighbors  neighbour rows (ids, distances) as a teacher's top scores
  table_loss_forward, table_loss_backward, table_loss
                     cross entropy against every row of a table, without the scores in memory: its
                     passes and the differentiable function
  gradient_norm, clip_gradients
                     the norm of many gradients together; the gradients scaled to a largest norm

linear_fp8, distill_loss and table_loss are differentiable, once; the passes and the 8-bit floating
products return results without a graph, and the results of top_scores, of the 8-bit whole numbers'
calls and of gradient_norm raise when they are differentiated.  Scores may have any row stride; bfloat16, float16 and float32.  A wrong argument raises
``ValueError`` or ``UngHipError``; there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
from array import array

import torch  # before libung_hip.so is loaded: one HIP runtime for both

from . import _lib
from ._lib import check

BLOCK = 128      # columns a scale stands for
MAX_K = 128      # longest list of top_scores and of the distillation
FP8 = torch.float8_e4m3fn
_BYTES = (FP8, torch.uint8)
_SAVED = 8       # floats a row that the backward pass of the distillation needs

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ready = None


def _library():
    """libung_hip.so, once it is known to share torch's HIP runtime: a process that loaded the
    library before torch has two of them, and neither knows the other's memory or streams."""
    global _ready
    if _ready is None:
        lib = _lib.load()
        with open("/proc/self/maps") as f:
            runtimes = {line.split()[-1] for line in f if "libamdhip64" in line}
        if len(runtimes) > 1:
            raise RuntimeError("import torch (or filtervectorcode_refactor_amd.scores) before libung_hip.so is "
                               f"loaded: two HIP runtimes are in this process ({', '.join(sorted(runtimes))})")
        _ready = lib
    return _ready


# The raw handle of a device's current stream, without making a torch.cuda.Stream of it (0.1
# against 2.6 us, a fifth of a small call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


class _On:
    """The device of a tensor made current for a call (HIP calls go to the current device)."""

    __slots__ = ("index", "before")

    def __init__(self, t):
        self.index = t.get_device()

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _need(ok, message):
    if not ok:
        raise ValueError(message)


# Messages are made only for an error: making one costs more than its check.
def _on_gpu(name, t, like=None):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ValueError(f"{name}: a tensor on the GPU is needed")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{name} is on another GPU")


def _matrix(name, t, like=None):
    """Checks a matrix of scores or rows; returns its type code and row stride."""
    _on_gpu(name, t, like)
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name}: float32, float16 or bfloat16 is needed, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name}: a matrix is needed, got {t.dim()} dimensions")
    rows, cols = t.shape
    stride, side = t.stride()
    if cols > 1 and side != 1:
        raise ValueError(f"{name}: elements of a row have to lie side by side")
    if rows > 1 and stride < cols:
        raise ValueError(f"{name}: rows overlap")
    return kind, max(stride, cols)


def _vector(name, t, n, like):
    """A row-wise float32 vector; one value for all rows (an expanded scalar) is laid out."""
    _on_gpu(name, t, like)
    if t.dtype != torch.float32 or tuple(t.shape) != (n,):
        raise ValueError(f"{name}: {n} float32 values are needed, got {tuple(t.shape)} of {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def _blocks(n):
    return -(-n // BLOCK)


def _workspace(fn, *args, device):
    """(tensor, address, bytes) of a call's workspace, from torch's allocator on its stream."""
    need = C.c_uint64()
    check(fn(*args, C.byref(need)))
    if not need.value:
        return None, None, 0
    t = torch.empty(need.value, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), need.value


class _Underivable(torch.autograd.Function):
    """Results that depend on `of` by kernels that autograd does not see: whoever differentiates
    them gets an error instead of a gradient without that part."""

    @staticmethod
    def forward(ctx, message, of, *results):
        ctx.message = message
        ctx.set_materialize_grads(False)
        return tuple(r if r is None else r.detach() for r in results)  # as themselves they could not be changed in place

    @staticmethod
    def backward(ctx, *grads):
        if any(g is not None for g in grads):
            raise RuntimeError(ctx.message)
        return (None,) * (len(grads) + 2)


def _once(name, *grads):
    """Gradients out of a backward pass; with create_graph they are marked as underivable."""
    if not torch.is_grad_enabled():
        return grads
    return _Underivable.apply(f"{name} has no second derivative", torch.zeros((), requires_grad=True), *grads)


def _marked(name, results, *of):
    """The results, of which none has a derivative by `of`: marked where one of those requires a gradient."""
    if torch.is_grad_enabled():
        for t in of:
            if t.requires_grad:
                return _Underivable.apply(f"{name} has no gradient: detach its result", t, *results)
    return results


# ---- 8-bit operands and their product -----------------------------------------------------
def quantize_fp8(x, block="row", transpose=False):
    """Rows as an 8-bit operand: (q, scale), with ``transpose`` (q, scale, qt, scale_t).

    q [n, columns rounded up to whole blocks of 128] float8_e4m3fn, padded with zeros; scale
    float32 [n, blocks] for ``block="row"`` (a scale for 128 columns of a row) or [blocks of n,
    blocks] for ``"square"`` (128 x 128).  qt [columns, n rounded up] is the transposed operand:
    quantised along its own rows (``"row"``), or the same values turned (``"square"``)."""
    kind, stride = _matrix("x", x)
    if block not in ("row", "square"):
        raise ValueError(f'block: "row" or "square" is needed, got {block!r}')
    with _On(x) as stream:
        return _quantize(x, kind, stride, block == "square", transpose, _library(), stream)


def _quantize(x, kind, row_stride, square, transpose, lib, stream):
    n, d = x.shape
    nb, db, device = _blocks(n), _blocks(d), x.device
    q = torch.empty(n, db * BLOCK, dtype=FP8, device=device)
    scale = torch.empty(nb if square else n, db, device=device)
    if not transpose:
        check(lib.ung_hip_fp8_quantize(x.data_ptr(), kind, n, d, row_stride, square, q.data_ptr(), scale.data_ptr(),
                                       None, None, stream))
        return q, scale
    qt = torch.empty(d, nb * BLOCK, dtype=FP8, device=device)
    scale_t = torch.empty(db if square else d, nb, device=device)
    check(lib.ung_hip_fp8_quantize(x.data_ptr(), kind, n, d, row_stride, square, q.data_ptr(), scale.data_ptr(),
                                   qt.data_ptr(), scale_t.data_ptr(), stream))
    return q, scale, qt, scale_t


def _transposed(x):
    """(qt, scale_t) of quantize_fp8(x, transpose=True) alone: the rows' own bytes are not written."""
    kind, stride = _matrix("x", x)
    n, d = x.shape
    qt = torch.empty(d, _blocks(n) * BLOCK, dtype=FP8, device=x.device)
    scale_t = torch.empty(d, _blocks(n), device=x.device)
    with _On(x) as stream:
        check(_library().ung_hip_fp8_quantize(x.data_ptr(), kind, n, d, stride, False, None, None, qt.data_ptr(),
                                              scale_t.data_ptr(), stream))
    return qt, scale_t


def _operand(name, q, scale, like=None):
    """Checks an operand; returns its rows, their length and whether its scales are by square."""
    _on_gpu(name, q, like)
    if q.dim() != 2 or q.dtype not in _BYTES or q.shape[1] % BLOCK or not q.is_contiguous():
        raise ValueError(f"{name}: contiguous float8_e4m3fn rows of a multiple of {BLOCK} bytes are needed, got "
                         f"{tuple(q.shape)} of {q.dtype}")
    _on_gpu(f"{name}_scale", scale, q)
    if scale.dtype != torch.float32 or not scale.is_contiguous():
        raise ValueError(f"{name}_scale: contiguous float32 is needed")
    (rows, kp), shape = q.shape, tuple(scale.shape)
    if shape == (rows, kp // BLOCK):
        return rows, kp, False
    if shape != (_blocks(rows), kp // BLOCK):
        raise ValueError(f"{name}_scale: ({rows}, {kp // BLOCK}) or ({_blocks(rows)}, {kp // BLOCK}) is needed, got "
                         f"{shape}")
    return rows, kp, True


def matmul_fp8(a, a_scale, b, b_scale, dtype=torch.bfloat16):
    """a b^T of two 8-bit operands (quantize_fp8) in ``dtype``; a with row scales, b with row
    or square ones.  Results are rounded once; float32 ones are summed in 32 bits throughout,
    16-bit ones by the 8-bit matrix instruction (errors of 1.4e-5 of their norm)."""
    m, kp, a_square = _operand("a", a, a_scale)
    n, b_kp, square = _operand("b", b, b_scale, a)
    if a_square:
        raise ValueError("a: row scales are needed")
    if dtype not in _TYPES:
        raise ValueError(f"dtype: float32, float16 or bfloat16 is needed, got {dtype}")
    if b_kp != kp:
        raise ValueError(f"a and b: rows of {kp} and {b_kp} bytes do not go together")
    with _On(a) as stream:
        return _product(a, a_scale, b, b_scale, square, m, n, kp, dtype, _library(), stream)


def _product(a, a_scale, b, b_scale, square, m, n, kp, dtype, lib, stream):
    kind, device = _TYPES[dtype], a.device
    c = torch.empty(m, n, dtype=dtype, device=device)
    keep, at, size = _workspace(lib.ung_hip_fp8_matmul_workspace, m, n, kp, kind, device=device)
    check(lib.ung_hip_fp8_matmul(a.data_ptr(), a_scale.data_ptr(), b.data_ptr(), b_scale.data_ptr(), square, m, n, kp,
                                 c.data_ptr(), kind, n, at, size, stream))
    return c


def matmul_fp8_grad(g, xt, xt_scale, wt, wt_scale):
    """Gradients of y = x w^T from g = dy: (dx in g's type, dw in float32).  xt, wt: the
    transposed operands of x (row scales along its rows) and of w (square or row scales), as
    quantize_fp8 gives them; g is brought to 8 bits both ways round in one pass."""
    kind, stride = _matrix("g", g)
    d, xt_len, xt_square = _operand("xt", xt, xt_scale, g)
    wt_rows, wt_len, wt_square = _operand("wt", wt, wt_scale, g)
    m, n = g.shape
    if wt_rows != d:
        raise ValueError("xt and wt: the same number of rows is needed")
    if xt_len != _blocks(m) * BLOCK:
        raise ValueError(f"xt: rows of {_blocks(m) * BLOCK} bytes are needed for {m} rows of g")
    if wt_len != _blocks(n) * BLOCK:
        raise ValueError(f"wt: rows of {_blocks(n) * BLOCK} bytes are needed for {n} columns of g")
    lib = _library()
    with _On(g) as stream:
        q, scale, qt, scale_t = _quantize(g, kind, stride, False, True, lib, stream)
        return (_product(q, scale, wt, wt_scale, wt_square, m, d, wt_len, g.dtype, lib, stream),
                _product(qt, scale_t, xt, xt_scale, xt_square, n, d, xt_len, torch.float32, lib, stream))


class _LinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, dtype):
        turn_x, turn_w = ctx.needs_input_grad[1], ctx.needs_input_grad[0]
        q, scale, *xt = quantize_fp8(x, transpose=turn_x)
        wq, w_scale, *wt = quantize_fp8(w, block="square", transpose=turn_w)
        ctx.save_for_backward(*xt, *wt)
        ctx.types = x.dtype, w.dtype
        return matmul_fp8(q, scale, wq, w_scale, dtype=dtype)

    @staticmethod
    def backward(ctx, g):
        g = g if g.stride(1) == 1 and g.stride(0) >= g.shape[1] else g.contiguous()
        saved, (x_type, w_type) = ctx.saved_tensors, ctx.types
        need_x, need_w = ctx.needs_input_grad[:2]
        dx = dw = None
        if need_x and need_w:
            xt, xt_scale, wt, wt_scale = saved
            dx, dw = matmul_fp8_grad(g, xt, xt_scale, wt, wt_scale)
        elif need_x:
            q, scale = quantize_fp8(g)
            dx = matmul_fp8(q, scale, *saved, dtype=g.dtype)
        elif need_w:
            dw = matmul_fp8(*_transposed(g), *saved, dtype=torch.float32)
        return *_once("linear_fp8", dx.to(x_type) if need_x else None, dw.to(w_type) if need_w else None), None


def linear_fp8(x, w, dtype=torch.bfloat16):
    """x w^T with both brought to 8 bits (x by rows, w by 128 x 128 squares), differentiable in
    both, once; its gradients are products in 8 bits too."""
    _matrix("x", x)
    _matrix("w", w, x)
    _need(x.shape[1] == w.shape[1], f"x and w: rows of {x.shape[1]} and {w.shape[1]} do not go together")
    return _LinearFp8.apply(x, w, dtype)


# ---- 8-bit whole numbers ------------------------------------------------------------------
def quantize_int8(x):
    """Rows in 8-bit whole numbers: (q int8 [n, columns rounded up to whole chunks of 128], padded
    with zeros; scale float32 [n]).  A row's scale is its largest magnitude / 127, an element's
    number the quotient by it to the nearest, ties to even.  A row with an infinity or NaN gets
    the scale NaN and zeros.  There is no gradient: of an x that requires one, differentiating the scale
    raises."""
    kind, stride = _matrix("x", x)
    n, d = x.shape
    q = torch.empty(n, _blocks(d) * BLOCK, dtype=torch.int8, device=x.device)
    scale = torch.empty(n, device=x.device)
    with _On(x) as stream:
        check(_library().ung_hip_int8_quantize(x.data_ptr(), kind, n, d, stride, q.data_ptr(), scale.data_ptr(), stream))
    return (q, *_marked("quantize_int8", (scale,), x))


def _numbers(name, q, scale, like=None):
    """Checks rows of whole numbers; returns how many there are and their length."""
    _on_gpu(name, q, like)
    if q.dim() != 2 or q.dtype != torch.int8 or q.shape[1] % BLOCK or not q.is_contiguous():
        raise ValueError(f"{name}: contiguous int8 rows of a multiple of {BLOCK} are needed, got {tuple(q.shape)} of "
                         f"{q.dtype}")
    _on_gpu(f"{name}_scale", scale, q)
    if scale.dtype != torch.float32 or tuple(scale.shape) != (q.shape[0],) or not scale.is_contiguous():
        raise ValueError(f"{name}_scale: contiguous float32 ({q.shape[0]},) is needed, got {tuple(scale.shape)} of "
                         f"{scale.dtype}")
    return q.shape


def matmul_int8(a, a_scale, b, b_scale, dtype=torch.bfloat16):
    """a b^T of rows in 8-bit whole numbers (quantize_int8) in ``dtype``: the sums are exact whole
    numbers, times both rows' scales in float32, rounded once to ``dtype``.  There is no gradient: of scales
    that require one, differentiating the result raises."""
    m, kp = _numbers("a", a, a_scale)
    n, b_kp = _numbers("b", b, b_scale, a)
    if dtype not in _TYPES:
        raise ValueError(f"dtype: float32, float16 or bfloat16 is needed, got {dtype}")
    if b_kp != kp:
        raise ValueError(f"a and b: rows of {kp} and {b_kp} bytes do not go together")
    kind, lib = _TYPES[dtype], _library()
    c = torch.empty(m, n, dtype=dtype, device=a.device)
    with _On(a) as stream:
        keep, at, size = _workspace(lib.ung_hip_int8_matmul_workspace, m, n, kp, kind, device=a.device)
        check(lib.ung_hip_int8_matmul(a.data_ptr(), a_scale.data_ptr(), b.data_ptr(), b_scale.data_ptr(), m, n, kp,
                                      c.data_ptr(), kind, n, at, size, stream))
    return _marked("matmul_int8", (c,), a_scale, b_scale)[0]


FEW_ROWS, FEW_LONG, FEW_TABLE = 4, 512, 200_000  # what linear_int8 takes in one launch, without a workspace


def _in_one_launch(m, d, n):
    return m <= FEW_ROWS and 0 < d <= FEW_LONG and n <= FEW_TABLE


def linear_int8(x, q, scale, dtype=torch.bfloat16):
    """x w^T with x brought to 8-bit whole numbers on the way and w kept in them (q, scale =
    quantize_int8(w), made once).  For answering: it has no gradient, and of an x or a scale that requires
    one, differentiating the result raises."""
    kind, stride = _matrix("x", x)
    n, kp = _numbers("q", q, scale, x)
    if dtype not in _TYPES:
        raise ValueError(f"dtype: float32, float16 or bfloat16 is needed, got {dtype}")
    m, d = x.shape
    if _blocks(d) * BLOCK != kp:
        raise ValueError(f"x and q: rows of {d} and {kp} do not go together")
    lib = _library()
    c = torch.empty(m, n, dtype=dtype, device=x.device)
    with _On(x) as stream:
        keep, at, size = (None, None, 0) if _in_one_launch(m, d, n) else \
            _workspace(lib.ung_hip_int8_linear_workspace, m, d, n, _TYPES[dtype], device=x.device)
        check(lib.ung_hip_int8_linear(x.data_ptr(), kind, m, d, stride, q.data_ptr(), scale.data_ptr(), n, c.data_ptr(),
                                      _TYPES[dtype], n, at, size, stream))
    return _marked("linear_int8", (c,), x, scale)[0]


# ---- the first scores of a row ------------------------------------------------------------
def top_scores(scores, k, temperature=1.0):
    """(values [n, k] float32, ids [n, k] int32, lse [n] float32): the first k scores of each
    row, larger first and of equal ones the lower id, and log sum exp(score / temperature) of
    the whole row.  Columns at -inf are not listed; missing entries are (-inf, -1).  There is no
    gradient: of scores that require one, differentiating values or lse raises."""
    kind, stride = _matrix("scores", scores)
    n, v = scores.shape
    if not 1 <= k <= MAX_K:
        raise ValueError(f"k={k} outside 1..{MAX_K}")
    values = torch.empty(n, k, device=scores.device)
    ids = torch.empty(n, k, dtype=torch.int32, device=scores.device)
    lse = torch.empty(n, device=scores.device)
    lib = _library()
    with _On(scores) as stream:
        keep, at, size = _workspace(lib.ung_hip_top_scores_workspace, scores.data_ptr(), kind, n, v, stride, k,
                                    device=scores.device)
        check(lib.ung_hip_top_scores(scores.data_ptr(), kind, n, v, stride, k, temperature, values.data_ptr(),
                                     ids.data_ptr(), lse.data_ptr(), at, size, stream))
    if scores.requires_grad and torch.is_grad_enabled():
        values, lse = _Underivable.apply("top_scores has no gradient: detach its values and log-sum-exp", scores,
                                         values, lse)
    return values, ids, lse


# ---- distillation ---------------------------------------------------------------------------
def entries_of_neighbors(ids, distances):
    """Neighbour rows (ids uint32/int32, missing ones UINT32_MAX / -1; squared distances, missing
    ones +inf) as a teacher's top scores: (ids int32, -distance float32)."""
    if str(ids.dtype).split(".")[-1] not in ("uint32", "int32"):
        raise ValueError(f"ids: uint32 or int32 is needed, got {ids.dtype}")
    ids = ids.view(torch.int32) if isinstance(ids, torch.Tensor) else torch.from_numpy(ids.view("int32"))
    distances = distances if isinstance(distances, torch.Tensor) else torch.from_numpy(distances)
    return ids, -distances.float()


def _teacher(scores, ids, values, lse):
    _on_gpu("ids", ids, scores)
    _on_gpu("values", values, scores)
    n, shape = scores.shape[0], ids.shape
    if len(shape) != 2 or shape[0] != n or ids.dtype != torch.int32:
        raise ValueError(f"ids: int32 [{n}, k] is needed, got {tuple(shape)} of {ids.dtype}")
    if values.shape != shape or values.dtype != torch.float32:
        raise ValueError(f"values: float32 {tuple(shape)} is needed, got {tuple(values.shape)} of {values.dtype}")
    if shape[1] > MAX_K:
        raise ValueError(f"k={shape[1]} outside 0..{MAX_K}")
    ids = ids if ids.is_contiguous() else ids.contiguous()
    values = values if values.is_contiguous() else values.contiguous()
    return ids, values, lse if lse is None else _vector("teacher_lse", lse, n, scores)


def _address(t):
    return None if t is None else t.data_ptr()


def _like_rows(scores, stride):
    """A tensor for the gradient whose rows lie as the scores' do; where those are slices of much
    wider ones (more than an eighth of a row lies between them), as close together as rows that
    begin at the same places of 16-byte vectors can."""
    n, v = scores.shape
    if stride - v > v // 8:
        stride = v + (stride - v) % (16 // scores.element_size())
    return torch.empty_strided((n, v), (stride, 1), dtype=scores.dtype, device=scores.device), stride


def distill_forward(scores, ids, values, teacher_lse=None, temperature=1.0):
    """(loss [n], saved): the loss of each row of the student's ``scores`` against the
    teacher's entries, and what distill_backward needs.

    Without ``teacher_lse`` the entries are the teacher's whole distribution (softmax over
    values / temperature); with it (log sum exp of all the teacher's scores / temperature, as
    top_scores returns) the rest of the teacher's mass stands against the student's mass outside
    the list.  Rows without an entry or without a score have loss 0."""
    kind, stride = _matrix("scores", scores)
    ids, values, lse = _teacher(scores, ids, values, teacher_lse)
    n, v = scores.shape
    loss = torch.empty(n, device=scores.device)
    saved = torch.empty(n, _SAVED, device=scores.device)
    lib = _library()
    with _On(scores) as stream:
        keep, at, size = _workspace(lib.ung_hip_distill_workspace, scores.data_ptr(), kind, n, v, stride,
                                    device=scores.device)
        check(lib.ung_hip_distill_forward(scores.data_ptr(), kind, n, v, stride, ids.data_ptr(), values.data_ptr(),
                                          ids.shape[1], _address(lse), temperature, loss.data_ptr(), saved.data_ptr(),
                                          at, size, stream))
    return loss, saved


def _written(out):
    """Tells autograd that a caller's tensor has been written: what was saved of it before is stale."""
    if out is not None and not out.is_inference():
        torch.autograd.graph.increment_version(out)


def _gradient(scores, stride, out):
    if out is None:
        return _like_rows(scores, stride)
    _need(out.dtype == scores.dtype and out.shape == scores.shape, "out: the scores' shape and type are needed")
    _, out_stride = _matrix("out", out, scores)
    _need(out.data_ptr() != scores.data_ptr() or out_stride == stride, "out: in place, the scores' rows are needed")
    return out, out_stride


def distill_backward(weight, scores, ids, values, saved, teacher_lse=None, temperature=1.0, out=None):
    """Gradient of sum(weight * loss) by the scores, in their type; the arguments are those of
    the forward call (teacher_lse is part of ``saved`` already).  ``out`` may be the scores
    themselves, which the gradient then replaces, but not overlap them otherwise; by default it is
    a new tensor whose rows lie as theirs, but without wide gaps."""
    kind, stride = _matrix("scores", scores)
    ids, values, _ = _teacher(scores, ids, values, teacher_lse)
    n, v = scores.shape
    _on_gpu("saved", saved, scores)
    _need(tuple(saved.shape) == (n, _SAVED) and saved.dtype == torch.float32 and saved.is_contiguous(),
          "saved: what distill_forward returned is needed")
    weight = None if weight is None else _vector("weight", weight, n, scores)
    grad, grad_stride = _gradient(scores, stride, out)
    with _On(scores) as stream:
        check(_library().ung_hip_distill_backward(scores.data_ptr(), kind, n, v, stride, ids.data_ptr(),
                                                  values.data_ptr(), ids.shape[1], saved.data_ptr(), _address(weight),
                                                  temperature, grad.data_ptr(), grad_stride, stream))
    _written(out)
    return grad


def distill_step(scores, ids, values, weight=None, teacher_lse=None, temperature=1.0, out=None):
    """(loss, gradient of sum(weight * loss)) in one call: where a row fits a block's registers,
    with one read of the scores and one write of the gradient."""
    kind, stride = _matrix("scores", scores)
    ids, values, lse = _teacher(scores, ids, values, teacher_lse)
    n, v = scores.shape
    weight = None if weight is None else _vector("weight", weight, n, scores)
    loss = torch.empty(n, device=scores.device)
    grad, grad_stride = _gradient(scores, stride, out)
    lib = _library()
    with _On(scores) as stream:
        keep, at, size = _workspace(lib.ung_hip_distill_workspace, scores.data_ptr(), kind, n, v, stride,
                                    device=scores.device)
        check(lib.ung_hip_distill_step(scores.data_ptr(), kind, n, v, stride, ids.data_ptr(), values.data_ptr(),
                                       ids.shape[1], _address(lse), _address(weight), temperature, loss.data_ptr(),
                                       grad.data_ptr(), grad_stride, at, size, stream))
    _written(out)
    return loss, grad


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, ids, values, teacher_lse, temperature):
        loss, saved = distill_forward(scores, ids, values, teacher_lse, temperature)
        ctx.save_for_backward(scores, ids, values, saved)
        ctx.temperature = temperature
        return loss

    @staticmethod
    def backward(ctx, g):
        scores, ids, values, saved = ctx.saved_tensors
        grad = distill_backward(g, scores, ids, values, saved, temperature=ctx.temperature)
        return *_once("distill_loss", grad), None, None, None, None


def distill_loss(scores, ids, values, teacher_lse=None, temperature=1.0):
    """The loss of each row (distill_forward), differentiable in the scores, once; the teacher's
    side is taken as given."""
    return _DistillLoss.apply(scores, ids, values, teacher_lse, temperature)


# ---- cross entropy against a table -----------------------------------------------------------
def _against(x, table, ids, without):
    kind, stride = _matrix("x", x)
    table_kind, table_stride = _matrix("table", table, x)
    n, d = x.shape
    if table_kind != kind or table.shape[1] != d:
        raise ValueError(f"table: rows of {d} elements of {x.dtype} are needed, got {table.shape[1]} of {table.dtype}")
    out = []
    for name, t in (("ids", ids), ("without", without)):
        if t is not None:
            _on_gpu(name, t, x)
            if t.dtype != torch.int32 or tuple(t.shape) != (n,):
                raise ValueError(f"{name}: int32 ({n},) is needed, got {tuple(t.shape)} of {t.dtype}")
            t = t if t.is_contiguous() else t.contiguous()
        out.append(t)
    if out[0] is None:
        raise ValueError("ids: a tensor on the GPU is needed")
    return (x.data_ptr(), stride, table.data_ptr(), table_stride, kind, n, table.shape[0], d), *out


def table_loss_forward(x, table, ids, without=None, temperature=1.0):
    """(loss [n], lse [n]) float32: cross entropy of each row of ``x`` with row ``ids`` of the table
    as its target, scores being x table^T / temperature, and the log-sum-exp of all its scores,
    which table_loss_backward needs.  A large batch's scores are never in memory.  Rows of x times rows of
    the table may be up to about 2.7e11 in float32, 5.4e11 in 16 bits; more are refused.

    ``without`` names one row of the table that each row of x leaves out (its own entry; -1: none).
    A row whose id is outside the table, or the one left out, has no target: its loss is 0."""
    sizes, ids, without = _against(x, table, ids, without)
    n, device = x.shape[0], x.device
    loss, lse = torch.empty(n, device=device), torch.empty(n, device=device)
    lib = _library()
    with _On(x) as stream:
        keep, at, size = _workspace(lib.ung_hip_table_loss_workspace, *sizes, False, device=device)
        check(lib.ung_hip_table_loss_forward(*sizes, ids.data_ptr(), _address(without), temperature, loss.data_ptr(),
                                             lse.data_ptr(), at, size, stream))
    return loss, lse


def table_loss_backward(weight, x, table, ids, lse, without=None, temperature=1.0, need=(True, True)):
    """Gradients of sum(weight * loss) by x and by the table, in their type; the arguments are those
    of the forward call and its log-sum-exp.  ``need``: which of the two to make (the other is
    None).  All weights of a row are off together by lse's one rounding: half its step, 1e-6 of
    themselves at scores of 20, 3e-5 at 1000 (and all of them past 1e7).  Rows without a target are not read: padding of any value, NaN too, may stand there."""
    sizes, ids, without = _against(x, table, ids, without)
    n, device = x.shape[0], x.device
    lse = _vector("lse", lse, n, x)
    weight = None if weight is None else _vector("weight", weight, n, x)
    dx = torch.empty(x.shape, dtype=x.dtype, device=device) if need[0] else None
    dtable = torch.empty(table.shape, dtype=x.dtype, device=device) if need[1] else None
    lib = _library()
    with _On(x) as stream:
        keep, at, size = _workspace(lib.ung_hip_table_loss_workspace, *sizes, True, device=device)
        check(lib.ung_hip_table_loss_backward(*sizes, ids.data_ptr(), _address(without), lse.data_ptr(),
                                              _address(weight), temperature, _address(dx), x.shape[1],
                                              _address(dtable), x.shape[1], at, size, stream))
    return dx, dtable


class _TableLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, table, ids, without, temperature):
        loss, lse = table_loss_forward(x, table, ids, without, temperature)
        ctx.save_for_backward(x, table, ids, without, lse)
        ctx.temperature = temperature
        return loss

    @staticmethod
    def backward(ctx, g):
        x, table, ids, without, lse = ctx.saved_tensors
        grads = table_loss_backward(g, x, table, ids, lse, without, ctx.temperature, ctx.needs_input_grad[:2])
        return *_once("table_loss", *grads), None, None, None


def table_loss(x, table, ids, without=None, temperature=1.0):
    """The loss of each row (table_loss_forward), differentiable in x and the table, once."""
    return _TableLoss.apply(x, table, ids, without, temperature)


# ---- gradients of a step -----------------------------------------------------------------------
def _side_by_side(t):
    """Whether a tensor's elements fill a stretch of memory, in any order of its dimensions."""
    if t.is_contiguous():
        return True
    room = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != room:
            return False
        room *= size
    return True


def _checked(name, tensors):
    """Why a list of tensors is refused."""
    for t in tensors:
        _on_gpu(name, t, tensors[0])
        if t.dtype not in _TYPES:
            raise ValueError(f"{name}: float32, float16 or bfloat16 is needed, got {t.dtype}")
        if not _side_by_side(t):
            raise ValueError(f"{name}: elements have to lie side by side, got strides {t.stride()} of {tuple(t.shape)}")


def _addresses(name, tensors):
    """(type codes, addresses) of tensors on one GPU whose elements lie side by side.  Many at a time:
    a call for each tensor and property costs more than the kernels of small ones."""
    try:
        kinds = [_TYPES[t.dtype] for t in tensors]
        fine = min(devices := set(map(torch.Tensor.get_device, tensors))) >= 0 and len(devices) == 1 and \
            all(map(torch.Tensor.is_contiguous, tensors))
    except (KeyError, TypeError, AttributeError):
        fine = False
    if not fine:
        _checked(name, tensors)
    return kinds, array("Q", map(torch.Tensor.data_ptr, tensors))


def _gradient_list(grads):
    grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("grads: at least one tensor is needed")
    kinds, at = _addresses("grads", grads)
    return grads, kinds, at, array("i", kinds), array("Q", map(torch.Tensor.numel, grads))


def _address_of(a):
    return a.buffer_info()[0]


def gradient_norm(grads):
    """The norm of all gradients together, a float32 tensor of no dimensions: the root of the sum
    of every element's square, made in 64 bits.  ``grads``: tensors on one GPU (None is skipped)
    of any types and shapes."""
    grads, _, at, types, sizes = _gradient_list(grads)
    norm, count, sizes_at = torch.empty((), device=grads[0].device), len(grads), _address_of(sizes)
    lib = _library()
    with _On(grads[0]) as stream:
        keep, work, size = _workspace(lib.ung_hip_gradient_workspace, sizes_at, count, device=norm.device)
        check(lib.ung_hip_gradient_norm(_address_of(at), _address_of(types), sizes_at, count, norm.data_ptr(), work, size,
                                        stream))
    if torch.is_grad_enabled():
        for g in grads:
            if g.requires_grad:
                return _Underivable.apply("gradient_norm has no gradient: detach it", g, norm)[0]
    return norm


def clip_gradients(grads, max_norm, out=None):
    """Scales the gradients by min(1, max_norm / norm) of their norm together, which it returns
    (gradient_norm).  In place, or to ``out``: as many tensors of the same types and shapes, laid out
    the same way.  Nothing waits for the norm.  Where it is infinite or NaN the gradients stay as
    they are, so that a program that asks later can leave the step out.  Tensors that require a gradient
    (parameters instead of their gradients) are refused but under torch.no_grad()."""
    given = list(grads)
    grads, kinds, at, types, sizes = _gradient_list(given)
    written, to, to_at = grads, None, None
    if out is not None:
        out = list(out)
        if len(out) != len(given):
            raise ValueError(f"out: {len(given)} tensors are needed, got {len(out)}")
        written = [o for o, g in zip(out, given) if g is not None]
        to_kinds, to = _addresses("out", written)
        to_at = _address_of(to)
        if kinds != to_kinds or list(map(torch.Tensor.size, written)) != list(map(torch.Tensor.size, grads)) or \
                written[0].get_device() != grads[0].get_device() or \
                not all(o.is_contiguous() and g.is_contiguous() or o.stride() == g.stride() for o, g in zip(written, grads)):
            raise ValueError("out: the gradients' shapes, types and strides are needed")
    if torch.is_grad_enabled():
        for t in (*grads, *written):
            if t.requires_grad:  # (parameters in their gradients' place among them)
                raise ValueError("grads: tensors that require a gradient themselves are clipped under torch.no_grad(); "
                                 "a parameter's gradient is its .grad")
    norm, count, sizes_at = torch.empty((), device=grads[0].device), len(grads), _address_of(sizes)
    lib = _library()
    with _On(grads[0]) as stream:
        keep, work, size = _workspace(lib.ung_hip_gradient_workspace, sizes_at, count, device=norm.device)
        check(lib.ung_hip_clip_gradients(_address_of(at), to_at, _address_of(types), sizes_at, count, max_norm,
                                         norm.data_ptr(), work, size, stream))
    torch.autograd.graph.increment_version(written)
    return norm
