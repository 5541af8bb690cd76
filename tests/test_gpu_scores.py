"""GPU tests of the score operators (filtervectorcode_refactor_amd.scores) against plain
implementations in 64 bits on the host, at the sizes, strides, types and masks where they can
go wrong.  Quantised bytes, scales, ids and listed scores are compared for equality; computed
values with bounds that follow from the number of roundings (stated at each)."""
import math

import numpy as np
import pytest
import torch

import filtervectorcode_refactor_amd as F
from filtervectorcode_refactor_amd import scores as S

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"fp32": 2.0 ** -126, "fp16": 2.0 ** -25, "bf16": 2.0 ** -126}  # below: absolute steps
EPS = 2.0 ** -23  # a 32-bit operation's error, rounding or truncating


def _say(*a):
    print(*a, flush=True)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- quantisation ---------------------------------------------------------------------------
def _blocks(n):
    return -(-n // 128)


def _quantized(x, block):
    """q (as float32 values) and scale of a float32 matrix, by numpy's IEEE division and torch's
    conversion on the CPU."""
    n, d = x.shape
    nb, db = _blocks(n), _blocks(d)
    hi = n if block == "row" else nb
    q, scale = torch.zeros(n, db * 128), torch.zeros(hi, db)
    for i in range(hi):
        rows = slice(i, i + 1) if block == "row" else slice(i * 128, (i + 1) * 128)
        for j in range(db):
            piece = x[rows, j * 128:(j + 1) * 128]
            most = max(float(piece.abs().max()), 2.0 ** -64)
            s = np.float32(most) * (np.float32(1) / np.float32(448))
            scale[i, j] = float(s)
            y = torch.from_numpy(piece.numpy() / s)
            q[rows, j * 128:j * 128 + piece.shape[1]] = y.to(torch.float8_e4m3fn).float()
    return q, scale


QUANT = [(1, 1), (1, 128), (3, 100), (128, 128), (129, 257), (77, 384), (300, 1000), (5, 130)]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,d", QUANT)
def test_quantize(n, d, kind):
    g = _gen(n * 1000 + d)
    x = (torch.randn(n, d, generator=g) * torch.exp(torch.randn(n, d, generator=g) * 2)).to(TYPES[kind])
    x[0, 0] = 0.0
    if n > 2:
        x[1] = 0.0  # a block of zeros
    for pad in (0, 8, 3):  # 3: rows off every 16-byte boundary
        whole = torch.full((n, d + pad), 7.0, dtype=TYPES[kind], device="cuda")
        whole[:, :d] = x
        view = whole[:, :d]
        for block in ("row", "square"):
            q, scale = S.quantize_fp8(view, block=block)
            want_q, want_s = _quantized(x.float(), block)
            assert torch.equal(q.float().cpu(), want_q) and torch.equal(scale.cpu(), want_s), (pad, block)
            q2, scale2, qt, scale_t = S.quantize_fp8(view, block=block, transpose=True)
            assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(scale2, scale)
            if block == "row":
                want_t, want_st = _quantized(x.float().t().contiguous(), "row")
            else:
                want_t = torch.zeros(d, _blocks(n) * 128)
                want_t[:, :n] = want_q[:, :d].t()
                want_st = want_s.t()
            assert torch.equal(qt.float().cpu(), want_t) and torch.equal(scale_t.cpu(), want_st), (pad, block)


def test_quantize_extremes():
    """Subnormals, values below the smallest scale, the type's largest, infinities and NaN."""
    x = torch.zeros(6, 256)
    x[0, 3], x[0, 200] = 2.0 ** -70, -1e-44
    x[1, :4] = torch.tensor([3.0e38, -1.0, 1e30, 2.0 ** -126])
    x[2, :3] = torch.tensor([math.inf, 1.0, 2.0])
    x[3, 5], x[3, 6] = math.nan, 1.0
    x[4, :2] = torch.tensor([-math.inf, math.inf])
    x[5, 250] = 5.0
    q, scale = S.quantize_fp8(x.cuda())
    q, scale = q.float().cpu(), scale.cpu()
    keep = [0, 1, 5]
    want_q, want_s = _quantized(x[keep], "row")
    assert torch.equal(q[keep], want_q) and torch.equal(scale[keep], want_s)
    values = q * scale.repeat_interleave(128, dim=1)
    for row in (2, 3, 4):  # the block is spoilt as a whole, the row's other block is not
        assert not torch.isfinite(values[row, :128]).any()
        assert torch.equal(values[row, 128:], torch.zeros(128))


# ---- product ----------------------------------------------------------------------------------
def _operand(n, d, block, g):
    x = torch.randn(n, d, generator=g) * torch.exp(torch.randn(n, 1, generator=g))
    q, scale = S.quantize_fp8(x.cuda(), block=block)
    s = scale.cpu().double()
    rows = torch.arange(n) if block == "row" else torch.arange(n) // 128
    return q, scale, q.float().cpu().double() * s[rows].repeat_interleave(128, dim=1)


def _product_bound(a, b, c, kind):
    """Error of the product: every term passes at most kp + 2 blocks + 2 operations of 32 bits
    on its way into the sum (its block's sum, the scales' product, the running sum), then the
    result is rounded once.  16-bit results: each of eight neighbouring products loses less
    than 2^-13 of the largest of them, 8 2^-13 of it in all, which is at most that of their sum."""
    kp = a.shape[1]
    inner = 2.0 ** -10 if kind != "fp32" else 0.0
    return ((kp + 2 * kp // 128 + 2) * EPS + inner) * (a.abs() @ b.abs().t()) + HALF_ULP[kind] * c.abs() * 1.001 + TINY[kind]


PRODUCTS = [(1, 1, 1), (1, 129, 100), (2, 1000, 768), (16, 16, 128), (17, 300, 384), (33, 77, 2000), (64, 130, 100),
            (65, 129, 768), (128, 128, 128), (130, 257, 384), (256, 300, 1000), (300, 511, 130), (5, 4100, 129),
            (3, 40, 5000), (48, 200, 9000), (700, 200, 64)]


@pytest.mark.parametrize("block", ["row", "square"])
@pytest.mark.parametrize("m,n,d", PRODUCTS)
def test_product(m, n, d, block):
    g = _gen(m * 7 + n * 3 + d)
    qa, sa, a = _operand(m, d, "row", g)
    qb, sb, b = _operand(n, d, block, g)
    want = a @ b.t()
    for kind, dtype in TYPES.items():
        got = S.matmul_fp8(qa, sa, qb, sb, dtype=dtype)
        assert got.dtype == dtype and tuple(got.shape) == (m, n)
        if kind == "fp16" and want.abs().max() > 60000:
            continue
        err = (got.cpu().double() - want).abs()
        assert (err <= _product_bound(a, b, want, kind)).all(), (kind, float((err - _product_bound(a, b, want, kind)).max()))


def test_product_is_the_same_every_time():
    g = _gen(5)
    for m, n, d in ((3, 500, 4096), (40, 128, 8192), (300, 300, 768)):
        qa, sa, _ = _operand(m, d, "row", g)
        qb, sb, _ = _operand(n, d, "row", g)
        one = S.matmul_fp8(qa, sa, qb, sb, dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(one, S.matmul_fp8(qa, sa, qb, sb, dtype=torch.float32))


def test_product_spoilt_rows_stay_apart():
    """Infinities and NaN of one row reach that row's results and no others'."""
    g = _gen(11)
    x, y = torch.randn(40, 300, generator=g), torch.randn(150, 300, generator=g)
    x[7, 200], y[140, 3] = math.inf, math.nan
    c = S.matmul_fp8(*S.quantize_fp8(x.cuda()), *S.quantize_fp8(y.cuda()), dtype=torch.float32).cpu()
    bad = torch.zeros(40, 150, dtype=torch.bool)
    bad[7], bad[:, 140] = True, True
    assert torch.equal(~torch.isfinite(c), bad)


def _operand_there(n, d, block, seed):
    """An operand and its values in 64 bits, all on the GPU."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, d, generator=g, device="cuda") * torch.exp(torch.randn(n, 1, generator=g, device="cuda"))
    q, scale = S.quantize_fp8(x, block=block)
    rows = torch.arange(n, device="cuda") // (1 if block == "row" else 128)
    return q, scale, q.double() * scale.double()[rows].repeat_interleave(128, dim=1)


# one and several rounds of large tiles, ragged both ways; rows of c that allow vectors and not;
# sums in shares, of large tiles, of small ones and of few rows
LARGE = [(2300, 5000, 130, "square"), (2300, 5002, 130, "row"), (130, 1002, 256, "row"), (2304, 5003, 100, "row"), (5000, 4504, 260, "row"), (6400, 7001, 128, "square"),
         (4000, 708, 20500, "square"), (4000, 703, 20500, "row"), (150, 150, 9000, "square"), (33, 1030, 6000, "row"),
         (20, 3000, 5000, "square"), (1, 65, 8192, "row")]


@pytest.mark.parametrize("m,n,d,block", LARGE)
def test_large_product(m, n, d, block):
    qa, sa, a = _operand_there(m, d, "row", m + d)
    qb, sb, b = _operand_there(n, d, block, n + d)
    want, wide = a @ b.t(), a.abs() @ b.abs().t()
    kp = a.shape[1]
    for kind in ("bf16", "fp32"):
        bound = ((kp + 2 * kp // 128 + 2) * EPS + (2.0 ** -10 if kind != "fp32" else 0.0)) * wide
        bound += HALF_ULP[kind] * want.abs() * 1.001 + TINY[kind]
        got = S.matmul_fp8(qa, sa, qb, sb, dtype=TYPES[kind])
        assert ((got.double() - want).abs() <= bound).all(), kind
        assert torch.equal(got, S.matmul_fp8(qa, sa, qb, sb, dtype=TYPES[kind])), kind


@pytest.mark.parametrize("pad", [8, 2, 3])
def test_large_product_into_wider_rows(pad):
    """c_stride above n, large tiles: what lies between the rows is left alone."""
    m, n, d = 2400, 4808, 256
    qa, sa, _ = _operand_there(m, d, "row", 1)
    qb, sb, _ = _operand_there(n, d, "square", 2)
    c = torch.full((m, n + pad), -5.0, device="cuda", dtype=torch.bfloat16)
    lib = F.load()
    rc = lib.ung_hip_fp8_matmul(qa.data_ptr(), sa.data_ptr(), qb.data_ptr(), sb.data_ptr(), 1, m, n, d, c.data_ptr(),
                                2, n + pad, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert (c[:, n:] == -5.0).all() and torch.equal(c[:, :n], S.matmul_fp8(qa, sa, qb, sb))


def test_large_product_spoilt_rows_stay_apart():
    g = torch.Generator(device="cuda").manual_seed(3)
    x, y = (torch.randn(n, 300, generator=g, device="cuda") for n in (3000, 4500))
    x[2999, 200], x[7, 0], y[140, 3] = math.inf, math.nan, math.nan
    c = S.matmul_fp8(*S.quantize_fp8(x), *S.quantize_fp8(y))
    bad = torch.zeros(3000, 4500, dtype=torch.bool, device="cuda")
    bad[2999], bad[7], bad[:, 140] = True, True, True
    assert torch.equal(~torch.isfinite(c), bad)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_products_of_no_length(kind):
    for m, n in ((1, 1), (40, 300), (300, 400), (2500, 4500)):
        a, b = (S.quantize_fp8(torch.empty(r, 0, device="cuda")) for r in (m, n))
        c = S.matmul_fp8(*a, *b, dtype=TYPES[kind])
        assert tuple(c.shape) == (m, n) and not c.any()


def test_product_needs_its_workspace():
    qa, sa, _ = _operand_there(150, 9000, "row", 1)
    qb, sb, _ = _operand_there(150, 9000, "row", 2)
    c = torch.full((150, 150), -5.0, device="cuda")
    lib = F.load()
    keep, at, size = S._workspace(lib.ung_hip_fp8_matmul_workspace, 150, 150, qa.shape[1], 0, device="cuda")
    assert size > 0
    for where, bytes_ in ((None, size), (at, size - 1), (at + 4, size)):
        rc = lib.ung_hip_fp8_matmul(qa.data_ptr(), sa.data_ptr(), qb.data_ptr(), sb.data_ptr(), 0, 150, 150,
                                    qa.shape[1], c.data_ptr(), 0, 150, where, bytes_,
                                    torch.cuda.current_stream().cuda_stream)
        assert rc == -1 and b"workspace" in lib.ung_hip_last_error()
    assert (c == -5.0).all()


@pytest.mark.parametrize("m,n,pad", [(5, 33, 3), (130, 129, 8), (20, 2000, 1)])
def test_product_into_wider_rows(m, n, pad):
    """c_stride above n: what lies between the rows is left alone."""
    g = _gen(m + n)
    qa, sa, a = _operand(m, 256, "row", g)
    qb, sb, b = _operand(n, 256, "square", g)
    c = torch.full((m, n + pad), -5.0, device="cuda")
    lib = F.load()
    keep, at, size = S._workspace(lib.ung_hip_fp8_matmul_workspace, m, n, 256, 0, device="cuda")
    rc = lib.ung_hip_fp8_matmul(qa.data_ptr(), sa.data_ptr(), qb.data_ptr(), sb.data_ptr(), 1, m, n, 256, c.data_ptr(),
                                0, n + pad, at, size, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    c = c.cpu()
    assert (c[:, n:] == -5.0).all()
    want = a @ b.t()
    assert ((c[:, :n].double() - want).abs() <= _product_bound(a, b, want, "fp32")).all()


def test_empty_products():
    q, s = S.quantize_fp8(torch.ones(4, 128, device="cuda"))
    none, none_s = q[:0], s[:0]
    assert S.matmul_fp8(none, none_s, q, s).shape == (0, 4) and S.matmul_fp8(q, s, none, none_s).shape == (4, 0)
    flat, flat_s = S.quantize_fp8(torch.empty(4, 0, device="cuda"))
    assert torch.equal(S.matmul_fp8(flat, flat_s, flat, flat_s, dtype=torch.float32).cpu(), torch.zeros(4, 4))
    assert S.quantize_fp8(torch.empty(0, 5, device="cuda"))[0].shape == (0, 128)


@pytest.mark.parametrize("m,n,d", [(1, 1, 1), (20, 300, 100), (129, 130, 257), (300, 64, 128)])
def test_product_gradients(m, n, d):
    """dx and dw against 64-bit products of the operands that the formula names."""
    g = _gen(m + n + d)
    x, w, up = (torch.randn(s, generator=g).bfloat16() for s in ((m, d), (n, d), (m, n)))
    _, _, xt, xts = S.quantize_fp8(x.cuda(), transpose=True)
    _, _, wt, wts = S.quantize_fp8(w.cuda(), block="square", transpose=True)
    dx, dw = S.matmul_fp8_grad(up.cuda(), xt, xts, wt, wts)

    def values(q, s, block="row"):
        s = s if block == "row" else s.repeat_interleave(128, dim=0)[:q.shape[0]]
        return q.double() * s.double().repeat_interleave(128, dim=1)

    gq, gs = _quantized(up.float(), "row")
    gt, gts = _quantized(up.float().t().contiguous(), "row")
    wq, ws = _quantized(w.float(), "square")
    turned = torch.zeros(d, _blocks(n) * 128)
    turned[:, :n] = wq[:, :d].t()
    a, b = values(gq, gs), values(turned, ws.t().contiguous(), "square")
    assert ((dx.cpu().double() - a @ b.t()).abs() <= _product_bound(a, b, a @ b.t(), "bf16")).all()
    a, b = values(gt, gts), values(*_quantized(x.float().t().contiguous(), "row"))
    assert ((dw.cpu().double() - a @ b.t()).abs() <= _product_bound(a, b, a @ b.t(), "fp32")).all()


def test_linear_gradients_against_differences():
    """Inputs of 0, +-1, +-2 that 8 bits hold exactly (each block has a 2): the layer is linear
    there, so differences of sum(g y) over a unit step are its gradient, and all of them are
    whole numbers."""
    g = _gen(3)
    m, n, d = 9, 140, 200
    x, w, up = (torch.randint(-2, 3, s, generator=g).float() for s in ((m, d), (n, d), (m, n)))
    x[:, 0] = x[:, 199] = w[:, 0] = w[:, 199] = up[:, 0] = up[:, 139] = up[0] = x[0] = 2.0
    x, w, up = x.cuda().requires_grad_(), w.cuda().requires_grad_(), up.cuda()
    y = S.linear_fp8(x, w, dtype=torch.float32)
    # whole numbers; the scales 2 / 448 round, each product by a few units of 2^-24
    assert (y - x @ w.t()).abs().max() < 1e-4
    y.backward(up)
    assert (x.grad - up @ w).abs().max() < 1e-4 and (w.grad - up.t() @ x).abs().max() < 1e-4
    with torch.no_grad():
        for t, i, j in ((x, 3, 50), (x, 8, 150), (w, 5, 20), (w, 139, 130)):
            old = float(t[i, j])
            t[i, j] = old + 1 if old < 1 else old - 1
            step = (S.linear_fp8(x, w, dtype=torch.float32).double() * up).sum() - (y.double() * up).sum()
            step = float(step) * (1 if old < 1 else -1)
            t[i, j] = old
            assert abs(step - float(t.grad[i, j])) < 1e-3
    for need in ((True, False), (False, True)):
        a, b = x.detach().requires_grad_(need[0]), w.detach().requires_grad_(need[1])
        S.linear_fp8(a, b, dtype=torch.float32).backward(up)
        assert a.grad is None if not need[0] else torch.equal(a.grad, x.grad)
        assert b.grad is None if not need[1] else torch.equal(b.grad, w.grad)


# ---- the first scores ---------------------------------------------------------------------------
def _top(x, k):
    """(values, ids) of float32 rows by a stable sort; NaN first, -inf not at all."""
    n, v = x.shape
    val, ids = np.full((n, k), -np.inf, np.float32), np.full((n, k), -1, np.int32)
    for r in range(n):
        row = x[r].astype(np.float64) + 0.0
        key = np.where(np.isnan(row), np.inf, row)
        order = np.lexsort((np.arange(v), -key, ~np.isnan(row)))
        order = [j for j in order if not row[j] == -np.inf][:k]
        ids[r, :len(order)] = order
        val[r, :len(order)] = x[r, order]
    return val, ids


def _lse(x, t):
    x = x.astype(np.float64) / t
    top = x.max(axis=1)
    with np.errstate(invalid="ignore", divide="ignore"):
        out = top + np.log(np.exp(x - np.where(np.isfinite(top), top, 0)[:, None]).sum(axis=1))
    return np.where(np.isinf(top), top, out)


def _scores(n, v, kind, pad, seed, masked=0.0, spread=3.0):
    g = _gen(seed)
    x = (torch.randn(n, v, generator=g) * spread)
    if masked:
        x[torch.rand(n, v, generator=g) < masked] = -math.inf
    x = x.to(TYPES[kind])
    whole = torch.full((n, v + pad), 50.0, dtype=TYPES[kind], device="cuda")
    whole[:, :v] = x.cuda()
    return x.float().numpy(), whole, whole[:, :v]


def _check_top(x, view, k, t=1.0):
    val, ids, lse = S.top_scores(view, k, temperature=t)
    want_val, want_ids = _top(x, k)
    val, ids, lse = val.cpu().numpy(), ids.cpu().numpy(), lse.cpu().numpy().astype(np.float64)
    assert np.array_equal(ids, want_ids), np.nonzero((ids != want_ids).any(axis=1))[0][:5]
    assert np.array_equal(val, want_val, equal_nan=True)
    want = _lse(x, t)
    # each weight exp(d) is off by at most (2 |d| + 4) eps of itself, |d| <= log v + 1 on the
    # sum's average; the sum by its depth; the result by its own rounding
    v = max(x.shape[1], 1)
    bound = (2 * math.log(v) + 8 + v / 256 + 64) * EPS + 2 * EPS * np.abs(np.where(np.isfinite(want), want, 0))
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(lse), np.isnan(want)) and np.array_equal(lse[np.isinf(want)], want[np.isinf(want)])
    assert (np.abs(lse - want)[fine] <= (bound if np.ndim(bound) else np.full(len(want), bound))[fine]).all()


TOPS = [(1, 1, 1), (3, 7, 5), (2, 50, 64), (5, 128, 128), (4, 1000, 32), (3, 2049, 100), (2, 33000, 128), (1, 100_003, 32),
        (700, 300, 20), (2, 300_001, 6)]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,v,k", TOPS)
def test_top_scores(n, v, k, kind):
    for pad, masked, t in ((0, 0.0, 1.0), (3, 0.5, 0.5), (8, 0.98, 2.0)):
        x, _, view = _scores(n, v, kind, pad, n + v + k, masked)
        _check_top(x, view, k, t)


@pytest.mark.parametrize("v", [40, 5000, 70_000])
def test_top_scores_ties_and_odd_values(v):
    """Rows of one value (ties go to the lowest id), of few values, of zeros of both signs, all
    filtered out, with infinities and with NaN; sorted rows, where one thread holds the best."""
    g = _gen(v)
    rows = [torch.full((v,), 1.5), torch.randint(0, 3, (v,), generator=g).float(), torch.zeros(v),
            torch.full((v,), -math.inf), torch.randn(v, generator=g), torch.randn(v, generator=g),
            torch.arange(v).float(), -torch.arange(v).float(), torch.randn(v, generator=g).abs().neg() * 1e30,
            torch.full((v,), torch.finfo(torch.float32).min), torch.full((v,), -math.inf)]
    rows[2][1::2] = -0.0
    rows[4][v // 2], rows[4][3] = math.inf, -math.inf
    rows[5][v // 3], rows[5][v - 1] = math.nan, -math.nan
    rows[9][v // 2] = 3.0
    rows[10][v - 1] = 2.0
    x = torch.stack(rows)
    for k in (1, 32, 128):
        _check_top(x.numpy(), x.cuda(), k)


def test_top_scores_empty():
    val, ids, lse = S.top_scores(torch.empty(3, 0, device="cuda"), 4)
    assert (val == -math.inf).all() and (ids == -1).all() and (lse == -math.inf).all()
    assert S.top_scores(torch.empty(0, 9, device="cuda"), 4)[0].shape == (0, 4)


def test_top_scores_past_32_bit_offsets():
    """The last rows of a block of more than 2^31 scores."""
    n, v = 33_000, 70_000
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 5 GB of free device memory")
    whole = torch.empty(n, v, dtype=torch.bfloat16, device="cuda")
    whole[:-2] = -math.inf
    x, _, view = _scores(2, v, "bf16", 0, 1)
    whole[-2:] = view
    val, ids, lse = S.top_scores(whole, 16)
    want_val, want_ids = _top(x, 16)
    assert np.array_equal(ids[-2:].cpu().numpy(), want_ids) and np.array_equal(val[-2:].cpu().numpy(), want_val)
    assert (ids[:-2] == -1).all()
    loss, grad = S.distill_step(whole, ids, val, out=whole)
    want = _distill(x, want_ids, want_val, None, np.ones(2), 1.0)
    assert np.allclose(loss[-2:].cpu().numpy(), want[0], rtol=1e-4, atol=1e-5) and not loss[:-2].any()
    assert np.abs(grad[-2:].float().cpu().numpy() - want[1]).max() < 0.01 and not grad[:10].any()


# ---- distillation ---------------------------------------------------------------------------------
def _distill(x, ids, val, lse, weight, t):
    """(loss, gradient, per-element error scale) in 64 bits, row by row from the definition."""
    n, v = x.shape
    loss, grad, scale = np.zeros(n), np.zeros((n, v)), np.zeros((n, v))
    for r in range(n):
        z = x[r].astype(np.float64) / t
        ok = [(int(i), float(a) / t) for i, a in zip(ids[r], val[r]) if 0 <= i < v and a != -np.inf]
        if not ok or not (z > -np.inf).any():
            continue
        m = z.max()
        e = np.exp(z - m)
        total = e.sum()
        a = np.array([b for _, b in ok])
        at = np.array([i for i, _ in ok])
        p = np.exp(a - (a.max() + np.log(np.exp(a - a.max()).sum()))) if lse is None else np.exp(a - float(lse[r]))
        log_q = z - m - np.log(total)
        used = p > 0
        loss[r] = (p[used] * (np.log(p[used]) - log_q[at[used]])).sum()
        dense = np.zeros(v)
        np.add.at(dense, at, p)
        q = e / total
        g = p.sum() * q - dense
        if lse is not None:
            out = np.ones(v, bool)
            out[at] = False
            rest_q, rest_p = q[out].sum(), max(0.0, 1 - p.sum())
            if rest_q > 0 and rest_p > 0:
                loss[r] += rest_p * (np.log(rest_p) - np.log(rest_q))
                g += rest_p * q
                g[out] -= rest_p * q[out] / rest_q
        grad[r] = g * weight[r] / t
        # p_r = 1 - sum p is off by the sum's error whatever its size, and enters over Q_r
        scale[r] = (q * (1 + np.minimum(np.abs(z - m), 100)) * (1 if lse is None else 1 + 1 / max(q[out].sum(), 1e-300))
                    + dense) * abs(weight[r]) / t
    return loss, grad, scale


def _teacher(n, v, k, seed, x=None, duplicates=False):
    g = np.random.default_rng(seed)
    ids = np.full((n, k), -1, np.int32)
    val = np.full((n, k), -np.inf, np.float32)
    for r in range(n):
        m = min(k, v)
        ids[r, :m] = g.choice(v, m, replace=duplicates)
        val[r] = np.sort(g.standard_normal(k).astype(np.float32) * 2)[::-1]
        if r % 5 == 1:
            ids[r, k // 2:] = -1       # a short list
        if r % 5 == 2:
            val[r, k // 3:] = -np.inf  # entries without a score
        if r % 7 == 3:
            ids[r] = -1                # no entry at all
        if r % 7 == 4:
            ids[r, :1] = v             # out of range: missing
    if x is not None:  # what the student has filtered out is not in the lists
        for r in range(n):
            for i in range(k):
                if 0 <= ids[r, i] < v and x[r, ids[r, i]] == -np.inf:
                    ids[r, i] = -1
    there = (ids >= 0) & (ids < v) & (val > -np.inf)
    lse = np.log(np.where(there, np.exp(val.astype(np.float64)), 0).sum(axis=1) + 0.5).astype(np.float32)
    return ids, val, lse


def _check_distill(x, view, ids, val, lse, t, kind, seed):
    n, v = x.shape
    w = np.random.default_rng(seed).random(n).astype(np.float32)
    args = [torch.from_numpy(a).cuda() for a in (ids, val)]
    t_lse = None if lse is None else torch.from_numpy(lse).cuda()
    tw = torch.from_numpy(w).cuda()
    want_loss, want_grad, scale = _distill(x, ids, val, lse, w.astype(np.float64), t)
    loss, saved = S.distill_forward(view, *args, teacher_lse=t_lse, temperature=t)
    grad = S.distill_backward(tw, view, *args, saved, teacher_lse=t_lse, temperature=t)
    loss2, grad2 = S.distill_step(view, *args, tw, teacher_lse=t_lse, temperature=t)
    over = view.clone(memory_format=torch.preserve_format)
    assert over.stride() == view.stride() or over.is_contiguous()
    loss3, grad3 = S.distill_step(over, *args, tw, teacher_lse=t_lse, temperature=t, out=over)
    assert grad3.data_ptr() == over.data_ptr()
    # a row's logarithms, weights and sums of v terms in 32 bits: each p (log p - log q) is off
    # by the error of log q <= (sum's depth + weights' error) and of the logarithms' roundings
    counts = np.isfinite(x) & (x > np.finfo(np.float32).min)  # the lowest value: no weight
    size = 40.0 if not counts.any() else np.abs(np.where(counts, x, 0)).max() / t + 20
    depth = 2 * math.log(v + 1) + v / 256 + 100
    for got in (loss, loss2, loss3):
        err = np.abs(got.cpu().numpy().astype(np.float64) - want_loss)
        assert (err <= EPS * (depth + 8 * size) * 2).all(), (err.max(), EPS * (depth + 8 * size) * 2)
    for got in (grad, grad2, grad3):
        assert got.dtype == view.dtype
        err = np.abs(got.float().cpu().numpy().astype(np.float64) - want_grad)
        bound = EPS * (depth + 8 * size) * scale + HALF_ULP[kind] * 1.001 * np.abs(want_grad) + TINY[kind]
        assert (err <= bound).all(), (np.argwhere(err > bound)[:4], (err - bound).max())
        assert not got.float().cpu().numpy()[x == -np.inf].any()  # nothing flows to filtered columns


DISTILLS = [(1, 1, 1), (3, 5, 8), (9, 50, 6), (12, 128, 128), (8, 1000, 32), (7, 4099, 64), (130, 5000, 20),
            (3, 33000, 128), (2, 300_001, 32)]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n,v,k", DISTILLS)
def test_distill(n, v, k, kind, tail):
    for pad, masked, t in ((0, 0.0, 1.0), (3, 0.6, 0.5), (8, 0.0, 2.0)):
        x, _, view = _scores(n, v, kind, pad, n + v + k, masked, spread=2.0)
        ids, val, lse = _teacher(n, v, k, v + k, x)
        if t != 1.0:
            there = (ids >= 0) & (ids < v) & (val > -np.inf)
            lse = np.log(np.where(there, np.exp(val.astype(np.float64) / t), 0).sum(axis=1) + 0.5).astype(np.float32)
        _check_distill(x, view, ids, val, lse if tail else None, t, kind, n)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("v", [200, 5000, 40000])
def test_top_of_a_row_with_nan_and_few_scores(v, kind):
    """A NaN, two scores and nothing else: NaN is first, the rest of a long list is missing."""
    x = torch.full((3, v), -math.inf)
    x[1, v // 2], x[1, 3], x[1, v - 1] = math.nan, -2.0, 5.0
    x[2, 7] = math.nan
    values, ids, lse = (t.cpu() for t in S.top_scores(x.to(TYPES[kind]).cuda(), 128))
    assert ids[1, :3].tolist() == [v // 2, v - 1, 3] and values[1, 1:3].tolist() == [5.0, -2.0]
    assert ids[2, 0] == 7 and torch.isnan(values[1:, 0]).all() and torch.isnan(lse[1:]).all()
    assert (ids[0] == -1).all() and (ids[1, 3:] == -1).all() and (ids[2, 1:] == -1).all() and lse[0] == -math.inf
    assert (values[0] == -math.inf).all() and (values[1, 3:] == -math.inf).all()


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("n,v,k", [(40, 849, 100), (9, 1000, 128), (5, 130, 128), (3, 100000, 128), (70, 3000, 128)])
def test_long_lists_of_short_rows(n, v, k, kind):
    """k close to the number of a block's threads that hold scores: nearly all are candidates."""
    x = torch.randn(n, v, generator=_gen(n + v)).to(TYPES[kind])
    values, ids, _ = S.top_scores(x.cuda(), k)
    order = np.lexsort((np.broadcast_to(np.arange(v), (n, v)), -x.double().numpy()))[:, :k]
    assert (ids.cpu().numpy() == order).all()
    assert torch.equal(values.cpu(), torch.gather(x.float(), 1, torch.from_numpy(order)))


@pytest.mark.parametrize("v", [300, 5000, 70000])
def test_distill_is_the_same_every_time(v):
    """Columns named many times over: sums keep their order whichever entry is seen first."""
    g = _gen(v)
    x = torch.randn(9, v, generator=g).cuda()
    ids = torch.randint(0, 20, (9, 100), generator=g, dtype=torch.int32).cuda()
    val = torch.randn(9, 100, generator=g).cuda()
    lse = torch.logsumexp(val, 1) + 0.3
    loss, grad = S.distill_step(x, ids, val, teacher_lse=lse)
    saved = S.distill_forward(x, ids, val, teacher_lse=lse)[1]
    for _ in range(10):
        again = S.distill_step(x, ids, val, teacher_lse=lse)
        assert torch.equal(loss, again[0]) and torch.equal(grad, again[1])
        assert torch.equal(saved[:, :6], S.distill_forward(x, ids, val, teacher_lse=lse)[1][:, :6])


@pytest.mark.parametrize("tail", [False, True])
def test_distill_columns_named_twice(tail):
    x, _, view = _scores(6, 40, "fp32", 0, 3)
    ids, val, lse = _teacher(6, 40, 60, 4, x, duplicates=True)
    ids[0] = np.tile([3, 7, 3], 20)
    val[0] = np.linspace(2, -2, 60)
    lse[0] = 4.0 + np.log(60)
    _check_distill(x, view, ids, val, lse if tail else None, 1.0, "fp32", 1)


@pytest.mark.parametrize("v", [64, 70_000])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_rows_at_the_edge(v, tail):
    """All scores filtered out; one left, listed or not; the list holds the student's whole mass
    or every column left; the type's lowest value as a mask; NaN and infinities."""
    x = np.full((9, v), -np.inf, np.float32)
    ids = np.full((9, 4), -1, np.int32)
    val = np.full((9, 4), -np.inf, np.float32)
    ids[:, 0], val[:, 0] = 5, 1.0
    x[1, 5] = 2.0                                  # one score, listed
    x[2, [5, 9]] = [1.0, 0.0]                      # half of the mass listed
    x[3], x[3, 5] = -80.0, 30.0                    # the rest's mass far below a rounding of 1
    x[4] = np.finfo(np.float32).min                # masked by the lowest value, all but two
    x[4, [5, 6]] = [0.5, 0.25]
    x[5, :] = np.finfo(np.float32).min             # ... all of them
    ids[6, :3], val[6, :3] = [5, 6, 7], [1.0, 0.0, -1.0]
    x[6, 5:8] = [0.1, 0.2, 0.3]                    # every column left is listed
    x[7], x[7, 11] = 0.0, np.nan
    x[8], x[8, 11] = 0.0, np.inf
    lse = np.log(np.where(val > -np.inf, np.exp(val.astype(np.float64)), 0).sum(axis=1) + 0.7).astype(np.float32)
    lse = lse if tail else None
    fine = slice(0, 7)
    _check_distill(x[fine], torch.from_numpy(x[fine]).cuda(), ids[fine], val[fine], None if lse is None else lse[fine],
                   1.0, "fp32", 2)
    args = [torch.from_numpy(a).cuda() for a in (x, ids, val)]
    t_lse = None if lse is None else torch.from_numpy(lse).cuda()
    loss, grad = S.distill_step(*args, teacher_lse=t_lse)
    assert torch.isfinite(loss[fine]).all() and torch.isfinite(grad[fine]).all()
    assert loss[7:].isnan().all() and grad[7:].isnan().all()
    assert float(loss[0]) == 0.0 and not grad[0].any()


def test_distill_without_entries():
    x = torch.randn(4, 100, device="cuda")
    ids, val = torch.empty(4, 0, dtype=torch.int32, device="cuda"), torch.empty(4, 0, device="cuda")
    loss, grad = S.distill_step(x, ids, val)
    assert not loss.any() and not grad.any()
    loss, grad = S.distill_step(x[:, :0], ids, val)
    assert not loss.any() and grad.shape == (4, 0)
    loss, grad = S.distill_step(x[:0], ids[:0], val[:0])
    assert loss.shape == (0,) and grad.shape == (0, 100)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_gradient_against_differences(tail):
    """Central differences of the loss with step h: off by the loss's error / h and by h^2 / 6
    of the third derivative, at most 1 / T^3 here."""
    n, v, k, t, h = 3, 300, 12, 1.0, 0.03
    x, _, view = _scores(n, v, "fp32", 0, 8, spread=1.0)
    ids, val, lse = _teacher(n, v, k, 9)
    ids[:, 0], val[:, 0] = [4, 5, 6], 2.0
    lse = torch.from_numpy(lse + 2.0).cuda() if tail else None
    args = [torch.from_numpy(a).cuda() for a in (ids, val)]
    s = view.clone().requires_grad_()
    S.distill_loss(s, *args, teacher_lse=lse, temperature=t).sum().backward()
    for r, j in ((0, 4), (0, 17), (1, 5), (1, 299), (2, 6), (2, 0)):
        ends = []
        for d in (h, -h):
            y = view.clone()
            y[r, j] += d
            ends.append(float(S.distill_forward(y, *args, teacher_lse=lse, temperature=t)[0][r].double()))
        assert abs((ends[0] - ends[1]) / (2 * h) - float(s.grad[r, j])) < 300 * EPS / h + h * h / 6


# ---- together, streams, graphs, refusals ------------------------------------------------------------
def test_teacher_and_student_together():
    """A teacher's top scores from the 8-bit product, the student's loss against them, and the
    gradients back to the student's rows and table: equal to the operators called apart."""
    g = _gen(21)
    x, w, teacher = (torch.randn(s, generator=g).cuda() for s in ((50, 200), (700, 200), (700, 200)))
    t_scores = S.matmul_fp8(*S.quantize_fp8(x), *S.quantize_fp8(teacher))
    values, ids, lse = S.top_scores(t_scores, 20, temperature=2.0)
    x, w = x.requires_grad_(), w.requires_grad_()
    loss = S.distill_loss(S.linear_fp8(x, w), ids, values, teacher_lse=lse, temperature=2.0)
    loss.mean().backward()
    with torch.no_grad():
        s = S.linear_fp8(x, w)
        loss2, ds = S.distill_step(s, ids, values, torch.full((50,), 1 / 50, device="cuda"), teacher_lse=lse, temperature=2.0)
        xt = S.quantize_fp8(x.detach(), transpose=True)[2:]
        wt = S.quantize_fp8(w.detach(), block="square", transpose=True)[2:]
        dx, dw = S.matmul_fp8_grad(ds, *xt, *wt)
    assert torch.equal(loss, loss2)
    assert torch.allclose(x.grad, dx.float(), rtol=0.02, atol=1e-4) and torch.allclose(w.grad, dw, rtol=0.02, atol=1e-4)


def test_side_stream_and_graph():
    g = _gen(31)
    x, w = torch.randn(40, 256, generator=g).cuda(), torch.randn(900, 256, generator=g).cuda()
    ids, val, lse = (torch.from_numpy(a).cuda() for a in _teacher(40, 900, 16, 2))
    lse = lse + 1.0

    def step():
        q, s, qt, st = S.quantize_fp8(x, transpose=True)
        wq, ws, wt, wts = S.quantize_fp8(w, block="square", transpose=True)
        y = S.matmul_fp8(q, s, wq, ws)
        top = S.top_scores(y, 16)
        loss, ds = S.distill_step(y, ids, val, teacher_lse=lse)
        return (y, *top, loss, ds, *S.matmul_fp8_grad(ds, qt, st, wt, wts))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        x.copy_(torch.randn(40, 256, generator=_gen(seed)))
        w.copy_(torch.randn(900, 256, generator=_gen(seed + 50)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_neighbor_lists_as_teacher():
    """The exact lists of a small base set as the teacher's entries; groups' rows that hold
    fewer neighbours than the list is long are short lists."""
    rng = np.random.default_rng(4)
    X = rng.standard_normal((300, 48)).astype(np.float32)
    with F.HipContext(0) as ctx:
        ctx.prepare_vectors(X)
        lists, dist, _ = ctx.group_knn([0], [300], 16)
    ids, values = (t.cuda() for t in S.entries_of_neighbors(lists, dist))
    student = (torch.from_numpy(X[:, :24]) @ torch.from_numpy(X[:, :24]).t())
    loss, grad = S.distill_step(student.cuda(), ids, values, temperature=4.0)
    want = _distill(student.numpy(), ids.cpu().numpy(), values.cpu().numpy(), None, np.ones(300), 4.0)
    assert np.allclose(loss.cpu().numpy(), want[0], rtol=1e-5, atol=1e-5)
    assert np.allclose(grad.cpu().numpy(), want[1], rtol=1e-4, atol=1e-6)


def test_refusals():
    x = torch.randn(8, 128, device="cuda")
    q, s = S.quantize_fp8(x)
    ids, val = torch.zeros(8, 4, dtype=torch.int32, device="cuda"), torch.zeros(8, 4, device="cuda")
    bad = [
        lambda: S.quantize_fp8(x.cpu()), lambda: S.quantize_fp8(x.double()), lambda: S.quantize_fp8(x.t()),
        lambda: S.quantize_fp8(x, block="column"), lambda: S.quantize_fp8(x[0]),
        lambda: S.quantize_fp8(x[:1].expand(8, 128)),
        lambda: S.matmul_fp8(q, s, q[:, :64], s), lambda: S.matmul_fp8(q, s[:2], q, s),
        lambda: S.matmul_fp8(q, s, q, s.half()), lambda: S.matmul_fp8(q, s, q, s, dtype=torch.int32),
        lambda: S.matmul_fp8(q, s, q.cpu(), s), lambda: S.matmul_fp8(q, s, torch.cat([q, q], 1), torch.cat([s, s], 1)),
        lambda: S.matmul_fp8_grad(torch.randn(8, 200, device="cuda"), q, s, q, s),
        lambda: S.linear_fp8(x, x[:, :64]),
        lambda: S.top_scores(x, 0), lambda: S.top_scores(x, 129), lambda: S.top_scores(x, 4, temperature=0.0),
        lambda: S.top_scores(x, 4, temperature=math.nan), lambda: S.top_scores(x.cpu(), 4),
        lambda: S.distill_forward(x, ids[:4], val), lambda: S.distill_forward(x, ids.long(), val),
        lambda: S.distill_forward(x, ids, val.half()), lambda: S.distill_forward(x, ids, val, temperature=-1.0),
        lambda: S.distill_forward(x, ids, val, teacher_lse=torch.zeros(3, device="cuda")),
        lambda: S.distill_step(x, ids, val, weight=torch.zeros(8)),
        lambda: S.distill_step(x, ids, val, out=torch.empty(8, 64, device="cuda")),
        lambda: S.distill_backward(None, x, ids, val, torch.empty(8, 3, device="cuda")),
        lambda: S.distill_step(x, torch.zeros(8, 129, dtype=torch.int32, device="cuda"), torch.zeros(8, 129, device="cuda")),
    ]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, F.UngHipError)):
            f()
            _say("not refused:", i)


@pytest.mark.parametrize("m", [32, 33, 63, 64, 65, 95, 96, 97, 128, 129, 192, 193, 385])
@pytest.mark.parametrize("n,d,block", [(257, 300, "row"), (1003, 4000, "square")])
def test_product_at_the_tiles_heights(m, n, d, block):
    """Tiles of 32, 64, 96 and 128 rows, at and beside their bounds, sums in shares too."""
    qa, sa, a = _operand_there(m, d, "row", m)
    qb, sb, b = _operand_there(n, d, block, n)
    want, wide = a @ b.t(), a.abs() @ b.abs().t()
    kp = a.shape[1]
    for kind in ("bf16", "fp32"):
        bound = ((kp + 2 * kp // 128 + 2) * EPS + (2.0 ** -10 if kind != "fp32" else 0.0)) * wide
        bound += HALF_ULP[kind] * want.abs() * 1.001 + TINY[kind]
        got = S.matmul_fp8(qa, sa, qb, sb, dtype=TYPES[kind])
        assert ((got.double() - want).abs() <= bound).all(), kind
