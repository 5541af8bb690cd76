"""GPU tests of the 8-bit whole numbers (scores.quantize_int8, matmul_int8, linear_int8): both are
defined to the last bit, so results are compared for equality with plain forms."""
import math

import numpy as np
import pytest
import torch

import filtervectorcode_refactor_amd as F
from filtervectorcode_refactor_amd import scores as S

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _numbers(x):
    """(numbers padded to whole chunks, scales) of float32 rows on the CPU; a row with an infinity
    or NaN has zeros and the scale NaN."""
    x = x.numpy()
    n, d = x.shape
    spoilt = ~np.isfinite(x).all(axis=1)
    x = np.where(spoilt[:, None], np.float32(0), x)
    most = np.maximum(np.abs(x).max(axis=1, initial=0.0), np.float32(2.0 ** -64)).astype(np.float32)
    scale = most * np.float32(1.0 / 127.0)
    q = np.zeros((n, -(-d // 128) * 128), np.int8)
    q[:, :d] = np.rint(x / scale[:, None]).astype(np.int8)
    return torch.from_numpy(q), torch.from_numpy(np.where(spoilt, np.float32(np.nan), scale))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,d", [(1, 1), (1, 128), (3, 127), (5, 129), (4, 512), (130, 100), (7, 1000), (6, 2049),
                                 (2, 4097), (3, 9000), (300, 384), (40_000, 24)])
def test_quantize(n, d, kind):
    g = _gen(n * 1000 + d)
    x = (torch.randn(n, d, generator=g) * torch.exp(torch.randn(n, 1, generator=g) * 4)).to(TYPES[kind])
    x[0, 0] = 0.0
    if n > 2:
        x[1] = 0.0
    want_q, want_s = _numbers(x.float())
    for pad in (0, 8, 3):
        whole = torch.full((n, d + pad), 99.0, dtype=TYPES[kind], device="cuda")
        whole[:, :d] = x
        q, scale = S.quantize_int8(whole[:, :d])
        assert torch.equal(q.cpu(), want_q) and torch.allclose(scale.cpu(), want_s, rtol=0, atol=0, equal_nan=True), pad


def test_quantize_extremes():
    """Subnormals, the type's largest, ties, infinities and NaN."""
    x = torch.zeros(8, 300)
    x[0, 3], x[0, 200] = 2.0 ** -70, -1e-44
    x[1, :3] = torch.tensor([3.4e38, -1.7e38, 1e30])
    x[2, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -2.5])  # scale 1 within rounding: ties to even
    x[5, 250] = -5.0
    x[6, 299] = 1e-30
    want_q, want_s = _numbers(x)
    x[3, 7], x[4, 5], x[7, 299] = math.inf, math.nan, -math.inf
    q, scale = (t.cpu() for t in S.quantize_int8(x.cuda()))
    keep = [0, 1, 2, 5, 6]
    assert torch.equal(q[keep], want_q[keep]) and torch.equal(scale[keep], want_s[keep])
    assert scale[[3, 4, 7]].isnan().all() and not q[[3, 4, 7]].any()


def _product(qa, sa, qb, sb, dtype):
    """The definition: exact sums (64 bits), to 32 bits, times the scales' product, to the type."""
    sums = (qa.double() @ qb.double().t().contiguous()).long()  # below 2^53: exact
    return (sums.float() * (sa[:, None] * sb[None, :])).to(dtype)


def _operand(n, kp, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(-128, 128, (n, kp), device="cuda", generator=g, dtype=torch.int8)
    return q, torch.rand(n, device="cuda", generator=g) + 0.01


PRODUCTS = [(1, 1, 128), (1, 129, 256), (2, 1000, 768), (16, 16, 128), (17, 300, 384), (33, 77, 2048), (64, 130, 128),
            (65, 129, 768), (128, 128, 128), (130, 257, 384), (256, 300, 1024), (300, 511, 256), (5, 4100, 256),
            (3, 40, 5120), (48, 200, 9088), (700, 200, 128), (1, 70_000, 384), (100, 20_000, 256), (2300, 5003, 256),
            (4000, 703, 2048), (150, 150, 16_384), (513, 2049, 640), (4097, 4099, 384)]


@pytest.mark.parametrize("m,n,kp", PRODUCTS)
def test_product(m, n, kp):
    qa, sa = _operand(m, kp, m + kp)
    qb, sb = _operand(n, kp, n + kp + 1)
    for kind, dtype in TYPES.items():
        by = 2.0 ** -18 if kind == "fp16" else 1.0  # in fp16's range
        got = S.matmul_int8(qa, sa * by, qb, sb, dtype=dtype)
        assert got.dtype == dtype and torch.equal(got, _product(qa, sa * by, qb, sb, dtype)), kind
        assert torch.equal(got, S.matmul_int8(qa, sa * by, qb, sb, dtype=dtype))


def test_longest_sums_are_exact():
    """The largest length of the smallest numbers: 2145386496, 2^31 less 2 million."""
    q = torch.full((3, 130_944), -128, dtype=torch.int8, device="cuda")
    q[1] = 127
    one = torch.ones(3, device="cuda")
    c = S.matmul_int8(q, one, q, one, dtype=torch.float32)
    assert torch.equal(c, _product(q, one, q, one, torch.float32)) and c[0, 0] == 130_944 * 128 * 128
    more = torch.zeros(3, 131_072, dtype=torch.int8, device="cuda")
    with pytest.raises(F.UngHipError, match="131072"):
        S.matmul_int8(more, one, more, one)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("m,n,pad", [(5, 33, 3), (130, 129, 8), (20, 2000, 1), (2400, 4808, 2), (2400, 4808, 3), (300, 1000, 4)])
def test_product_into_wider_rows(m, n, pad, kind):
    """c_stride above n: what lies between the rows is left alone."""
    qa, sa = _operand(m, 256, 1)
    qb, sb = _operand(n, 256, 2)
    sa = sa * 2.0 ** -16
    c = torch.full((m, n + pad), -5.0, device="cuda", dtype=TYPES[kind])
    code = {"fp32": 0, "fp16": 1, "bf16": 2}[kind]
    lib = F.load()
    keep, at, size = S._workspace(lib.ung_hip_int8_matmul_workspace, m, n, 256, code, device="cuda")
    rc = lib.ung_hip_int8_matmul(qa.data_ptr(), sa.data_ptr(), qb.data_ptr(), sb.data_ptr(), m, n, 256, c.data_ptr(),
                                 code, n + pad, at, size, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert (c[:, n:] == -5.0).all() and torch.equal(c[:, :n], _product(qa, sa, qb, sb, TYPES[kind]))


def test_product_needs_its_workspace():
    qa, sa = _operand(20, 16_384, 1)
    c = torch.full((20, 20), -5.0, device="cuda")
    lib = F.load()
    keep, at, size = S._workspace(lib.ung_hip_int8_matmul_workspace, 20, 20, 16_384, 0, device="cuda")
    assert size > 0  # shares of the inner length
    for where, bytes_ in ((None, size), (at, size - 1), (at + 4, size)):
        rc = lib.ung_hip_int8_matmul(qa.data_ptr(), sa.data_ptr(), qa.data_ptr(), sa.data_ptr(), 20, 20, 16_384,
                                     c.data_ptr(), 0, 20, where, bytes_, torch.cuda.current_stream().cuda_stream)
        assert rc == -1 and b"workspace" in lib.ung_hip_last_error()
    assert (c == -5.0).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("m,n,d", [(1, 1, 1), (1, 5000, 100), (2, 300, 384), (16, 1000, 768), (17, 129, 257), (33, 77, 2000),
                                   (77, 3001, 768), (300, 1000, 64), (8, 40_000, 128), (4, 200, 9000), (1000, 900, 500)])
def test_linear(m, n, d, kind):
    """Rows brought to whole numbers on the way: quantize_int8 and matmul_int8 one after the other."""
    g = torch.Generator(device="cuda").manual_seed(m + n + d)
    x = torch.randn(m, d + 3, device="cuda", generator=g).to(TYPES[kind])
    w = torch.randn(n, d, device="cuda", generator=g)
    q, scale = S.quantize_int8(w)
    for view in (x[:, :d], x[:, 3:], x[:, :d].contiguous()):
        xq, xs = S.quantize_int8(view)
        for dtype in TYPES.values():
            assert torch.equal(S.linear_int8(view, q, scale, dtype=dtype), _product(xq, xs, q, scale, dtype))


def test_values_near_the_products_of_the_rows():
    """Each factor is off by at most half a step of its row's 127: the product of two rows by
    d (|a|max |b|max) (1 / 254 (1 + 1) + 1 / 254^2) at most, and the roundings of 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x, w = torch.randn(50, 300, device="cuda", generator=g), torch.randn(400, 300, device="cuda", generator=g)
    y = S.linear_int8(x, *S.quantize_int8(w), dtype=torch.float32)
    step = (x.abs().amax(1)[:, None] / 254 * w.abs().sum(1) + w.abs().amax(1) / 254 * x.abs().sum(1)[:, None]
            + 300 * x.abs().amax(1)[:, None] * w.abs().amax(1) / 254 ** 2)
    assert ((y.double() - x.double() @ w.double().t().contiguous()).abs() <= 1.001 * step).all()


def test_spoilt_rows_stay_apart():
    g = _gen(11)
    x, y = torch.randn(40, 300, generator=g), torch.randn(150, 300, generator=g)
    x[7, 200], y[140, 3] = math.inf, math.nan
    c = S.linear_int8(x.cuda(), *S.quantize_int8(y.cuda()), dtype=torch.float32).cpu()
    bad = torch.zeros(40, 150, dtype=torch.bool)
    bad[7], bad[:, 140] = True, True
    assert torch.equal(c.isnan(), bad)


def test_empty():
    q, s = S.quantize_int8(torch.ones(4, 128, device="cuda"))
    assert S.matmul_int8(q[:0], s[:0], q, s).shape == (0, 4) and S.matmul_int8(q, s, q[:0], s[:0]).shape == (4, 0)
    flat, flat_s = S.quantize_int8(torch.empty(4, 0, device="cuda"))
    assert flat.shape == (4, 0) and not S.matmul_int8(flat, flat_s, flat, flat_s).any()
    assert S.quantize_int8(torch.empty(0, 5, device="cuda"))[0].shape == (0, 128)
    assert S.linear_int8(torch.empty(0, 128, device="cuda"), q, s).shape == (0, 4)
    assert S.linear_int8(torch.ones(3, 128, device="cuda"), q[:0], s[:0]).shape == (3, 0)


def test_rows_past_32_bit_offsets():
    """A table of 4.6 GB of whole numbers: rows at both ends."""
    n, kp = 6_000_000, 768
    q = torch.empty(n, kp, dtype=torch.int8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(2)
    for i in range(0, n, 1 << 20):
        q[i:i + (1 << 20)] = torch.randint(-127, 128, (min(1 << 20, n - i), kp), device="cuda", generator=g, dtype=torch.int8)
    scale = torch.rand(n, device="cuda", generator=g)
    a, sa = _operand(3, kp, 5)
    c = S.matmul_int8(a, sa, q, scale, dtype=torch.float32)
    for first in (0, 2_796_000, 5_592_000, n - 500):
        rows = slice(first, first + 500)
        assert torch.equal(c[:, rows], _product(a, sa, q[rows], scale[rows], torch.float32))
    x = torch.randn(6_000, kp, device="cuda", generator=g)
    c = S.matmul_int8(*S.quantize_int8(x), q[:400_000], scale[:400_000])  # results past 2^31 elements
    xq, xs = S.quantize_int8(x[-2:])
    assert torch.equal(c[-2:, -3000:], _product(xq, xs, q[397_000:400_000], scale[397_000:400_000], torch.bfloat16))


def test_a_graph_replays_with_new_inputs():
    x = torch.randn(70, 500, device="cuda")
    q, scale = S.quantize_int8(torch.randn(3000, 500, device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        S.linear_int8(x, q, scale)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = S.linear_int8(x, q, scale)
    for _ in range(4):
        x.copy_(torch.randn(70, 500, device="cuda"))
        want = S.linear_int8(x, q, scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_no_gradient():
    x = torch.randn(5, 128, device="cuda", requires_grad=True)
    q, scale = S.quantize_int8(torch.randn(7, 128, device="cuda"))
    y = S.linear_int8(x, q, scale)
    with pytest.raises(RuntimeError, match="linear_int8 has no gradient"):
        y.float().sum().backward()
    with torch.no_grad():
        assert not S.linear_int8(x, q, scale).requires_grad


def test_refusals():
    x = torch.randn(5, 128, device="cuda")
    q, s = S.quantize_int8(x)
    bad = [
        (lambda: S.quantize_int8(x.cpu()), "x: a tensor on the GPU"),
        (lambda: S.quantize_int8(x.double()), "x: float32"),
        (lambda: S.quantize_int8(x.t()), "side by side"),
        (lambda: S.matmul_int8(q[:, :64], s, q, s), "a: contiguous int8"),
        (lambda: S.matmul_int8(q.view(torch.uint8), s, q, s), "a: contiguous int8"),
        (lambda: S.matmul_int8(q, s[:4], q, s), "a_scale"),
        (lambda: S.matmul_int8(q, s.double(), q, s), "a_scale"),
        (lambda: S.matmul_int8(q, s, q.cpu(), s), "b: a tensor on the GPU"),
        (lambda: S.matmul_int8(q, s, torch.cat([q, q], 1), s), "do not go together"),
        (lambda: S.matmul_int8(q, s, q, s, dtype=torch.float64), "dtype"),
        (lambda: S.linear_int8(x, q, s, dtype=torch.int32), "dtype"),
        (lambda: S.linear_int8(torch.randn(5, 129, device="cuda"), q, s), "do not go together"),
        (lambda: S.linear_int8(x, q.cpu(), s), "q: a tensor on the GPU"),
    ]
    for call, words in bad:
        with pytest.raises(ValueError, match=words):
            call()


@pytest.mark.parametrize("kind", list(TYPES))
def test_few_rows_in_one_launch(kind):
    """Up to 4 rows of up to 512 columns against up to 200000, and the first sizes past each bound, with
    a spoilt row among them."""
    g = torch.Generator(device="cuda").manual_seed(7)
    q, scale = _operand(200_001, 512, 9)
    for m, n, d in ((1, 1, 1), (4, 63, 130), (3, 65, 512), (2, 129, 127), (5, 300, 512), (4, 300, 513), (4, 200_000, 100),
                    (4, 200_001, 100), (3, 130_000, 512), (4, 64, 129)):
        kp = -(-d // 128) * 128
        b = torch.zeros(n, kp, dtype=torch.int8, device="cuda")
        b[:, :min(d, 512)] = q[:n, :min(d, 512)]
        x = torch.randn(m, d + 1, device="cuda", generator=g).to(TYPES[kind])[:, 1:]
        if m > 2:
            x[1, d - 1] = math.nan
        xq, xs = S.quantize_int8(x)
        for dtype in TYPES.values():
            got = S.linear_int8(x, b, scale[:n] * 2.0 ** -8, dtype=dtype)
            want = _product(xq, xs, b, scale[:n] * 2.0 ** -8, dtype)
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num()), (m, n, d)
            if m > 2:
                assert got[1].isnan().all() and not got[0].isnan().any()


def test_rows_without_columns():
    """Sums over nothing are 0, for few rows as for many, as matmul_int8 has them."""
    for kind in TYPES.values():
        q, scale = S.quantize_int8(torch.empty(6, 0, device="cuda"))
        for m in (1, 3, 4, 5, 40):
            for dtype in TYPES.values():
                y = S.linear_int8(torch.empty(m, 0, dtype=kind, device="cuda"), q, scale, dtype=dtype)
                assert y.shape == (m, 6) and y.dtype == dtype and not y.any()


def test_no_gradient_is_lost_in_silence():
    """Results that depend on a tensor that requires a gradient raise when they are differentiated."""
    w = torch.randn(7, 128, device="cuda", requires_grad=True)
    x = torch.randn(5, 128, device="cuda")
    q, scale = S.quantize_int8(w)
    with pytest.raises(RuntimeError, match="quantize_int8 has no gradient"):
        scale.sum().backward()
    xq, xs = S.quantize_int8(x)
    assert not xs.requires_grad and not q.requires_grad
    factor = torch.full((7,), 2.0, device="cuda", requires_grad=True)
    by = scale.detach() * factor
    for call, name in ((lambda: S.linear_int8(x, q, by), "linear_int8"), (lambda: S.matmul_int8(xq, xs, q, by), "matmul_int8"),
                       (lambda: S.matmul_int8(q, by, xq, xs), "matmul_int8")):
        with pytest.raises(RuntimeError, match=f"{name} has no gradient"):
            call().float().sum().backward()
    want = S.linear_int8(x, q, by.detach())
    assert not want.requires_grad and torch.equal(S.linear_int8(x, q, by), want)
    with torch.no_grad():
        assert not S.quantize_int8(w)[1].requires_grad and not S.matmul_int8(xq, xs, q, by).requires_grad
