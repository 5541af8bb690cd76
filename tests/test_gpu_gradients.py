"""GPU tests of gradient_norm and clip_gradients against 64 bits: one rounding of the norm, one of
the factor, one of each element."""
import math

import pytest
import torch

import filtervectorcode_refactor_amd as F
from filtervectorcode_refactor_amd import scores as S

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def _grads(lengths, kind, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    types = list(TYPES.values()) if kind == "mixed" else [TYPES[kind]]
    return [(torch.randn(n, device="cuda", generator=g) * size * 2.0 ** (i % 5)).to(types[i % len(types)])
            for i, n in enumerate(lengths)]


def _norm(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def _check(got, grads, norm, most):
    """out = g * by, by = most / norm in 64 bits rounded to 32, the product rounded to 32 bits and
    then to the type: two roundings of 32 bits and one of the type."""
    by = min(1.0, most / norm) if norm else 1.0
    for a, g in zip(got, grads):
        assert a.dtype == g.dtype and a.shape == g.shape
        want = g.double() * by
        bound = want.abs() * (HALF_ULP[g.dtype] * 1.001 + 2.0 ** -23) + TINY[g.dtype]
        assert ((a.double() - want).abs() <= bound).all()


LENGTHS = [[1], [7], [8192], [8193], [3, 0, 5], [100_000, 1, 17], [8192 * 3 + 5, 8191, 2], [3_000_001], [1] * 70,
           [64 + 37 * i for i in range(300)], [0, 4], [20_000_000, 9]]


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16", "mixed"])
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda l: f"{len(l)}x{max(l)}")
def test_against_64_bits(lengths, kind):
    grads = _grads(lengths, kind)
    norm = _norm(grads)
    got = S.gradient_norm(grads)
    assert got.dtype == torch.float32 and got.shape == ()
    # 64-bit sums in either order are within 2^-40 for these lengths; the norm is rounded once
    assert abs(float(got) - norm) <= norm * (2.0 ** -24 + 2.0 ** -40)
    for ratio in (0.25, 0.999, 1.5):
        most = norm * ratio
        out = [torch.full_like(g, 7.0) for g in grads]
        before = [g.clone() for g in grads]
        assert torch.equal(S.clip_gradients(grads, most, out=out), got)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        _check(out, grads, norm, torch.tensor(most, dtype=torch.float32).item())
        mine = [g.clone() for g in grads]
        assert torch.equal(S.clip_gradients(mine, most), got)
        assert all(torch.equal(a, b) for a, b in zip(mine, out))
        if ratio > 1:
            assert all(torch.equal(a, b) for a, b in zip(mine, grads))


@pytest.mark.parametrize("size", [1e30, 1e-30, 1e-40])
def test_squares_past_32_bits(size):
    grads = _grads([1000, 20_000], "fp32", size=size)
    norm = _norm(grads)
    assert abs(float(S.gradient_norm(grads)) - norm) <= norm * 2.0 ** -23 + 2.0 ** -149
    out = [torch.empty_like(g) for g in grads]
    S.clip_gradients(grads, 1.0, out=out)
    _check(out, grads, norm, 1.0)


def test_norms_that_are_not_finite_leave_the_gradients():
    for bad in (math.inf, -math.inf, math.nan):
        grads = _grads([100, 9000, 3], "mixed")
        grads[1][8500] = bad
        before = [g.clone() for g in grads]
        out = [torch.empty_like(g) for g in grads]
        norm = S.clip_gradients(grads, 0.5, out=out)
        assert not torch.isfinite(norm) and bool(norm.isnan()) == math.isnan(bad)
        S.clip_gradients(grads, 0.5)
        for a in (out, grads):
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, before))


def test_largest_norms_of_0_and_infinity():
    grads = _grads([100, 9000], "fp32")
    before = [g.clone() for g in grads]
    S.clip_gradients(grads, math.inf)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    S.clip_gradients(grads, 0.0)
    assert not any(g.any() for g in grads)
    assert float(S.clip_gradients(grads, 0.0)) == 0.0  # and of zeros
    for bad in (-1.0, math.nan):
        with pytest.raises(F.UngHipError, match="negative or NaN"):
            S.clip_gradients(grads, bad)


def test_views_of_any_alignment_and_order():
    """Elements side by side in any order of dimensions, from addresses aligned to an element alone;
    what lies around them is left alone."""
    for kind in TYPES.values():
        whole = torch.randn(40_000, device="cuda").to(kind)
        keep = whole.clone()
        views = [whole[1:9_000], whole[9_001:9_004], whole[10_003:10_003 + 64 * 33].view(64, 33).t(),
                 whole[20_001:20_001 + 4 * 5 * 6].view(4, 5, 6).permute(2, 0, 1), whole[30_000:30_001]]
        grads = [v.clone() for v in views]
        norm = _norm(grads)
        S.clip_gradients(views, norm / 3)
        _check(views, grads, norm, torch.tensor(norm / 3, dtype=torch.float32).item())
        changed = torch.zeros(40_000, dtype=torch.bool, device="cuda")
        for a, b in ((1, 9_000), (9_001, 9_004), (10_003, 10_003 + 64 * 33), (20_001, 20_121), (30_000, 30_001)):
            changed[a:b] = True
        assert torch.equal(whole[~changed], keep[~changed])


def test_none_is_skipped_and_order_does_not_show():
    grads = _grads([100, 9000, 3], "mixed")
    norm = S.gradient_norm(grads)
    assert torch.equal(S.gradient_norm([None, grads[0], None, *grads[1:]]), norm)
    out = [torch.empty_like(g) for g in grads]
    S.clip_gradients([None, *grads], 0.1, out=[None, *out])
    _check(out, grads, _norm(grads), torch.tensor(0.1).item())
    # 64-bit sums: the order of the tensors moves the last of 53 bits, the norm has 24
    assert abs(float(S.gradient_norm(grads[::-1])) - float(norm)) <= float(norm) * 2.0 ** -23


def test_overlaps_are_refused():
    a = torch.randn(1000, device="cuda")
    b = torch.randn(1000, device="cuda")
    keep = a.clone(), b.clone()
    for grads, out in (([a, a], None), ([a[:600], a[500:]], None), ([a, b], [b, a]), ([a[:500]], [a[1:501]]),
                       ([a, b], [b, b])):
        with pytest.raises(F.UngHipError, match="overlap"):
            S.clip_gradients(grads, 0.1, out=out)
    assert torch.equal(a, keep[0]) and torch.equal(b, keep[1])
    S.gradient_norm([a, a])  # read twice: counts twice
    assert abs(float(S.gradient_norm([a, a])) - math.sqrt(2) * _norm([a])) < 1e-4


def test_autograd_sees_that_gradients_were_written():
    w = torch.randn(50, device="cuda", requires_grad=True)
    y = w * 2
    z = (y * y).sum()
    S.clip_gradients([y.detach()], 1e-3)  # the saved y changes under autograd's eyes
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        z.backward()
    with pytest.raises(ValueError, match="no_grad"):
        S.clip_gradients([y], 1.0)
    with pytest.raises(RuntimeError, match="gradient_norm has no gradient"):
        S.gradient_norm([w * 3]).backward()


def test_a_training_step():
    """As a program does: a model's gradients clipped in place, the same as by the formula."""
    g = torch.Generator(device="cuda").manual_seed(2)
    w = [torch.randn(300, 200, device="cuda", generator=g).requires_grad_(),
         torch.randn(300, device="cuda", generator=g).bfloat16().requires_grad_()]
    ((w[0].sum(1) + w[1].float()) ** 2).mean().backward()
    before = [p.grad.clone() for p in w]
    norm = S.clip_gradients([p.grad for p in w], 0.01)
    _check([p.grad for p in w], before, _norm(before), torch.tensor(0.01).item())
    assert abs(float(norm) - _norm(before)) <= _norm(before) * 2.0 ** -23


def test_a_graph_replays_with_new_inputs():
    grads = _grads([5000, 3, 90_000] + [50] * 80, "mixed")
    out = [torch.empty_like(g) for g in grads]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        S.clip_gradients(grads, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = S.clip_gradients(grads, 1.0, out=out)
    for seed in range(4):
        for a, b in zip(grads, _grads([5000, 3, 90_000] + [50] * 80, "mixed", seed, size=10.0 ** (1 - seed * 2))):
            a.copy_(b)
        mine = [torch.empty_like(g) for g in grads]
        want = S.clip_gradients(grads, 1.0, out=mine)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(out, mine))


def test_the_same_every_time():
    grads = _grads([5_000_000, 77], "bf16")
    first = S.gradient_norm(grads)
    assert all(torch.equal(first, S.gradient_norm(grads)) for _ in range(5))


def test_refusals():
    a = torch.randn(10, 10, device="cuda")
    bad = [
        (lambda: S.gradient_norm([]), "at least one"),
        (lambda: S.gradient_norm([None]), "at least one"),
        (lambda: S.gradient_norm([a.cpu()]), "a tensor on the GPU"),
        (lambda: S.gradient_norm([a, a.cpu()]), "a tensor on the GPU"),
        (lambda: S.gradient_norm([a.double()]), "float32"),
        (lambda: S.gradient_norm([a[:, :5]]), "side by side"),
        (lambda: S.gradient_norm([a[:1].expand(10, 10)]), "side by side"),
        (lambda: S.clip_gradients([a], 1.0, out=[]), "out: 1 tensors"),
        (lambda: S.clip_gradients([a], 1.0, out=[a.half()]), "out: the gradients'"),
        (lambda: S.clip_gradients([a], 1.0, out=[a.t()]), "out: the gradients'"),
        (lambda: S.clip_gradients([a], 1.0, out=[torch.empty(100, device="cuda")]), "out: the gradients'"),
    ]
    for call, words in bad:
        with pytest.raises(ValueError, match=words):
            call()


def test_inference_tensors():
    """Tensors of inference mode have no versions that autograd counts."""
    with torch.inference_mode():
        grads = _grads([100, 9000], "mixed")
        before = [g.clone() for g in grads]
        S.clip_gradients(grads, 0.5)
        _check(grads, before, _norm(before), 0.5)


def test_more_partial_sums_than_a_block_adds_up():
    """Three lists of 64 tensors each: the partial sums are joined by a launch of their own."""
    grads = _grads([9000 * 16] * 150, "bf16")
    norm = S.gradient_norm(grads)
    assert abs(float(norm) - _norm(grads)) <= _norm(grads) * (2.0 ** -24 + 2.0 ** -40)
    out = [torch.empty_like(g) for g in grads]
    assert torch.equal(S.clip_gradients(grads, 10.0, out=out), norm)
    _check(out, grads, _norm(grads), 10.0)


def test_parameters_in_their_gradients_place_are_refused():
    """An in-place operation on a leaf that requires a gradient is an error, and changes nothing."""
    layer = torch.nn.Linear(30, 20).cuda()
    layer(torch.randn(5, 30, device="cuda")).square().sum().backward()
    before = [p.detach().clone() for p in layer.parameters()]
    grads = [p.grad for p in layer.parameters()]
    mine = [torch.empty_like(g) for g in grads]
    for call in (lambda: S.clip_gradients(layer.parameters(), 1e-3), lambda: S.clip_gradients(list(layer.parameters()), 1e-3),
                 lambda: S.clip_gradients(layer.parameters(), 1e-3, out=mine),
                 lambda: S.clip_gradients(grads, 1e-3, out=layer.parameters())):
        with pytest.raises(ValueError, match="no_grad"):
            call()
    assert all(torch.equal(p, b) for p, b in zip(layer.parameters(), before))
    S.clip_gradients(grads, 1e-3)
    with torch.no_grad():  # where torch's own in-place operations work too
        S.clip_gradients(layer.parameters(), 1e-3)
    _check([p.detach() for p in layer.parameters()], before, _norm(before), torch.tensor(1e-3).item())


@pytest.mark.parametrize("lengths", [[100, 9000], [30_000, 70_000], [500_000] * 3])
def test_a_norm_past_32_bits_leaves_the_gradients(lengths):
    """Finite gradients whose norm no 32-bit number holds: the norm that the caller sees is infinite, and the
    gradients stay as they are, as with any infinite norm."""
    grads = [torch.full((n,), 3e38, device="cuda") for n in lengths]
    before = [g.clone() for g in grads]
    out = [torch.empty_like(g) for g in grads]
    assert float(S.gradient_norm(grads)) == math.inf
    assert float(S.clip_gradients(grads, 1.0, out=out)) == math.inf
    assert float(S.clip_gradients(grads, 1.0)) == math.inf
    assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(grads, before, out))
