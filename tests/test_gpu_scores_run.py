"""The operators of a training and serving run together, as the program of the narrow embedding
calls them: embeddings in 8 bits, cross entropy against the whole table, the gradients clipped,
and lists from the table in 8-bit whole numbers."""
import math

import pytest
import torch  # before the library is loaded

from filtervectorcode_refactor_amd import scores as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("loss", ["lists", "nearest"])
def test_training_and_serving(loss):
    from filtervectorcode_refactor_amd import compact

    X = compact.vectors(700, 96, seed=5)
    student, x, ids, losses, before = compact.fit(X, k=12, narrow=24, steps=6, loss=loss, clip=0.05)
    assert len(losses) == 6 and all(math.isfinite(l) and l >= 0 for l in losses)
    norm = S.gradient_norm([p.grad for p in student.parameters()])
    # scaled by a factor that is rounded once, each element rounded once
    assert float(norm) <= 0.05 * (1 + 2.0 ** -22)
    again = compact.fit(X, k=12, narrow=24, steps=6, loss=loss, clip=0.05)
    assert again[3] == losses and all(torch.equal(a, b) for a, b in zip(student.parameters(), again[0].parameters()))
    served = compact.served_lists(student, x, 12)
    own = torch.arange(700, device="cuda")[:, None]
    assert served.shape == (700, 12) and ((served >= 0) & (served < 700) & (served != own)).all()
    assert (served.sort(dim=1).values.diff(dim=1) > 0).all()  # no id twice


def test_gradients_of_the_step_against_64_bits():
    """One step's gradients by the two matrices: through table_loss and linear_fp8, whose own
    gradients are the products of operands in 8 bits."""
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(200, 32, device="cuda", generator=g).bfloat16().requires_grad_()
    t = torch.randn(300, 32, device="cuda", generator=g).bfloat16().requires_grad_()
    ids = torch.randint(0, 300, (200,), device="cuda", generator=g).int()
    own = ((ids + 7) % 300).int()
    S.table_loss(q, t, ids, without=own, temperature=2.0).mean().backward()
    a, b = q.detach().double().requires_grad_(), t.detach().double().requires_grad_()
    z = (a @ b.t() / 2.0).scatter(1, own.long()[:, None], -math.inf)
    torch.nn.functional.cross_entropy(z, ids.long()).backward()
    p = torch.softmax(z.detach(), dim=1)
    p[torch.arange(200), ids.long()] += 1  # magnitudes of what a gradient sums
    # half a step of bf16 on each weight, half on the result, and 32-bit errors well below a tenth of them
    for got, want, size in ((q.grad, a.grad, p @ b.detach().abs()), (t.grad, b.grad, p.t().contiguous() @ a.detach().abs())):
        assert ((got.double() - want).abs() <= 1.1 * 2.0 ** -8 * (size / 400 + want.abs())).all()


def test_lists_from_whole_numbers_are_those_of_their_scores():
    """quantize_int8, linear_int8 and top_scores one after the other, against the exact product of
    the numbers and a stable sort."""
    g = torch.Generator(device="cuda").manual_seed(2)
    x, table = torch.randn(50, 100, device="cuda", generator=g), torch.randn(3000, 100, device="cuda", generator=g)
    q, scale = S.quantize_int8(table)
    xq, xs = S.quantize_int8(x)
    values, ids, _ = S.top_scores(S.linear_int8(x, q, scale, dtype=torch.float32), 20)
    want = (xq.double() @ q.double().t().contiguous()).float() * (xs[:, None] * scale[None, :])
    order = want.sort(dim=1, descending=True, stable=True)
    assert torch.equal(values, order.values[:, :20]) and torch.equal(ids, order.indices[:, :20].int())
