"""The score operators together: a narrow embedding trained on the stage's own exact lists."""
import pytest
import torch  # before the library is loaded

pytestmark = pytest.mark.gpu


def test_training_on_exact_neighbours():
    from filtervectorcode_refactor_amd import compact

    X = compact.vectors(1500, 96, seed=3)
    losses, before, after = compact.train(X, k=16, narrow=24, steps=40)
    assert all(l == l and l >= 0 for l in losses)
    assert losses[-1] < 0.8 * losses[0]
    assert after > before
    again, _, _ = compact.train(X, k=16, narrow=24, steps=3)
    assert again == losses[:3]  # the same every time
