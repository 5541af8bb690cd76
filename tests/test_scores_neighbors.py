"""Neighbour rows as a teacher's entries: types that are taken, and those that are not.  No GPU."""
import numpy as np
import pytest
import torch

from filtervectorcode_refactor_amd import scores as S

IDS = [[3, 0, 0xFFFFFFFF], [1, 2, 7]]
DIST = [[0.5, 2.0, np.inf], [0.0, 1.0, 4.0]]


@pytest.mark.parametrize("make", [lambda: np.array(IDS, np.uint32), lambda: np.array(IDS, np.uint32).view(np.int32),
                                  lambda: np.asfortranarray(np.array(IDS, np.uint32)),
                                  lambda: torch.from_numpy(np.array(IDS, np.uint32).view(np.int32)),
                                  lambda: torch.from_numpy(np.array(IDS, np.uint32))])
def test_ids_of_32_bits(make):
    ids, values = S.entries_of_neighbors(make(), np.array(DIST, np.float32))
    assert ids.dtype == torch.int32 and ids.tolist() == [[3, 0, -1], [1, 2, 7]]
    assert values.dtype == torch.float32 and values.tolist() == [[-0.5, -2.0, -np.inf], [0.0, -1.0, -4.0]]


@pytest.mark.parametrize("dtype", [np.int64, np.uint64, np.int16, np.float32])
def test_other_ids_are_refused(dtype):
    """Read as 32-bit words, 64-bit ids were twice as many columns, every other one 0 or -1."""
    ids = np.array([[3, 0, 5]]).astype(dtype)
    for given in (ids, torch.from_numpy(ids)):
        with pytest.raises(ValueError, match="ids"):
            S.entries_of_neighbors(given, np.zeros((1, 3), np.float32))
