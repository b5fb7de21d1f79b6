"""Dropout of everything: nothing of x is left, whatever dimension the mask is shared along."""

import pytest
import torch

from oracle import block_oracle as oracle
from tests.block_helpers import DTYPES, normal
from tests.test_dropout_add_gpu import check


@pytest.mark.parametrize("shared", [None, -3, -2, -1])
def test_oracle_keeps_the_shape(shared):
    x = torch.ones(3, 4, 5)
    for p in (0.0, 0.5, 1.0):
        for residual in (None, x):
            y = oracle.dropout_add(x, residual, oracle.keep_mask(x.shape, p, 3, 0, shared), p)
            assert y.shape == x.shape and (p < 1 or torch.equal(y, x.double() if residual is not None else 0 * x.double()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shared", [None, -3, -2, -1])
@pytest.mark.parametrize("shape", [(5, 7, 24), (9, 4, 33), (1, 14, 51), (46, 2, 13)])
def test_everything_dropped(shape, shared, dtype):
    x, r = normal(*shape, seed=1, dtype=dtype), normal(*shape, seed=2, dtype=dtype)
    check(x, r, 1.0, 5, 1, shared)
    check(x, None, 1.0, 5, 1, shared)
