"""Layer norm without an eps: what a block computes for the rows that it does not have enters nothing."""

import pytest
import torch

from tests.block_helpers import DTYPES, normal
from tests.test_layer_norm_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 64), (33, 64), (1, 128), (33, 128), (130, 256), (7, 512), (1, 101), (41, 101), (5, 203), (3, 1000),
                                        (149, 1000), (3, 1999), (301, 2048), (2, 4095), (3, 8192), (66, 8200)])
def test_gradients_without_eps(rows, width, dtype, eps):
    """The definition's values, for numbers of rows that leave places of a block's turn empty (1e-60 is 0 in fp32)."""
    x, dy = normal(rows, width, seed=1, dtype=dtype), normal(rows, width, seed=2, dtype=dtype)
    check(x, (1 + 0.3 * normal(width, seed=3)).to(dtype), (0.3 * normal(width, seed=4)).to(dtype), dy, eps=eps)


def test_row_of_one_value_without_eps():
    """Its deviation is 0: not finite in its own row and in the weight's gradient, by the definition; no other row sees it."""
    from trifast_b200 import layer_norm
    x = normal(40, 96, seed=1)
    x[7] = 2.0
    y = layer_norm(x, eps=0.0)
    keep = torch.arange(40, device="cuda") != 7
    assert y[7].isnan().all() and torch.isfinite(y[keep]).all()
