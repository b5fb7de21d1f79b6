"""The operators around the attention under torch.vmap: as a call for each entry."""

import pytest
import torch

from tests.block_helpers import normal

pytestmark = pytest.mark.gpu


@pytest.mark.filterwarnings("ignore:There is a performance drop")
def test_vmap():
    from trifast_b200 import dropout_add, gated_feed_forward, layer_norm
    x, w, b = normal(3, 5, 24, seed=1), normal(24, seed=2), normal(24, seed=3)
    g, u, d = normal(40, 24, seed=4), normal(40, 24, seed=5), normal(24, 40, seed=6)
    for f in (lambda v: layer_norm(v, w, b), lambda v: gated_feed_forward(v, g, u, d), lambda v: dropout_add(v, v, 0.5, 3)):
        assert torch.equal(torch.vmap(f)(x), torch.stack([f(v) for v in x]))
        # (its transforms of gradients do not take native autograd functions)
        with pytest.raises(RuntimeError, match="functorch transforms"):
            torch.func.grad(lambda v: f(v).square().sum())(x[0])
