"""Sizes that the operators around the attention refuse, before anything is cut to a narrower type."""

import ctypes as C

import pytest
import torch

from tests.test_block_run_gpu import on_cuda_kernel

WIDTHS = [(1 << 20) + 1, 1 << 31, (1 << 32) + 8, (1 << 33) + 64]


@pytest.mark.parametrize("width", WIDTHS)
def test_layer_norm_refuses_wide_rows(width):
    x = torch.empty(0, width)
    with pytest.raises(ValueError, match=f"width must be at most 1048576; got {width}"):
        on_cuda_kernel("layer_norm", x, None, None, 1e-5)
    with pytest.raises(ValueError, match=f"width must be at most 1048576; got {width}"):
        on_cuda_kernel("layer_norm_grads", x, x, None, 1e-5, True, False, False)


@pytest.mark.parametrize("width", [65537, (1 << 32) + 8])
def test_feed_forward_refuses_wide_rows(width):
    x, g, d = torch.empty(0, width), torch.empty(1, 1).expand(1, width), torch.zeros(4, 1)
    with pytest.raises(ValueError, match="at most 65536"):
        on_cuda_kernel("gated_feed_forward", x, g, g, d)
