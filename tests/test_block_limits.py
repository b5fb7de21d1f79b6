"""Sizes that the operators around the attention refuse, before anything is cut to a narrower type."""

import ctypes as C

import pytest
import torch

from tests.test_block_run_gpu import on_cuda_kernel
from trifast_b200 import _lib

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


def test_weight_sums_have_a_share_of_the_workspace_for_each_run():
    """Without a device: rows of a chunk beyond 128 tiles have partial sums of their own."""
    lib = _lib.load()
    size = lambda rows, w, h, dt: lib.trifast_feed_forward_backward_workspace_bytes(C.byref(_lib.FeedForward(rows, w, w, w, h, w, dt)))
    for width, hidden in ((136, 8), (200, 16)):
        stride = 4 * (2 * hidden * width + width * hidden)
        for rows in (128 * 128 * 40, 128 * 128 * 100):
            values = 3 * 2 * hidden * (-(-rows // 128) * 128)      # h, da, db of the chunk
            assert size(rows, width, hidden, 2) - values >= stride * (rows // (128 * 128))


@pytest.mark.parametrize("width,dtype,rc", [(8192, 1, -1), (8188, 0, -1), (8192, 0, -1), (8185, 2, -1), (8184, 1, -1), (8186, 1, -12), (8190, 0, -12),
                                            (8193, 0, -12), (8200, 2, -12)])
def test_row_limit_of_layer_norm_is_that_of_long_rows(width, dtype, rc):
    """Rows that a block holds in registers have none: the call goes on to its pointers."""
    lib = _lib.load()
    n = _lib.Norm(rows=4_194_241, ld_x=width, ld_dy=width, width=width, dtype=dtype, affine_dtype=0, eps=1e-5)
    assert lib.trifast_layer_norm(C.byref(n), None, None, None, None, None) == rc
    assert lib.trifast_layer_norm_backward(C.byref(n), *[None] * 7, 0, None) == rc
    n.rows -= 1
    assert lib.trifast_layer_norm(C.byref(n), None, None, None, None, None) == -1
