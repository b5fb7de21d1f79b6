"""Dropout with the residual sum against the 64-bit definition and the generator's."""

import pytest
import torch

from tests.block_helpers import DTYPES, STEP, U, assert_bounded, normal
from oracle import block_oracle as oracle

pytestmark = pytest.mark.gpu


def check(x, residual, p, seed, offset=0, shared=None, op_seed=None):
    from trifast_b200 import dropout_add
    keep = oracle.keep_mask(x.shape, p, seed, offset, shared).to(x.device)
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, residual)]
    y = dropout_add(*leaves, p, seed if op_seed is None else op_seed, offset=offset, shared_dim=shared)
    want = oracle.dropout_add(x, residual, keep, p)
    # the scale, its product and the sum in fp32, then the type
    size = oracle.dropout_add(x.abs(), None if residual is None else residual.abs(), keep, p)
    assert y.dtype == x.dtype and y.is_contiguous()
    assert_bounded(y, want, U[x.dtype] * want.abs() + 2 * STEP * size, "y")
    dy = normal(*x.shape, seed=77, dtype=x.dtype, device=x.device)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    want = oracle.dropout_add(dy, None, keep, p)
    assert_bounded(grads[0], want, (U[x.dtype] + STEP) * want.abs(), "dx")
    if residual is not None:
        assert torch.equal(grads[1], dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shared", [None, -3, -2, -1])
@pytest.mark.parametrize("shape", [(1, 1, 1), (5, 7, 24), (9, 4, 33), (3, 130, 8), (65, 3, 16)])
def test_shapes(shape, shared, dtype):
    x, r = normal(*shape, seed=1, dtype=dtype), normal(*shape, seed=2, dtype=dtype)
    check(x, r, 0.3, 0x1234567890ABCDE, 3, shared)
    check(x, None, 0.15, 5, 0, shared)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shared", [-3, -2])
@pytest.mark.parametrize("shape", [(2, 9, 1), (40, 37, 5), (3, 11, 9), (70, 17, 9), (17, 65, 10), (6, 200, 23), (1, 301, 12), (301, 3, 31),
                                   (33, 41, 127), (5, 90, 130), (3, 3, 2047)])
def test_rows_inside_pieces(shape, shared, dtype):
    """Rows of every alignment, tiny ones, several turns and steps of a thread; the other rows of a piece keep their own."""
    x, r = normal(*shape, seed=1, dtype=dtype), normal(*shape, seed=2, dtype=dtype)
    check(x, r, 0.3, -7, 1, shared)
    check(x, None, 0.6, 5, 0, shared)


def test_nothing_behind_a_map_is_written():
    """Results of rows that end inside a piece, in a larger buffer of the caller's."""
    from trifast_b200 import _lib
    n, c = 5, 27
    x = normal(n, n, c, seed=1, dtype=torch.bfloat16)
    y = torch.full((x.numel() + 16,), 3.0, device="cuda", dtype=x.dtype)
    keep = oracle.keep_mask(x.shape, 0.5, 3, 0, -2).cuda()
    d = _lib.Dropout(outer=n, mid=n, inner=c, dtype=_lib.DTYPE_CODE[x.dtype], p=0.5, seed=3, offset=0)
    rc = _lib.load().trifast_dropout_add(d, None, x.data_ptr(), None, y.data_ptr(), torch.cuda.current_stream().cuda_stream)
    _lib.check(rc, "dropout")
    assert torch.equal(y[:x.numel()].view_as(x), torch.where(keep, 2 * x, torch.zeros_like(x)))
    assert (y[x.numel():] == 3).all()


@pytest.mark.parametrize("shared", [None, 0, 1, 2, 3])
def test_batched_maps_and_strides(shared):
    x = normal(2, 6, 5, 40, seed=1, dtype=torch.bfloat16)
    check(x.transpose(1, 2), x.transpose(1, 2), 0.25, 11, 1, shared)
    check(x[..., 1:25], x[..., :24], 0.25, 11, 1, shared)     # a base that is not on 16 bytes


@pytest.mark.parametrize("p", [0.0, 2.0 ** -33, 0.5, 1 - 2.0 ** -20, 1.0])
def test_ends_of_p(p):
    from trifast_b200 import dropout_add
    x, r = normal(40, 48, seed=1), normal(40, 48, seed=2)
    check(x, r, p, 9)
    if p == 1:
        x[:] = float("nan")     # nothing of x enters
        assert torch.equal(dropout_add(x, r, p, 9), r)


def test_dropped_values_do_not_enter():
    from trifast_b200 import dropout_add
    keep = oracle.keep_mask((64, 64), 0.5, 3).cuda()
    x = normal(64, 64, seed=1, dtype=torch.float16)
    x[~keep] = torch.tensor([float("inf"), float("nan")], device="cuda", dtype=x.dtype).repeat(2048)[:int((~keep).sum())]
    y = dropout_add(x, None, 0.5, 3)
    assert torch.equal(y[~keep], torch.zeros_like(y[~keep])) and torch.isfinite(y).all()


def test_seeds():
    """64-bit seeds and offsets, negative ones as their bits; a seed in device memory."""
    x = normal(30, 32, seed=1)
    for seed, offset in ((1 << 62, 0), (-1, 1 << 40), (0, -5), (123, 7)):
        check(x, x, 0.4, seed, offset)
        check(x, x, 0.4, seed, offset, op_seed=torch.tensor([seed], device="cuda"))


def test_share_of_dropped_elements():
    """2^22 entries with p = 0.1: the count is within six standard deviations (a chance of 2e-9)."""
    from trifast_b200 import dropout_add
    n, p = 1 << 22, 0.1
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    for seed in range(3):
        dropped = int((dropout_add(x, None, p, seed) == 0).sum())
        assert abs(dropped - n * p) <= 6 * (n * p * (1 - p)) ** 0.5


def test_large_map_and_far_entries():
    """Every thread's walk along the shared dimension, and a mask of more than 2^22 entries, against a mask drawn
    by the operator on ones, whose first and last entries are the generator's."""
    from trifast_b200 import dropout_add
    for shape, shared in (((300, 200, 128), 0), ((300, 200, 128), 1), ((5, 9, 100003), 0), ((2200, 2500), None)):
        x, r = normal(*shape, seed=1, dtype=torch.bfloat16), normal(*shape, seed=2, dtype=torch.bfloat16)
        small = list(shape)
        if shared is not None:
            small[shared] = 1
        keep = dropout_add(torch.ones(small, device="cuda"), None, 0.5, 21, offset=2) > 0
        first = torch.tensor([w >= 1 << 31 for w in oracle.random_words(4000, 21, 2)])
        assert torch.equal(keep.flatten()[:4000].cpu(), first)
        want = oracle.dropout_add(x, r, keep, 0.5)
        y = dropout_add(x, r, 0.5, 21, offset=2, shared_dim=shared)
        assert_bounded(y, want, U[x.dtype] * want.abs() + 2 * STEP * (2 * x.abs() + r.abs()).double(), str(shape))


def test_no_elements():
    from trifast_b200 import dropout_add
    x = torch.empty(3, 0, 8, device="cuda", requires_grad=True)
    y = dropout_add(x, x.detach(), 0.5, 1, shared_dim=0)
    assert y.shape == x.shape
    assert torch.autograd.grad(y, x, torch.empty_like(y))[0].shape == x.shape


def test_second_gradient():
    """The operator is linear in x: the gradient of its gradient is itself."""
    from trifast_b200 import dropout_add
    x = normal(8, 16, seed=1).requires_grad_()
    dy = normal(8, 16, seed=2).requires_grad_()
    dx, = torch.autograd.grad(dropout_add(x, None, 0.5, 4), x, dy, create_graph=True)
    v = normal(8, 16, seed=3)
    ddy, = torch.autograd.grad(dx, dy, v)
    assert torch.equal(ddy, dropout_add(v, None, 0.5, 4))
