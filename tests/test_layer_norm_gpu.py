"""Layer norm and its gradients against the 64-bit definition."""

import pytest
import torch

from tests.block_helpers import DTYPES, STEP, U, assert_bounded, normal
from oracle import block_oracle as oracle

pytestmark = pytest.mark.gpu


def bounds(x, w, b, dy, eps, wt):
    """Worst cases.  A row lies in threads of 16 elements at most (rows beyond 8192: of width / 512), joined in
    9 steps, so a row's sums are off by k = 32 + width / 256 steps of their magnitudes; mean, deviation and r
    make that a relative error of xh of d = k (max|x| r + 3) steps per element."""
    t = x.dtype
    x, dy = x.double(), dy.double()
    width = x.shape[-1]
    k = 32 + width / 256
    _, xh, r = oracle.layer_norm(x, None, None, eps)
    wd = torch.ones(width, dtype=torch.float64, device=x.device) if w is None else w.double()
    bd = 0 * wd if b is None else b.double()
    top = lambda v: v.abs().amax(-1, keepdim=True)
    dxh = k * STEP * (top(x) * r + 3 * (xh.abs() + 1)) * (1 + xh.abs())
    y = xh * wd + bd
    by = U[t] * y.abs() + wd.abs() * dxh + 2 * STEP * (y.abs() + (xh * wd).abs())
    g = dy * wd
    m2 = (g * xh).mean(-1, keepdim=True)
    dm = k * STEP * (top(g) * (1 + top(xh))) + (g.abs() * dxh).mean(-1, keepdim=True)
    dx, dw, db = oracle.layer_norm_grads(dy, x, w, eps)
    bdx = U[t] * dx.abs() + r * (dm * (1 + xh.abs()) + m2.abs() * dxh) + \
        4 * STEP * r * (g.abs() + top(g) * (1 + xh.abs())) * (1 + k * (top(x) * r + 4))
    flat = lambda v: v.reshape(-1, width)
    # a thread adds its rows one by one: one of 2 x 8 or more row groups of each block, 64 rows of a long one;
    # then at most 1184 blocks in 32 lanes
    rows = flat(x).shape[0]
    n = 64 + rows / 16 + 1184 / 32
    bdw = U[wt] * dw.abs() + n * STEP * flat(dy * xh).abs().sum(0) + flat(dy.abs() * dxh).sum(0)
    bdb = U[wt] * db.abs() + n * STEP * flat(dy).abs().sum(0)
    return y, by, (dx, dw, db), (bdx, bdw, bdb)


def check(x, w, b, dy, eps=1e-5):
    from trifast_b200 import layer_norm
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    wanted = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, wanted, dy)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    want_y, by, want, bound = bounds(x, w, b, dy, eps, x.dtype if w is None else w.dtype)
    assert_bounded(y, want_y, by, "y")
    for name, g, e, bd, t in zip(("dx", "dw", "db"), grads, want, bound, wanted):
        assert g.dtype == t.dtype and g.shape == t.shape
        assert_bounded(g, e, bd, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (2, 7), (5, 8), (33, 64), (9, 65), (1000, 128), (17, 130), (40, 256), (21, 500),
                                        (33, 512), (7, 1000), (5, 1024), (9, 1999), (4, 2048), (3, 4096), (2, 8190), (3, 8192), (2, 8193),
                                        (130, 8200)])
def test_widths(rows, width, dtype):
    x, dy = normal(rows, width, seed=1, dtype=dtype), normal(rows, width, seed=2, dtype=dtype)
    check(x, (1 + 0.3 * normal(width, seed=3)).to(dtype), (0.3 * normal(width, seed=4)).to(dtype), dy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("affine", ["none", "fp32", "weight"])
@pytest.mark.parametrize("width", [100, 128, 1280])
def test_affine_types(affine, width, dtype):
    x, dy = normal(2, 5, 6, width, seed=1, dtype=dtype), normal(2, 5, 6, width, seed=2, dtype=dtype)
    w = None if affine == "none" else normal(width, seed=3, dtype=torch.float32 if affine == "fp32" else dtype)
    b = normal(width, seed=4) if affine == "fp32" else None
    check(x, w, b, dy, eps=1e-3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_and_rows_of_one_value(dtype):
    """More rows than the blocks take in one go; rows whose variance is 0 are eps alone."""
    rows, width = 70001, 32
    x, dy = normal(rows, width, seed=1, dtype=dtype), normal(rows, width, seed=2, dtype=dtype)
    x[5::1000] = 3.0
    check(x, normal(width, seed=3, dtype=dtype), normal(width, seed=4, dtype=dtype), dy, eps=1e-2)


def test_values_far_from_zero():
    """The variance is that of the deviations: a mean of 1000 deviations costs no more than its digits."""
    x = normal(64, 256, seed=1) + 1000.0
    check(x, normal(256, seed=2), normal(256, seed=3), normal(64, 256, seed=4))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strided_rows_and_gradients(dtype):
    """Rows of a wider tensor, a transposed map, a base that is not on 16 bytes, an expanded gradient."""
    from trifast_b200 import layer_norm
    wide = normal(6, 7, 96, seed=1, dtype=dtype)
    w, b = normal(40, seed=2, dtype=dtype), normal(40, seed=3, dtype=dtype)
    for x in (wide[..., 8:48], wide[..., 3:43], wide.transpose(0, 1)[..., 8:48], wide[:, ::2, 16:56], wide[:, :1, :40]):
        check(x, w, b, normal(*x.shape, seed=5, dtype=dtype))
    x = wide[..., :40].contiguous().requires_grad_()
    layer_norm(x, w, b).sum().backward()
    dy = torch.ones_like(x)
    want_y, by, want, bound = bounds(x.detach(), w, b, dy, 1e-5, dtype)
    assert_bounded(x.grad, want[0], bound[0], "dx of an expanded gradient")


def test_nonfinite_rows_stay_in_their_rows():
    from trifast_b200 import layer_norm
    x = normal(64, 128, seed=1, dtype=torch.bfloat16)
    clean = layer_norm(x)
    x[3, 5], x[40, 0] = float("inf"), float("nan")
    y = layer_norm(x)
    assert not torch.isfinite(y[3]).any() and y[40].isnan().all()
    keep = torch.ones(64, dtype=torch.bool, device="cuda")
    keep[[3, 40]] = False
    assert torch.equal(y[keep], clean[keep])



# widths of each way of sharing a row among threads, whose rows begin and end inside 16-byte pieces
ODD_WIDTHS = [1, 2, 3, 5, 7, 9, 25, 27, 33, 59, 65, 91, 101, 129, 249, 251, 257, 301, 505, 507, 777, 1023, 1273, 1275, 1999, 2553, 2555,
              2901, 4089, 4091, 5001, 5113, 5115, 8001, 8185]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", ODD_WIDTHS)
def test_rows_inside_pieces(width, dtype):
    """Every class of rows, more than one turn of a block, a mean of many deviations."""
    rows = max(21, min(5003, 400_000 // width))
    x, dy = normal(rows, width, seed=1, dtype=dtype), normal(rows, width, seed=2, dtype=dtype)
    x[::3] += 30.0
    check(x, (1 + 0.3 * normal(width, seed=3)).to(dtype), (0.3 * normal(width, seed=4)).to(dtype), dy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [3, 9, 65, 301, 1023, 1999, 2901, 4091, 5001, 8001])
def test_neighbours_of_rows_inside_pieces(width, dtype):
    """What lies in a row's first and last piece beside it (rows that are not finite, here) is not seen."""
    from trifast_b200 import layer_norm
    x, dy = normal(24, width, seed=1, dtype=dtype), normal(24, width, seed=2, dtype=dtype)

    def run(x, dy):
        leaf = x.clone().requires_grad_()
        y = layer_norm(leaf)
        return y.detach(), torch.autograd.grad(y, leaf, dy)[0]
    clean = run(x, dy)
    bad, bad_dy = x.clone(), dy.clone()
    bad[::2] = float("nan")
    bad_dy[::2] = float("inf")
    got = run(bad, bad_dy)
    for c, g in zip(clean, got):
        assert torch.equal(c[1::2], g[1::2]) and g[::2].isnan().all()


def test_only_what_is_asked_for():
    from trifast_b200 import layer_norm
    x, w, b = normal(50, 96, seed=1), normal(96, seed=2), normal(96, seed=3)
    dy = normal(50, 96, seed=4)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(layer_norm(*full), full, dy)
    for i in range(3):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(layer_norm(*leaves), [leaves[i]], dy)
        assert torch.equal(got, want[i])
        got, = torch.autograd.grad(layer_norm(*full), [full[i]], dy)
        assert torch.equal(got, want[i])
    assert not layer_norm(x, w, b).requires_grad


def test_no_rows():
    from trifast_b200 import layer_norm
    x = torch.empty(0, 4, 24, device="cuda", requires_grad=True)
    w = torch.ones(24, device="cuda", requires_grad=True)
    y = layer_norm(x, w, w.detach())
    assert y.shape == x.shape
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(w))


def test_same_bits_again():
    """No order of additions depends on timing."""
    from trifast_b200 import layer_norm
    x, w = normal(30011, 128, seed=1, dtype=torch.bfloat16).requires_grad_(), normal(128, seed=2).requires_grad_()
    b, dy = normal(128, seed=3).requires_grad_(), normal(30011, 128, seed=4, dtype=torch.bfloat16)
    run = lambda: torch.autograd.grad(layer_norm(x, w, b), (x, w, b), dy)
    first = run()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, run()))


def test_gradient_against_differences():
    """Central differences of the operator itself along a random direction: off by at most what halving the step
    changes, and by the rounding of the two sums."""
    from trifast_b200 import layer_norm
    x, w, b, dy = normal(20, 48, seed=1), normal(48, seed=2), normal(48, seed=3), normal(20, 48, seed=4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    for i, g in enumerate(grads):
        v = normal(*g.shape, seed=9)
        def along(e):
            f = lambda s: (layer_norm(*(t + s * e * v if j == i else t for j, t in enumerate((x, w, b)))).double() * dy.double()).sum()
            return float(f(1) - f(-1)) / (2 * e)
        e = 2.0 ** -6
        d, d2 = along(e), along(2 * e)
        noise = 64 * 2.0 ** -24 * float((dy.abs() * (1 + layer_norm(x, w, b).abs())).sum()) / e
        assert abs(float((g.double() * v.double()).sum()) - d) <= abs(d - d2) + noise
