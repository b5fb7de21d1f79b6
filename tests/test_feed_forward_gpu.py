"""The gated feed-forward block and its gradients against the 64-bit definition."""

import pytest
import torch

from tests.block_helpers import DTYPES, STEP, TINY, U, assert_bounded, assert_norm, normal
from oracle import block_oracle as oracle

pytestmark = pytest.mark.gpu


def bounds(dy, x, wg, wu, wd):
    """The 64-bit result of the call and its gradients with their worst-case errors: sums over k products are off
    by k(n) of the sum of magnitudes, hidden values and their gradients by a rounding to the type on top."""
    t = x.dtype
    fp32 = t == torch.float32
    u, uh = U[t], 2.0 ** -22 if fp32 else U[t]      # (sigmoid: two approximations of 2^-22 or so)
    # fp32: six products of parts, what is left out is below 2^-21; 16 products are one addition
    k = lambda n: ((6 * n / 16 + 8) * STEP + 2.0 ** -21) if fp32 else (n / 16 + 8) * STEP
    dy, x, wg, wu, wd = (v.double().reshape(-1, v.shape[-1]) for v in (dy, x, wg, wu, wd))
    (rows, c), (o, h_) = x.shape, wd.shape
    a, b = x @ wg.T, x @ wu.T
    s = torch.sigmoid(a)
    silu, slope = a * s, s * (1 + a * (1 - s))
    h, dh = silu * b, dy @ wd
    da, db = dh * b * slope, dh * silu
    ea, eb = k(c) * (x.abs() @ wg.abs().T), k(c) * (x.abs() @ wu.abs().T)
    sig = 8 * 2.0 ** -22 * (1 + a.abs())
    eh = TINY[t] + uh * h.abs() + 1.1 * b.abs() * ea + silu.abs() * eb + sig * (a * b).abs()
    edh = k(o) * (dy.abs() @ wd.abs())
    edb = TINY[t] + uh * db.abs() + silu.abs() * edh + 1.1 * dh.abs() * ea + sig * (a * dh).abs()
    eda = TINY[t] + uh * da.abs() + (b * slope).abs() * edh + 1.1 * dh.abs() * eb + 0.5 * (dh * b).abs() * ea + sig * (dh * b).abs()
    y = h @ wd.T
    ey = u * y.abs() + eh @ wd.abs().T + k(h_) * (h.abs() @ wd.abs().T)
    dx = da @ wg + db @ wu
    ex = u * dx.abs() + eda @ wg.abs() + edb @ wu.abs() + k(2 * h_) * (da.abs() @ wg.abs() + db.abs() @ wu.abs())
    weight = lambda d, e, v: (d.T @ v, u * (d.T @ v).abs() + e.T @ v.abs() + (k(rows) + 64 * STEP) * (d.abs().T @ v.abs()))
    dg, eg = weight(da, eda, x)
    du, eu = weight(db, edb, x)
    dd = dy.T @ h
    ed = u * dd.abs() + dy.abs().T @ eh + (k(rows) + 64 * STEP) * (dy.abs().T @ h.abs())
    return (y, dx, dg, du, dd), (ey, ex, eg, eu, ed)


NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down")


def draw(rows, c, h, o, dtype, lead=None):
    lead = lead or (rows,)
    x, dy = normal(*lead, c, seed=1, dtype=dtype), normal(*lead, o, seed=2, dtype=dtype)
    wg, wu = normal(h, c, seed=3, dtype=dtype, std=c ** -0.5), normal(h, c, seed=4, dtype=dtype, std=c ** -0.5)
    return dy, x, wg, wu, normal(o, h, seed=5, dtype=dtype, std=h ** -0.5)


def run(dy, x, *w):
    from trifast_b200 import gated_feed_forward
    leaves = [t.detach().requires_grad_() for t in (x, *w)]
    y = gated_feed_forward(*leaves)
    return [y, *torch.autograd.grad(y, leaves, dy)]


def check(dy, x, wg, wu, wd, norm=True):
    got = run(dy, x, wg, wu, wd)
    want, bound = bounds(dy, x, wg, wu, wd)
    # (typical, not worst: independent roundings of hidden values and results, each below u, add up in squares)
    rel = 4e-6 if x.dtype == torch.float32 else 1.5 * U[x.dtype]
    for name, g, e, b, like in zip(NAMES, got, want, bound, (dy, x, wg, wu, wd)):
        assert g.dtype == x.dtype and g.shape == like.shape
        assert_bounded(g.reshape(e.shape), e, b, name)
        if norm and e.numel() >= 256:
            assert_norm(g.reshape(e.shape), e, rel, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,h,o", [
    (1, 128, 512, 128),      # one token
    (1, 1, 1, 1), (2, 3, 5, 7), (129, 8, 16, 8), (129, 8, 520, 8), (65, 128, 1000, 100),
    (127, 64, 256, 64), (128, 128, 128, 128), (300, 128, 512, 128),
    (257, 100, 290, 100),    # rows that TMA cannot address
    (200, 130, 70, 66), (64, 72, 200, 264), (130, 264, 130, 40), (333, 256, 384, 128),
    (40, 520, 520, 520),
])
def test_sizes(rows, c, h, o, dtype):
    check(*draw(rows, c, h, o, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", range(1, 10))
@pytest.mark.parametrize("c,h,o", [(128, 512, 128), (33, 70, 5), (520, 1032, 264), (8, 8, 1)])
def test_few_rows(rows, c, h, o, dtype):
    """A few tokens: rows alone, of a wider tensor and at odd distances."""
    from trifast_b200 import gated_feed_forward
    dy, x, *w = draw(rows, c, h, o, dtype)
    wide = normal(rows, c + 13, seed=9, dtype=dtype)
    for v in (x, wide[:, 8:8 + c], wide[:, 1:1 + c]):
        want, bound = bounds(dy, v, *w)
        assert_bounded(gated_feed_forward(v, *w), want[0], bound[0], "y")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 3, 8])
@pytest.mark.parametrize("c,h,o", [(289, 909, 301), (520, 1024, 1300), (601, 2048, 40), (1500, 24, 1200), (1111, 601, 7)])
def test_few_rows_of_wide_blocks(rows, c, h, o, dtype):
    """Two kernels: a warp or a block to a result, pieces or elements."""
    from trifast_b200 import gated_feed_forward
    dy, x, *w = draw(rows, c, h, o, dtype)
    want, bound = bounds(dy, x, *w)
    y = gated_feed_forward(x, *w)
    assert_bounded(y, want[0], bound[0], "y")
    assert torch.equal(y, gated_feed_forward(x, *w))


@pytest.mark.parametrize("rows,c,dtype", [(45001, 136, torch.bfloat16), (45001, 131, torch.float16), (15003, 24, torch.float32)])
def test_several_chunks_of_hidden_values(rows, c, dtype):
    """Three chunks of rows in the workspace, whose weight gradients are added up, the same bits each time."""
    from trifast_b200 import gated_feed_forward
    dy, x, *w = draw(rows, c, 2048, c, dtype)
    check(dy, x, *w)
    leaves = [t.clone().requires_grad_() for t in (x, *w)]
    run = lambda: torch.autograd.grad(gated_feed_forward(*leaves), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(run(), run()))


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("rows,c,h,o", [
    (9472, 128, 512, 128), (9601, 128, 64, 128), (18945, 128, 130, 40), (20011, 40, 200, 128), (40003, 128, 64, 128),
    (38017, 64, 256, 64), (9999, 64, 70, 24), (37889, 100, 290, 100), (12001, 8, 8, 8), (57000, 128, 384, 128),
])
def test_rows_of_up_to_128_elements(rows, c, h, o, dtype):
    """The kernels that keep the hidden values on chip: one and two row tiles to an item, one chunk of hidden units
    and several, ragged ends of everything."""
    check(*draw(rows, c, h, o, dtype))


def test_sums_of_many_rows_in_one_block():
    """More row tiles to one block than a run of sums holds."""
    check(*draw(66001, 16, 4737, 16, torch.bfloat16))


@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_padded_rows_in_chunks(dtype):
    """Rows that have to be laid out anew, of more than one chunk, by the kernels that keep the hidden values on chip."""
    check(*draw(400001, 33, 40, 33, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c,h", [(64, 128), (192, 320)])
def test_many_rows(c, h, dtype):
    """More rows than a chunk of the workspace holds, the last chunk ragged; weight gradients over all of them."""
    rows = 60001 if c == 64 else 30011
    check(*draw(rows, c, h, c, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_leading_dimensions_and_strides(dtype):
    """Rows of a wider tensor, odd offsets, a transposed map, transposed weights, an expanded gradient."""
    from trifast_b200 import gated_feed_forward
    dy, x, wg, wu, wd = draw(0, 32, 48, 24, dtype, lead=(5, 6))
    wide = normal(5, 6, 80, seed=7, dtype=dtype)
    check(dy, wide[..., 16:48], wg, wu, wd)
    check(dy, wide[..., 3:35], wg, wu, wd)
    check(dy.transpose(0, 1), wide.transpose(0, 1)[..., :32], wg, wu, wd)
    check(dy, x, wg.T.contiguous().T, wu, wd.T.contiguous().T)
    check(dy[:1, :1], wide[:1, :1, 1:33], wg, wu, wd)
    x = x.clone().requires_grad_()
    gated_feed_forward(x, wg, wu, wd).sum().backward()
    want, bound = bounds(torch.ones_like(dy), x.detach(), wg, wu, wd)
    assert_bounded(x.grad.reshape(-1, 32), want[1], bound[1], "dx of an expanded gradient")


@pytest.mark.parametrize("dtype", DTYPES)
def test_gate_far_from_zero(dtype):
    """Gates beyond where an exponential overflows: silu is 0 or the value itself."""
    from trifast_b200 import gated_feed_forward
    x = torch.tensor([[-30000.0], [-200.0], [-90.0], [0.0], [90.0], [200.0], [1000.0]], device="cuda").to(dtype)
    one = torch.ones(1, 1, device="cuda", dtype=dtype)
    y = gated_feed_forward(x, one, one / 1024, one)
    a = x.double()
    want = a * torch.sigmoid(a) * a / 1024
    assert_bounded(y, want, 2.5 * U[dtype] * want.abs() + 2.0 ** -20 * want.abs() + 1e-30, "y")


def test_nonfinite_rows_stay_in_their_rows():
    from trifast_b200 import gated_feed_forward
    for dtype in DTYPES:
        dy, x, wg, wu, wd = draw(300, 64, 128, 64, dtype)
        clean = gated_feed_forward(x, wg, wu, wd)
        x[7, 3], x[299, 0] = float("nan"), float("inf")
        y = gated_feed_forward(x, wg, wu, wd)
        assert y[7].isnan().all() and not torch.isfinite(y[299]).any()
        keep = torch.ones(300, dtype=torch.bool, device="cuda")
        keep[[7, 299]] = False
        assert torch.equal(y[keep], clean[keep])


def test_only_what_is_asked_for():
    from trifast_b200 import gated_feed_forward
    dy, *ts = draw(200, 64, 96, 64, torch.bfloat16)
    full = [t.clone().requires_grad_() for t in ts]
    want = torch.autograd.grad(gated_feed_forward(*full), full, dy)
    for i in range(4):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate(ts)]
        got, = torch.autograd.grad(gated_feed_forward(*leaves), [leaves[i]], dy)
        assert torch.equal(got, want[i])
    assert not gated_feed_forward(*ts).requires_grad


def test_no_rows():
    from trifast_b200 import gated_feed_forward
    _, _, *w = (t.requires_grad_() for t in draw(3, 16, 24, 8, torch.float16))
    x = torch.empty(4, 0, 16, device="cuda", dtype=torch.float16, requires_grad=True)
    y = gated_feed_forward(x, *w)
    assert y.shape == (4, 0, 8)
    dx, *dw = torch.autograd.grad(y, (x, *w), torch.empty_like(y))
    assert dx.shape == x.shape and all(torch.equal(g, torch.zeros_like(p)) for g, p in zip(dw, w))


def test_same_bits_again():
    """No order of additions depends on timing."""
    case = draw(20011, 128, 256, 128, torch.bfloat16)
    first = run(*case)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, run(*case)))


@pytest.mark.parametrize("hidden", [256, 576])
def test_rows_do_not_depend_on_their_neighbours(hidden):
    """A row's result is the same in a batch of any size (of more than eight rows) and at any place of it."""
    from trifast_b200 import gated_feed_forward
    _, x, *w = draw(400, 128, hidden, 128, torch.bfloat16)
    y = gated_feed_forward(x, *w)
    for i in (0, 120, 128, 391):
        assert torch.equal(gated_feed_forward(x[i:i + 9], *w), y[i:i + 9])
    assert torch.equal(gated_feed_forward(x[37:], *w), y[37:])
    # nor on how many there are
    many = normal(40000, 128, seed=8, dtype=torch.bfloat16)
    many[:400] = x
    assert torch.equal(gated_feed_forward(many, *w)[:400], y)


def test_gradient_against_differences():
    """Central differences of the operator itself along a random direction: off by at most what halving the step
    changes, and by the rounding of the two sums."""
    from trifast_b200 import gated_feed_forward
    dy, *ts = draw(30, 24, 40, 16, torch.float32)
    leaves = [t.clone().requires_grad_() for t in ts]
    y = gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    for i, g in enumerate(grads):
        v = normal(*g.shape, seed=9, std=float(ts[i].std()))
        def along(e):
            f = lambda s: (gated_feed_forward(*(t + s * e * v if j == i else t for j, t in enumerate(ts))).double() * dy.double()).sum()
            return float(f(1) - f(-1)) / (2 * e)
        e = 2.0 ** -6
        d, d2 = along(e), along(2 * e)
        noise = 64 * 2.0 ** -24 * float((dy.abs() * (1 + y.detach().abs())).sum()) / e
        assert abs(float((g.double() * v.double()).sum()) - d) <= abs(d - d2) + noise
