"""The gated feed-forward block where its arithmetic ends: gates whose exponential overflows, hidden values beyond
the largest fp16 number, gradients near the smallest, and sums over millions of rows."""

import pytest
import torch

from tests.block_helpers import DTYPES, STEP, TINY, U, assert_bounded, normal
from tests.test_feed_forward_gpu import bounds, draw, run
from oracle import block_oracle as oracle

pytestmark = pytest.mark.gpu

GATES = [-30000.0, -200.0, -90.0, 0.0, 90.0, 200.0, 1000.0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [7, 8, 9, 40, 300])
@pytest.mark.parametrize("width", [64, 128, 136, 264])
def test_gates_far_from_zero_in_every_kernel(width, rows, dtype):
    """Weights that are the identity (w_up: over 1024): silu is 0 or the value itself, its slope 0 or 1.  Few rows, both
    kernels that keep the hidden values on chip and those that do not, one CTA a tile and two; and their gradients."""
    eye = torch.eye(width, device="cuda")
    x = torch.tensor(GATES, device="cuda")[torch.randint(7, (rows, width), generator=torch.Generator().manual_seed(3)).cuda()].to(dtype)
    dy = normal(rows, width, seed=4, dtype=dtype, std=0.01)
    w = [eye.to(dtype), (eye / 1024).to(dtype), eye.to(dtype)]
    got = run(dy, x, *w)
    a, d = x.double(), dy.double()
    b, on = a / 1024, (a > 0).double() + 0.5 * (a == 0)
    silu, slope = a * (a > 0), on
    h, da, db = silu * b, d * b * slope, d * silu
    # what each kernel rounds: h, da and db to the type, a sigmoid off by 2^-20 in all (its limits are exact), the result
    near = lambda t: 2.0 ** -20 * t.abs() + U[dtype] * t.abs() + TINY[dtype]
    dx = da + db / 1024
    eda, edb, eh = near(da), near(db), near(h)
    k = (rows / 16 + 72) * STEP
    total = lambda e, v: e.T @ v.abs()
    want = (h, dx, da.T @ a, db.T @ a, d.T @ h)
    bound = (eh + near(h), eda + edb / 1024 + near(dx) + near(da) + near(db / 1024),
             total(eda, a) + U[dtype] * (da.T @ a).abs() + k * total(da.abs(), a),
             total(edb, a) + U[dtype] * (db.T @ a).abs() + k * total(db.abs(), a),
             total(d.abs(), eh) + U[dtype] * (d.T @ h).abs() + k * total(d.abs(), h))
    for name, g, e, t in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), got, want, bound):
        if dtype == torch.float16:    # sums beyond the type's largest number (65504; from 65520 on, rounded) are infinite
            beyond = e.abs() - t >= 65520
            assert torch.equal(g[beyond].double(), torch.sign(e[beyond]) * float("inf")), name
            unsure = ~beyond & (e.abs() + t > 65504)
            g, e = (torch.where(beyond | unsure, 0, v) for v in (g, e))
        assert_bounded(g, e, t, name)


@pytest.mark.parametrize("width", [64, 136])
def test_hidden_values_beyond_fp16(width):
    """A hidden value beyond 65504 is infinite between two fp16 products, and finite with the fp32 hidden values of up to
    eight rows; other rows are as they were."""
    from trifast_b200 import gated_feed_forward
    x = torch.zeros(9, width, device="cuda", dtype=torch.float16)
    x[:, 1] = 1.0
    x[4, 0] = 300.0                                    # silu(300) 300 = 90,000
    eye = torch.eye(width, device="cuda", dtype=torch.float16)
    y = gated_feed_forward(x, eye, eye, eye / 4)
    assert y[4, 0] == float("inf") and torch.isfinite(y[[0, 1, 2, 3, 5, 6, 7, 8]]).all()
    y = gated_feed_forward(x[:8], eye, eye, eye / 4)
    assert torch.isfinite(y).all() and abs(float(y[4, 0]) - 22500) <= 22500 * 2.0 ** -10


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [64, 136])
@pytest.mark.parametrize("std", [1e-4, 1e-6])
def test_small_gradients(std, c, dtype):
    """Hidden gradients about fp16's smallest numbers are off by half of the smallest, no more."""
    dy, x, *w = draw(200, c, 96, c, dtype)
    dy = (dy.float() * std).to(dtype)
    want, bound = bounds(dy, x, *w)
    for name, g, e, b in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), run(dy, x, *w), want, bound):
        assert_bounded(g, e, b, name)


@pytest.mark.parametrize("c,hidden", [(136, 8), (128, 64), (64, 40)])
def test_sums_of_millions_of_rows_do_not_drift(c, hidden):
    """Weight gradients over 5.5 million rows, every term positive.  The accumulators of TMEM round towards zero, so that a
    long sum drifts.  A run of sums there is 128 row tiles, 1024 additions of 16 products; if each loses two steps of 2^-23,
    of an accumulator that is half its last value on average, the mean over the entries is off by 1024 2^-23 = 1.22e-4, a
    quarter of fp16's rounding.  What the entries' own roundings (u = 2^-11, a uniform error of u / sqrt 3) leave in that mean is
    below 6 u / sqrt(3 count)."""
    from trifast_b200 import gated_feed_forward
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    rows = 5_500_000
    g = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")
    x, dy = (0.5 + rand(rows, c)).half(), (0.004 + 0.002 * rand(rows, c)).half()
    wg, wu = ((rand(hidden, c) / 64).half() for _ in range(2))
    wd = (rand(c, hidden) / 32).half()
    leaves = [t.requires_grad_() for t in (wg, wu, wd)]
    got = torch.autograd.grad(gated_feed_forward(x, *leaves), leaves, dy)
    want = [torch.zeros(t.shape, dtype=torch.float64, device="cuda") for t in leaves]
    for r in range(0, rows, 500_000):
        for s, v in zip(want, oracle.feed_forward_grads(dy[r:r + 500_000], x[r:r + 500_000], *(t.detach() for t in leaves))[1:]):
            s += v
    off = torch.cat([((p.double() - q) / q).flatten() for p, q in zip(got, want)])
    assert max(float(q.max()) for q in want) * (1 + 2.0 ** -10) < 65504 and min(float(q.min()) for q in want) > 1
    mean = float(off.mean())
    print(f"mean relative error of {off.numel()} sums: {mean:.3g}")
    assert abs(mean) <= 1024 * 2.0 ** -23 + 6 * U[torch.float16] / (3 * off.numel()) ** 0.5
