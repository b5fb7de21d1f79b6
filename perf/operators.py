"""Timed cases of the operators that stand around triangle attention in a pair stack: layer norm, the
gated feed-forward block, and dropout with the residual sum; and their plain forms.

A case names one call, or one training step (the call and all of its gradients):

    op           "layer_norm", "feed_forward" or "dropout_add"
    dtype        "bf16", "fp16" or "fp32"
    train        the call and its gradients, or the call alone
  layer_norm:    rows, width; affine "same" (weight and bias in x's type), "fp32" or "none"
  feed_forward:  rows, width, hidden
  dropout_add:   n, width (x is (n, n, width)); p; shared "none", "rows" (one mask for all first
                 pair indices) or "columns" (one for all second ones); residual

``own`` false: the plain forms below, in 32 bits and rounded once at the end.  ``own`` true: the
framework's operators.
"""

import math

import numpy as np
import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SHARED = {"none": None, "rows": -3, "columns": -2}


# ------------------------------------------------------------------ cases
def listed():
    ln = lambda name, rows, width, dtype, affine, train: dict(
        name=name, op="layer_norm", rows=rows, width=width, dtype=dtype, affine=affine, train=train)
    ff = lambda name, rows, width, hidden, dtype, train: dict(
        name=name, op="feed_forward", rows=rows, width=width, hidden=hidden, dtype=dtype, train=train)
    do = lambda name, n, width, dtype, p, shared, residual, train: dict(
        name=name, op="dropout_add", n=n, width=width, dtype=dtype, p=p, shared=shared, residual=residual, train=train)
    return [
        # the norm before each block of a large complex's pair stack, 4 heads of 32
        ln("ln_train_pair1024_c128_bf16", 1024 * 1024, 128, "bf16", "same", True),
        # a ragged pair map with the affine part kept in 32 bits
        ln("ln_train_pair191_c64_fp16", 191 * 191, 64, "fp16", "fp32", True),
        # long rows, of odd length: a wide token representation
        ln("ln_train_4096x1999_bf16", 4096, 1999, "bf16", "same", True),
        # a few tokens in inference
        ln("ln_forward_33x512_fp32", 33, 512, "fp32", "same", False),
        # one token through the block: latency
        ff("ff_forward_1_c128_bf16", 1, 128, 512, "bf16", False),
        # the block in inference on a middle-sized pair map of 8 heads of 64
        ff("ff_forward_pair256_c512_bf16", 256 * 256, 512, 1024, "bf16", False),
        # a training step of a large complex (the largest case)
        ff("ff_train_pair1024_c128_bf16", 1024 * 1024, 128, 512, "bf16", True),
        # a wide token representation
        ff("ff_train_8192_c512_fp16", 8192, 512, 2048, "fp16", True),
        # full precision, sizes that no tile divides
        ff("ff_train_5041_c100_fp32", 71 * 71, 100, 290, "fp32", True),
        # after the attention around the starting node: one mask for all rows
        do("dropout_train_pair1024_c128_bf16", 1024, 128, "bf16", 0.25, "rows", True, True),
        # every element its own, no residual
        do("dropout_train_pair383_c64_fp16", 383, 64, "fp16", 0.1, "none", False, True),
        # a small map in full precision
        do("dropout_forward_pair25_c32_fp32", 25, 32, "fp32", 0.15, "columns", True, False),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "feed_forward", "dropout_add"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    train = rng.random() < 0.7
    if op == "layer_norm":
        width = _log_uniform(rng, 16, 8192)
        rows = _log_uniform(rng, 1, min(1 << 20, (1 << 27) // width))
        return dict(op=op, rows=rows, width=width, dtype=dtype, affine=rng.choice(["same", "fp32", "none"]), train=train)
    if op == "feed_forward":
        width = _log_uniform(rng, 16, 1024)
        hidden = int(width * rng.uniform(1.0, 4.0))
        most = (1 << 36) // (width * hidden) // (16 if dtype == "fp32" else 1)
        return dict(op=op, rows=_log_uniform(rng, 1, min(1 << 20, most)), width=width, hidden=hidden, dtype=dtype, train=train)
    n, shared = _log_uniform(rng, 8, 1024), rng.choice(["none", "rows", "columns"])
    # (a mask that is not shared has to be drawn in whole by exact())
    width = _log_uniform(rng, 8, min(512, max(8, ((1 << 25) if shared == "none" else (1 << 27)) // (n * n))))
    return dict(op=op, n=n, width=width, dtype=dtype, p=round(rng.uniform(0.05, 0.5), 3), shared=shared,
                residual=rng.random() < 0.7, train=train)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")
    if case["op"] == "layer_norm":
        rows, c = case["rows"], case["width"]
        # a residual stream: rows of different scale and mean
        x = normal(rows, c).mul_(0.5 + 2.5 * torch.rand(rows, 1, generator=g, device="cuda")).add_(0.5 * normal(rows, 1)).to(dt)
        wt = torch.float32 if case["affine"] == "fp32" else dt
        w, b = (None, None) if case["affine"] == "none" else ((1 + 0.2 * normal(c)).to(wt), (0.2 * normal(c)).to(wt))
        leaves = [t for t in (x, w, b) if t is not None]
        state = dict(x=x, w=w, b=b, dy=normal(rows, c).to(dt) if case["train"] else None)
    elif case["op"] == "feed_forward":
        rows, c, h = case["rows"], case["width"], case["hidden"]
        x = normal(rows, c).to(dt)
        wg, wu = ((normal(h, c) * c ** -0.5).to(dt) for _ in range(2))
        wd = (normal(c, h) * h ** -0.5).to(dt)
        leaves = [x, wg, wu, wd]
        state = dict(x=x, wg=wg, wu=wu, wd=wd, dy=normal(rows, c).to(dt) if case["train"] else None)
    else:
        shape = (case["n"], case["n"], case["width"])
        x = normal(*shape).to(dt)
        res = normal(*shape).to(dt) if case["residual"] else None
        leaves = [t for t in (x, res) if t is not None]
        state = dict(x=x, res=res, seed=(seed * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 62),
                     dy=normal(*shape).to(dt) if case["train"] else None)
    if case["train"]:
        for t in leaves:
            t.requires_grad_(True)
    return dict(state, case=case, leaves=leaves)


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        return {"layer_norm": _plain_layer_norm, "feed_forward": _plain_feed_forward,
                "dropout_add": _plain_dropout_add}[case["op"]](case, state)


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    train = case["train"]
    if case["op"] == "layer_norm":
        rows, c = case["rows"], case["width"]
        affine = {"same": es, "fp32": 4, "none": 0}[case["affine"]] * 2 * c
        # x (and dy) in, y (and dx) out; the affine part in (and its gradients out)
        return {"bytes": rows * c * es * (4 if train else 2) + affine * (2 if train else 1),
                "flops": rows * c * (18 if train else 7)}
    if case["op"] == "feed_forward":
        rows, c, h = case["rows"], case["width"], case["hidden"]
        # three products; in training six more (the hidden gradient, two for dx, three for the weights)
        return {"bytes": rows * c * es * (4 if train else 2) + 3 * c * h * es * (2 if train else 1),
                "flops": 2 * rows * c * h * (9 if train else 3)}
    e = case["n"] ** 2 * case["width"]
    # x (and the residual) in, y out; in training dy in and dx out (the residual's gradient is dy)
    return {"bytes": e * es * (2 + case["residual"] + 2 * train), "flops": e * (2 + train)}


# ------------------------------------------------------------------ the framework's operators
def _run_own(case, s):
    from trifast_b200 import dropout_add, gated_feed_forward, layer_norm
    if case["op"] == "layer_norm":
        y = layer_norm(s["x"], s["w"], s["b"], EPS)
    elif case["op"] == "feed_forward":
        y = gated_feed_forward(s["x"], s["wg"], s["wu"], s["wd"])
    else:
        y = dropout_add(s["x"], s["res"], case["p"], s["seed"], shared_dim=SHARED[case["shared"]])
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, s["leaves"], s["dy"])]


# ------------------------------------------------------------------ the plain forms
def _plain_layer_norm(case, s):
    x32 = s["x"].float()
    c = x32.shape[-1]
    xc = x32 - x32.mean(-1, keepdim=True)
    rstd = ((xc * xc).mean(-1, keepdim=True) + EPS).rsqrt()
    xhat = xc * rstd
    y = xhat if s["w"] is None else xhat * s["w"].float() + s["b"].float()
    out = [y.to(s["x"].dtype)]
    if not case["train"]:
        return out
    dy = s["dy"].float()
    gy = dy if s["w"] is None else dy * s["w"].float()
    dx = rstd * (gy - gy.mean(-1, keepdim=True) - xhat * ((gy * xhat).sum(-1, keepdim=True) / c))
    out.append(dx.to(s["x"].dtype))
    if s["w"] is not None:
        out += [(dy * xhat).sum(0, dtype=torch.float64).to(s["w"].dtype), dy.sum(0, dtype=torch.float64).to(s["b"].dtype)]
    return out


def _plain_feed_forward(case, s):
    x, wg, wu, wd = (s[k].float() for k in ("x", "wg", "wu", "wd"))
    a, b = x @ wg.t(), x @ wu.t()
    sig = 1 / (1 + torch.exp(-a))
    h = a * sig * b
    dt = s["x"].dtype
    out = [(h @ wd.t()).to(dt)]
    if not case["train"]:
        return out
    dy = s["dy"].float()
    dwd = dy.t() @ h
    del h
    dh = dy @ wd
    db = dh * a * sig
    da = dh * b * (sig * (1 + a * (1 - sig)))
    del a, b, sig, dh
    dx = da @ wg + db @ wu
    return out + [dx.to(dt), (da.t() @ x).to(dt), (db.t() @ x).to(dt), dwd.to(dt)]


def _random_words(count, seed, device):
    """``count`` 32-bit words, as int64, of the counter-based generator Philox-4x32 with ten rounds
    (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011): word i is word i % 4 of the block
    with counter (i // 4, 0) and the seed as its key."""
    m32 = 0xFFFFFFFF
    q = torch.arange((count + 3) // 4, dtype=torch.int64, device=device)
    c0, c1 = q & m32, q >> 32
    c2, c3 = torch.zeros_like(q), torch.zeros_like(q)
    k0, k1 = seed & m32, (seed >> 32) & m32

    def product(c, m):      # high and low word; the 64-bit product wraps into the sign, its bits are right
        p = c * m
        return (p >> 32) & m32, p & m32

    for _ in range(10):
        h0, l0 = product(c0, 0xD2511F53)
        h1, l1 = product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    return torch.stack([c0, c1, c2, c3], 1).flatten()[:count]


def _plain_dropout_add(case, s):
    x, dt = s["x"], s["x"].dtype
    shape = list(x.shape)
    if SHARED[case["shared"]] is not None:
        shape[SHARED[case["shared"]]] = 1
    keep = (_random_words(math.prod(shape), s["seed"], x.device) >= int(round(case["p"] * 2 ** 32))).reshape(shape)
    scale = 1 / (1 - case["p"])
    kept = lambda t: torch.where(keep, t.float() * scale, 0.0)
    y = kept(x)
    if s["res"] is not None:
        y = y + s["res"].float()
    out = [y.to(dt)]
    if case["train"]:
        out.append(kept(s["dy"]).to(dt))
        if s["res"] is not None:
            out.append(s["dy"].clone())
    return out


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    up = lambda t: None if t is None else t.detach().double().requires_grad_(case["train"])
    if case["op"] == "layer_norm":
        leaves = [up(s["x"]), up(s["w"]), up(s["b"])]
        x, w, b = leaves
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS)
        if w is not None:
            y = w * y + b
    elif case["op"] == "feed_forward":
        leaves = [up(s[k]) for k in ("x", "wg", "wu", "wd")]
        x, wg, wu, wd = leaves
        y = torch.nn.functional.linear(torch.nn.functional.silu(torch.nn.functional.linear(x, wg))
                                       * torch.nn.functional.linear(x, wu), wd)
    else:
        leaves = [up(s["x"]), up(s["res"])]
        n, c = case["n"], case["width"]
        shape = {"none": (n, n, c), "rows": (1, n, c), "columns": (n, 1, c)}[case["shared"]]
        keep = _exact_words(math.prod(shape), s["seed"]) >= np.uint64(round(case["p"] * 2 ** 32))
        keep = torch.from_numpy(keep.reshape(shape)).cuda()
        y = leaves[0] * keep / (1 - case["p"])
        if leaves[1] is not None:
            y = y + leaves[1]
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [t for t in leaves if t is not None], s["dy"].double())]


def _exact_words(count, seed):
    low = np.uint64(0xFFFFFFFF)
    ctr = np.zeros((4, -(-count // 4)), dtype=np.uint64)
    ctr[0] = np.arange(ctr.shape[1], dtype=np.uint64)
    for r in range(10):
        key = [np.uint64((((seed >> s) & 0xFFFFFFFF) + r * w) & 0xFFFFFFFF) for s, w in ((0, 0x9E3779B9), (32, 0xBB67AE85))]
        p, q = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = np.stack([(q >> np.uint64(32)) ^ ctr[1] ^ key[0], q & low, (p >> np.uint64(32)) ^ ctr[3] ^ key[1], p & low])
    return ctr.T.reshape(-1)[:count]
