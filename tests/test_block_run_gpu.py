"""The operators of a pair stack's block together, as a model runs them: with the attention, captured in a graph,
on other streams, and what they refuse."""

import pytest
import torch

from tests.block_helpers import U, assert_norm, normal
from oracle import block_oracle, triangle_oracle

N, H, D, HID = 40, 4, 16, 96
C = H * D


def parameters(dtype, device="cuda"):
    w = lambda i, o, *s: normal(*s, seed=10 + i, dtype=dtype, device=device, std=o ** -0.5)
    return dict(g0=1 + w(0, 25, C), b0=w(1, 25, C), qkv=w(2, C, 3 * C, C), bias=w(3, C, H, C), out=w(4, C, C, C),
                g1=1 + w(5, 25, C), b1=w(6, 25, C), wg=w(7, C, HID, C), wu=w(8, C, HID, C), wd=w(9, HID, C, HID))


def block(z, p, mask, drop, attention, norm, ff, add):
    """z + dropout(attention(norm(z))), then z + dropout(feed_forward(norm(z)))."""
    x = norm(z, p["g0"], p["b0"])
    q, k, v = (x @ p["qkv"].T).reshape(N, N, 3, H, D).permute(2, 3, 0, 1, 4)[:, None]
    bias = (x @ p["bias"].T).permute(2, 0, 1)[None]
    o = attention(q, k, v, bias, mask[None])[0].permute(1, 2, 0, 3).reshape(N, N, C)
    z = add(o @ p["out"].T, z, 0)
    return add(ff(norm(z, p["g1"], p["b1"]), p["wg"], p["wu"], p["wd"]), z, 1)


def ours(z, p, mask, seed, drop=0.25):
    from trifast_b200 import dropout_add, gated_feed_forward, layer_norm, triangle_attention
    return block(z, p, mask, drop, triangle_attention, layer_norm, gated_feed_forward,
                 lambda x, r, i: dropout_add(x, r, drop, seed, offset=i, shared_dim=-3))


def plain(z, p, mask, seed, drop=0.25):
    norm = lambda x, w, b: block_oracle.layer_norm(x, w, b, 1e-5)[0]
    keep = [block_oracle.keep_mask(z.shape, drop, seed, i, -3).to(z.device) for i in (0, 1)]
    return block(z.double(), p, mask, drop, lambda *a: triangle_oracle.attention_reference_port(*a), norm,
                 block_oracle.feed_forward, lambda x, r, i: block_oracle.dropout_add(x, r, keep[i], drop))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_and_its_gradients(dtype):
    z = normal(N, N, C, seed=1, dtype=dtype)
    mask = torch.zeros(N, N, dtype=torch.bool, device="cuda")
    mask[:, -5:] = True
    p = parameters(dtype)
    dy = normal(N, N, C, seed=2, dtype=dtype)
    leaves = [t.clone().requires_grad_() for t in (z, *p.values())]
    y = ours(leaves[0], dict(zip(p, leaves[1:])), mask, 5)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    leaves = [t.double().requires_grad_() for t in (z, *p.values())]
    y = plain(leaves[0], dict(zip(p, leaves[1:])), mask, 5)
    want = [y, *torch.autograd.grad(y, leaves, dy.double())]
    # some twelve roundings one after the other, each below u; the plain products' TF32 is off
    rel = 1e-4 if dtype == torch.float32 else 12 * U[dtype]
    for name, a, b in zip(("y", "dz", *p), got, want):
        assert_norm(a, b.detach(), rel, name)


@pytest.mark.gpu
def test_step_in_a_graph_draws_anew():
    """A captured step equals the eager one bit for bit, and draws new masks when the seed's tensor changes; two
    graphs of the same leaves do not disturb one another."""
    dtype = torch.bfloat16
    p = {k: v.requires_grad_() for k, v in parameters(dtype).items()}
    z, dy = normal(N, N, C, seed=1, dtype=dtype).requires_grad_(), normal(N, N, C, seed=2, dtype=dtype)
    mask = torch.zeros(N, N, dtype=torch.bool, device="cuda")
    seed = torch.tensor([5], device="cuda")

    def step():
        y = ours(z, p, mask, seed)
        return [y.detach(), *torch.autograd.grad(y, [z, *p.values()], dy)]

    eager = {}
    for s in (5, 6):
        seed.fill_(s)
        eager[s] = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for s in (6, 5, 6):
        seed.fill_(s)
        for g, _ in graphs:
            g.replay()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager[s]))


@pytest.mark.gpu
def test_on_another_stream():
    dtype = torch.bfloat16
    p, z = parameters(dtype), normal(N, N, C, seed=1, dtype=dtype)
    mask = torch.zeros(N, N, dtype=torch.bool, device="cuda")
    want = ours(z, p, mask, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ours(z, p, mask, 5) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls on two streams have workspaces of their own."""
    from trifast_b200 import gated_feed_forward
    xs = [normal(30000, 128, seed=s, dtype=torch.bfloat16) for s in (1, 2)]
    p = parameters(torch.bfloat16)
    w = [normal(256, 128, seed=3, dtype=torch.bfloat16), normal(256, 128, seed=4, dtype=torch.bfloat16), normal(128, 256, seed=5, dtype=torch.bfloat16)]
    want = [gated_feed_forward(x, *w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for _ in range(4):
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(gated_feed_forward(x, *w))
    torch.cuda.synchronize()
    assert p and all(torch.equal(g, want[i % 2]) for i, g in enumerate(got))


@pytest.mark.gpu
def test_from_a_thread_that_has_not_used_the_device():
    """With all memory from the allocator's cache, the first thing such a thread does is to encode a tensor map."""
    import threading

    from trifast_b200 import gated_feed_forward, triangle_attention
    x = normal(9600, 64, seed=1, dtype=torch.bfloat16)
    w = [normal(64, 64, seed=i, dtype=torch.bfloat16) for i in (2, 3, 4)]
    q, b = normal(1, 2, 64, 64, 32, seed=5, dtype=torch.bfloat16), normal(1, 2, 64, 64, seed=6, dtype=torch.bfloat16)
    m = torch.zeros(1, 64, 64, dtype=torch.bool, device="cuda")
    for call in (lambda: gated_feed_forward(x, *w), lambda: triangle_attention(q, q, q, b, m)):
        want, got = call(), []
        call()

        def run():
            try:
                got.append(call())
            except Exception as e:   # seen by the assertion below
                got.append(e)
        t = threading.Thread(target=run)
        t.start()
        t.join()
        assert isinstance(got[0], torch.Tensor), got[0]
        assert torch.equal(got[0], want)


@pytest.mark.gpu
def test_gradients_have_no_gradient():
    from trifast_b200 import gated_feed_forward, layer_norm
    x = normal(4, 8, seed=1).requires_grad_()
    w = normal(8, 8, seed=2).requires_grad_()
    for y in (layer_norm(x), gated_feed_forward(x, w, w, w)):
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):
            g.sum().backward()


# ------------------------------------------------------------------ refusals
def on_cuda_kernel(op, *args):
    """The CUDA implementation itself, which checks its arguments before it touches a device."""
    import trifast_b200  # noqa: F401
    return getattr(torch.ops.trifast_b200, op).default.redispatch(torch._C.DispatchKeySet(torch._C.DispatchKey.CUDA), *args)


X = torch.zeros(2, 3, 8)
W = torch.zeros(8)
G, D_ = torch.zeros(5, 8), torch.zeros(4, 5)


@pytest.mark.parametrize("args,error,text", [
    ((torch.zeros(()), None, None, 1e-5), ValueError, "x must be"),
    ((torch.zeros(3, 0), None, None, 1e-5), ValueError, "x must be"),
    ((X, torch.zeros(7), None, 1e-5), ValueError, "weight must be [8]; got [7]"),
    ((X, W, torch.zeros(1, 8), 1e-5), ValueError, "bias must be [8]; got [1, 8]"),
    ((X, None, W, 1e-5), ValueError, "a bias needs a weight"),
    ((X, W.half(), None, 1e-5), TypeError, "weight must be float32 or of x's type"),
    ((X.half(), W, W.half(), 1e-5), TypeError, "must share one dtype"),
    ((X, W, None, -1.0), ValueError, "eps must be"),
    ((X, W, None, float("nan")), ValueError, "eps must be"),
    ((X.double(), None, None, 1e-5), TypeError, "unsupported dtype"),
    ((X, W, W, 1e-5), RuntimeError, "CUDA devices only"),
])
def test_layer_norm_refuses(args, error, text):
    with pytest.raises(error) as e:
        on_cuda_kernel("layer_norm", *args)
    assert text in str(e.value)


@pytest.mark.parametrize("args,error,text", [
    ((torch.zeros(()), G, G, D_), ValueError, "x must be"),
    ((X, torch.zeros(5, 7), G, D_), ValueError, "w_gate must be (hidden, 8); got [5, 7]"),
    ((X, torch.zeros(0, 8), G, D_), ValueError, "w_gate must be"),
    ((X, G, torch.zeros(6, 8), D_), ValueError, "w_up must be [5, 8]; got [6, 8]"),
    ((X, G, G, torch.zeros(4, 6)), ValueError, "w_down must be (width_out, 5); got [4, 6]"),
    ((X, G.half(), G, D_), TypeError, "must share one dtype"),
    ((X.double(), G.double(), G.double(), D_.double()), TypeError, "unsupported dtype"),
    ((X, torch.zeros(65537, 8), torch.zeros(65537, 8), torch.zeros(1, 65537)), ValueError, "at most 65536"),
    ((X, G, G, D_), RuntimeError, "CUDA devices only"),
])
def test_feed_forward_refuses(args, error, text):
    with pytest.raises(error) as e:
        on_cuda_kernel("gated_feed_forward", *args)
    assert text in str(e.value)


@pytest.mark.parametrize("args,error,text", [
    ((X, None, -0.1, 1, 0, None, None), ValueError, "p must be in [0, 1]"),
    ((X, None, 1.5, 1, 0, None, None), ValueError, "p must be in [0, 1]"),
    ((X, None, float("nan"), 1, 0, None, None), ValueError, "p must be in [0, 1]"),
    ((X, None, 0.5, 1, 0, None, 3), ValueError, "shared_dim 3 is not a dimension of x"),
    ((X, None, 0.5, 1, 0, None, -4), ValueError, "shared_dim -4 is not a dimension of x"),
    ((X, torch.zeros(2, 3, 1), 0.5, 1, 0, None, None), ValueError, "residual must be [2, 3, 8]; got [2, 3, 1]"),
    ((X, X.half(), 0.5, 1, 0, None, None), TypeError, "must share one dtype"),
    ((X, None, 0.5, 0, 0, torch.zeros(1), None), TypeError, "must be int64"),
    ((X, None, 0.5, 0, 0, torch.zeros(2, dtype=torch.int64), None), ValueError, "one element"),
    ((X.double(), None, 0.5, 1, 0, None, None), TypeError, "unsupported dtype"),
    ((X, X, 0.5, 1, 0, None, None), RuntimeError, "CUDA devices only"),
])
def test_dropout_refuses(args, error, text):
    with pytest.raises(error) as e:
        on_cuda_kernel("dropout_add", *args)
    assert text in str(e.value)


@pytest.mark.parametrize("op,args,text", [
    ("layer_norm_grads", (torch.zeros(2, 8), X, None, 1e-5, True, False, False), "dy must be [2, 3, 8]"),
    ("layer_norm_grads", (X.half(), X, None, 1e-5, True, False, False), "dy must be [2, 3, 8]"),
    ("layer_norm_grads", (X, X, None, 1e-5, True, True, False), "without a weight"),
    ("gated_feed_forward_grads", (X, X, G, G, D_, True, True), "dy must be [2, 3, 4]"),
])
def test_gradients_refuse(op, args, text):
    with pytest.raises(ValueError) as e:
        on_cuda_kernel(op, *args)
    assert text in str(e.value)


def test_shapes_without_a_device():
    """Tracing sees shapes and types only."""
    from trifast_b200 import dropout_add, gated_feed_forward, layer_norm
    x = torch.empty(2, 3, 8, device="meta", dtype=torch.bfloat16)
    g, d = torch.empty(5, 8, device="meta", dtype=x.dtype), torch.empty(4, 5, device="meta", dtype=x.dtype)
    assert layer_norm(x).shape == x.shape and dropout_add(x, x, 0.5, 1).shape == x.shape
    assert gated_feed_forward(x, g, g, d).shape == (2, 3, 4)


def test_c_entries_check_their_arguments():
    """Without a device: every argument is checked before the first launch."""
    import ctypes as C

    from trifast_b200 import _lib
    lib = _lib.load()
    ok = C.c_void_p(0x1000)
    norm = lambda **kw: C.byref(_lib.Norm(**{**dict(rows=4, ld_x=64, ld_dy=64, width=64, dtype=1, affine_dtype=0, eps=1e-5), **kw}))
    fwd = lambda n, x=ok, y=ok: lib.trifast_layer_norm(n, x, ok, ok, y, None)
    assert fwd(None) == -1 and fwd(norm(), x=None) == -1 and fwd(norm(), y=C.c_void_p(0x1008)) == -6
    for kw, rc in ((dict(rows=-1), -2), (dict(width=0), -2), (dict(width=(1 << 20) + 1), -2), (dict(eps=-1.0), -2), (dict(eps=float("inf")), -2),
                   (dict(dtype=5), -4), (dict(affine_dtype=2), -4), (dict(ld_x=63), -5), (dict(rows=1 << 23, width=9000, ld_x=9000), -12)):
        assert fwd(norm(**kw)) == rc, kw
    assert fwd(norm(rows=0), x=None, y=None) == 0
    bwd = lambda n, ws=ok, size=1 << 30: lib.trifast_layer_norm_backward(n, ok, ok, ok, ok, ok, ok, ws, size, None)
    assert bwd(norm(ld_dy=63)) == -5 and bwd(norm(), ws=None) == -7 and bwd(norm(), size=16) == -7 and bwd(norm(), ws=C.c_void_p(0x1010)) == -6

    ff = lambda **kw: C.byref(_lib.FeedForward(**{**dict(rows=4, ld_x=64, ld_dy=32, width=64, hidden=96, width_out=32, dtype=1), **kw}))
    fwd = lambda f, x=ok, ws=ok, size=1 << 30: lib.trifast_feed_forward(f, x, ok, ok, ok, ok, ws, size, None)
    assert fwd(None) == -1 and fwd(ff(), x=None) == -1 and fwd(ff(), x=C.c_void_p(0x1002)) == -6 and fwd(ff(rows=64, dtype=0), size=1) == -7
    for kw, rc in ((dict(rows=-1), -2), (dict(hidden=0), -2), (dict(width_out=65537), -2), (dict(dtype=-1), -4), (dict(ld_x=60), -5)):
        assert fwd(ff(**kw)) == rc, kw
        assert lib.trifast_feed_forward_workspace_bytes(ff(**kw)) == 0
    bwd = lambda f, dw=ok: lib.trifast_feed_forward_backward(f, ok, ok, ok, ok, ok, ok, ok, dw, ok, ok, 1 << 30, None)
    assert bwd(ff(ld_dy=31)) == -5 and bwd(ff(), dw=None) == -1

    drop = lambda **kw: C.byref(_lib.Dropout(**{**dict(outer=1, mid=2, inner=8, dtype=1, seed=1, offset=0, p=0.5), **kw}))
    call = lambda d, x=ok, seed=None: lib.trifast_dropout_add(d, seed, x, None, ok, None)
    assert call(None) == -1 and call(drop(), x=None) == -1 and call(drop(), x=C.c_void_p(0x1004)) == -6
    assert call(drop(), seed=C.c_void_p(0x1004)) == -6
    for kw, rc in ((dict(outer=-1), -2), (dict(p=1.01), -2), (dict(p=float("nan")), -2), (dict(dtype=3), -4), (dict(outer=1 << 30, mid=1 << 30), -2)):
        assert call(drop(**kw)) == rc, kw
    assert call(drop(mid=0), x=None) == 0


def test_workspace_of_the_feed_forward_does_not_grow_with_the_rows():
    from ctypes import byref

    from trifast_b200 import _lib
    lib = _lib.load()
    for dtype in (0, 1):
        size = [lib.trifast_feed_forward_backward_workspace_bytes(byref(_lib.FeedForward(r, 128, 128, 128, 512, 128, dtype)))
                for r in (1 << 20, 1 << 24, 1 << 30)]
        assert all(0 < s < 320 << 20 for s in size)


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Tensors of more than 2^31 elements: the last rows are those of a call of their own."""
    from trifast_b200 import dropout_add, gated_feed_forward, layer_norm
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free device memory")
    for width, hidden in ((8, 8), (136, 8)):
        rows = (1 << 31) // width + 1001
        x = torch.zeros(rows, width, device="cuda", dtype=torch.bfloat16)
        x[-600:] = normal(600, width, seed=1, dtype=x.dtype)
        w = normal(width, seed=2)
        g, u, d = (normal(*s, seed=3 + i, dtype=x.dtype) for i, s in enumerate(((hidden, width), (hidden, width), (width, hidden))))
        tail = x[-600:].clone()
        assert torch.equal(layer_norm(x, w)[-600:], layer_norm(tail, w))
        assert torch.equal(gated_feed_forward(x, g, u, d)[-600:], gated_feed_forward(tail, g, u, d))
        dy = torch.zeros_like(x)
        dy[-600:] = normal(600, width, seed=9, dtype=x.dtype)
        grads = torch.ops.trifast_b200
        for op, args in ((grads.layer_norm_grads, (w, 1e-5, True, False, False)), (grads.gated_feed_forward_grads, (g, u, d, True, False))):
            a, b = op(dy, x, *args)[0], op(dy[-600:].clone(), tail, *args)[0]
            assert torch.equal(a[-600:], b) and not a[:-600].any()
            del a
        y = dropout_add(x, dy, 0.5, 7, shared_dim=0)
        assert torch.equal(y[-600:], dropout_add(tail, dy[-600:].clone(), 0.5, 7, shared_dim=0))
        # every element its own: the last mask entries against those of the same counters at a small place
        y = dropout_add(torch.ones_like(x), None, 0.5, 7)
        blocks = [(x.numel() - 1) // 4 - i for i in range(3)]
        for q in blocks:
            want = torch.tensor([v >= 1 << 31 for v in block_oracle.random_words_at(q, 7)])
            got = (y.view(-1)[4 * q:4 * q + 4] > 0).cpu()
            assert torch.equal(got, want[:got.numel()])
        del x, dy, y


@pytest.mark.gpu
def test_operators_pass_the_checks_of_tracing():
    """Schema, fake kernels and autograd registration as torch.compile expects them."""
    import trifast_b200  # noqa: F401
    from torch.library import opcheck
    ops = torch.ops.trifast_b200
    t = lambda *s, i=0: normal(*s, seed=i, dtype=torch.float32).requires_grad_()
    x, dy = t(2, 9, 16), normal(2, 9, 16, seed=7)
    what = ("test_schema", "test_autograd_registration", "test_faketensor")
    for op, args in ((ops.layer_norm, (x, t(16, i=1), t(16, i=2), 1e-5)), (ops.layer_norm, (x, None, None, 1e-5)),
                     (ops.layer_norm_grads, (dy, x.detach(), normal(16, seed=1), 1e-5, True, True, False)),
                     (ops.gated_feed_forward, (x, t(24, 16, i=1), t(24, 16, i=2), t(8, 24, i=3))),
                     (ops.gated_feed_forward_grads, (normal(2, 9, 8, seed=4), x.detach(), *(normal(*s, seed=5) for s in ((24, 16), (24, 16), (8, 24))), True, True)),
                     (ops.dropout_add, (x, t(2, 9, 16, i=3), 0.3, 5, 1, None, 1)),
                     (ops.dropout_add, (x, None, 0.3, 0, 1, torch.tensor([4], device="cuda"), None))):
        opcheck(op.default, args, test_utils=what)


@pytest.mark.gpu
@pytest.mark.parametrize("width,hidden", [(64, 64), (136, 64)])
def test_after_a_kernel_that_gave_up(width, hidden):
    """With the device's status set, a call raises; a kernel launched all the same writes nothing and ends."""
    import ctypes as C

    from trifast_b200 import _lib, gated_feed_forward
    lib = _lib.load()
    x = normal(300, width, seed=1, dtype=torch.bfloat16)
    w = [normal(*s, seed=2, dtype=torch.bfloat16) for s in ((hidden, width), (hidden, width), (width, hidden))]
    want = gated_feed_forward(x, *w)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(lib.trifast_debug_wait_probe(1000, stream), "trifast_debug_wait_probe")
    y = torch.full_like(x, 7.0)
    ff = _lib.FeedForward(300, width, width, width, hidden, width, 1)
    size = lib.trifast_feed_forward_workspace_bytes(C.byref(ff))
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    args = [C.c_void_p(t.data_ptr()) for t in (x, *w, y, ws)]
    _lib.check(lib.trifast_feed_forward(C.byref(ff), *args, size, stream), "trifast_feed_forward")
    torch.cuda.synchronize()
    assert torch.equal(y, torch.full_like(y, 7.0))
    with pytest.raises(RuntimeError, match="gave up"):
        gated_feed_forward(x, *w)
    assert torch.equal(gated_feed_forward(x, *w), want)      # the status has been cleared
