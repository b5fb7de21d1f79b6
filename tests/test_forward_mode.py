"""Forward-mode derivatives: no operator has one, and a tangent is refused instead of being lost.  (Shapes without a
device take the same way through autograd.)"""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import trifast_b200
from trifast_b200 import dropout_add, gated_feed_forward, layer_norm

meta = lambda *s, dtype=torch.float32: torch.empty(*s, device="meta", dtype=dtype)
X, W, G, D_ = meta(2, 3, 8), meta(8), meta(5, 8), meta(4, 5)
ops = torch.ops.trifast_b200

# operator, its arguments, the places of those that a tangent may come with
BLOCK = {
    "layer_norm": (lambda *a: layer_norm(*a), (X, W, W), (0, 1, 2)),
    "layer_norm_grads": (lambda dy, x, w: ops.layer_norm_grads(dy, x, w, 1e-5, True, True, True), (X, X, W), (0, 1, 2)),
    "gated_feed_forward": (lambda *a: gated_feed_forward(*a), (X, G, G, D_), (0, 1, 2, 3)),
    "gated_feed_forward_grads": (lambda *a: ops.gated_feed_forward_grads(*a, True, True), (meta(2, 3, 4), X, G, G, D_), (0, 1, 2, 3, 4)),
    "dropout_add": (lambda x, r: dropout_add(x, r, 0.5, 1), (X, X), (0, 1)),
}
CASES = [(n, i, g) for n, (_, _, places) in BLOCK.items() for i in places for g in (False, True)]


def refused(call, args, place, requires_grad):
    args = [a.clone() for a in args]
    if requires_grad:
        for a in args:
            if a.is_floating_point():
                a.requires_grad_()
    with fwd.dual_level():
        args[place] = fwd.make_dual(args[place], torch.empty_like(args[place]))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                call(*args)
    # without a tangent it runs
    call(*(a.detach() for a in args))


@pytest.mark.parametrize("name,place,requires_grad", CASES)
def test_tangents_are_refused(name, place, requires_grad):
    call, args, _ = BLOCK[name]
    refused(call, args, place, requires_grad)


@pytest.mark.parametrize("name", BLOCK)
def test_jvp_is_refused(name):
    call, args, _ = BLOCK[name]
    with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
        torch.func.jvp(call, args, tuple(torch.empty_like(a) for a in args))


def test_forward_over_reverse_is_refused():
    """An upstream gradient with a tangent reaches the gradients' operator."""
    x = X.clone().requires_grad_()
    y = layer_norm(x)
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
        torch.autograd.grad(y, x, fwd.make_dual(torch.empty_like(y), torch.empty_like(y)))


# ------------------------------------------------------------------ the attention
Q, B, M = meta(1, 2, 5, 5, 16), meta(1, 2, 5, 5), meta(1, 5, 5, dtype=torch.bool)
SAVED = (Q, Q, Q, Q, B, Q, meta(1, 2, 5, 5))
ATTENTION = {
    "triangle_attention": (lambda *a: trifast_b200.triangle_attention(*a, M), (Q, Q, Q, B)),
    "triangle_attention_ending_node": (lambda *a: trifast_b200.triangle_attention_ending_node(*a, M), (Q, Q, Q, B)),
    "triangle_attention_grads": (lambda *a: ops.triangle_attention_grads(*a, M), SAVED),
    "triangle_attention_backward": (lambda *a: ops.triangle_attention_backward(*a, M), SAVED),
}


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name,place", [(n, i) for n, (_, args) in ATTENTION.items() for i in range(len(args))])
def test_attention_refuses_tangents(name, place, requires_grad):
    call, args = ATTENTION[name]
    refused(call, args, place, requires_grad)


@pytest.mark.parametrize("name", ATTENTION)
def test_attention_refuses_jvp(name):
    call, args = ATTENTION[name]
    with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
        torch.func.jvp(call, args, tuple(torch.empty_like(a) for a in args))
