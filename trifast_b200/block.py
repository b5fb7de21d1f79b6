"""The operators around triangle attention in a pair stack's blocks: layer norm, the gated feed-forward
block ("transition"), and dropout with the residual sum.

Native like the attention (``csrc/torch_block_ops.cpp``): argument checks, allocation and autograd run
without Python, all compute in the CUDA library behind the C ABI, on the caller's stream; nothing
synchronises, and calls can be captured in a CUDA graph.  Gradients are those of reverse mode; an input with
a forward-mode tangent is refused (NotImplementedError).  A pre-norm block of a pair map ``z`` of shape
(*batch, n, n, width)::

    z = dropout_add(attention(layer_norm(z, w0, b0)), z, p, seed, shared_dim=-3)
    z = dropout_add(gated_feed_forward(layer_norm(z, w1, b1), w_gate, w_up, w_down), z, p, seed, offset=1)
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from .torch import _triangle_attention as _  # noqa: F401  (loads the operators)


def _op(name):
    try:
        return getattr(torch.ops.trifast_b200, name).default
    except AttributeError:
        from .torch import triangle_attention_bwd

        def missing(*_args):
            triangle_attention_bwd()     # raises with the build instructions
        return missing


def _register_fakes():
    register = torch.library.register_fake

    @register("trifast_b200::layer_norm")
    def _(x, weight, bias, eps):
        return torch.empty_like(x, memory_format=torch.contiguous_format)

    @register("trifast_b200::layer_norm_grads")
    def _(dy, x, weight, eps, want_x, want_weight, want_bias):
        like = lambda t, wanted: torch.empty_like(t, memory_format=torch.contiguous_format) if wanted else x.new_empty(0)
        return like(x, want_x), like(weight, want_weight), like(weight, want_bias)

    @register("trifast_b200::gated_feed_forward")
    def _(x, w_gate, w_up, w_down):
        return x.new_empty((*x.shape[:-1], w_down.shape[0]))

    @register("trifast_b200::gated_feed_forward_grads")
    def _(dy, x, w_gate, w_up, w_down, want_x, want_weights):
        like = lambda t, wanted: torch.empty_like(t, memory_format=torch.contiguous_format) if wanted else x.new_empty(0)
        return like(x, want_x), *(like(w, want_weights) for w in (w_gate, w_up, w_down))

    @register("trifast_b200::dropout_add")
    def _(x, residual, p, seed, offset, seed_tensor, shared_dim):
        return torch.empty_like(x, memory_format=torch.contiguous_format)


_layer_norm, _gated_feed_forward, _dropout_add = map(_op, ("layer_norm", "gated_feed_forward", "dropout_add"))
if hasattr(torch.ops.trifast_b200, "layer_norm"):
    _register_fakes()


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    x: (..., width), fp32, bf16 or fp16, with width at most 2**20; weight and bias: (width,), both of x's type or both fp32, or None
    (no affine part; a bias needs a weight).  Arithmetic is in fp32 and the result, of x's shape and type,
    is rounded once.  Differentiable, once, in x, weight and bias.  Rows may be strided; a tensor whose
    leading dimensions cannot be walked with one stride is copied.  Rows of more than 8192 elements (8185 where they are
    not whole 16-byte pieces; fp32 8189): at most 4,194,240 of them.
    """
    return _layer_norm(x, weight, bias, eps)


def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor) -> torch.Tensor:
    """The gated feed-forward block ``(silu(x w_gate^T) * (x w_up^T)) w_down^T``.

    x: (..., width); w_gate, w_up: (hidden, width); w_down: (width_out, hidden), as a linear layer holds
    them; all fp32, bf16 or fp16, at most 65536 wide.  Returns (..., width_out) in x's type.  Sums are fp32; the hidden
    values are rounded to x's type between the two products (fp16: a hidden value beyond 65504 is infinite),
    and so are their gradients in the backward (fp16: those below 2**-25 are 0), which computes the hidden values
    again instead of keeping them: nothing but the arguments is saved, and the workspace of a call does not
    grow with the number of rows beyond a chunk of them.  fp32 products are as exact as fp32 sums, but an infinite
    value in x, a weight or between the products gives NaN there.  The forward pass of up to eight rows runs on the
    CUDA cores with fp32 hidden values: its last bits may differ from those of the same rows in a larger batch, where
    an fp16 hidden value beyond 65504 is infinite.  Differentiable, once, in all four.
    """
    return _gated_feed_forward(x, w_gate, w_up, w_down)


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor], p: float, seed: Union[int, torch.Tensor], *,
                offset: int = 0, shared_dim: Optional[int] = None) -> torch.Tensor:
    """``residual + dropout(x)``: each element of x is dropped with probability p, else scaled by 1 / (1 - p).

    The mask is never stored: element i of it comes from a counter-based generator (Philox-4x32-10, word i % 4
    of counter (i // 4, offset) under the key ``seed``; kept if the word, of 2**32, is not below round(p 2**32)),
    so that equal arguments drop the same elements, in the backward too.  Calls of one step take the same
    seed and different offsets.  ``seed`` may be a one-element int64 CUDA tensor, read when the kernel runs: a
    captured graph draws anew at each replay if the tensor is changed in between.

    shared_dim: a dimension of x along which the mask is shared (mask entries are then counted over the other
    dimensions): -3 gives all rows of a pair map (..., n, n, width) one mask, -2 all columns; None: none is shared.
    residual: like x, or None for 0.  Differentiable in x and residual.  A dropped element does not enter
    the result, whatever it is (an infinity or NaN either).
    """
    if isinstance(seed, torch.Tensor):
        return _dropout_add(x, residual, p, 0, offset, seed, shared_dim)
    return _dropout_add(x, residual, p, seed, offset, None, shared_dim)
