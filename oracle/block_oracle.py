"""64-bit definitions of the operators around the attention: layer norm, the gated feed-forward block and
dropout with the residual sum, each with its gradients written out, on torch tensors of any device."""

from __future__ import annotations

import math

import torch


def layer_norm(x, weight, bias, eps):
    """y, and the normalised rows and 1 / standard deviation that the gradients need."""
    x = x.double()
    xc = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    xh = xc * r
    y = xh if weight is None else xh * weight.double()
    return (y if bias is None else y + bias.double()), xh, r


def layer_norm_grads(dy, x, weight, eps):
    """dx, dweight, dbias."""
    _, xh, r = layer_norm(x, None, None, eps)
    dy = dy.double()
    g = dy if weight is None else dy * weight.double()
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    flat = lambda t: t.reshape(-1, t.shape[-1])
    return dx, flat(dy * xh).sum(0), flat(dy).sum(0)


def feed_forward(x, w_gate, w_up, w_down):
    x, wg, wu, wd = (t.double() for t in (x, w_gate, w_up, w_down))
    a, b = x @ wg.T, x @ wu.T
    return (a * torch.sigmoid(a) * b) @ wd.T


def feed_forward_grads(dy, x, w_gate, w_up, w_down):
    """dx, dw_gate, dw_up, dw_down."""
    dy, x, wg, wu, wd = (t.double() for t in (dy, x, w_gate, w_up, w_down))
    dy2, x2 = dy.reshape(-1, dy.shape[-1]), x.reshape(-1, x.shape[-1])
    a, b = x2 @ wg.T, x2 @ wu.T
    s = torch.sigmoid(a)
    h, dh = a * s * b, dy2 @ wd
    da, db = dh * b * s * (1 + a * (1 - s)), dh * a * s
    return (da @ wg + db @ wu).reshape(x.shape), da.T @ x2, db.T @ x2, dy2.T @ h


def random_words_at(block, seed, offset=0):
    """The four words of Philox-4x32-10 (Salmon et al., 2011) at counter (block, offset) under the key ``seed``."""
    mask = 0xFFFFFFFF
    c = [block & mask, (block >> 32) & mask, offset & mask, (offset >> 32) & mask]
    k = [seed & mask, (seed >> 32) & mask]
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & mask, (p >> 32) ^ c[3] ^ k[1], p & mask]
        k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
    return c


def random_words(count, seed, offset=0):
    """Words 0 .. count - 1 as a list of ints: word i is number i % 4 at counter (i // 4, offset)."""
    return [w for block in range((count + 3) // 4) for w in random_words_at(block, seed, offset)][:count]


def keep_mask(shape, p, seed, offset=0, shared_dim=None):
    """Bool tensor that broadcasts to ``shape``: the elements that dropout keeps."""
    shape = list(shape)
    if shared_dim is not None:
        shape[shared_dim] = 1
    words = torch.tensor(random_words(math.prod(shape), seed, offset), dtype=torch.int64)
    return (words >= round(p * 2 ** 32)).reshape(shape)


def dropout_add(x, residual, keep, p):
    y = torch.where(keep, x.double() / (1 - p) if p < 1 else 0.0, 0.0).expand(x.shape)
    return y if residual is None else y + residual.double()
