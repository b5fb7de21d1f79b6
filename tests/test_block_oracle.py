"""The 64-bit definitions of the operators around the attention: known answers, autograd and differences."""

import pytest
import torch

from oracle import block_oracle as oracle


def test_generator_known_answers():
    """The published vectors: counter and key of zeros, and of ones."""
    assert oracle.random_words(4, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = (1 << 64) - 1
    assert oracle.random_words_at(ones, ones, ones) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    a, b = oracle.random_words(8, 5, 9), oracle.random_words(8, 5, 10)
    assert a != b and a[:4] != a[4:]
    assert oracle.random_words(5, (1 << 64) - 1, 3) == oracle.random_words(8, -1, 3)[:5]


def draw(*shape, seed):
    return torch.randn(*shape, dtype=torch.float64, generator=torch.Generator().manual_seed(seed))


def differences(f, t, e=1e-5):
    g = torch.zeros_like(t)
    for i in range(t.numel()):
        up, down = t.clone(), t.clone()
        up.view(-1)[i] += e
        down.view(-1)[i] -= e
        g.view(-1)[i] = (f(up) - f(down)) / (2 * e)
    return g


def test_layer_norm_gradients():
    x, w, b, dy = draw(3, 5, seed=0), draw(5, seed=1), draw(5, seed=2), draw(3, 5, seed=3)
    loss = lambda x, w, b: (oracle.layer_norm(x, w, b, 1e-3)[0] * dy).sum()
    got = oracle.layer_norm_grads(dy, x, w, 1e-3)
    for i, t in enumerate((x, w, b)):
        f = lambda v: loss(*(v if j == i else u for j, u in enumerate((x, w, b))))
        # differences: e^2 times a third derivative of order 10, and 1e-16 / e
        torch.testing.assert_close(got[i], differences(f, t), rtol=1e-6, atol=1e-8)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = torch.nn.functional.layer_norm(leaves[0], (5,), leaves[1], leaves[2], 1e-3)
    torch.testing.assert_close(oracle.layer_norm(x, w, b, 1e-3)[0], y.detach())
    for a, c in zip(got, torch.autograd.grad(y, leaves, dy)):
        torch.testing.assert_close(a, c)


def test_feed_forward_gradients():
    ts = [draw(2, 3, 4, seed=0), draw(6, 4, seed=1), draw(6, 4, seed=2), draw(5, 6, seed=3)]
    dy = draw(2, 3, 5, seed=4)
    got = oracle.feed_forward_grads(dy, *ts)
    for i, t in enumerate(ts):
        f = lambda v: (oracle.feed_forward(*(v if j == i else u for j, u in enumerate(ts))) * dy).sum()
        torch.testing.assert_close(got[i], differences(f, t), rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("shared", [None, 0, -2, -1])
def test_dropout_mask(shared):
    keep = oracle.keep_mask((4, 5, 6), 0.5, 7, 1, shared)
    want = [4, 5, 6]
    if shared is not None:
        want[shared] = 1
    assert list(keep.shape) == want and 0.2 < keep.double().mean() < 0.8
    assert not oracle.keep_mask((4, 4), 1.0, 3).any() and oracle.keep_mask((4, 4), 0.0, 3).all()
