"""Inputs and error bounds of the tests of the operators around the attention.

The bounds are worst cases, element by element, of the arithmetic that the operators promise:
U[t] is the rounding of a result to its type (half a step, eps / 2); a sum of k terms in fp32 is off by
at most k 2^-23 of the sum of magnitudes (a step and not half of one: the tensor cores' accumulators need not
round to nearest).
"""

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
STEP = 2.0 ** -23
# What a rounding is off by below the type's smallest normal number, where U's relative bound does not hold: half
# of the smallest number above 0 (fp16: 2^-24 / 2; the other types share fp32's exponents, down to 2^-126, and the
# kernels may flush what lies below).
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def assert_bounded(got, want, bound, what):
    """|got - want| <= bound element by element (fp64), and what rounding adds to it near 0."""
    bound = bound + TINY[got.dtype]
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)      # NaN is bad
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; first at {i}: "
                             f"{float(got[i])!r}, want {float(want[i])!r} +- {float(bound[i]):.3g}")


def assert_norm(got, want, rel, what):
    """2-norm of the difference against that of the result."""
    err = float((got.detach().double() - want).norm() / want.norm().clamp_min(1e-300))
    assert err <= rel, f"{what}: relative error {err:.3g} > {rel:.3g}"


def normal(*shape, seed, dtype=torch.float32, device="cuda", std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(device)
