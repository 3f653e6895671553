"""Bounds of the products of 16-bit operands, used by their tests.

A sum of k products of 16-bit numbers in fp32: the products are exact, each of the k additions is off by at most 2^-23 of the largest partial sum (a matrix
instruction may cut where it adds, so twice the half step of 2^-24), and no partial sum passes S = sum |a| |b|: |error| <= k 2^-23 S.  Rounding to 16 bits: at most half a step,
eps / 2 of the value, and for half half of the smallest number, 2^-25, where it is subnormal."""
import torch


def sum_error(a, b):
    """Bound of the error of a @ b (float64 operands), before the last rounding."""
    return a.shape[1] * 2.0 ** -23 * (a.abs() @ b.abs())


def rounded(y, before, dtype):
    """Bound of the error of y, known up to `before`, after its rounding to dtype."""
    return before + torch.finfo(dtype).eps / 2 * (y.abs() + before) + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def check(got, want, bound, what=""):
    got = got.double().cpu()
    want, bound = want.cpu(), bound.cpu()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what + ": not finite"
    off = (got - want).abs() - bound
    at = int(off.argmax()) if off.numel() else 0
    assert off.numel() == 0 or float(off.max()) <= 0, "%s: element %d is %r, should be %r within %r" % (
        what, at, float(got.flatten()[at]), float(want.flatten()[at]), float(bound.flatten()[at]))
