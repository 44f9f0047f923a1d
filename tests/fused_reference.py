"""Plain 64-bit form of the products around a transformer block, with a bound on what a correct kernel may be off.

The bounds follow from the arithmetic, not from runs. With u = 2^-11 (half), 2^-8 (bfloat16) or 2^-24 (single):
  - a product of 16-bit operands is exact in fp32; a tensor core adds 16 of them at a time to a fp32 accumulator and may
    cut off instead of rounding, so a sum of K products is off by at most (K / 16 + 4) * 2^-22 of sum |a||b|;
  - the single-precision kernels keep 2^-21 of every product (two parts of 11 bits) and add in fp32: at most
    2^-20 + (K + 8) * 2^-24 of sum |a||b|;
  - activations and their slopes have a slope of at most 1.2 and 1.2 in their argument, and are evaluated to 2^-19 of
    |z| and of 1;
  - a stored value is off by u relative, or by half the type's smallest subnormal.
"""
import math

import torch

STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
ACTS = {161: "identity", 162: "relu", 163: "gelu", 164: "gelu_tanh", 165: "silu"}


def value(act, z):
    if act == 162:
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == 163:
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if act == 164:
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if act == 165:
        return z * torch.sigmoid(z)
    return z


def slope(act, z):
    if act == 162:
        return (z > 0).double()
    if act == 163:
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == 164:
        s = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return s + z * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if act == 165:
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def sum_error(k, dtype):
    return 2.0 ** -20 + (k + 8) * 2.0 ** -24 if dtype == torch.float32 else (k / 16 + 4) * 2.0 ** -22


def stored(exact, error, dtype):
    """Bound on a stored value whose unrounded form is within `error` of `exact`."""
    return STEP[dtype] * (exact.abs() + error) + error + TINY[dtype]


def product(x, w, alpha):
    """x (rows x k) times w (k x n) in 64 bits, and sum |x||w|."""
    x, w = x.double(), w.double()
    return alpha * (x @ w), abs(alpha) * (x.abs() @ w.abs())


def forward(x, w, alpha, bias, act, beta, d, dtype, c_dtype):
    """(C, bound, Z, bound) of act(alpha x w + bias) + beta d."""
    z, mag = product(x, w, alpha)
    err = sum_error(x.shape[1], dtype) * mag
    if bias is not None:
        z = z + bias.double()
        err = err + 2.0 ** -22 * (mag + bias.double().abs())
    y = value(act, z)
    y_err = 1.2 * err + 2.0 ** -19 * z.abs()
    if beta != 0:
        y = y + beta * d.double()
        y_err = y_err + 2.0 ** -22 * (y.abs() + abs(beta) * d.double().abs())
    z_err = err
    if dtype == torch.float32:  # single precision rounds the product before the pass over it
        y_err = y_err + 2.0 ** -22 * mag
    return y, stored(y, y_err, c_dtype), z, stored(z, z_err, dtype)


def backward(x, w, alpha, beta, d, act, z, dtype):
    """(C, bound, column sums, bound) of (alpha x w + beta d) * slope(z)."""
    g, mag = product(x, w, alpha)
    err = sum_error(x.shape[1], dtype) * mag + 2.0 ** -22 * mag
    if beta != 0:
        g = g + beta * d.double()
        err = err + 2.0 ** -22 * abs(beta) * d.double().abs()
    return gradient(g, err, act, z, dtype)


def gradient(g, err, act, z, dtype):
    c = g * slope(act, z.double()) if z is not None else g
    c_err = 1.2 * err + 2.0 ** -19 * g.abs()
    total = c.sum(0)
    total_err = c_err.sum(0) + (c.shape[0] + 8) * 2.0 ** -24 * c.abs().sum(0)
    return c, stored(c, c_err, dtype), total, stored(total, total_err, dtype)


def check(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        i = int(torch.argmax((off / bound).nan_to_num(nan=float("inf")).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values outside the bound; worst at {i}: got "
                             f"{got.flatten()[i].item()!r}, want {want.flatten()[i].item()!r}, bound {bound.flatten()[i].item():.3g}")
