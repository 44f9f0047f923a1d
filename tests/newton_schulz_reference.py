"""The Newton-Schulz iteration in 64 bits, with and without the roundings that the kernels document, and a check of a result
entry by entry that no lost line, strip or tile passes.

What a correct kernel may be off follows from the iteration itself run in 64 bits with every kept matrix rounded:
  - 16-bit types: X, G and the bracket are kept in half precision, off by at most 2^-11 of an entry; sums in fp32 lie far
    below. The last product is stored in the caller's type, whose rounding has a root mean square of at most STEP / sqrt 3.
  - single precision: a matrix kept as two halves is off by 2^-22, and so are both operands of a product; leaving out lo lo
    costs another 2^-22; eight truncating additions to an accumulator 8 * 2^-24.6; together 2^-20 of an entry.
The roundings of kernel and model are not the same draws, so the norms of their errors are compared: a kernel's error may be
1.5 times the model's. It stays below that at any size with more than some thousand entries, and one bit less in any of the
kept matrices doubles its own share. Errors spread like the roundings that they stem from: over a line or a block of 8 x 8
their root mean square may be four times that over the whole matrix, and a lost one is off by its own size, hundreds of
times more.
"""
import math

import torch

STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def rounded(x, bits):
    """x with `bits` binary digits, to nearest."""
    mantissa, exponent = torch.frexp(x)
    return torch.ldexp(torch.round(mantissa * 2.0 ** bits) * 2.0 ** -bits, exponent)


def iterate(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7, bits=None, last=False, plant=None):
    """The result for one matrix; `bits` that every kept matrix holds, the last X too if `last`. `plant` (name, step, matrix)
    may spoil one of them: x, gram, poly."""
    keep = (lambda x: x) if bits is None else (lambda x: rounded(x, bits))
    spoil = plant or (lambda name, step, x: x)
    x = g.double()
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    x = keep(x.mT if tall else x)
    for i in range(steps):
        a, b, c = coefficients
        gram = spoil("gram", i, keep(x @ x.mT))
        poly = spoil("poly", i, keep(b * gram + c * gram @ gram))
        x = a * x + poly @ x
        if i + 1 < steps or last:
            x = keep(x)
        x = spoil("x", i, x)
    return x.mT if tall else x


def allowed(g, dtype, steps=5, coefficients=COEFFICIENTS):
    """(the exact result, the root mean square that a kernel's error may have relative to the result's)."""
    want = iterate(g, steps, coefficients)
    single = dtype == torch.float32
    model = iterate(g, steps, coefficients, bits=20 if single else 11, last=single)
    return want, float(1.5 * (model - want).norm() / want.norm()) + STEP[dtype] / math.sqrt(3)


def check(got, want, limit):
    off = got.double() - want
    rms = want.norm() / math.sqrt(want.numel())
    assert off.norm() <= limit * want.norm(), f"whole matrix off by {float(off.norm() / want.norm()):.3g}, may be {limit:.3g}"
    squares = (off / rms) ** 2
    for name, mean in (("row", squares.mean(1)), ("column", squares.mean(0))):
        i = int(mean.argmax())
        assert mean[i] <= (4 * limit) ** 2, f"{name} {i} off by {float(mean[i]) ** 0.5:.3g} of the matrix's mean, may be {4 * limit:.3g}"
    padded = torch.nn.functional.pad(squares, (0, -squares.shape[1] % 8, 0, -squares.shape[0] % 8))
    blocks = padded.view(padded.shape[0] // 8, 8, padded.shape[1] // 8, 8).mean((1, 3)).sqrt()
    i = int(blocks.argmax())
    assert blocks.flatten()[i] <= 4 * limit, (f"block {divmod(i, blocks.shape[1])} off by {float(blocks.max()):.3g} of the matrix's mean, "
                                              f"may be {4 * limit:.3g}")
