"""Activations and slopes at every finite half and bfloat16 number, and in single precision at the same places.

An exponential 2^x carries the rounding of its argument: x is off by at most four roundings of 2^-24 relative, so 2^x by
|x| ln 2 2^-22 < |x| 2^-22 relative; the exponential itself, the reciprocal and the fitted polynomial add less than 2^-20.
(x = z^2 / 2 log2 e for gelu, 2 |u| log2 e for its tanh form, |z| log2 e for silu, 128 at most: beyond, the value is zero.)
A product of such factors keeps that relative error, a sum takes it on the size of its terms. Where the exponential leaves
the range of fp32 results below 2^-118 become zero."""
import math

import pytest

import clblast_b200 as cb
from tests import fused_reference as R

pytestmark = pytest.mark.gpu

ROW, NO = 101, 111
OK = cb.StatusCode.kSuccess
LOG2E = math.log2(math.e)


def numbers(torch, dtype):
    bits = torch.arange(-32768, 32768, device="cuda", dtype=torch.int32).to(torch.int16)
    z = bits.view(torch.bfloat16 if dtype == torch.float32 else dtype)
    return z[torch.isfinite(z)].to(dtype)


def relative(torch, act, z):
    if act == 162:
        return torch.zeros_like(z)
    x = {163: z * z / 2, 164: (2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)).abs(), 165: z.abs()}[act] * LOG2E
    return 2.0 ** -20 + x.clamp(max=128.0) * 2.0 ** -22


def slope_terms(torch, act, z):
    """The size of the terms that the slope is a sum of."""
    if act == 162:
        return torch.ones_like(z)
    if act == 163:
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z.abs() * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3) if act == 164 else z
    s, rest = torch.sigmoid(u), torch.sigmoid(-u)
    du = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z) if act == 164 else 1
    return s + z.abs() * s * rest * du


@pytest.mark.parametrize("name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("act", [162, 163, 164, 165])
@pytest.mark.parametrize("v", [None, "0", "3,2"])
def test_every_number(cuda, monkeypatch, name, act, v):
    torch = cuda
    if v:
        monkeypatch.setenv("B200BLAS_FUSED", v)
    dtype = getattr(torch, name)
    z = numbers(torch, dtype)
    n, stream = z.numel(), torch.cuda.current_stream()
    one, c = torch.ones(1, device="cuda", dtype=dtype), torch.full_like(z, float("nan"))
    assert cb.GemmEpilogue(ROW, NO, NO, 1, n, 1, 1.0, one, 0, 1, z, 0, n, None, 0, act, None, 0, n, 0.0, None, 0, n, c, 0, n, stream=stream) == OK
    exact = z.double()
    want = R.value(act, exact)
    most = torch.finfo(dtype).max
    e = relative(torch, act, exact)
    R.check(c, want.clamp(-most, most), R.stored(want, e * want.abs(), dtype) + 2.0 ** -118, "value")
    dy, dz = torch.ones_like(z), torch.full_like(z, float("nan"))
    want = R.slope(act, exact)
    want = torch.where(exact.abs() > 1e4, (exact > 0).double(), want)  # the formula's inf * 0
    bound = R.stored(want, 2 * e * slope_terms(torch, act, exact.clamp(-1e4, 1e4)), dtype) + 2.0 ** -118
    assert cb.ActivationGrad(1, n, act, dy, 0, n, z, 0, n, dz, 0, n, None, 0, stream=stream) == OK
    R.check(dz, want, bound, "slope")
    # the same slopes in a product's epilogue: C = (1 * 1) act'(Z)
    ones = torch.ones_like(z)
    dz.fill_(float("nan"))
    assert cb.GemmEpilogueGrad(ROW, NO, NO, 1, n, 1, 1.0, one, 0, 1, ones, 0, n, 0.0, None, 0, n, act, z, 0, n, dz, 0, n, None, 0, stream=stream) == OK
    R.check(dz, want, bound, "slope in the epilogue")
