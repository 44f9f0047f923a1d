"""The check of Newton-Schulz results notices what a kernel could lose. Mistakes are planted in the 64-bit model."""
import pytest
import torch

from tests import newton_schulz_reference as N


def matrix(m, n, seed=0):
    return torch.randn(m, n, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).float()


def model(g, dtype, plant=None, bits=None):
    single = dtype == torch.float32
    return N.iterate(g, bits=bits or (20 if single else 11), last=single, plant=plant).to(dtype)


TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(129, 300), (300, 129), (264, 264)])
def test_the_documented_roundings_pass(m, n, dtype):
    g = matrix(m, n).to(dtype)
    want, limit = N.allowed(g, dtype)
    assert limit < 0.01
    # the same roundings on other draws: the matrix with its columns in another order and one sign turned
    order = torch.randperm(n, generator=torch.Generator().manual_seed(1))
    N.check(model(-g[:, order] * 1.3, dtype)[:, torch.argsort(order)].neg(), want, limit)


def zero(name, where, at=None):
    def plant(which, step, x):
        if which == name and (at is None or step == at):
            x = x.clone()
            x[where] = 0
        return x
    return plant


MISTAKES = {
    "last row of the result": zero("x", (slice(-1, None), slice(None)), 4),
    "eight entries of one row": zero("x", (5, slice(8, 16)), 4),
    "a block of the result": zero("x", (slice(120, 128), slice(64, 72)), 4),
    "the last columns of the result": zero("x", (slice(None), slice(-1, None)), 4),
    "last row of X between two steps": zero("x", (slice(-1, None), slice(None)), 2),
    "a mirrored strip of G": zero("gram", (slice(0, 8), slice(128, None)), 4),
    "a mirrored strip of the bracket": zero("poly", (slice(0, 8), slice(128, None)), 3),
    "the last row of the bracket": zero("poly", (slice(-1, None), slice(None)), 4),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mistake", MISTAKES)
def test_a_lost_part_is_noticed(mistake, dtype):
    g = matrix(264, 520).to(dtype)
    want, limit = N.allowed(g, dtype)
    with pytest.raises(AssertionError):
        N.check(model(g, dtype, MISTAKES[mistake]), want, limit)


@pytest.mark.parametrize("dtype,bits", [(torch.float16, 9), (torch.bfloat16, 9), (torch.float32, 18)])
def test_two_bits_less_are_noticed(dtype, bits):
    g = matrix(264, 520).to(dtype)
    want, limit = N.allowed(g, dtype)
    with pytest.raises(AssertionError):
        N.check(model(g, dtype, bits=bits), want, limit)
