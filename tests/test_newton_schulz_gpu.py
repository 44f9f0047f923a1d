"""Newton-Schulz orthogonalisation against a 64-bit form of the same iteration.

The bounds hold for the Frobenius norm of the difference. 16-bit types: X, G and the bracket are rounded to half between
the products. An entry's rounding is at most 2^-11 relative, so a rounded matrix is off by at most 2^-11 of its
Frobenius norm. One step X' = a X + B X with B = b G + c G G takes an error E of X to at most (the largest slope of
the polynomial on [0, 1.2]) |E|; directions orthogonal to X's own grow by at most the polynomial's slope at 0. With the
default coefficients (3.4445, -4.7750, 2.0315) the slope p'(0) = 3.4445 is the largest, and small singular values grow by
the same factor as their errors: an error of relative size e in a direction that has not saturated stays of relative
size e. Directions that have saturated have singular values in [0.68, 1.13], where |p'| < 2.2. A step adds at most
2^-11 (|X'| + |B|_2 ... ) <= 8 * 2^-11 of |X'|, so after five steps the error is bounded by 5 * 8 * 2.2 * 2^-11 of |X|;
random signs keep the measured error far below. Single precision: the same with 2^-20 in place of 2^-11.
Results are compared through their norms, entries through a multiple of the root mean square.
"""
import pytest

import clblast_b200 as cb

pytestmark = pytest.mark.gpu

ROW, COL = 101, 102
OK = cb.StatusCode.kSuccess
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
LIMIT = {"half": 5 * 8 * 2.2 * 2.0 ** -11, "bf16": 5 * 8 * 2.2 * 2.0 ** -11 + 2.0 ** -8, "single": 5 * 8 * 2.2 * 2.0 ** -20}


def dt(torch, name):
    return {"half": torch.float16, "bf16": torch.bfloat16, "single": torch.float32}[name]


def exact(torch, g, scale, steps, coefficients, eps):
    x = g.double()
    x = x / (x.norm(dim=(-2, -1), keepdim=True) + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for i in range(steps):
        a, b, c = coefficients[i] if not isinstance(coefficients[0], float) else coefficients
        m = x @ x.mT
        x = a * x + (b * m + c * m @ m) @ x
    return scale * (x.mT if tall else x)


def run(torch, name, layout, m, n, batch=1, *, steps=5, coefficients=COEFFICIENTS, eps=1e-7, alpha=1.0, scale=1.0, pad=0, inplace=False, seed=0):
    dtype = dt(torch, name)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lines, one = (m, n) if layout == ROW else (n, m)
    g = (torch.randn(batch, lines, one, generator=gen, device="cuda") * scale).to(dtype)
    ld, stride = one + pad, lines * (one + pad) + 3 * pad
    size = pad + batch * stride + 64
    a = torch.full((size,), -7.0, device="cuda", dtype=dtype)
    a.as_strided((batch, lines, one), (stride, ld, 1), pad).copy_(g)
    b = a if inplace else torch.full((size,), -7.0, device="cuda", dtype=dtype)
    st = cb.NewtonSchulz(layout, m, n, alpha, a, pad, ld, stride, b, pad, ld, stride, batch, steps=steps, coefficients=coefficients,
                         epsilon=eps, stream=torch.cuda.current_stream())
    assert st == OK, st
    got = b.as_strided((batch, lines, one), (stride, ld, 1), pad).double()
    want = exact(torch, g, alpha, steps, coefficients, eps)
    for i in range(batch):
        norm = want[i].norm()
        off = (got[i] - want[i]).norm() / norm
        assert off <= LIMIT[name], (name, m, n, i, float(off))
        rms = norm / want[i].numel() ** 0.5
        assert (got[i] - want[i]).abs().max() <= 40 * LIMIT[name] * max(rms, want[i].abs().max())
    rest = b.clone()
    rest.as_strided((batch, lines, one), (stride, ld, 1), pad).fill_(-7.0)
    assert (rest == -7.0).all(), "written outside of B"
    code, where = cb.tensor_core_status()
    assert code == OK, where
    return got


@pytest.mark.parametrize("name", ["half", "bf16", "single"])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 64), (64, 1), (8, 24), (65, 63), (128, 128), (129, 300), (300, 129), (256, 520), (520, 256),
                                 (700, 700), (1000, 333)])
def test_sizes(cuda, name, m, n):
    run(cuda, name, ROW, m, n)
    run(cuda, name, COL, m, n)


@pytest.mark.parametrize("v", ["0", "2", "3"])
@pytest.mark.parametrize("m,n", [(512, 768), (768, 512), (600, 600), (264, 1000)])
def test_variants(cuda, monkeypatch, v, m, n):
    monkeypatch.setenv("B200BLAS_FUSED", v)
    run(cuda, "bf16", ROW, m, n, 2)


@pytest.mark.parametrize("name", ["half", "bf16", "single"])
def test_batches_strides_and_scales(cuda, name):
    run(cuda, name, ROW, 136, 264, 3, pad=8)
    run(cuda, name, ROW, 136, 264, 3, pad=3, alpha=-0.25)
    run(cuda, name, ROW, 264, 136, 2, pad=1, inplace=True)
    run(cuda, name, ROW, 100, 100, steps=1)
    run(cuda, name, ROW, 100, 100, steps=3, coefficients=[(4.0, -6.0, 3.0), (3.5, -5.0, 2.2), (3.0, -4.0, 2.0)])
    run(cuda, name, ROW, 200, 100, scale=1e-3)
    if name != "half":
        run(cuda, name, ROW, 200, 100, scale=1e-12, eps=0.0)
        run(cuda, name, ROW, 200, 100, scale=1e25, eps=0.0)


@pytest.mark.parametrize("name", ["half", "bf16", "single"])
def test_zero_and_nan(cuda, name):
    torch = cuda
    g = torch.zeros(3, 64, 72, device="cuda", dtype=dt(torch, name))
    g[1].normal_()
    g[2].normal_()
    g[2, 5, 7] = float("nan")
    out = torch.full_like(g, 9.0)
    st = cb.NewtonSchulz(ROW, 64, 72, 1.0, g, 0, 72, 64 * 72, out, 0, 72, 64 * 72, 3, stream=torch.cuda.current_stream())
    assert st == OK
    assert (out[0] == 0).all() and torch.isfinite(out[1]).all() and torch.isnan(out[2]).all()


def test_repeats_bit_for_bit(cuda):
    torch = cuda
    a = run(torch, "bf16", ROW, 700, 520, 2)
    b = run(torch, "bf16", ROW, 700, 520, 2)
    assert torch.equal(a, b)
