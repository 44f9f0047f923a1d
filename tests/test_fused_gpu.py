"""Products with an epilogue and products grouped by expert, forward and backward, against a 64-bit form of the same.

Sizes are chosen around the tiles (128 or 256 features, 32 to 256 vectors, 64 inner elements): one below, at and above
them, single rows, sizes that are multiples of nothing. B200BLAS_FUSED forces a kernel variant where a small problem
would not reach it by itself."""
import itertools

import pytest

import clblast_b200 as cb
from tests import fused_reference as R

pytestmark = pytest.mark.gpu

ROW, COL, NO, YES = 101, 102, 111, 112
OK = cb.StatusCode.kSuccess
VARIANTS = ["0", "1", "2", "3", "4", "5", "2,2", "2,4", "3,2", "3,8", "4,2", "4,8", "1,2"]


def force(monkeypatch, v):
    if v is None:
        monkeypatch.delenv("B200BLAS_FUSED", raising=False)
    else:
        monkeypatch.setenv("B200BLAS_FUSED", v)


def dt(torch, name):
    return {"half": torch.float16, "bf16": torch.bfloat16, "single": torch.float32}[name]


def randn(torch, g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


class Padded:
    """A matrix inside a larger buffer of a sentinel, so that writes outside of it are seen."""

    def __init__(self, torch, rows, cols, ld, offset, dtype, fill=None, planes=1, stride=0):
        self.rows, self.cols, self.ld, self.offset, self.planes, self.stride = rows, cols, ld, offset, planes, stride
        size = offset + (planes - 1) * stride + (rows - 1) * ld + cols + 67
        self.buf = torch.full((size,), 0.0, dtype=dtype, device="cuda")
        self.sentinel = -77.0
        self.buf.fill_(self.sentinel)
        if fill is not None:
            self.view().copy_(fill if planes > 1 else fill.reshape(rows, cols))

    def view(self):
        if self.planes > 1:
            return self.buf.as_strided((self.planes, self.rows, self.cols), (self.stride, self.ld, 1), self.offset)
        return self.buf.as_strided((self.rows, self.cols), (self.ld, 1), self.offset)

    def outside_untouched(self):
        copy = self.buf.clone()
        if self.planes > 1:
            copy.as_strided((self.planes, self.rows, self.cols), (self.stride, self.ld, 1), self.offset).fill_(self.sentinel)
        else:
            copy.as_strided((self.rows, self.cols), (self.ld, 1), self.offset).fill_(self.sentinel)
        return bool((copy == self.sentinel).all())


def linear(torch, monkeypatch, v, name, c_name, layout, ta, tb, rows, n, k, *, bias=True, act=161, keep=True, beta=0.0, alpha=1.0,
           grad=False, pads=(0, 0, 0, 0, 0), offs=(0, 0, 0, 0, 0), inplace=None, seed=0, bias_grad=True):
    """One call in the caller's layout. rows / n are vectors / features: the row-major view of C is rows x n."""
    force(monkeypatch, v)
    dtype, c_dtype = dt(torch, name), dt(torch, c_name)
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, w = randn(torch, g, (rows, k), dtype), randn(torch, g, (k, n), dtype, k ** -0.5)
    d = randn(torch, g, (rows, n), c_dtype)
    z = randn(torch, g, (rows, n), dtype)
    b = randn(torch, g, (n,), dtype, 0.5)
    # row-major: A is x (rows x k), B is w (k x n). Column-major: the same memory is B and A, transposed.
    t_x, t_w = (ta, tb) if layout == ROW else (tb, ta)
    xs, ws = (x, w) if layout == ROW else (x.t().contiguous(), w.t().contiguous())

    def stored(mat, trans, pad, off):
        # memory lines of op(mat)'s storage: row-major stores rows, column-major columns
        m = mat if trans == NO else mat.t()
        m = m if layout == ROW else m.t()
        m = m.contiguous()
        return Padded(torch, m.shape[0], m.shape[1], m.shape[1] + pad, off, mat.dtype, m), m.shape[1] + pad

    px, ldx = stored(xs, t_x, pads[0], offs[0])
    pw, ldw = stored(ws, t_w, pads[1], offs[1])
    pd = Padded(torch, rows, n, n + pads[2], offs[2], c_dtype, d)
    pz = Padded(torch, rows, n, n + pads[3], offs[3], dtype, z if grad else None)
    pc = Padded(torch, rows, n, n + pads[4], offs[4], c_dtype, torch.full((rows, n), float("nan"), device="cuda", dtype=c_dtype))
    if inplace == "d":
        pc = pd
    if inplace == "z":
        pc = pz
    pb = Padded(torch, 1, n, n, 3, dtype, b)
    pg = Padded(torch, 1, n, n, 5, dtype)
    m_, n_ = (rows, n) if layout == ROW else (n, rows)
    (A, lda, oa), (B, ldb, ob) = ((px, ldx, offs[0]), (pw, ldw, offs[1])) if layout == ROW else ((pw, ldw, offs[1]), (px, ldx, offs[0]))
    stream = torch.cuda.current_stream()
    if grad:
        st = cb.GemmEpilogueGrad(layout, ta, tb, m_, n_, k, alpha, A.buf, oa, lda, B.buf, ob, ldb, beta, pd.buf if beta else None,
                                 offs[2], pd.ld, act, pz.buf if act != 161 else None, offs[3], pz.ld, pc.buf, pc.offset, pc.ld,
                                 pg.buf if bias_grad else None, 5, stream=stream)
        assert st == OK, st
        c, c_tol, total, t_tol = R.backward(x, w, alpha, beta, d, act, z if act != 161 else None, dtype)
        R.check(pc.view(), c, c_tol, "C")
        if bias_grad:
            R.check(pg.view()[0], total, t_tol, "bias gradient")
            assert pg.outside_untouched()
    else:
        st = cb.GemmEpilogue(layout, ta, tb, m_, n_, k, alpha, A.buf, oa, lda, B.buf, ob, ldb, pb.buf if bias else None, 3, act,
                             pz.buf if keep else None, offs[3], pz.ld, beta, pd.buf if beta else None, offs[2], pd.ld, pc.buf,
                             pc.offset, pc.ld, stream=stream)
        assert st == OK, st
        c, c_tol, zz, z_tol = R.forward(x, w, alpha, b if bias else None, act, beta, d, dtype, c_dtype)
        R.check(pc.view(), c, c_tol, "C")
        if keep:
            R.check(pz.view(), zz, z_tol, "Z")
            assert pz.outside_untouched()
    assert pc.outside_untouched()
    assert px.outside_untouched() and pw.outside_untouched()
    code, where = cb.tensor_core_status()
    assert code == OK, where


@pytest.mark.parametrize("v", VARIANTS)
@pytest.mark.parametrize("name", ["half", "bf16"])
def test_every_variant(cuda, monkeypatch, v, name):
    linear(cuda, monkeypatch, v, name, name, ROW, NO, YES, 70, 264, 200, act=165, beta=0.5)
    assert cb.last_kernel().startswith("fused_")
    linear(cuda, monkeypatch, v, name, name, ROW, NO, YES, 300, 520, 1000, act=163)
    linear(cuda, monkeypatch, v, name, name, ROW, NO, YES, 300, 520, 1000, act=164, grad=True, beta=1.0)
    linear(cuda, monkeypatch, v, name, "single", ROW, NO, YES, 300, 520, 128, act=162, beta=-1.5)


@pytest.mark.parametrize("layout,ta,tb", list(itertools.product((ROW, COL), (NO, YES), (NO, YES))))
@pytest.mark.parametrize("v", [None, "0", "2", "3,4"])
def test_layouts(cuda, monkeypatch, layout, ta, tb, v):
    linear(cuda, monkeypatch, v, "half", "half", layout, ta, tb, 136, 264, 320, act=163, beta=2.0, alpha=0.5)
    linear(cuda, monkeypatch, v, "bf16", "bf16", layout, ta, tb, 136, 264, 320, act=165, beta=2.0, alpha=0.5, grad=True)


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 8, 8), (1, 129, 65), (2, 1000, 63), (31, 127, 64), (32, 128, 128), (33, 129, 192),
                                      (64, 256, 64), (65, 255, 8), (128, 257, 72), (255, 384, 96), (257, 136, 1032), (1000, 24, 520),
                                      (3, 4104, 40), (515, 1, 16)])
@pytest.mark.parametrize("name", ["half", "bf16", "single"])
def test_sizes(cuda, monkeypatch, rows, n, k, name):
    linear(cuda, monkeypatch, None, name, name, ROW, NO, YES, rows, n, k, act=163, beta=1.0)
    linear(cuda, monkeypatch, None, name, name, ROW, NO, NO, rows, n, k, act=164, beta=1.0, grad=True)


@pytest.mark.parametrize("rows,n,k", [(5, 33, 130), (16, 100, 1025), (17, 65, 515), (32, 520, 2050), (33, 64, 31), (64, 400, 300), (65, 129, 777),
                                      (130, 130, 2048), (700, 1000, 900), (1030, 257, 2400)])
@pytest.mark.parametrize("layout,ta,tb", [(ROW, NO, YES), (ROW, NO, NO), (COL, NO, NO), (COL, YES, YES), (ROW, YES, NO)])
def test_single_precision(cuda, monkeypatch, rows, n, k, layout, ta, tb):
    """Few vectors, one tile, ragged tiles, an inner extent split over blocks, and products with many tiles."""
    for pads, offs in (((0, 0, 0, 0, 0), (0, 0, 0, 0, 0)), ((4, 4, 1, 2, 3), (4, 8, 1, 2, 3)), ((1, 3, 0, 0, 0), (0, 5, 0, 0, 0))):
        linear(cuda, monkeypatch, None, "single", "single", layout, ta, tb, rows, n, k, act=163, beta=1.0, alpha=0.75, pads=pads, offs=offs)
        linear(cuda, monkeypatch, None, "single", "single", layout, ta, tb, rows, n, k, act=165, beta=-0.5, grad=True, pads=pads, offs=offs)
        linear(cuda, monkeypatch, None, "single", "single", layout, ta, tb, rows, n, k, act=164, grad=True, pads=pads, offs=offs, bias_grad=False)
    linear(cuda, monkeypatch, None, "single", "single", layout, ta, tb, rows, n, k, act=165, beta=1.0, inplace="d")
    linear(cuda, monkeypatch, None, "single", "single", layout, ta, tb, rows, n, k, act=165, beta=1.0, grad=True, inplace="z", bias_grad=False)
    linear(cuda, monkeypatch, None, "single", "single", layout, ta, tb, rows, n, k, act=165, beta=1.0, grad=True, inplace="z")


@pytest.mark.parametrize("act", [161, 162, 163, 164, 165])
@pytest.mark.parametrize("name,c_name", [("half", "half"), ("bf16", "bf16"), ("half", "single"), ("bf16", "single"), ("single", "single")])
@pytest.mark.parametrize("bias,keep,beta", [(False, False, 0.0), (True, True, 0.0), (True, False, 1.0), (False, True, -0.25)])
def test_epilogues(cuda, monkeypatch, act, name, c_name, bias, keep, beta):
    linear(cuda, monkeypatch, None, name, c_name, ROW, NO, YES, 200, 392, 256, act=act, bias=bias, keep=keep, beta=beta, alpha=1.5)
    if name == c_name:
        linear(cuda, monkeypatch, None, name, name, ROW, NO, YES, 200, 392, 256, act=act, grad=True, beta=beta, bias_grad=bias)


@pytest.mark.parametrize("pads,offs", [((8, 8, 8, 8, 8), (8, 16, 24, 8, 8)), ((1, 0, 0, 0, 0), (0, 0, 0, 0, 0)), ((0, 3, 0, 0, 0), (0, 1, 0, 0, 0)),
                                       ((0, 0, 1, 0, 0), (0, 0, 0, 0, 0)), ((0, 0, 0, 5, 0), (0, 0, 0, 2, 0)), ((0, 0, 0, 0, 3), (0, 0, 0, 0, 1)),
                                       ((7, 7, 7, 7, 7), (1, 3, 5, 7, 9))])
@pytest.mark.parametrize("v", [None, "0", "3", "4,4"])
def test_strides_and_offsets(cuda, monkeypatch, pads, offs, v):
    linear(cuda, monkeypatch, v, "half", "half", ROW, NO, YES, 161, 272, 136, act=165, beta=1.0, pads=pads, offs=offs)
    linear(cuda, monkeypatch, v, "bf16", "bf16", ROW, NO, YES, 161, 272, 136, act=165, beta=1.0, pads=pads, offs=offs, grad=True)
    linear(cuda, monkeypatch, v, "bf16", "single", ROW, NO, YES, 161, 272, 136, act=165, beta=1.0, pads=pads, offs=offs)


@pytest.mark.parametrize("v", [None, "0", "2", "4,8"])
def test_in_place(cuda, monkeypatch, v):
    for name in ("half", "bf16", "single"):
        linear(cuda, monkeypatch, v, name, name, ROW, NO, YES, 300, 392, 256, act=163, beta=1.0, inplace="d", keep=False)
        linear(cuda, monkeypatch, v, name, name, ROW, NO, YES, 300, 392, 256, act=163, beta=1.0, inplace="z", grad=True)
        linear(cuda, monkeypatch, v, name, name, ROW, NO, YES, 300, 392, 256, act=163, beta=1.0, inplace="d", grad=True)


@pytest.mark.parametrize("v", ["0", "1", "2", "3", "4", "5"])
def test_many_tiles_per_cta(cuda, monkeypatch, v):
    """More tiles than SMs: both accumulators, the operand ring and the staging rings go round several times."""
    linear(cuda, monkeypatch, v, "bf16", "bf16", ROW, NO, YES, 3000, 4104, 136, act=165, beta=1.0)
    linear(cuda, monkeypatch, v, "bf16", "bf16", ROW, NO, YES, 3000, 4104, 136, act=165, grad=True, beta=1.0)


def test_infinities_and_nan(cuda, monkeypatch):
    """An infinity or NaN reaches its own row or feature and nothing else; activations take their limits."""
    torch = cuda
    force(monkeypatch, None)
    rows, n, k = 96, 272, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    for act in (161, 162, 163, 164, 165):
        x, w = randn(torch, g, (rows, k), torch.float16), randn(torch, g, (n, k), torch.float16, 0.1)
        bias = torch.zeros(n, device="cuda", dtype=torch.float16)
        bias[3], bias[5], bias[7] = float("inf"), float("-inf"), float("nan")
        c = torch.empty(rows, n, device="cuda", dtype=torch.float16)
        x[10, 4] = float("nan")
        st = cb.GemmEpilogue(ROW, NO, YES, rows, n, k, 1.0, x, 0, k, w, 0, k, bias, 0, act, None, 0, n, 0.0, None, 0, n, c, 0, n,
                             stream=torch.cuda.current_stream())
        assert st == OK
        plain = torch.ones(n, dtype=torch.bool, device="cuda")
        plain[[3, 5, 7]] = False
        others = torch.arange(rows, device="cuda") != 10
        assert torch.isfinite(c[others][:, plain]).all()
        assert torch.isnan(c[10]).all() and torch.isnan(c[:, 7]).all()
        assert (c[others, 3] == float("inf")).all()
        assert (c[others, 5] == (float("-inf") if act == 161 else 0.0)).all()


# ---- grouped ---------------------------------------------------------------------------------------------------------

def spans(torch, sizes, rows, first=0):
    ends = [first]
    for s in sizes:
        ends.append(ends[-1] + s)
    assert ends[-1] <= rows
    return torch.tensor(ends, dtype=torch.int64, device="cuda"), list(zip(ends[:-1], ends[1:]))


def grouped(torch, monkeypatch, v, name, c_name, sizes, rows, n, k, *, first=0, trans=YES, bias=True, act=165, keep=True, beta=0.0,
            alpha=1.0, grad=False, pad=0, w_pad=0, seed=0, w_shared=False):
    force(monkeypatch, v)
    dtype, c_dtype = dt(torch, name), dt(torch, c_name)
    g = torch.Generator(device="cuda").manual_seed(seed)
    G = len(sizes)
    x, w = randn(torch, g, (rows, k), dtype), randn(torch, g, (G, k, n), dtype, k ** -0.5)
    if w_shared:
        w[:] = w[0].clone()
    d, z, b = randn(torch, g, (rows, n), c_dtype), randn(torch, g, (rows, n), dtype), randn(torch, g, (G, n), dtype)
    off, parts = spans(torch, sizes, rows, first)
    ws = w if trans == NO else w.transpose(1, 2).contiguous()
    w_ld = ws.shape[2] + w_pad
    w_stride = ws.shape[1] * w_ld + w_pad
    pw = Padded(torch, ws.shape[1], ws.shape[2], w_ld, 0, dtype, ws if G > 1 else ws[0], planes=G, stride=w_stride)
    px = Padded(torch, rows, k, k + pad, pad, dtype, x)
    pd, pz = Padded(torch, rows, n, n + pad, pad, c_dtype, d), Padded(torch, rows, n, n + pad, pad, dtype, z if grad else None)
    pc = Padded(torch, rows, n, n + pad, pad, c_dtype)
    pc.view().fill_(55.0)
    if not grad:
        pz.view().fill_(55.0)
    pb, pg = Padded(torch, G, n, n + 3, 1, dtype, b), Padded(torch, G, n, n + 5, 2, dtype)
    stream = torch.cuda.current_stream()
    if grad:
        st = cb.GemmGroupedGrad(trans, G, rows, n, k, alpha, px.buf, pad, k + pad, pw.buf, 0, w_ld, 0 if w_shared else w_stride, off, beta,
                                pd.buf if beta else None, pad, n + pad, act, pz.buf if act != 161 else None, pad, n + pad, pc.buf, pad,
                                n + pad, pg.buf, 2, n + 5, stream=stream)
    else:
        st = cb.GemmGrouped(trans, G, rows, n, k, alpha, px.buf, pad, k + pad, pw.buf, 0, w_ld, 0 if w_shared else w_stride, off,
                            pb.buf if bias else None, 1, n + 3, act, pz.buf if keep else None, pad, n + pad, beta,
                            pd.buf if beta else None, pad, n + pad, pc.buf, pad, n + pad, stream=stream)
    assert st == OK, st
    assert cb.last_kernel().startswith("fused_")
    inside = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for i, (lo, hi) in enumerate(parts):
        inside[lo:hi] = True
        if grad:
            c, tol, total, t_tol = R.backward(x[lo:hi], w[i], alpha, beta, d[lo:hi], act, z[lo:hi] if act != 161 else None, dtype)
            R.check(pg.view()[i] if G > 1 else pg.view()[0], total, t_tol, f"bias gradient of group {i}")
        else:
            c, tol, zz, z_tol = R.forward(x[lo:hi], w[i], alpha, b[i] if bias else None, act, beta, d[lo:hi], dtype, c_dtype)
            if keep:
                R.check(pz.view()[lo:hi], zz, z_tol, f"Z of group {i}")
        R.check(pc.view()[lo:hi], c, tol, f"C of group {i}")
    assert (pc.view()[~inside] == 55.0).all(), "rows of no group were written"
    if keep and not grad:
        assert (pz.view()[~inside] == 55.0).all()
    assert pc.outside_untouched() and pz.outside_untouched() and pg.outside_untouched() and pw.outside_untouched()
    code, where = cb.tensor_core_status()
    assert code == OK, where


SIZES = [([5], 5), ([0], 4), ([0, 0, 7, 0], 7), ([1, 1, 1, 1, 1], 5), ([3, 0, 64, 33, 0, 1, 129], 240), ([257, 31, 0, 300], 600)]


@pytest.mark.parametrize("sizes,rows", SIZES)
@pytest.mark.parametrize("v", [None, "0", "1", "2", "3", "4", "5", "4,8", "2,2"])
def test_groups(cuda, monkeypatch, sizes, rows, v):
    grouped(cuda, monkeypatch, v, "bf16", "bf16", sizes, rows, 264, 200, act=165, beta=1.0)
    grouped(cuda, monkeypatch, v, "half", "half", sizes, rows, 264, 200, act=163, beta=1.0, grad=True)


@pytest.mark.parametrize("trans", [NO, YES])
@pytest.mark.parametrize("n,k", [(8, 8), (127, 64), (129, 65), (384, 333), (40, 1000)])
def test_grouped_sizes(cuda, monkeypatch, trans, n, k):
    grouped(cuda, monkeypatch, None, "half", "half", [3, 0, 64, 33, 0, 1, 129], 250, n, k, first=2, trans=trans, beta=-1.0, alpha=0.5)
    grouped(cuda, monkeypatch, None, "bf16", "bf16", [3, 0, 64, 33, 0, 1, 129], 250, n, k, first=2, trans=trans, beta=-1.0, grad=True)
    grouped(cuda, monkeypatch, None, "bf16", "single", [3, 0, 64, 33, 0, 1, 129], 250, n, k, first=2, trans=trans, beta=1.0)


@pytest.mark.parametrize("pad,w_pad", [(8, 8), (1, 0), (0, 1), (3, 5)])
def test_grouped_strides(cuda, monkeypatch, pad, w_pad):
    grouped(cuda, monkeypatch, None, "half", "half", [50, 0, 70], 130, 272, 136, pad=pad, w_pad=w_pad, beta=1.0)
    grouped(cuda, monkeypatch, None, "half", "half", [50, 0, 70], 130, 272, 136, pad=pad, w_pad=w_pad, beta=1.0, grad=True)
    grouped(cuda, monkeypatch, None, "bf16", "single", [50, 0, 70], 130, 272, 136, pad=pad, w_pad=w_pad, beta=1.0, trans=NO)


def test_many_groups(cuda, monkeypatch):
    sizes = [(7 * i) % 13 for i in range(1024)]
    for v in (None, "0", "2"):
        grouped(cuda, monkeypatch, v, "bf16", "bf16", sizes, sum(sizes) + 9, 24, 32, first=9)
        grouped(cuda, monkeypatch, v, "bf16", "bf16", sizes, sum(sizes) + 9, 24, 32, first=9, grad=True)


def test_shared_weights(cuda, monkeypatch):
    grouped(cuda, monkeypatch, None, "bf16", "bf16", [20, 0, 41], 61, 136, 72, w_shared=True)


def test_offsets_out_of_range(cuda, monkeypatch):
    """Offsets that leave [0, rows] or descend lose rows and touch nothing else."""
    torch = cuda
    force(monkeypatch, None)
    rows, n, k, G = 100, 136, 64, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = randn(torch, g, (rows, k), torch.float16), randn(torch, g, (G, n, k), torch.float16, 0.1)
    off = torch.tensor([-5, 40, 30, 2 ** 40, 60], dtype=torch.int64, device="cuda")
    spans_ = [(0, 40), (40, 40), (40, 100), (100, 100)]
    c = Padded(torch, rows, n, n, 0, torch.float16)
    st = cb.GemmGrouped(YES, G, rows, n, k, 1.0, x, 0, k, w, 0, k, n * k, off, None, 0, n, 161, None, 0, n, 0.0, None, 0, n, c.buf, 0, n,
                        stream=torch.cuda.current_stream())
    assert st == OK
    for i, (lo, hi) in enumerate(spans_):
        want, tol, _, _ = R.forward(x[lo:hi], w[i].t(), 1.0, None, 161, 0.0, None, torch.float16, torch.float16)
        R.check(c.view()[lo:hi], want, tol, "C")
    assert c.outside_untouched()
    dw = Padded(torch, k, n, n, 0, torch.float32, planes=G, stride=k * n)
    y = randn(torch, g, (rows, n), torch.float16)
    st = cb.GemmGroupedWeight(G, rows, k, n, 1.0, x, 0, k, y, 0, n, off, 0.0, dw.buf, 0, n, k * n, stream=torch.cuda.current_stream())
    assert st == OK
    torch.cuda.synchronize()
    assert dw.outside_untouched()


def weight(torch, monkeypatch, v, name, c_name, sizes, rows, m, n, *, first=0, alpha=1.0, beta=0.0, pad=0, seed=0, poison=False):
    force(monkeypatch, v)
    dtype, c_dtype = dt(torch, name), dt(torch, c_name)
    g = torch.Generator(device="cuda").manual_seed(seed)
    G = len(sizes)
    x, y, c = randn(torch, g, (rows, m), dtype), randn(torch, g, (rows, n), dtype), randn(torch, g, (G, m, n), c_dtype)
    off, parts = spans(torch, sizes, rows, first)
    if poison:  # rows of no group may hold anything
        inside = torch.zeros(rows, dtype=torch.bool, device="cuda")
        for lo, hi in parts:
            inside[lo:hi] = True
        x[~inside], y[~inside] = float("nan"), float("inf")
    px, py = Padded(torch, rows, m, m + pad, pad, dtype, x), Padded(torch, rows, n, n + pad, pad, dtype, y)
    stride = m * (n + pad) + pad
    start = c if beta else torch.full_like(c, float("nan"))
    pc = Padded(torch, m, n, n + pad, pad, c_dtype, start if G > 1 else start[0], planes=G, stride=stride)
    st = cb.GemmGroupedWeight(G, rows, m, n, alpha, px.buf, pad, m + pad, py.buf, pad, n + pad, off, beta, pc.buf, pad, n + pad, stride,
                              stream=torch.cuda.current_stream())
    assert st == OK, st
    for i, (lo, hi) in enumerate(parts):
        want, mag = R.product(x[lo:hi].t(), y[lo:hi], alpha)
        err = R.sum_error(hi - lo, dtype) * mag
        if beta:
            want = want + beta * c[i].double()
            err = err + 2.0 ** -22 * (want.abs() + abs(beta) * c[i].double().abs())
        R.check(pc.view()[i] if G > 1 else pc.view(), want, R.stored(want, err, c_dtype), f"C of group {i}")
    assert pc.outside_untouched()
    code, where = cb.tensor_core_status()
    assert code == OK, where


@pytest.mark.parametrize("sizes,rows", SIZES)
@pytest.mark.parametrize("v", [None, "0", "1", "2", "3", "5", "2,2", "3,4"])
def test_weight_gradients(cuda, monkeypatch, sizes, rows, v):
    weight(cuda, monkeypatch, v, "bf16", "single", sizes, rows, 136, 264, beta=1.0)
    weight(cuda, monkeypatch, v, "half", "half", sizes, rows, 136, 264)
    weight(cuda, monkeypatch, v, "bf16", "single", sizes, rows + 20, 64, 128, first=11, poison=True, alpha=-2.0)


@pytest.mark.parametrize("v", ["0", "1", "2", "3", "5", "3,2"])
def test_weight_gradients_of_many_short_groups(cuda, monkeypatch, v):
    """Many tiles per CTA, each with a cut-off last block: several of them are in the operand ring at once."""
    sizes = [(13 * i) % 131 for i in range(40)]
    weight(cuda, monkeypatch, v, "bf16", "bf16", sizes, sum(sizes), 520, 776)
    weight(cuda, monkeypatch, v, "half", "single", sizes, sum(sizes) + 5, 520, 776, first=5, poison=True, beta=1.0)


@pytest.mark.parametrize("m,n,pad", [(1, 1, 0), (8, 8, 8), (65, 127, 0), (129, 257, 3), (200, 333, 1)])
def test_weight_gradient_sizes(cuda, monkeypatch, m, n, pad):
    for name, c_name in (("half", "half"), ("bf16", "bf16"), ("half", "single")):
        weight(cuda, monkeypatch, None, name, c_name, [3, 0, 64, 33, 0, 1, 129], 250, m, n, first=2, beta=0.5, pad=pad)


@pytest.mark.parametrize("name", ["half", "bf16", "single"])
@pytest.mark.parametrize("rows,n,pad", [(1, 1, 0), (7, 1000, 0), (64, 256, 8), (65, 257, 1), (1000, 40, 0), (70000, 8, 0)])
def test_activation_grad(cuda, monkeypatch, name, rows, n, pad):
    torch = cuda
    dtype = dt(torch, name)
    g = torch.Generator(device="cuda").manual_seed(2)
    for act in (161, 162, 163, 164, 165):
        dy, z = randn(torch, g, (rows, n), dtype), randn(torch, g, (rows, n), dtype, 2.0)
        py, pz = Padded(torch, rows, n, n + pad, pad, dtype, dy), Padded(torch, rows, n, n + pad, pad, dtype, z)
        pc, pg = Padded(torch, rows, n, n + pad, pad, dtype), Padded(torch, 1, n, n, 1, dtype)
        st = cb.ActivationGrad(rows, n, act, py.buf, pad, n + pad, pz.buf if act != 161 else None, pad, n + pad, pc.buf, pad, n + pad,
                               pg.buf, 1, stream=torch.cuda.current_stream())
        assert st == OK, st
        c, tol, total, t_tol = R.gradient(dy.double(), torch.zeros_like(dy, dtype=torch.float64), act, z if act != 161 else None, dtype)
        R.check(pc.view(), c, tol, "DZ")
        R.check(pg.view()[0], total, t_tol, "bias gradient")
        assert pc.outside_untouched() and pg.outside_untouched()
    # in place, without the sums; the sums alone
    st = cb.ActivationGrad(rows, n, act, py.buf, pad, n + pad, pz.buf, pad, n + pad, py.buf, pad, n + pad, None, 0,
                           stream=torch.cuda.current_stream())
    assert st == OK and torch.equal(py.view(), pc.view())
    again = Padded(torch, 1, n, n, 1, dtype)
    py2 = Padded(torch, rows, n, n + pad, pad, dtype, dy)
    st = cb.ActivationGrad(rows, n, act, py2.buf, pad, n + pad, pz.buf, pad, n + pad, None, 0, n, again.buf, 1,
                           stream=torch.cuda.current_stream())
    assert st == OK and torch.equal(again.buf, pg.buf)


def test_activation_grad_by_group(cuda):
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(4)
    sizes, rows, n = [3, 0, 64, 200, 0, 1], 300, 136
    off, parts = spans(torch, sizes, rows, 5)
    dy, z = randn(torch, g, (rows, n), torch.bfloat16), randn(torch, g, (rows, n), torch.bfloat16)
    dz, bg = torch.full_like(dy, 55.0), Padded(torch, len(sizes), n, n + 3, 0, torch.bfloat16)
    st = cb.ActivationGrad(rows, n, 163, dy, 0, n, z, 0, n, dz, 0, n, bg.buf, 0, groups=len(sizes), group_offsets=off, bias_grad_ld=n + 3,
                           stream=torch.cuda.current_stream())
    assert st == OK
    inside = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for i, (lo, hi) in enumerate(parts):
        inside[lo:hi] = True
        c, tol, total, t_tol = R.gradient(dy[lo:hi].double(), torch.zeros(hi - lo, n, device="cuda", dtype=torch.float64), 163, z[lo:hi],
                                          torch.bfloat16)
        R.check(dz[lo:hi], c, tol, "DZ")
        R.check(bg.view()[i], total, t_tol, "bias gradient")
    assert (dz[~inside] == 55.0).all() and bg.outside_untouched()
