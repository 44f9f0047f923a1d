"""The products around a transformer block as a program uses them: run after one another through a training step, on other
streams than the default, captured and replayed, beside one another; and the calls they refuse on a device.

Bounds are those of the plain 64-bit form of each product on the operands that it was really given. Where a whole chain
is compared, an error E of an operand reaches a product's result as at most |E| |W| entry by entry."""
import pytest

import clblast_b200 as cb
from tests import fused_reference as R

pytestmark = pytest.mark.gpu

ROW, NO, YES = 101, 111, 112
S = cb.StatusCode
OK = S.kSuccess


def randn(torch, seed, shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def healthy():
    code, where = cb.tensor_core_status()
    assert code == OK, where


# ---- one after another ---------------------------------------------------------------------------------------------

class Experts:
    """A training step of experts over rows sorted by expert: two grouped products with a residual, their gradients, and
    the orthogonalised update of the first weights. Rows behind the last group are padding."""

    def __init__(self, torch, sizes, rows, n, h, dtype, act, seed=0):
        self.torch, self.rows, self.n, self.h, self.act, self.G, self.dtype = torch, rows, n, h, act, len(sizes), dtype
        ends = [0]
        for s in sizes:
            ends.append(ends[-1] + s)
        self.spans = list(zip(ends[:-1], ends[1:]))
        self.used = ends[-1]
        self.offsets = torch.tensor(ends, dtype=torch.int64, device="cuda")
        G = self.G
        self.x, self.g = randn(torch, seed, (rows, n), dtype), randn(torch, seed + 1, (rows, n), dtype)
        self.w1, self.w2 = randn(torch, seed + 2, (G, h, n), dtype, n ** -0.5), randn(torch, seed + 3, (G, n, h), dtype, h ** -0.5)
        self.b1, self.b2 = randn(torch, seed + 4, (G, h), dtype, 0.1), randn(torch, seed + 5, (G, n), dtype, 0.1)
        new = lambda *shape, t=dtype: torch.full(shape, 9.0, dtype=t, device="cuda")
        self.z, self.a, self.y = new(rows, h), new(rows, h), new(rows, n)
        self.da, self.dx = new(rows, h), new(rows, n)
        self.db1, self.db2 = new(G, h), new(G, n)
        self.dw1, self.dw2 = new(G, h, n, t=torch.float32), new(G, n, h, t=torch.float32)
        self.update = new(G, h, n, t=torch.float32)
        self.results = [self.z, self.a, self.y, self.da, self.dx, self.db1, self.db2, self.dw1, self.dw2, self.update]

    def step(self, stream):
        G, rows, n, h = self.G, self.rows, self.n, self.h
        st = [
            cb.GemmGrouped(YES, G, rows, h, n, 1.0, self.x, 0, n, self.w1, 0, n, h * n, self.offsets, self.b1, 0, h, self.act, self.z, 0, h,
                           0.0, None, 0, h, self.a, 0, h, stream=stream),
            cb.GemmGrouped(YES, G, rows, n, h, 1.0, self.a, 0, h, self.w2, 0, h, n * h, self.offsets, self.b2, 0, n, 161, None, 0, n, 1.0,
                           self.x, 0, n, self.y, 0, n, stream=stream),
            cb.ActivationGrad(rows, n, 161, self.g, 0, n, None, 0, n, None, 0, n, self.db2, 0, groups=G, group_offsets=self.offsets,
                              bias_grad_ld=n, stream=stream),
            cb.GemmGroupedGrad(NO, G, rows, h, n, 1.0, self.g, 0, n, self.w2, 0, h, n * h, self.offsets, 0.0, None, 0, h, self.act, self.z, 0,
                               h, self.da, 0, h, self.db1, 0, h, stream=stream),
            cb.GemmGroupedGrad(NO, G, rows, n, h, 1.0, self.da, 0, h, self.w1, 0, n, h * n, self.offsets, 1.0, self.g, 0, n, 161, None, 0, n,
                               self.dx, 0, n, None, 0, n, stream=stream),
            cb.GemmGroupedWeight(G, rows, n, h, 1.0, self.g, 0, n, self.a, 0, h, self.offsets, 0.0, self.dw2, 0, h, n * h, stream=stream),
            cb.GemmGroupedWeight(G, rows, h, n, 1.0, self.da, 0, h, self.x, 0, n, self.offsets, 0.0, self.dw1, 0, n, h * n, stream=stream),
            cb.NewtonSchulz(ROW, h, n, 1.0, self.dw1, 0, n, h * n, self.update, 0, n, h * n, G, stream=stream),
        ]
        assert st == [OK] * len(st), st

    def check(self):
        """Each result against the 64-bit form on what its product was given."""
        torch, d = self.torch, self.dtype
        for i, (lo, hi) in enumerate(self.spans):
            s = slice(lo, hi)
            a, a_tol, z, z_tol = R.forward(self.x[s], self.w1[i].t(), 1.0, self.b1[i], self.act, 0.0, None, d, d)
            R.check(self.z[s], z, z_tol, "Z")
            R.check(self.a[s], a, a_tol, "hidden")
            y, tol, _, _ = R.forward(self.a[s], self.w2[i].t(), 1.0, self.b2[i], 161, 1.0, self.x[s], d, d)
            R.check(self.y[s], y, tol, "Y")
            total = self.g[s].double().sum(0)
            R.check(self.db2[i], total, R.stored(total, (hi - lo + 8) * 2.0 ** -24 * self.g[s].double().abs().sum(0), d), "db2")
            c, tol, total, t_tol = R.backward(self.g[s], self.w2[i], 1.0, 0.0, None, self.act, self.z[s], d)
            R.check(self.da[s], c, tol, "dZ")
            R.check(self.db1[i], total, t_tol, "db1")
            c, tol, _, _ = R.backward(self.da[s], self.w1[i], 1.0, 1.0, self.g[s], 161, None, d)
            R.check(self.dx[s], c, tol, "dX")
            for got, p, q in ((self.dw2[i], self.g[s], self.a[s]), (self.dw1[i], self.da[s], self.x[s])):
                want, mag = R.product(p.t(), q, 1.0)
                R.check(got, want, R.stored(want, R.sum_error(hi - lo, d) * mag, torch.float32), "dW")
        for t in (self.z, self.a, self.y, self.da, self.dx):
            assert (t[self.used:] == 9.0).all(), "padding was written"
        empty = torch.tensor([lo == hi for lo, hi in self.spans], device="cuda")
        assert (self.dw1[empty] == 0).all() and (self.update[empty] == 0).all() and (self.db1[empty] == 0).all()

    def whole(self):
        """The same step by 64-bit automatic differentiation, from the inputs alone."""
        torch = self.torch
        leaf = lambda t: t.double().clone().requires_grad_()
        x, w1, w2, b1, b2 = leaf(self.x), leaf(self.w1), leaf(self.w2), leaf(self.b1), leaf(self.b2)
        loss = 0.0
        for i, (lo, hi) in enumerate(self.spans):
            s = slice(lo, hi)
            a = R.value(self.act, x[s] @ w1[i].t() + b1[i])
            loss = loss + ((a @ w2[i].t() + b2[i] + x[s]) * self.g[s].double()).sum()
        return torch.autograd.grad(loss, [x, w1, w2, b1, b2])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("act", [163, 164, 165])
def test_training_step_of_experts(cuda, dtype, act):
    torch = cuda
    e = Experts(torch, [70, 0, 33, 1, 160], 270, 136, 264, getattr(torch, dtype), act)
    e.step(torch.cuda.current_stream())
    torch.cuda.synchronize()
    e.check()
    # The whole chain, in Frobenius norms with u the rounding. Z is off by u |Z|, which changes a slope by at most
    # 1.2 u |Z|; entries of Z are about 1 and below 4, so dZ is off by at most (1 + 1.2 * 4) u relative. Hidden values
    # are off by (1.2 + 1) u. A product of either with an exact operand of independent entries keeps the ratio of norms
    # and adds one rounding: below 8 u.
    u = R.STEP[getattr(torch, dtype)]
    dx, dw1, dw2, db1, db2 = e.whole()
    for got, want in ((e.dx[:e.used], dx[:e.used]), (e.dw1, dw1), (e.dw2, dw2), (e.db1, db1), (e.db2, db2)):
        assert (got.double() - want).norm() <= 8 * u * want.norm()
    # Orthogonal directions: the polynomial's extremes keep saturated singular values in [0.68, 1.203]. Group 0 has 70
    # rows, so 70 directions, the larger half of which are far above 3.4445^-5.
    sv = torch.linalg.svdvals(e.update[0].double())
    assert sv[0] < 1.25 and (sv[:35] > 0.6).all()
    healthy()


def test_gradients_against_differences(cuda):
    """A dense block in single precision: gradients from the kernels against central differences of its 64-bit loss.

    The differences have a relative error of h^2 and 2^-52 / h, below 1e-8 at h = 1e-5 times the third derivative. The
    gradients are off by at most 2^-20 + (k + 8) 2^-24 of sum |a||b| per product, 2^-19 per slope; three products
    follow one another, and |slope| <= 1.2."""
    torch = cuda
    rows, n, h = 37, 72, 136
    x, w1, w2 = randn(torch, 1, (rows, n), torch.float32), randn(torch, 2, (h, n), torch.float32, n ** -0.5), randn(torch, 3, (n, h), torch.float32, h ** -0.5)
    b1, b2, g = randn(torch, 4, (h,), torch.float32, 0.1), randn(torch, 5, (n,), torch.float32, 0.1), randn(torch, 6, (rows, n), torch.float32)
    stream = torch.cuda.current_stream()
    for act in (163, 164, 165):
        z, a, y = torch.empty(rows, h, device="cuda"), torch.empty(rows, h, device="cuda"), torch.empty(rows, n, device="cuda")
        dz, dx, db1, db2 = torch.empty_like(z), torch.empty_like(x), torch.empty_like(b1), torch.empty_like(b2)
        dw1 = torch.empty_like(w1)
        st = [
            cb.GemmEpilogue(ROW, NO, YES, rows, h, n, 1.0, x, 0, n, w1, 0, n, b1, 0, act, z, 0, h, 0.0, None, 0, h, a, 0, h, stream=stream),
            cb.GemmEpilogue(ROW, NO, YES, rows, n, h, 1.0, a, 0, h, w2, 0, h, b2, 0, 161, None, 0, n, 1.0, x, 0, n, y, 0, n, stream=stream),
            cb.ActivationGrad(rows, n, 161, g, 0, n, None, 0, n, None, 0, n, db2, 0, stream=stream),
            cb.GemmEpilogueGrad(ROW, NO, NO, rows, h, n, 1.0, g, 0, n, w2, 0, h, 0.0, None, 0, h, act, z, 0, h, dz, 0, h, db1, 0, stream=stream),
            cb.GemmEpilogueGrad(ROW, NO, NO, rows, n, h, 1.0, dz, 0, h, w1, 0, n, 1.0, g, 0, n, 161, None, 0, n, dx, 0, n, None, 0, stream=stream),
            cb.Gemm(ROW, YES, NO, h, n, rows, 1.0, dz, 0, h, x, 0, n, 0.0, dw1, 0, n, stream=stream),
        ]
        assert st == [OK] * 6
        torch.cuda.synchronize()

        def loss(x, w1, b1, b2):
            return ((R.value(act, x @ w1.t() + b1) @ w2.double().t() + b2 + x) * g.double()).sum()

        leaves = [x.double(), w1.double(), b1.double(), b2.double()]
        big = ((x.double().abs() @ w1.double().abs().t() + 1) * (g.double().abs() @ w2.double().abs()))  # of dZ's terms
        scale = [g.double().abs() + 1.2 * big @ w1.double().abs(), 1.2 * big.t() @ x.double().abs(), 1.2 * big.sum(0), g.double().abs().sum(0)]
        e = 3 * (2.0 ** -20 + (h + 8) * 2.0 ** -24) + 2 * 2.0 ** -19
        for i, got in enumerate((dx, dw1, db1, db2)):
            v = randn(torch, 20 + i, got.shape, torch.float64)
            step = 1e-5
            up, down = list(leaves), list(leaves)
            up[i], down[i] = leaves[i] + step * v, leaves[i] - step * v
            want = (loss(*up) - loss(*down)) / (2 * step)
            bound = (scale[i] * v.abs()).sum()
            assert abs((got.double() * v).sum() - want) <= (e + 1e-8) * bound, (act, i)


# ---- streams and graphs ----------------------------------------------------------------------------------------------

def make(torch, seed=0):
    return Experts(torch, [70, 0, 133, 1, 300], 520, 264, 392, torch.bfloat16, 165, seed)


def test_other_streams_and_synchronous_calls(cuda):
    torch = cuda
    a, b, c, d = make(torch), make(torch), make(torch), make(torch, 50)
    torch.cuda.synchronize()
    a.step(torch.cuda.current_stream())
    torch.cuda.synchronize()
    b.step(None)  # complete on return
    for p, q in zip(a.results, b.results):
        assert torch.equal(p, q)
    # two streams at once, several times over
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        c.step(s)
        d.step(t)
    torch.cuda.synchronize()
    for p, q in zip(a.results, c.results):
        assert torch.equal(p, q)
    d.check()
    healthy()


def test_streams_of_the_caller_order_the_work(cuda):
    """Work in front of a call on its stream is waited for, and work behind it waits."""
    torch = cuda
    e, ref = make(torch), make(torch)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    x = e.x.clone()
    e.x.fill_(float("nan"))
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        e.x.copy_(x)
        e.step(s)
        after = e.update.clone()
    ref.step(torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert torch.equal(after, ref.update) and torch.equal(e.dx, ref.dx)


def test_captured_and_replayed(cuda):
    """Two graphs of the same and of different leaves, alive together, replayed in turn and at once, with new inputs and
    new group offsets; results are those of plain calls bit for bit."""
    torch = cuda
    a, b = make(torch), make(torch, 50)
    pool = torch.cuda.Stream()
    graphs = []
    for e in (a, b, a):
        e.step(torch.cuda.current_stream())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=pool):
            e.step(torch.cuda.current_stream())
        graphs.append(graph)
    before = [[t.clone() for t in e.results] for e in (a, b)]
    for e in (a, b):
        for t in e.results:
            t.fill_(9.0)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s):
            graphs[0].replay()
        with torch.cuda.stream(t):
            graphs[1].replay()
    torch.cuda.synchronize()
    for e, want in zip((a, b), before):
        for got, w in zip(e.results, want):
            assert torch.equal(got, w)
    # new values in the same places; an eager call between two replays of the other graph over the same leaves
    a.x.copy_(randn(torch, 90, a.x.shape, a.x.dtype))
    a.offsets.copy_(torch.tensor([0, 0, 200, 333, 333, 400], device="cuda"))
    a.spans, a.used = [(0, 0), (0, 200), (200, 333), (333, 333), (333, 400)], 400
    for e in a.results:
        e.fill_(9.0)
    graphs[2].replay()
    torch.cuda.synchronize()
    a.check()
    first = [e.clone() for e in a.results]
    b.step(torch.cuda.current_stream())
    graphs[0].replay()
    torch.cuda.synchronize()
    for p, q in zip(first, a.results):
        assert torch.equal(p, q)
    for got, w in zip(b.results, before[1]):
        assert torch.equal(got, w)
    healthy()


def test_capture_of_copies_and_single_precision(cuda):
    """Calls that take scratch (operands off 16 bytes, partial sums, single precision) while a graph records."""
    torch = cuda
    rows, n, k = 65, 131, 77
    x, w = randn(torch, 1, (rows, k), torch.float16), randn(torch, 2, (n, k), torch.float16, 0.1)
    z, c, sums = (torch.zeros(rows, n, device="cuda", dtype=torch.float16) for _ in range(3))
    z.normal_()
    sums = torch.zeros(n, device="cuda", dtype=torch.float16)
    xs, ws, cs = x.float(), w.float(), torch.zeros(rows, n, device="cuda")
    m, o = randn(torch, 5, (63, 90), torch.float32), torch.zeros(63, 90, device="cuda")

    def work(stream):
        st = [cb.GemmEpilogueGrad(ROW, NO, YES, rows, n, k, 1.0, x, 0, k, w, 0, k, 0.0, None, 0, n, 164, z, 0, n, c, 0, n, sums, 0, stream=stream),
              cb.GemmEpilogue(ROW, NO, YES, rows, n, k, 1.0, xs, 0, k, ws, 0, k, None, 0, 163, None, 0, n, 0.0, None, 0, n, cs, 0, n, stream=stream),
              cb.NewtonSchulz(ROW, 63, 90, 1.0, m, 0, 90, 63 * 90, o, 0, 90, 63 * 90, 1, stream=stream),
              cb.NewtonSchulz(ROW, 63, 90, 1.0, m, 0, 90, 63 * 90, m, 0, 90, 63 * 90, 1, steps=2, coefficients=(3.0, 2.0, 1.0), stream=stream)]
        assert st == [OK] * 4

    start = m.clone()
    work(torch.cuda.current_stream())
    torch.cuda.synchronize()
    want = [t.clone() for t in (c, sums, cs, o, m)]
    m.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work(torch.cuda.current_stream())
    for t in (c, sums, cs, o):
        t.zero_()
    m.copy_(start)
    graph.replay()
    torch.cuda.synchronize()
    for got, before in zip((c, sums, cs, o, m), want):
        assert torch.equal(got, before)
    assert cb.ClearCache() == OK  # the graph keeps its scratch
    m.copy_(start)
    graph.replay()
    torch.cuda.synchronize()
    for got, before in zip((c, sums, cs, o, m), want):
        assert torch.equal(got, before)
    healthy()


def test_host_threads(cuda):
    """Several host threads, each with a stream and leaves of its own, at once: results are those of one thread alone."""
    import threading
    torch = cuda
    steps = [make(torch, 100 * i) for i in range(4)]
    alone = [make(torch, 100 * i) for i in range(4)]
    for e in alone:
        e.step(torch.cuda.current_stream())
    torch.cuda.synchronize()
    failures = []

    def work(e, i):
        try:
            stream = torch.cuda.Stream()
            for j in range(5):
                e.step(stream if i % 2 else None)  # synchronous calls among them
            stream.synchronize()
        except BaseException as error:  # noqa: BLE001
            failures.append(error)

    threads = [threading.Thread(target=work, args=(e, i)) for i, e in enumerate(steps)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures, failures
    for e, want in zip(steps, alone):
        for p, q in zip(e.results, want.results):
            assert torch.equal(p, q)
    healthy()


def test_first_calls_of_a_process_captured(cuda):
    """Nothing has to run before a capture: what the library sets up at first use can be set up while a graph records."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
from tests.test_fused_use_gpu import make
e, ref = make(torch), make(torch)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    e.step(torch.cuda.current_stream())
graph.replay()
torch.cuda.synchronize()
ref.step(torch.cuda.current_stream())
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(e.results, ref.results))
print("same")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


# ---- few vectors -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("dtype,c_dtype", [("float16", "float16"), ("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float32", "float32")])
@pytest.mark.parametrize("n,k,act,beta,off", [(1000, 4104, 165, 1.0, 0), (8, 520, 163, -0.5, 3), (4104, 64, 164, 0.0, 0), (1, 1, 162, 1.0, 1),
                                              (777, 333, 161, 2.0, 0), (2048, 2048, 162, 1.0, 8)])
def test_few_vectors(cuda, rows, dtype, c_dtype, n, k, act, beta, off):
    """Single tokens up to five, every epilogue; C in D's place; the first layer's operands at odd places."""
    torch = cuda
    dtype, c_dtype = getattr(torch, dtype), getattr(torch, c_dtype)
    xb, wb = randn(torch, 1, (off + rows * k,), dtype), randn(torch, 2, (off + n * k,), dtype, k ** -0.5)
    x, w = xb[off:].view(rows, k), wb[off:].view(n, k)
    bias, d = randn(torch, 3, (n,), dtype), randn(torch, 4, (rows, n), c_dtype)
    z, c = torch.zeros(rows, n, device="cuda", dtype=dtype), d.clone()
    stream = torch.cuda.current_stream()
    st = cb.GemmEpilogue(ROW, NO, YES, rows, n, k, 1.5, xb, off, k, wb, off, k, bias, 0, act, z, 0, n, beta, c, 0, n, c, 0, n, stream=stream)
    assert st == OK
    want, tol, zz, z_tol = R.forward(x, w.t(), 1.5, bias, act, beta, d, dtype, c_dtype)
    R.check(c, want, tol, "C")
    R.check(z, zz, z_tol, "Z")
    if c_dtype == dtype:
        zi = randn(torch, 5, (rows, n), dtype)
        g, sums = zi.clone(), torch.zeros(n, device="cuda", dtype=dtype)
        st = cb.GemmEpilogueGrad(ROW, NO, YES, rows, n, k, 1.5, xb, off, k, wb, off, k, beta, d, 0, n, act, g, 0, n, g, 0, n, sums, 0, stream=stream)
        assert st == OK
        want, tol, total, t_tol = R.backward(x, w.t(), 1.5, beta, d, act, zi if act != 161 else None, dtype)
        R.check(g, want, tol, "C of the gradient")
        R.check(sums, total, t_tol, "bias gradient")
    healthy()


# ---- far offsets -----------------------------------------------------------------------------------------------------

def test_offsets_past_32_bits(cuda):
    """Leading dimensions, strides and offsets that take element numbers past 2^32, on every matrix."""
    torch = cuda
    dtype, far = torch.bfloat16, 2 ** 32 + 8
    rows, n, k = 300, 136, 72
    ld = 2 ** 24  # the last line begins past 2^32
    buf = torch.empty(far + rows * ld, dtype=dtype, device="cuda")
    lane = lambda first, cols: buf.as_strided((rows, cols), (ld, 1), first)
    x, z, d, c = lane(far, k), lane(far + 1024, n), lane(far + 2048, n), lane(far + 4096, n)
    x.copy_(randn(torch, 1, (rows, k), dtype))
    d.copy_(randn(torch, 2, (rows, n), dtype))
    w = randn(torch, 3, (n, k), dtype, k ** -0.5)
    stream = torch.cuda.current_stream()
    st = cb.GemmEpilogue(ROW, NO, YES, rows, n, k, 1.0, buf, far, ld, w, 0, k, None, 0, 165, buf, far + 1024, ld, 1.0, buf, far + 2048, ld,
                         buf, far + 4096, ld, stream=stream)
    assert st == OK
    want, tol, zz, z_tol = R.forward(x, w.t(), 1.0, None, 165, 1.0, d, dtype, dtype)
    R.check(c, want, tol, "C")
    R.check(z, zz, z_tol, "Z")
    sums = torch.zeros(n, device="cuda", dtype=dtype)
    st = cb.ActivationGrad(rows, n, 165, buf, far + 2048, ld, buf, far + 1024, ld, buf, far + 4096, ld, sums, 0, stream=stream)
    assert st == OK
    want, tol, total, t_tol = R.gradient(d.double(), torch.zeros_like(d, dtype=torch.float64), 165, z, dtype)
    R.check(c, want, tol, "DZ")
    R.check(sums, total, t_tol, "bias gradient")
    # operands off 16 bytes, which are copied first
    st = cb.GemmEpilogueGrad(ROW, NO, YES, rows, n, k - 1, 1.0, buf, far + 1, ld, w, 1, k, 0.0, None, 0, ld, 161, None, 0, ld, buf, far + 4097,
                             ld, None, 0, stream=stream)
    assert st == OK
    want, tol, _, _ = R.backward(x[:, 1:], w[:, 1:].t(), 1.0, 0.0, None, 161, None, dtype)
    R.check(lane(far + 4097, n), want, tol, "C")
    # weights and weight gradients whose groups lie more than 2^31 elements apart
    G, stride = 3, 2 ** 31 + 8
    off = torch.tensor([0, 100, 100, 300], dtype=torch.int64, device="cuda")
    wide = buf.as_strided((G, n, k), (stride, k, 1), 0)
    x0 = x.contiguous()
    y0 = d.contiguous()
    wide.copy_(randn(torch, 4, (G, n, k), dtype, k ** -0.5))
    y = torch.empty(rows, n, device="cuda", dtype=dtype)
    st = cb.GemmGrouped(YES, G, rows, n, k, 1.0, x0, 0, k, buf, 0, k, stride, off, None, 0, n, 161, None, 0, n, 0.0, None, 0, n, y, 0, n,
                        stream=stream)
    assert st == OK
    for i, (lo, hi) in enumerate(((0, 100), (100, 100), (100, 300))):
        want, tol, _, _ = R.forward(x0[lo:hi], wide[i].t(), 1.0, None, 161, 0.0, None, dtype, dtype)
        R.check(y[lo:hi], want, tol, "grouped C")
    st = cb.GemmGroupedWeight(G, rows, n, k, 1.0, y0, 0, n, x0, 0, k, off, 0.0, buf, 0, k, stride, stream=stream)
    assert st == OK
    for i, (lo, hi) in enumerate(((0, 100), (100, 100), (100, 300))):
        want, mag = R.product(y0[lo:hi].t(), x0[lo:hi], 1.0)
        R.check(wide[i], want, R.stored(want, R.sum_error(hi - lo, dtype) * mag, dtype), "weight gradient")
    healthy()


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_many_vectors(cuda, dtype):
    """More vectors than a grid has rows of blocks: products, their gradients and the sums over all vectors. Values are
    small integers, so that sums over four million of them are exact in single precision below 2^24."""
    torch = cuda
    dtype = getattr(torch, dtype)
    rows, n, k = 4_300_000, 8, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(-1, 2, (rows, k), generator=g, device="cuda").to(dtype)
    w = torch.randint(-1, 2, (n, k), generator=g, device="cuda").to(dtype)
    c, sums = torch.zeros(rows, n, device="cuda", dtype=dtype), torch.zeros(n, device="cuda", dtype=dtype)
    stream = torch.cuda.current_stream()
    want = x.double() @ w.double().t()
    total = want.sum(0)
    assert cb.GemmEpilogue(ROW, NO, YES, rows, n, k, 1.0, x, 0, k, w, 0, k, None, 0, 162, None, 0, n, 0.0, None, 0, n, c, 0, n, stream=stream) == OK
    assert torch.equal(c.double(), want.clamp(min=0))
    assert cb.GemmEpilogueGrad(ROW, NO, YES, rows, n, k, 1.0, x, 0, k, w, 0, k, 0.0, None, 0, n, 161, None, 0, n, c, 0, n, sums, 0, stream=stream) == OK
    assert torch.equal(c.double(), want) and torch.equal(sums, total.to(dtype))
    sums.zero_()
    assert cb.ActivationGrad(rows, n, 161, c, 0, n, None, 0, n, None, 0, n, sums, 0, stream=stream) == OK
    assert torch.equal(sums, total.to(dtype))
    if dtype == torch.float16:
        off = torch.tensor([0, 1, 1, 4_000_000, rows], dtype=torch.int64, device="cuda")
        y = torch.zeros_like(c)
        wg = torch.stack([w, -w, w, -w])
        assert cb.GemmGrouped(YES, 4, rows, n, k, 1.0, x, 0, k, wg, 0, k, n * k, off, None, 0, n, 161, None, 0, n, 0.0, None, 0, n, y, 0, n,
                              stream=stream) == OK
        want[4_000_000:] *= -1
        assert torch.equal(y.double(), want)
        dw = torch.zeros(4, n, k, device="cuda")
        assert cb.GemmGroupedWeight(4, rows, n, k, 1.0, y, 0, n, x, 0, k, off, 0.0, dw, 0, k, n * k, stream=stream) == OK
        for i, (lo, hi) in enumerate(((0, 1), (1, 1), (1, 4_000_000), (4_000_000, rows))):
            exact = y[lo:hi].double().t() @ x[lo:hi].double()
            bound = R.sum_error(hi - lo, dtype) * (y[lo:hi].double().abs().t() @ x[lo:hi].double().abs())
            R.check(dw[i], exact, R.stored(exact, bound, torch.float32), "weight gradient")
    healthy()


def test_leading_dimension_of_a_single_line(cuda):
    """Of a matrix with one line the leading dimension is never walked, however large."""
    torch = cuda
    n, k, far = 136, 72, 2 ** 40
    x, w = randn(torch, 1, (1, k), torch.float16), randn(torch, 2, (n, k), torch.float16, k ** -0.5)
    z, c, sums = randn(torch, 3, (1, n), torch.float16), torch.zeros(1, n, device="cuda", dtype=torch.float16), torch.zeros(n, device="cuda", dtype=torch.float16)
    stream = torch.cuda.current_stream()
    want, tol, total, t_tol = R.backward(x, w.t(), 1.0, 0.0, None, 165, z, torch.float16)
    for bias_grad in (sums, None):
        c.zero_()
        assert cb.GemmEpilogueGrad(ROW, NO, YES, 1, n, k, 1.0, x, 0, far, w, 0, k, 0.0, None, 0, n, 165, z, 0, far, c, 0, far, bias_grad, 0,
                                   stream=stream) == OK
        R.check(c, want, tol, "C")
    R.check(sums, total, t_tol, "bias gradient")
    healthy()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("act", [162, 163, 164, 165])
def test_limits_of_activations(cuda, dtype, act):
    """At infinities and the type's largest numbers: the value tends to z and 0, the slope to 1 and 0; NaN stays NaN."""
    torch = cuda
    dtype = getattr(torch, dtype)
    most = torch.finfo(dtype).max
    z = torch.tensor([[float("inf"), most, 1e4, 100.0, float("-inf"), -most, -1e4, -100.0, float("nan"), 0.0]], device="cuda", dtype=dtype)
    n, stream = z.numel(), torch.cuda.current_stream()
    one, dy, dz, c = torch.ones(1, 1, device="cuda", dtype=dtype), torch.ones_like(z), torch.zeros_like(z), torch.zeros_like(z)
    assert cb.ActivationGrad(1, n, act, dy, 0, n, z, 0, n, dz, 0, n, None, 0, stream=stream) == OK
    assert (dz[0, :4] == 1).all() and (dz[0, 4:8] == 0).all() and torch.isnan(dz[0, 8]) and dz[0, 9] == (0.0 if act == 162 else 0.5)
    assert cb.GemmEpilogue(ROW, NO, NO, 1, n, 1, 1.0, one, 0, 1, z, 0, n, None, 0, act, None, 0, n, 0.0, None, 0, n, c, 0, n, stream=stream) == OK
    assert torch.equal(c[0, :4], z[0, :4]) and (c[0, 4:8] == 0).all() and torch.isnan(c[0, 8]) and c[0, 9] == 0


# ---- refusals --------------------------------------------------------------------------------------------------------

def test_refused_on_a_device(cuda):
    """Buffers that are too small, that meet, or that live elsewhere: refused, and nothing is written."""
    torch = cuda
    rows, n, k = 16, 32, 24
    half = lambda *shape: torch.zeros(*shape, device="cuda", dtype=torch.float16)
    far = 2 ** 40  # past any allocation
    big = torch.zeros(8 << 20, device="cuda", dtype=torch.float16)
    x, w, c = half(rows, k), half(n, k), half(rows, n).fill_(5.0)
    z, d = half(rows, n), half(rows, n)
    stream = torch.cuda.current_stream()

    def forward(c_buf=c, c_off=0, z_buf=z, z_off=0, d_buf=d, d_off=0, x_buf=x, bias=None, bias_off=0, ld=n, beta=1.0):
        return cb.GemmEpilogue(ROW, NO, YES, rows, n, k, 1.0, x_buf, 0, k, w, 0, k, bias, bias_off, 161, z_buf, z_off, ld, beta, d_buf, d_off, ld,
                               c_buf, c_off, ld, stream=stream)

    end = big.numel()
    assert forward(c_buf=big, c_off=end - rows * n) == OK
    assert forward(c_buf=big, c_off=far) == S.kInsufficientMemoryC
    assert forward(z_buf=big, z_off=far) == S.kInsufficientMemoryC
    assert forward(bias=big, bias_off=end - n) == OK
    assert forward(bias=big, bias_off=far) == S.kInsufficientMemoryX
    assert forward(z_buf=c) == S.kInvalidMatrixC       # two results in one place
    assert forward(c_buf=big, z_buf=big, z_off=8) == S.kInvalidMatrixC
    assert forward(c_buf=big, d_buf=big, d_off=8) == S.kInvalidMatrixC
    assert forward(c_buf=big, x_buf=big) == S.kInvalidMatrixC
    assert forward(z_buf=big, x_buf=big) == S.kInvalidMatrixC
    assert forward(z_buf=z, d_buf=z) == S.kInvalidMatrixC
    assert forward(c_buf=big, bias=big) == S.kInvalidMatrixC
    assert forward(c_buf=big, c_off=0, z_buf=big, z_off=64, d_buf=big, d_off=128, ld=192) == OK  # columns of the same lines
    assert forward(d_buf=big, c_buf=big) == OK         # D in C's place
    assert (c == 0).all()
    c.fill_(5.0)

    def gradient(c_buf=c, z_buf=z, d_buf=None, sums=None, sums_off=0):
        return cb.GemmEpilogueGrad(ROW, NO, YES, rows, n, k, 1.0, x, 0, k, w, 0, k, 0.0 if d_buf is None else 1.0, d_buf, 0, n, 163, z_buf, 0, n,
                                   c_buf, 0, n, sums, sums_off, stream=stream)

    assert gradient(sums=big, sums_off=far) == S.kInsufficientMemoryY
    assert gradient(sums=c) == S.kInvalidVectorY
    assert gradient(sums=z) == S.kInvalidVectorY
    assert gradient(c_buf=z, z_buf=z, sums=big) == OK
    off = torch.tensor([0, 4, 16], dtype=torch.int64, device="cuda")
    wg = half(2, n, k)

    def experts(offsets=off, c_buf=c, stride=n * k, G=2, x_buf=x, w_buf=wg):
        return cb.GemmGrouped(YES, G, rows, n, k, 1.0, x_buf, 0, k, w_buf, 0, k, stride, offsets, None, 0, n, 161, None, 0, n, 0.0, None, 0, n,
                              c_buf, 0, n, stream=stream)

    assert (c == 5.0).all()
    assert experts(c_buf=big, w_buf=big) == S.kInvalidMatrixC
    assert experts(c_buf=big, x_buf=big) == S.kInvalidMatrixC
    assert experts(offsets=torch.zeros_like(off)) == OK  # every group empty
    assert (c == 5.0).all()
    weights = lambda c_buf, stride, x_buf=x: cb.GemmGroupedWeight(2, rows, k, k, 1.0, x_buf, 0, k, x, 0, k, off, 0.0, c_buf, 0, k, stride, stream=stream)
    assert weights(big, k * k - 1) == S.kInvalidDimension
    assert weights(big, k * k, big) == S.kInvalidMatrixC
    assert weights(big, k * k) == OK
    torch.cuda.synchronize()
    with pytest.raises(ValueError):
        forward(x_buf=torch.zeros(rows, k, dtype=torch.float16))
    healthy()


@pytest.mark.parametrize("name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("coefficients,steps,kernel", [((3.0, 2.0, 1.0), 2, "newton_schulz_single"), ((70.0, 0.0, 0.0), 1, "newton_schulz_single"),
                                                       ((0.5, 0.0, 5000.0), 1, "newton_schulz_single"), ((1.5, 0.25, 0.125), 2, None),
                                                       ((60.0, 0.0, 0.0), 1, None), ((0.0, 3.0, 0.0), 1, None)])
def test_newton_schulz_with_other_coefficients(cuda, name, coefficients, steps, kernel):
    """No coefficient negative: the relative error grows by at most 5 a step (s p'(s) / p(s) <= 5) and a step adds at most
    8 roundings, so two steps stay within 8 * 6 of them. 2^-20 in single precision, 2^-11 for the halves, and the stored
    type's own rounding. Which kernels run follows from the largest value that the polynomial can reach."""
    torch = cuda
    dtype = getattr(torch, name)
    m, n = 100, 136
    a = randn(torch, 1, (2, m, n), dtype)
    b = torch.zeros_like(a)
    st = cb.NewtonSchulz(ROW, m, n, 0.5, a, 0, n, m * n, b, 0, n, m * n, 2, steps=steps, coefficients=coefficients,
                         stream=torch.cuda.current_stream())
    assert st == OK
    assert cb.last_kernel().startswith(kernel or ("newton_schulz_parts" if name == "float32" else "fused"))
    x = a.double() / (a.double().norm(dim=(1, 2), keepdim=True) + 1e-7)
    for _ in range(steps):
        g = x @ x.mT
        x = coefficients[0] * x + (coefficients[1] * g + coefficients[2] * g @ g) @ x
    rounding = 2.0 ** -20 if kernel or name == "float32" else 2.0 ** -11
    for i in range(2):
        assert (b[i].double() - 0.5 * x[i]).norm() <= (48 * rounding + R.STEP[dtype]) * 0.5 * x[i].norm()
    healthy()
