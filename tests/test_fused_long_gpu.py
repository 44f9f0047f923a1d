"""Long inner extents into 16-bit results. The tensor cores cut off when they add to an accumulator; with products of one
sign that adds up, so an accumulator takes 16384 inner elements at most and the rest is added rounded. The bound is that of
the other tests for one such accumulator, (16384 / 16 + 4) * 2^-22, and half a step of fp32 for each addition of them: half
a step of half precision beside the rounding itself, whatever the extent."""
import pytest

import clblast_b200 as cb
from tests import fused_reference as R
from tests import test_fused_gpu as F

pytestmark = pytest.mark.gpu

ROW, COL, NO, YES = 101, 102, 111, 112
SUM_ERROR = R.sum_error


@pytest.fixture
def one_sign(monkeypatch):
    def positive(torch, g, shape, dtype, scale=1.0):
        return ((torch.rand(shape, generator=g, device="cuda") + 0.5) * scale).to(dtype)

    monkeypatch.setattr(F, "randn", positive)
    monkeypatch.setattr(R, "sum_error", lambda k, dtype: SUM_ERROR(min(k, 16384), dtype) + (k / 16384 + 8) * 2.0 ** -24)


FORMS = [None, "0", "1", "2", "3", "4", "5", "2,2", "1,4", "3,8"]


@pytest.mark.parametrize("v", FORMS)
def test_products(cuda, monkeypatch, one_sign, v):
    for n in (264, 259):  # 16-byte and element-wise epilogues
        F.linear(cuda, monkeypatch, v, "half", "half", ROW, NO, YES, 300, n, 131172, act=165, beta=1.0, alpha=2.0 ** -6)
        F.linear(cuda, monkeypatch, v, "half", "half", ROW, YES, NO, 300, n, 131172, grad=True, act=165, beta=1.0, alpha=2.0 ** -6)
    F.linear(cuda, monkeypatch, v, "bf16", "bf16", COL, NO, YES, 136, 72, 1048600, act=161, alpha=2.0 ** -6)


@pytest.mark.parametrize("v", ["0", "1", "2", "3,2"])
def test_several_tiles_per_cta(cuda, monkeypatch, one_sign, v):
    cb.set_sm_budget(4)
    try:
        F.linear(cuda, monkeypatch, v, "half", "half", ROW, NO, YES, 520, 776, 49200, act=165, beta=1.0, alpha=2.0 ** -6)
        F.linear(cuda, monkeypatch, v, "half", "half", ROW, NO, YES, 520, 776, 32768, act=165, alpha=2.0 ** -6)
        F.linear(cuda, monkeypatch, v, "half", "half", ROW, NO, YES, 520, 776, 16385, grad=True, act=165, alpha=2.0 ** -6)
    finally:
        cb.set_sm_budget(0)


@pytest.mark.parametrize("v", [None, "0", "1", "2", "3", "5", "2,2", "3,4"])
def test_weight_gradients(cuda, monkeypatch, one_sign, v):
    """Groups below, at and far above the limit in one call."""
    sizes = [100, 0, 131171, 16384, 1, 16385, 40000]
    F.weight(cuda, monkeypatch, v, "half", "half", sizes, sum(sizes) + 20, 136, 264, first=11, alpha=2.0 ** -8, beta=1.0)
    F.weight(cuda, monkeypatch, v, "half", "half", sizes, sum(sizes) + 20, 65, 129, first=11, alpha=2.0 ** -8)
    F.weight(cuda, monkeypatch, v, "bf16", "bf16", [0, 1048577], 1048577, 64, 72, alpha=2.0 ** -8)


@pytest.mark.parametrize("v", [None, "0", "3,4"])
def test_grouped_products(cuda, monkeypatch, one_sign, v):
    F.grouped(cuda, monkeypatch, v, "half", "half", [3, 0, 40, 131], 180, 136, 66000, act=165, beta=1.0, alpha=2.0 ** -6)
    F.grouped(cuda, monkeypatch, v, "half", "half", [3, 0, 40, 131], 180, 136, 66000, grad=True, act=165, beta=1.0, alpha=2.0 ** -6)


def test_captured_beside_another(cuda, monkeypatch, one_sign):
    """Two recorded calls and a plain one, each with sums of its own, at once; the same bits as alone."""
    torch = cuda
    monkeypatch.delenv("B200BLAS_FUSED", raising=False)
    m, n, k = 264, 520, 70000
    g = torch.Generator(device="cuda").manual_seed(0)
    operands = [(torch.rand(k, m, generator=g, device="cuda").half(), torch.rand(k, n, generator=g, device="cuda").half()) for _ in range(3)]
    outs = [torch.zeros(m, n, device="cuda", dtype=torch.half) for _ in range(3)]

    def work(i, stream):
        x, y = operands[i]
        assert cb.GemmEpilogue(ROW, YES, NO, m, n, k, 2.0 ** -8, x, 0, m, y, 0, n, None, 0, 161, None, 0, n, 0.0, None, 0, n, outs[i], 0, n,
                               stream=stream) == cb.StatusCode.kSuccess

    for i in range(3):
        work(i, torch.cuda.current_stream())
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            work(i, torch.cuda.current_stream())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        work(2, streams[2])
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(outs, want))
    code, where = cb.tensor_core_status()
    assert code == cb.StatusCode.kSuccess, where


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,n", [(64, 300000), (300000, 64)])
def test_newton_schulz_of_a_long_matrix(cuda, name, m, n):
    """The diagonal of X X^T is a sum of squares over the long side."""
    torch = cuda
    from tests.newton_schulz_reference import allowed, check
    gen = torch.Generator(device="cuda").manual_seed(0)
    g = torch.randn(m, n, generator=gen, device="cuda").to(getattr(torch, name))
    out = torch.zeros_like(g)
    assert cb.NewtonSchulz(ROW, m, n, 1.0, g, 0, n, m * n, out, 0, n, m * n, 1, stream=torch.cuda.current_stream()) == cb.StatusCode.kSuccess
    want, limit = allowed(g, g.dtype)
    check(out, want, limit)
