"""Newton-Schulz results line by line and block by block, under bounds from the documented roundings."""
import pytest

import clblast_b200 as cb
from tests import newton_schulz_reference as N

pytestmark = pytest.mark.gpu

ROW, COL = 101, 102
OK = cb.StatusCode.kSuccess
LAST = {"0": "fused_pair_256x256", "2": "fused_128x128", "3": "fused_128x64", "5": "fused_pair_256x128"}


def run(torch, dtype, layout, m, n, batch=1, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = torch.randn(batch, m, n, generator=gen, device="cuda").to(dtype)
    stored = g if layout == ROW else g.mT.contiguous()
    ld = stored.shape[2]
    out = torch.full_like(stored, float("nan"))
    st = cb.NewtonSchulz(layout, m, n, 1.0, stored, 0, ld, m * n, out, 0, ld, m * n, batch, stream=torch.cuda.current_stream())
    assert st == OK, st
    for i in range(batch):
        want, limit = N.allowed(g[i], dtype)
        N.check(out[i] if layout == ROW else out[i].mT, want, limit)
    code, where = cb.tensor_core_status()
    assert code == OK, where


@pytest.mark.parametrize("name", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("m,n", [(129, 300), (300, 129), (256, 520), (700, 700), (1000, 333), (1029, 2050), (2305, 1300), (2048, 2048)])
def test_entries(cuda, name, m, n):
    run(cuda, getattr(cuda, name), ROW, m, n)
    run(cuda, getattr(cuda, name), COL, m, n)


@pytest.mark.parametrize("name", ["float16", "bfloat16", "float32"])
def test_a_large_square_and_a_batch(cuda, name):
    run(cuda, getattr(cuda, name), ROW, 4096, 4096)
    run(cuda, getattr(cuda, name), ROW, 520, 1000, 4)


@pytest.mark.parametrize("v", ["0", "2", "3", "5"])
@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,n", [(600, 600), (768, 512), (264, 1000)])
def test_entries_of_every_variant(cuda, monkeypatch, v, name, m, n):
    """The tiles that are asked for serve the last product; the symmetric ones need square tiles and may have others."""
    monkeypatch.setenv("B200BLAS_FUSED", v)
    run(cuda, getattr(cuda, name), ROW, m, n, 2)
    assert cb.last_kernel().startswith(LAST[v])
