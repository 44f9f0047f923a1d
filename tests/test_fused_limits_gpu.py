"""Fused products at the limits of what their kernels hold, against the same 64-bit forms as their other tests."""
import pytest

import clblast_b200 as cb
from tests.test_fused_gpu import NO, ROW, YES, grouped, linear, weight

pytestmark = pytest.mark.gpu


def test_groups_beside_the_sums_of_split_tiles(cuda, monkeypatch):
    """192 groups and more leave 128 x 256 tiles with a split no room for two ring stages: other tiles serve the call."""
    grouped(cuda, monkeypatch, None, "bf16", "bf16", [161] * 192, 30912, 16, 4096)  # takes 128 x 256 tiles with fewer groups
    for groups in (191, 192, 1024):
        sizes = [(5 * i) % 9 for i in range(groups)]
        for v in ("1,2", "1,4"):
            grouped(cuda, monkeypatch, v, "bf16", "bf16", sizes, sum(sizes) + 3, 72, 264, first=3, beta=1.0)
            grouped(cuda, monkeypatch, v, "half", "single", sizes, sum(sizes) + 3, 72, 264, beta=1.0)
            grouped(cuda, monkeypatch, v, "half", "half", sizes, sum(sizes) + 3, 72, 264, grad=True, beta=1.0)
            weight(cuda, monkeypatch, v, "bf16", "single", sizes, sum(sizes) + 3, 72, 40, first=3, poison=True, beta=1.0)


def test_first_calls_of_threads_with_different_sizes(cuda):
    """The first calls of a process, on threads that start together and whose launches of the same kernels need different
    amounts of shared memory (with and without Z, few and many groups); then every call again."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import threading
import torch
import clblast_b200 as cb
ROW, NO, YES = 101, 111, 112
rows, n, k = 1024, 264, 128
half = lambda *shape: torch.randn(*shape, device="cuda").half()
x, w, wg = half(rows, k), half(n, k), half(1024, n, k)
z = torch.empty(rows, n, device="cuda", dtype=torch.half)
calls = []
for keep in (True, False):
    calls.append(lambda c, s, keep=keep: cb.GemmEpilogue(ROW, NO, YES, rows, n, k, 1.0, x, 0, k, w, 0, k, None, 0, 161, z if keep else None, 0, n,
                                                         0.0, None, 0, n, c, 0, n, stream=s))
for groups in (1024, 2, 300, 40):
    off = torch.linspace(0, rows, groups + 1, device="cuda").long()
    calls.append(lambda c, s, groups=groups, off=off: cb.GemmGrouped(YES, groups, rows, n, k, 1.0, x, 0, k, wg, 0, k, n * k, off, None, 0, n, 161,
                                                                     None, 0, n, 0.0, None, 0, n, c, 0, n, stream=s))
outs = [torch.empty(rows, n, device="cuda", dtype=torch.half) for _ in calls]
torch.cuda.synchronize()
start, states = threading.Barrier(len(calls)), []
def work(f, c):
    stream = torch.cuda.Stream()
    start.wait()
    states.append(int(f(c, stream)))
    stream.synchronize()
threads = [threading.Thread(target=work, args=p) for p in zip(calls, outs)]
[t.start() for t in threads]
[t.join() for t in threads]
for f, c in zip(calls, outs):
    again = torch.empty_like(c)
    states.append(int(f(again, torch.cuda.current_stream())))
    torch.cuda.synchronize()
    assert torch.equal(c, again)
assert states == [0] * (2 * len(calls)), states
print("same")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "same" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("budget", [1, 2, 5])
def test_few_multiprocessors(cuda, monkeypatch, budget):
    """A limit below what a pair or a split tile takes: tiles of one SM serve the call, one after another."""
    cb.set_sm_budget(budget)
    try:
        for v in (None, "0", "3,8"):
            linear(cuda, monkeypatch, v, "half", "half", ROW, NO, YES, 70, 264, 200, act=165, beta=0.5)
            linear(cuda, monkeypatch, v, "bf16", "bf16", ROW, NO, YES, 300, 520, 1000, act=164, grad=True, beta=1.0)
            grouped(cuda, monkeypatch, v, "bf16", "single", [3, 0, 64, 33, 0, 1, 129], 240, 264, 200, beta=1.0)
            weight(cuda, monkeypatch, v, "half", "single", [3, 0, 64, 33, 0, 1, 129], 240, 136, 264, beta=1.0)
    finally:
        cb.set_sm_budget(0)


def test_results_that_meet_the_group_offsets_are_refused(cuda):
    """Nothing is launched, and nothing written; right beside them is allowed."""
    torch = cuda
    S = cb.StatusCode
    rows, n, k, G = 64, 24, 16, 3
    table = torch.tensor([0, 10, 10, rows], dtype=torch.int64, device="cuda")
    space = torch.zeros(4096, dtype=torch.int64, device="cuda")
    half = space.view(torch.float16)  # the same memory
    x, w, z = (torch.ones(s, device="cuda", dtype=torch.float16) for s in ((rows, k), (G, n, k), (rows, n)))
    y, stream = torch.ones(rows, n, device="cuda", dtype=torch.float16), torch.cuda.current_stream()

    def grouped_(off, c, c_off=0, zz=None, z_off=0):
        return cb.GemmGrouped(YES, G, rows, n, k, 1.0, x, 0, k, w, 0, k, n * k, off, None, 0, n, 161, zz, z_off, n, 0.0, None, 0, n, c, c_off, n,
                              stream=stream)

    def gradient(off, c, c_off=0, sums=None, s_off=0):
        return cb.GemmGroupedGrad(YES, G, rows, n, k, 1.0, x, 0, k, w, 0, k, n * k, off, 0.0, None, 0, n, 165, z, 0, n, c, c_off, n, sums, s_off, n,
                                  stream=stream)

    def weight_(off, c, c_off=0):
        return cb.GemmGroupedWeight(G, rows, k, n, 1.0, x, 0, k, y, 0, n, off, 0.0, c, c_off, n, k * n, stream=stream)

    def activation(off, c, c_off=0, sums=None, s_off=0):
        return cb.ActivationGrad(rows, n, 165, y, 0, n, z, 0, n, c, c_off, n, sums, s_off, groups=G, group_offsets=off, bias_grad_ld=n,
                                 stream=stream)

    c = torch.zeros(rows, n, device="cuda", dtype=torch.float16)
    at = 2048  # where the offsets lie, counted in halves
    space[at // 4:at // 4 + G + 1] = table
    before, off = space.clone(), space[at // 4:at // 4 + G + 1]
    for c_off in (at - rows * n + 1, at, at + 4 * (G + 1) - 1):
        assert grouped_(off, half, c_off) == S.kInvalidMatrixC
        assert grouped_(off, c, 0, half, c_off) == S.kInvalidMatrixC
        assert gradient(off, half, c_off) == S.kInvalidMatrixC
        assert activation(off, half, c_off) == S.kInvalidMatrixC
    for s_off in (at - G * n + 1, at, at + 4 * (G + 1) - 1):
        assert gradient(off, c, 0, half, s_off) == S.kInvalidVectorY
        assert activation(off, c, 0, half, s_off) == S.kInvalidVectorY
        assert activation(off, None, 0, half, s_off) == S.kInvalidVectorY
    for c_off in (at - G * k * n + 1, at, at + 4 * (G + 1) - 1):
        assert weight_(off, half, c_off) == S.kInvalidMatrixC
    torch.cuda.synchronize()
    assert torch.equal(space, before)
    for c_off in (at - rows * n, at + 4 * (G + 1)):
        assert grouped_(off, half, c_off) == S.kSuccess
        assert gradient(off, c, 0, half, c_off) == S.kSuccess
        torch.cuda.synchronize()
        assert torch.equal(off, table)
    code, where = cb.tensor_core_status()
    assert code == S.kSuccess, where
