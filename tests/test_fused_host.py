"""Host half of the fused products, compiled with g++ against launchers that only note what they would enqueue
(tests/host): which kernel a call gets, and that it gets one."""
import itertools
import random
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "clblast_b200" / "csrc"
MAX_SMEM = 232448  # bytes that a block of this architecture may have
HALF, BF16, SINGLE = 16, 1016, 32
PLAIN, COLS, INNER = 0, 1, 2
FORMS = ["0", "1", "2", "3", "4", "5"] + [f"{v},{s}" for v in (1, 2, 3, 4) for s in (2, 4, 8)]


def compiled(tmp_path_factory, name, *sources):
    exe = tmp_path_factory.mktemp("host") / name
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", CSRC, "-I", ROOT / "include", "-I", "/usr/local/cuda/include", *sources, "-o", exe,
                    "-lpthread"], check=True)
    return exe


@pytest.fixture(scope="module")
def selection(tmp_path_factory):
    return compiled(tmp_path_factory, "fused_selection", ROOT / "tests" / "host" / "fused_selection.cpp", CSRC / "fused_host.cpp")


def call(kind, problems, m, n, k, type=BF16, c_type=None, grad=0, z=0, bias_grad=0, beta=0.0, a_mn=0, b_mn=0, tri=0, parts=0, budget=0):
    return (kind, problems, m, n, k, type, c_type or type, grad, z, bias_grad, beta, a_mn, b_mn, tri, parts, budget)


def choices(exe, calls, form=None):
    """(error, variant, split, stages, smem, grid) of each call."""
    text = "\n".join(" ".join(map(str, c)) for c in calls)
    done = subprocess.run([exe], input=text, capture_output=True, text=True, check=True, env={"B200BLAS_FUSED": form} if form else {})
    rows = [tuple(map(int, line.split())) for line in done.stdout.splitlines()]
    assert len(rows) == len(calls)
    return rows


def launched(exe, calls, form=None):
    rows = choices(exe, calls, form)
    for c, (error, variant, split, stages, smem, grid) in zip(calls, rows):
        assert error == 0 and variant >= -1 and stages >= 2 and smem <= MAX_SMEM and grid >= 1, (c, form, error, variant, split, stages, smem)
    return rows


def test_many_groups_find_a_kernel(selection):
    """Groups take shared memory from the operand ring: 128 x 256 tiles with a split have room for 191 of them."""
    launched(selection, [call(COLS, 192, 16, 30912, 4096), call(COLS, 200, 16, 38400, 4096), call(COLS, 200, 384, 40000, 4096),
                         call(COLS, 256, 384, 131072, 7168)])
    for form, groups in itertools.product(FORMS, (1, 191, 192, 1024)):
        rows = launched(selection, [call(COLS, groups, 384, 40000, 4096, z=1), call(COLS, groups, 384, 40000, 4096, c_type=SINGLE, z=1, beta=1.0),
                                    call(COLS, groups, 384, 40000, 4096, grad=1, z=1, bias_grad=1, beta=1.0),
                                    call(INNER, groups, 384, 512, 40000, c_type=SINGLE, a_mn=1, b_mn=1, beta=1.0)], form)
        if form == "1,2":  # taken where it has room
            assert all((r[1:3] == (1, 2)) == (groups <= 191) for r in rows)


def test_every_call_finds_a_kernel(selection):
    rng = random.Random(0)
    size = lambda most: max(1, int(most ** rng.random()))
    calls = []
    for _ in range(4000):
        kind = rng.choice([PLAIN, COLS, INNER])
        problems = rng.choice([1, 1, size(64)]) if kind == PLAIN else size(1024)
        yes = lambda: int(rng.random() < 0.5)
        kw = dict(type=rng.choice([HALF, BF16]), beta=rng.choice([0.0, 1.0]))
        if kind == INNER:
            kw.update(a_mn=1, b_mn=1)
        else:
            kw.update(grad=yes(), z=yes(), a_mn=yes(), b_mn=yes() if kind == PLAIN else 0)
            kw.update(bias_grad=yes() if kw["grad"] and problems == 1 or kw["grad"] and kind == COLS else 0)
        if not kw.get("grad"):
            kw.update(c_type=rng.choice([kw["type"], SINGLE]))
        calls.append(call(kind, problems, size(16384), size(65536), size(65536), **kw))
    launched(selection, calls)


def test_kernel_attributes_are_never_lowered(tmp_path_factory):
    """A kernel is launched with sizes that vary from call to call, from several threads: once a size is recorded as set,
    no other call may set a smaller one."""
    exe = compiled(tmp_path_factory, "kernel_ready", ROOT / "tests" / "host" / "kernel_ready.cpp", CSRC / "runtime_state.cpp")
    for _ in range(3):
        done = subprocess.run([exe], capture_output=True, text=True, check=True, timeout=60)
        assert done.stdout.split() == ["230000", "230000", "77"]


def test_limit_on_multiprocessors(selection):
    """No more CTAs than the SMs that the caller leaves, whatever the tiles: pairs and split tiles take several each."""
    rng = random.Random(1)
    size = lambda most: max(1, int(most ** rng.random()))
    calls = []
    for _ in range(1500):
        budget = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 33, 100, 147])
        rows = 5 + size(8192)
        calls.append(rng.choice([
            call(PLAIN, 1, size(8192), rows, size(8192), budget=budget),
            call(PLAIN, 1, size(8192), rows, size(8192), grad=1, z=1, bias_grad=1, budget=budget),
            call(COLS, size(64), size(4096), rows, size(4096), budget=budget),
            call(INNER, size(64), size(4096), size(4096), rows, c_type=SINGLE, a_mn=1, b_mn=1, budget=budget)]))
    for side in (8, 256, 1024, 4096):
        calls += [call(PLAIN, 2, side, side, 512, type=HALF, tri=1, parts=parts, budget=budget) for budget in (1, 2, 5) for parts in (0, 1)]
    for c, row in zip(calls, launched(selection, calls)):
        assert row[5] <= c[-1] or row[1] == -1, (c, row)
    for form in ("0", "4,8"):  # asked for by name and too large
        assert all(row[5] <= c[-1] or row[1] == -1 for c, row in zip(calls, launched(selection, calls, form)))


def test_sums_of_two_halves_have_one_kernel(selection):
    sides = [(8, 8), (128, 304), (512, 1000), (4096, 4096), (1000, 70000)]  # padded to eights, as the iteration keeps them
    calls = []
    for side, long in sides:
        calls += [call(PLAIN, 3, side, side, long, type=HALF, tri=1, parts=1), call(PLAIN, 3, side, side, side, type=HALF, beta=1.0, tri=1, parts=1),
                  call(PLAIN, 3, side, long, side, type=HALF, beta=1.0, parts=1), call(PLAIN, 3, long, side, side, type=HALF, beta=1.0, a_mn=1, parts=1)]
    for form in (None, *FORMS):
        assert all(row[1:3] == (2, 1) for row in launched(selection, calls, form))
