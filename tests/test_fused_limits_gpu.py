"""Fused products at the limits of what their kernels hold, against the same 64-bit forms as their other tests."""
import pytest

from tests.test_fused_gpu import grouped, weight

pytestmark = pytest.mark.gpu


def test_groups_beside_the_sums_of_split_tiles(cuda, monkeypatch):
    """192 groups and more leave 128 x 256 tiles with a split no room for two ring stages: other tiles serve the call."""
    grouped(cuda, monkeypatch, None, "bf16", "bf16", [160] * 192, 30720, 16, 4096)  # takes 128 x 256 tiles with fewer groups
    for groups in (191, 192, 1024):
        sizes = [(5 * i) % 9 for i in range(groups)]
        for v in ("1,2", "1,4"):
            grouped(cuda, monkeypatch, v, "bf16", "bf16", sizes, sum(sizes) + 3, 72, 264, first=3, beta=1.0)
            grouped(cuda, monkeypatch, v, "half", "single", sizes, sum(sizes) + 3, 72, 264, beta=1.0)
            grouped(cuda, monkeypatch, v, "half", "half", sizes, sum(sizes) + 3, 72, 264, grad=True, beta=1.0)
            weight(cuda, monkeypatch, v, "bf16", "single", sizes, sum(sizes) + 3, 72, 40, first=3, poison=True, beta=1.0)
