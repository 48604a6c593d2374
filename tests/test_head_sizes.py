"""The query head's workspaces and kernels by size, on the CPU."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

L = fg.lib
F32, BF16 = 0, 1


@pytest.mark.parametrize("nq,nc", [(65536, 10_000_000), (1 << 20, 1 << 23), (1 << 20, 1 << 30), (1, 1 << 30), (40, 1 << 30)])
@pytest.mark.parametrize("dim", [136, 768])
def test_loss_workspace_does_not_grow_with_the_scores(nq, nc, dim):
    """A row's constants and at most 512 MB of parts (a row's few of them rounded up to whole tiles)."""
    assert 0 < L.fgpu_contrastive_loss_workspace_bytes(nq, nc, dim, BF16) <= (1 << 29) + (1 << 26)


def test_more_results_than_one_launch_are_refused():
    """No tile's grid fits (arrays of a terabyte): refused before anything is launched."""
    assert L.fgpu_linear(1 << 20, 1 << 20, None, None, 1 << 30, 8, 1 << 16, BF16, 0, 1 << 20, None, None, 0, None) == 2
