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


P = 1 << 20  # stands for a 16-byte-aligned device pointer: refused calls never read it


@pytest.mark.parametrize("call", [
    lambda: L.fgpu_linear(P, P, None, None, 1 << 16, 1023, 1024, BF16, 0, P, None, None, 1 << 40, None),
    lambda: L.fgpu_linear_backward(P, P, P, None, 1 << 16, 1024, 1024, F32, 0, P, P, P, None, 1 << 40, None),
    lambda: L.fgpu_layer_norm_backward(P, P, None, P, P, 4, 8, F32, P, P, None, None, 1 << 40, None),
    lambda: L.fgpu_contrastive_loss(P, P, P, None, None, 4, 8, 8, F32, 1.0, P, P, None, 1 << 40, None),
    lambda: L.fgpu_contrastive_loss_backward(P, P, P, P, P, None, None, 4, 8, 200, F32, 1.0, P, P, P, None, 1 << 40, None),
])
def test_no_workspace_whatever_its_stated_size(call):
    assert call() == 6
