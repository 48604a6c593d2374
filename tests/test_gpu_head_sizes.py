"""The query head's operators at sizes whose work does not fit one launch (HIP counts a launch in 32 bits of threads)."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,dim", [((1 << 28) + 5, 8), ((1 << 24) + 3, 1032), ((1 << 22) + 1, 4104)])
def test_layer_norm_many_rows(rows, dim):
    """2^32 threads and more, in each arrangement of a row over lanes; in place, so that one array is enough.  Rows of
    zeros stay zeros; a few that hold something, around every power of two from 2^20 rows on, agree with the same rows
    alone."""
    x = torch.zeros((rows, dim), dtype=torch.bfloat16, device="cuda")
    at = sorted({r for p in range(20, 29) for r in ((1 << p) - 1, 1 << p) if r < rows} | {0, rows - 1})
    at = torch.tensor(at, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x[at] = torch.randn((at.numel(), dim), generator=g, device="cuda").to(torch.bfloat16)
    gain = torch.randn(dim, generator=g, device="cuda").to(torch.bfloat16)
    want, wmean, wrstd = fg.layer_norm(x[at].clone(), gain)
    y, mean, rstd = fg.layer_norm(x, gain, out=x)
    assert torch.equal(y[at], want) and torch.equal(mean[at], wmean) and torch.equal(rstd[at], wrstd)
    y[at] = 0
    assert not any(part.any() for part in y.split(1 << 22))
