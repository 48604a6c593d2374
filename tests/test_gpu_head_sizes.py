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


def was_ones(*shape, dtype):
    """A freed block of ones, which the next tensor of the same size gets."""
    torch.ones(shape, dtype=dtype, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_queries_many_candidates(dtype):
    """An empty batch's gradients are zeros whatever their size (2^28 elements and more; 1 to 15 bytes past a multiple of 16)."""
    for nc, dim in (((1 << 21) + 1, 129), ((1 << 21) + 3, 128), (3, 1), (7, 1), (1, 1)):
        q = torch.empty((0, dim), dtype=dtype, device="cuda")
        c, none = torch.empty((nc, dim), dtype=dtype, device="cuda"), torch.empty(0, device="cuda")
        torch.cuda.empty_cache()
        was_ones(nc, dim, dtype=dtype)
        dq, dc, db = fg.contrastive_loss_backward(none, q, c, none.to(torch.int32), none)
        assert dq.shape == q.shape and dc.shape == c.shape and not dc.any() and not db.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows_large_weight(dtype):
    n, k = 1 << 16, 4099
    dy, x = torch.empty((0, n), dtype=dtype, device="cuda"), torch.empty((0, k), dtype=dtype, device="cuda")
    w = torch.empty((n, k), dtype=dtype, device="cuda")
    torch.cuda.empty_cache()
    was_ones(n, k, dtype=dtype)
    _, dw, db = fg.linear_backward(dy, x, w)
    assert not dw.any() and not db.any()


def test_zeros_stop_where_the_array_does():
    """Arrays that begin and end anywhere: what surrounds them stays."""
    for count in (1, 7, 8, 9, 2047, 4099):
        for dtype, code, first in ((torch.bfloat16, 1, 1), (torch.float32, 0, 3)):
            buf = torch.ones(count + 16, dtype=dtype, device="cuda")
            at = buf.data_ptr() + first * buf.element_size()
            assert fg.lib.fgpu_contrastive_loss_backward(None, None, None, None, None, None, None, 0, count, 1, code, 1.0,
                                                         None, at, None, None, 0, None) == 0
            torch.cuda.synchronize()
            assert buf[:first].all() and buf[first + count:].all() and not buf[first:first + count].any()
