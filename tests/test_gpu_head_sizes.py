"""The query head's operators at sizes whose work does not fit one launch (HIP counts a launch in 32 bits of threads)."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402
from tests.test_gpu_head import check_loss, loss_inputs  # noqa: E402

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


@pytest.mark.parametrize("nq,nc,dim,dtype", [(1 << 17, (1 << 22) + 77, 136, torch.bfloat16),
                                             ((1 << 15) + 77, (1 << 19) + 300, 136, torch.float32)])
def test_contrastive_loss_many_scores(nq, nc, dim, dtype):
    """More scores than one launch takes (2^39 and 2^34), against 64 bits in a sample of the rows.  Targets, masks and copies
    lie in the first launch's columns, the last one's and between.  Bound: a score's error is (dim + 14) 2^-24 of the
    magnitudes in it; the sum's, of at most nc / 16 terms in a row of additions whose errors are of random sign, below
    sqrt(nc) 2^-24 (times 8); and a few last places of the result."""
    u = 2.0**-24
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    c = torch.empty((nc, dim), dtype=dtype, device="cuda")
    for i in range(0, nc, 1 << 20):
        c[i:i + (1 << 20)] = torch.randn((min(1 << 20, nc - i), dim), generator=g, device="cuda").to(dtype)
    q = torch.randn((nq, dim), generator=g, device="cuda").to(dtype)
    t = torch.randint(nc, (nq,), generator=g, device="cuda", dtype=torch.int32)
    rows = torch.tensor([0, 1, 2, 255, 256, 4097, nq // 2, nq - 2, nq - 1], device="cuda")
    t[rows] = torch.tensor([0, nc - 1, nc // 2, 255, 256, 1 << 17, (1 << 17) - 1, -1, nc - 300], dtype=torch.int32, device="cuda")
    ids = torch.arange(nc, device="cuda", dtype=torch.int32) % (nc - 1000)  # the first thousand's copies are the last ones
    bias = torch.randn(nc, generator=g, device="cuda")
    bias[7::1000] = -torch.inf
    scale = 1 / dim**0.5
    loss, lse = fg.contrastive_loss(q, c, t, scale, bias=bias, ids=ids)
    for r in rows.tolist():
        qd = q[r].double()
        s, mag = torch.empty(nc, dtype=torch.float64, device="cuda"), 0.0
        for i in range(0, nc, 1 << 20):
            cd = c[i:i + (1 << 20)].double()
            s[i:i + (1 << 20)] = scale * torch.mv(cd, qd)
            mag = max(mag, (scale * torch.mv(cd.abs(), qd.abs())).max().item())
        s += bias.double()
        at = t[r].item()
        if at >= 0:
            same = ids == ids[at]
            same[at] = False
            s[same] = -torch.inf
        want = torch.logsumexp(s, 0).item()
        bound = (dim + 14) * u * mag + 8 * nc**0.5 * u + 16 * u * (mag + 8)
        assert abs(lse[r].item() - want) <= bound, r
        assert abs(loss[r].item() - (want - s[at].item() if at >= 0 else 0.0)) <= (2 * bound if at >= 0 else 0.0), r


def test_linear_most_rows():
    """2^30 rows, where the smallest tiles would be 2^32 threads."""
    x = torch.zeros((1 << 30, 8), dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, 63, 64, (1 << 24) + 1, (1 << 29) - 1, 1 << 29, (1 << 30) - 1], device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x[at] = torch.randn((8, 8), generator=g, device="cuda").to(torch.bfloat16)
    flip = torch.eye(8, device="cuda").flip(0).to(torch.bfloat16)
    y = fg.linear(x, flip)
    assert torch.equal(y[at], x[at].flip(1))
    y[at] = 0
    assert not any(part.any() for part in y.split(1 << 26))


def test_contrastive_backward_chunks_many_results():
    """A query gradient of 2^26 elements and more, added up over column chunks: more joining than one grid's workgroups hold."""
    q, c, t, scale, bias, ids = loss_inputs((1 << 16) + 5, 5000, 1032, "bf16")
    full = fg.lib.fgpu_contrastive_loss_backward_workspace_bytes((1 << 16) + 5, 5000, 1032, 1)
    check_loss(q, c, t, scale, bias, ids, "bf16", workspace=torch.empty(int(full * 0.95), dtype=torch.uint8, device="cuda"))
