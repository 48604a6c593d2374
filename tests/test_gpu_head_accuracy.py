"""What the query head's arithmetic holds beyond the bounds of a whole operator's sums: each piece alone, against 64 bits.

u = 2^-24, half a last place of float32 at most."""
import math

import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": U, "bf16": 2.0**-8}


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [70_000, 16])
def test_gelu_and_its_slope_keep_their_digits(dt, rows):
    """z Phi(z) relative to itself on the negative side as well, out to where it leaves float32's range.  The tail 1 -
    Phi(|z|): one u for its polynomial, 1.5 z^2 u for the exponential's argument (two roundings of z^2 / 2 log2 e and the
    constant's), 2 for the exponential, 4 for the reciprocal's part, 6 for the polynomial's and products' roundings: 13, and
    3 more to be safe against none; 3 u of the value for 1 - tail and the product with z."""
    t = TYPES[dt]
    z = torch.linspace(-13, 13, rows, device="cuda").to(t)[:, None].contiguous()
    one = torch.ones((1, 1), dtype=t, device="cuda")
    y, pre = fg.linear(z, one, act="gelu", save_pre=True)
    assert torch.equal(pre, z)
    zd = z.double()
    phi, tail = torch.special.erfc(-zd / math.sqrt(2)) / 2, torch.special.erfc(zd.abs() / math.sqrt(2)) / 2
    te = (16 + 1.5 * zd**2) * U * tail  # the tail's error
    want = zd * phi
    bound = zd.abs() * te + 3 * U * want.abs()
    assert ((y.double() - want).abs() <= bound + HALF[dt] * (want.abs() + bound) + 2.0**-126).all()
    # its slope Phi(z) + z exp(-z^2 / 2) / sqrt(2 pi): the density's error is the exponential's and four roundings
    dx, _, _ = fg.linear_backward(torch.ones_like(z), z, one, pre, act="gelu", want=("x",))
    dens = zd * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi)
    want = phi + dens
    bound = te + (8 + 1.5 * zd**2) * U * dens.abs() + 3 * U * (phi + dens.abs())
    assert ((dx.double() - want).abs() <= bound + HALF[dt] * (want.abs() + bound) + 2.0**-126).all()


@pytest.mark.parametrize("m,n,k", [(2, 1024, 64), (2, 100, 8), (2, 1 << 15, 2048)])
def test_bias_gradient_takes_dz_unrounded(m, n, k):
    """bfloat16: two rows whose dz nearly cancel, where dz rounded on its way to the sum would be most of the result.  dz:
    the reciprocal, exponential and products of the slope, 10 u, its sum 4 u more."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    a = (1 + torch.rand(n, generator=g, device="cuda")).bfloat16()
    z = (0.02 + 0.04 * torch.rand(n, generator=g, device="cuda")).bfloat16()
    dy, pre = torch.stack([a, -a]), torch.stack([z, (z.view(torch.int16) + 1).view(torch.bfloat16)])
    x, w = torch.randn((m, k), generator=g, device="cuda").bfloat16(), torch.randn((n, k), generator=g, device="cuda").bfloat16()
    p = pre.double()
    s = torch.sigmoid(p)
    dz = dy.double() * s * (1 + p * (1 - s))
    want, bound = dz.sum(0), 16 * U * dz.abs().sum(0)
    for names in (("x", "weight", "bias"), ("bias",)):
        db = fg.linear_backward(dy, x, w, pre, act="silu", want=names)[2].double()
        assert ((db - want).abs() <= bound + 2.0**-8 * (want.abs() + bound)).all()


@pytest.mark.parametrize("m", [1, 100, 4096])
def test_float32_products_of_one_term(m):
    """x w alone: the plane products left out are at most 4 u of it, the last addition rounds by two at most, the ones before
    by 2^-7 of that.  Among the values, those whose first eight bits leave most over, and the type's ends, where no finite
    product may become infinite."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    w = torch.randn((2048, 1), generator=g, device="cuda")
    w[:512, 0] = 1 + (65024 + torch.arange(512, device="cuda")) * 2.0**-23  # just below 1 + 2^-7
    w[512:1024, 0] = 1 + (32512 + torch.arange(512, device="cuda")) * 2.0**-23  # about half of it
    w[1024:1029, 0] = torch.tensor([3.4028235e38, -3.4028235e38, 3.3895314e38, 3.3961775e38, 2.0**-100], device="cuda")
    x = torch.cat([w[700:701], w[:1024], torch.randn((3071, 1), generator=g, device="cuda").clamp(-0.99, 0.99)])[:m].contiguous()
    want = x.double() @ w.double().t()
    keep = want.abs() <= 3.4028235e38  # the others' float32 is infinite
    y = fg.linear(x, w).double()
    assert ((y - want).abs() <= 6.1 * U * want.abs())[keep].all()
    dx, dw, _ = fg.linear_backward(x, torch.ones_like(x), w[:1], want=("x",))
    want = x.double() * w[0].double()
    assert ((dx.double() - want).abs() <= 6.1 * U * want.abs()).all() and dw is None


def rounding(v):
    """What rounding to bfloat16 takes from v."""
    return v.bfloat16().double() - v


def check_loss_gradient_error(nq, nc, dim, ids, weight, workspace=1.0):
    """bfloat16 queries half way to their targets: a target's score gradient is about as large as its row's others together,
    and no part of it may be lost.  The others are rounded, up to 2^-8 of each, with random signs: the gradients are as far
    from the exact ones, in norm, as the result's own rounding and those together, each at its most."""
    g = torch.Generator(device="cuda")
    g.manual_seed(nq + dim)
    c = torch.nn.functional.normalize(torch.randn((nc, dim), generator=g, device="cuda"))
    t = torch.randperm(nc, generator=g, device="cuda")[:nq] if nq <= nc else torch.randint(nc, (nq,), generator=g, device="cuda")
    if ids:  # some targets shared by several rows, near and far
        t[1::3] = t[0:-1:3][:t[1::3].numel()]
        t[nq // 2:nq // 2 + 5] = t[0]
        t[-1] = t[0]
    q = torch.nn.functional.normalize(0.35 * c[t] + 0.65 * torch.randn((nq, dim), generator=g, device="cuda") / dim**0.5)
    q, c, t, dl = q.bfloat16(), c.bfloat16(), t.to(torch.int32), torch.full((nq,), weight, device="cuda")
    t[::17] = -1
    loss, lse = fg.contrastive_loss(q, c, t, 20.0)
    size = int(fg.lib.fgpu_contrastive_loss_backward_workspace_bytes(nq, nc, dim, 1) * workspace)
    dq, dc, _ = fg.contrastive_loss_backward(dl, q, c, t, lse, 20.0, workspace=torch.empty(size, dtype=torch.uint8, device="cuda"))
    live, at, rows = t >= 0, t.clamp(min=0).long(), torch.arange(nq, device="cuda")
    qd, cd = q.double(), c.double()
    p = torch.softmax(20 * qd @ cd.t(), 1) * live[:, None] * weight
    hot = torch.zeros_like(p)
    hot[rows, at] = live.double() * weight
    grad = p - hot
    others = torch.where(hot > 0, 0.0, grad)
    if dim > 128:  # dc: only a target's first row
        first = torch.full((nc,), nq, device="cuda").scatter_reduce(0, at[live], rows[live], "amin")
        shared = torch.where((hot > 0) & (first[None, :] == rows[:, None]), 0.0, grad)
    else:
        shared = others
    for got, want, left, side in ((dq, grad @ cd, others, cd), (dc, grad.t() @ qd, shared.t(), qd)):
        lost = (2.0**-8 * 20 * left).square() @ side.square().sum(1)
        bound = (rounding(20 * want).square().sum() + lost.sum()).sqrt()
        assert (got.double() - 20 * want).norm() <= 1.02 * bound


@pytest.mark.parametrize("ids", [False, True])
@pytest.mark.parametrize("weight", [1 / 883, 1.0, 1 / 600])
@pytest.mark.parametrize("nq,nc,dim", [(883, 4707, 128), (1024, 1024, 96), (700, 700, 40), (3000, 30000, 61)])
def test_loss_gradients_lose_nothing_of_the_targets(nq, nc, dim, ids, weight):
    check_loss_gradient_error(nq, nc, dim, ids, weight)


@pytest.mark.parametrize("ids", [False, True])
@pytest.mark.parametrize("nq,nc,dim,weight,workspace", [
    (883, 4707, 200, 1 / 883, 1.0), (1024, 1024, 136, 1.0, 1.0), (300, 1500, 203, 1 / 600, 1.0), (3001, 30000, 256, 1 / 883, 1.0),
    (3000, 6001, 137, 1 / 600, 1.0), (1500, 2200, 768, 1.0, 1.0), (700, 9000, 200, 1 / 883, 0.7), (3000, 20000, 136, 1.0, 0.6),
    (2500, 700, 168, 1 / 883, 1.0)])
def test_wide_loss_gradients_lose_nothing_of_the_targets(nq, nc, dim, weight, workspace, ids):
    check_loss_gradient_error(nq, nc, dim, ids, weight, workspace)
