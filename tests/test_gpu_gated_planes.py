"""The gated layer's float32 products one term at a time, in every tile: operands with one entry a row that is not zero, so that
each result is one product (or of two factors one each) of two float32, whatever else the sum holds being zeros.

u = 2^-24.  x = h + m + l in three bf16, |m| < 2^-7 and |l| <= 2^-16 of x's power of two, so the three plane products that are
left out are at most 2 2^-23 + 2^-32 of a product: 4 u.  The six that are kept are summed by the matrix instruction, whose sums
are off by less than a last place rather than half of one: of -0x1.01e8e8p-1 times -0x1.09fafap-1 the six are 3.49 u short of the
product and come out another 1.73 u short, where a last place is 1.91 u and six sums each rounded to the nearest would be 0.18 u
off.  So 2 u for the last sum and 2^-5 of that for those before it, whose terms are below 2^-5: a product is good to 6.1 u.  One
that lost a third plane would be off by 2^-16 of it, 256 u."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0**-24
ONE = 6.1 * U  # of a product of two float32
SPLIT = 2048  # FGPU_TILE_SPLIT
PAIR = 1024  # FGPU_TILE_PAIR


def rnd(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def one_a_row(m, k, seed):
    """([m][k] with one normal number a row, its columns)"""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    at = torch.randint(k, (m,), generator=g, device="cuda")
    x = torch.zeros((m, k), device="cuda")
    x[torch.arange(m, device="cuda"), at] = rnd(seed + 1, m)
    return x, at


FORWARD = [(70, 200, 100), (300, 77, 260), (1500, 200, 999), (960, 643, 577), (5000, 600, 2050), (4555, 291, 1556),
           (4000, 1024, 2048)]


@pytest.mark.parametrize("m,k,n", FORWARD)
def test_forward(m, k, n):
    x, at = one_a_row(m, k, 1)
    w = rnd(3, 2 * n, k)
    h, pre = fg.gated_linear(x, w, act="none", save_pre=True)
    z = x.double().sum(1, keepdim=True) * w.double().t()[at]
    assert ((pre.double() - z).abs() <= ONE * z.abs()).all()
    want = z[:, :n] * z[:, n:]
    assert ((h.double() - want).abs() <= (2 * ONE + 1.1 * U) * want.abs() + 2.0**-140).all()


def test_forward_sizes_take_every_kernel():
    assert {fg.lib.fgpu_gated_linear_tile(*s, 0) for s in FORWARD} == {0, SPLIT + 64, SPLIT + 128, 256}


BACKWARD = [(40, 30, 20), (70, 200, 100), (4099, 771, 96), (3000, 700, 1030), (100, 2050, 3000), (20000, 2050, 33)]


@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("m,k,n", BACKWARD)
def test_backward(m, k, n, half):
    """act none and the gate's or the other factor's values zero: one half of dz is dh times the other's, the other half zero.  dh
    has one entry a row, so dx has one term; dw's rows as many as rows of dh share their column: those of one are
    looked at.  dz is off by u."""
    dh, at = one_a_row(m, n, 5)
    x, w, pre = rnd(7, m, k), rnd(8, 2 * n, k), rnd(9, m, 2 * n)
    pre[:, half * n:(half + 1) * n] = 0
    dx, dw, db = fg.gated_linear_backward(dh, x, w, pre, act="none")
    other = (1 - half) * n  # the factor that is there; dz's half for the factor that is not is dh times it
    rows = torch.arange(m, device="cuda")
    dz = dh[rows, at].double() * pre[rows, other + at].double()
    want = dz[:, None] * w.double()[half * n + at]
    assert ((dx.double() - want).abs() <= (ONE + 1.1 * U) * want.abs() + 2.0**-140).all()
    once = torch.bincount(at, minlength=n)[at] == 1
    got = dw[half * n + at[once]].double()
    want = dz[once, None] * x[once].double()
    assert ((got - want).abs() <= (ONE + 1.1 * U) * want.abs() + 2.0**-140).all()
    assert not dw[other:other + n].any() and not db[other:other + n].any()
    assert ((db[half * n + at[once]].double() - dz[once]).abs() <= 2 * U * dz[once].abs()).all()


def test_backward_sizes_take_tiles_of_every_form():
    seen = {fg.lib.fgpu_linear_tile(m, k, 2 * n, 0, product) for m, k, n in BACKWARD for product in (1, 2)}
    assert seen >= {64 + PAIR, 64, 256}, seen
