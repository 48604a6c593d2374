"""The orthogonalisation of an update against its definition in 64 bits.

Each step's X is off by what its products' operands and sums lose: operands 2^-22 (two planes), a float32 sum of k products
about sqrt(k) u (u = 2^-24, roundings of either sign), taken three times over, each times the magnitudes that enter: (|a| s +
|b| s^3 + |c| s^5) <= 16 |X| for singular values s up to 1.2.  A step hands an error on at most L = 3.4445 times (the largest
slope of a s + b s^3 + c s^5 on [0, 1.21]).  So the result is off, in the Frobenius norm, by at most the sum over the steps i
of 16 (2^-22 + 3 sqrt(k) u) |X_i| L^(steps - 1 - i), |X_i| from the definition; a result in bfloat16 adds 2^-8 of itself."""
import math

import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
COEF = (3.4445, -4.7750, 2.0315)


def rnd(seed, *shape, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def steps64(x, steps, coef=COEF, eps=1e-7):
    """All the X_i, of the shorter side first."""
    x = x.double().cpu()
    x = (x / (x.norm() + eps)).cuda()
    x = x.t().contiguous() if x.shape[0] > x.shape[1] else x
    every = [x]
    a, b, c = coef
    for _ in range(steps):
        g = x @ x.t().contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
        every.append(x)
    return every


def check(x, steps=5, dt="f32", got=None):
    y = fg.orthogonalize(x, steps=steps) if got is None else got
    assert y.dtype == x.dtype and y.shape == x.shape
    every = steps64(x, steps)
    k = max(x.shape)
    each = 16 * (2.0**-22 + 3 * math.sqrt(k) * U)
    bound = sum(each * every[i].norm().item() * 3.4445**(steps - 1 - i) for i in range(steps))
    want = every[-1].t() if x.shape[0] > x.shape[1] else every[-1]
    bound += (2.0**-8 if dt == "bf16" else U) * want.norm().item()
    off = (y.double() - want).norm().item()
    assert off <= bound, (x.shape, dt, off, bound, want.norm().item())


# One of everything, both orders, around the tiles, odd strides, long ones whose products are split.
SIZES = [(1, 1), (1, 40), (40, 1), (2, 3), (8, 8), (33, 33), (64, 64), (65, 200), (200, 65), (128, 771), (771, 128), (130, 1030),
         (300, 257), (257, 300), (64, 5000), (5000, 64), (520, 520), (1024, 1040), (9, 20000), (20000, 9), (2048, 520)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", SIZES)
def test_orthogonalize(m, n, dt):
    check(rnd(m + n, m, n, scale=1e-3, dtype=TYPES[dt]), dt=dt)


# A step in two launches and in three, of sides around both bounds and the waves' parts; rows of planes apart and not.
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(1, 8192), (8192, 1), (16, 8193), (31, 100), (32, 33), (97, 97), (96, 97), (97, 96), (101, 96),
                                 (127, 1024), (128, 128), (128, 1025), (129, 200), (200, 129), (65, 1600), (1600, 65), (64, 2048),
                                 (256, 1024), (1024, 256), (256, 1032), (192, 192)])
@pytest.mark.parametrize("steps", [1, 3, 5])
def test_few_launches(m, n, dt, steps):
    check(rnd(m * n + steps, m, n, dtype=torch.float32 if dt == "f32" else torch.bfloat16), steps=steps, dt=dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(96, 400), (400, 96), (256, 256)])
@pytest.mark.parametrize("power", [0.5, 1.0, 2.0])
def test_spectra(m, n, power, dt):
    """Singular values that fall off: what the steps multiply most is what a rounding reaches first."""
    s = min(m, n)
    q, _ = torch.linalg.qr(rnd(1, m, s).double().cpu())
    v, _ = torch.linalg.qr(rnd(2, n, s).double().cpu())
    x = (q * torch.arange(1, s + 1).double()**-power) @ v.t()
    check(x.to(TYPES[dt]).cuda(), dt=dt)


def test_singular_values_are_drawn_to_one():
    """From 64 x 200 normal numbers, whose singular values lie within a factor of about four, five steps bring all of them
    into [0.6, 1.25]: the map's image of [0.05, 1] after five steps."""
    y = fg.orthogonalize(rnd(3, 64, 200))
    s = torch.linalg.svdvals(y.double().cpu())
    assert s.min() > 0.6 and s.max() < 1.25


@pytest.mark.parametrize("steps", [1, 2, 3, 6, 9])
def test_steps(steps):
    check(rnd(5, 70, 100), steps=steps)
    check(rnd(5, 100, 70), steps=steps)


def test_other_coefficients():
    """The classic cubic and quintic maps, on singular values below one, which stay below one."""
    x = rnd(6, 50, 90)
    for coef in ((1.5, -0.5, 0.0), (1.875, -1.25, 0.375)):
        want = steps64(x, 8, coef)[-1]
        y = fg.orthogonalize(x, steps=8, coefficients=coef)
        assert (y.double() - want).norm() <= 1e-4 * want.norm()


@pytest.mark.parametrize("scale", [1e-30, 1e-10, 1.0, 1e10, 1e36])
def test_any_scale(scale):
    """float32 over its range: with eps zero the result does not depend on the scale beyond the roundings of x itself."""
    x = rnd(7, 60, 80)
    y = fg.orthogonalize((x.double() * scale).float(), eps=0.0)
    want = steps64(x, 5, eps=0.0)[-1]
    assert (y.double() - want).norm() <= 2e-4 * want.norm()


def test_eps_of_tiny_updates():
    x = rnd(8, 30, 40, scale=1e-9)
    want = steps64(x, 5, eps=1e-7)[-1]
    assert (fg.orthogonalize(x).double() - want).norm() <= 2e-4 * want.norm()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_zero_and_not_finite(dt):
    x = torch.zeros((40, 70), dtype=TYPES[dt], device="cuda")
    assert torch.equal(fg.orthogonalize(x), x) and torch.equal(fg.orthogonalize(x, eps=0.0), x)
    for bad in (math.nan, math.inf):
        x = rnd(1, 40, 70, dtype=TYPES[dt])
        x[3, 5] = bad
        assert torch.isnan(fg.orthogonalize(x)).all()
    assert fg.orthogonalize(x[:0]).shape == (0, 70) and fg.orthogonalize(x[:, :0]).shape == (40, 0)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_views_in_place_and_beside(dt):
    t = TYPES[dt]
    wide = rnd(1, 50, 100, dtype=t)
    x = wide[:, 13:86]
    y = fg.orthogonalize(x)
    assert torch.equal(y, fg.orthogonalize(x.contiguous()))
    tt = rnd(2, 73, 50, dtype=t).t()
    assert torch.equal(fg.orthogonalize(tt), fg.orthogonalize(tt.contiguous()))
    hold = torch.full((50 * 73 + 64,), 7.0, dtype=t, device="cuda")
    out = hold[32:32 + 50 * 73].view(50, 73)
    assert torch.equal(fg.orthogonalize(x, out=out), y)
    assert (hold[:32] == 7).all() and (hold[32 + 50 * 73:] == 7).all()
    z = x.contiguous()
    assert torch.equal(fg.orthogonalize(z, out=z), y)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(70, 100), (128, 3000), (3000, 128)])
def test_same_bits_on_another_stream_and_replayed(m, n, dt):
    x = rnd(1, m, n, dtype=TYPES[dt])
    first = fg.orthogonalize(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = fg.orthogonalize(x, stream=side)
    side.synchronize()
    assert torch.equal(first, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fg.orthogonalize(x)
    for k in range(3):
        x.copy_(rnd(100 + k, m, n, dtype=TYPES[dt]))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, fg.orthogonalize(x))
