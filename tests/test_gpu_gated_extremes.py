"""The gated, the 8-bit and the orthogonalising operators where calls go wrong that small ones never show: rows of very many, both
workspaces of two streams at once, precision beyond what a whole operator's bound tells."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0**-24


def rnd(seed, *shape, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_very_many_rows(dt):
    """2^28 rows of one column: grids near and past what one launch counts, in every kernel that takes rows."""
    m = (1 << 28) + 5
    x = torch.ones((m, 1), dtype=dt, device="cuda")
    x[-3:, 0] = torch.tensor([2.0, -1.0, 0.0], device="cuda")
    w = torch.tensor([[2.0], [3.0]], dtype=dt, device="cuda")
    h = fg.gated_linear(x, w, act="relu")
    assert (h[:-3] == 6).all() and h[-3:, 0].tolist() == [24.0, 0.0, 0.0]
    del h
    q, s = fg.quantize_rows(w)
    y = fg.gated_linear_int8(x, q, s, act="relu")
    assert ((y[:-3].float() - 6).abs() <= 0.05).all() and abs(y[-3, 0].item() - 24) <= 0.2 and y[-2:, 0].tolist() == [0.0, 0.0]
    del y
    z = fg.linear_int8(x, q, s)
    assert ((z[:-3, 0].float() - 2).abs() <= 0.02).all() and ((z[:-3, 1].float() - 3).abs() <= 0.03).all()


def test_gradients_of_very_many_rows():
    m = (1 << 24) + 5
    x, dh = torch.ones((m, 1), dtype=torch.bfloat16, device="cuda"), torch.ones((m, 1), dtype=torch.bfloat16, device="cuda")
    pre = torch.ones((m, 2), dtype=torch.bfloat16, device="cuda")
    w = torch.tensor([[2.0], [3.0]], dtype=torch.bfloat16, device="cuda")
    dx, dw, db = fg.gated_linear_backward(dh, x, w, pre, act="none")
    assert (dx == 5).all()
    for g in (dw, db):
        assert ((g.float() - m).abs() <= 2.0**-8 * m).all()


def test_two_streams_at_once():
    """The same calls on two streams without a wait between them: neither takes the other's workspace."""
    a, b = rnd(1, 700, 900), rnd(2, 700, 900)
    xa, xb = rnd(3, 3000, 600, dtype=torch.bfloat16), rnd(4, 3000, 600, dtype=torch.bfloat16)
    w, ws = fg.quantize_rows(rnd(5, 400, 600))
    dh, pre, wt = rnd(6, 3000, 100, dtype=torch.bfloat16), rnd(7, 3000, 200, dtype=torch.bfloat16), rnd(8, 200, 600, dtype=torch.bfloat16)

    def every(o, x):
        return (fg.orthogonalize(o), fg.linear_int8(x, w, ws), fg.gated_linear_int8(x, w, ws),
                *fg.gated_linear_backward(dh, x, wt, pre))

    want = every(a, xa), every(b, xb)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(one):
            first = every(a, xa)
        with torch.cuda.stream(two):
            second = every(b, xb)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(first, want[0]))
        assert all(torch.equal(p, q) for p, q in zip(second, want[1]))


def test_float32_gated_products_of_one_term():
    """k = 1: each factor is one product of two float32, good to 2^-22 of itself; h to twice that and a rounding."""
    x, w = rnd(1, 300, 1), rnd(2, 100, 1)
    h = fg.gated_linear(x, w, act="none").double()
    z = x.double() @ w.double().t()
    want = z[:, :50] * z[:, 50:]
    assert ((h - want).abs() <= (2 * 2.0**-22 + 2 * U) * want.abs() + 2.0**-140).all()


@pytest.mark.parametrize("m,n", [(96, 400), (400, 96), (500, 500), (1100, 300)])
@pytest.mark.parametrize("power", [0.0, 0.5, 1.0, 2.0])
def test_bfloat16_orthogonalisation_beside_its_rounding(m, n, power):
    """What several products in one plane leave, apart from the result's own rounding to bfloat16 (at most 2^-9 of the norm as
    a root mean square, 1.7e-3): 2e-3 at most, so that both together stay under 2.8e-3."""
    s = min(m, n)
    q, _ = torch.linalg.qr(rnd(1, m, s).double().cpu())
    v, _ = torch.linalg.qr(rnd(2, n, s).double().cpu())
    x = ((q * torch.arange(1, s + 1).double()**-power) @ v.t()).bfloat16()
    y = fg.orthogonalize(x.cuda()).double().cpu()
    z = x.double() / (x.double().norm() + 1e-7)
    z = z.t() if m > n else z
    for _ in range(5):
        g = z @ z.t()
        z = 3.4445 * z + (-4.7750 * g + 2.0315 * g @ g) @ z
    z = z.t() if m > n else z
    assert (y - z).norm() <= 2.8e-3 * z.norm()


@pytest.mark.parametrize("coef", [(3.5, -5.0, 2.2), (3.4445, -4.7750, 2.0315)])
@pytest.mark.parametrize("steps", [5, 12])
def test_bfloat16_steps_and_coefficients_that_take_two_planes(coef, steps):
    """Larger coefficients, or more steps, hold A in two planes: the result is off by little beside its rounding."""
    x = rnd(1, 60, 90, dtype=torch.bfloat16)
    y = fg.orthogonalize(x, steps=steps, coefficients=coef).double()
    z = x.double() / (x.double().norm() + 1e-7)
    a, b, c = coef
    for _ in range(steps):
        g = z @ z.t().contiguous()
        z = a * z + (b * g + c * (g @ g)) @ z
    assert (y - z).norm() <= 2.8e-3 * z.norm()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steps", [5, 12])
def test_coefficients_that_diverge(dt, steps):
    """(4, -6, 3) sends singular values past 64 before the fifth step (1.38, 1.56, 4.2, 3.5e3, ...): nothing finite comes back."""
    y = fg.orthogonalize(rnd(1, 60, 90, dtype=dt), steps=steps, coefficients=(4.0, -6.0, 3.0))
    assert not torch.isfinite(y).any()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(2110, 1317), (2300, 3100), (4351, 4049), (4004, 6054), (7300, 5606)])
def test_large_orthogonalisations(m, n, dt):
    """Every tile, whole products and joined triangles.  The bound of the operator's own tests: for each step 16 (2^-22 + 3
    sqrt(k) u) |X_i| 3.4445^(steps left), and of bfloat16 2.8e-3 of the result's norm as above."""
    x = rnd(m, m, n, dtype=dt)
    y = fg.orthogonalize(x).double()
    z = x.double()
    z = z / (z.norm() + 1e-7)
    if m > n:
        z, y = z.t().contiguous(), y.t()
    bound = 0.0
    for i in range(5):
        bound += 16 * (2.0**-22 + 3 * max(m, n)**0.5 * U) * z.norm().item() * 3.4445**(4 - i)
        g = z @ z.t().contiguous()
        z = 3.4445 * z + (-4.7750 * g + 2.0315 * (g @ g)) @ z
    assert (y - z).norm() <= (bound + U * z.norm() if dt is torch.float32 else 2.8e-3 * z.norm())
