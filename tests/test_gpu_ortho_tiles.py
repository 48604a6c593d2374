"""Every kernel of the orthogonalisation at the precision of its planes, each product of a step by itself: coefficients (0, b, 0)
give b A X, (0, 0, c) c A^2 X and (a, 0, 0) a^steps X, with b and c such that the results are of X's size."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

from . import _ortho  # noqa: E402

pytestmark = pytest.mark.gpu


def make(m, n, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(m * n)
    return torch.randn((m, n), generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", _ortho.SIZES)
def test_each_product(m, n, dt):
    x = make(m, n, dt)
    x0 = _ortho.start(x)
    for order in (1, 2):
        factor = float(min(m, n))**order
        want, error = _ortho.step_of_gram(x0, order, factor)
        y = fg.orthogonalize(x, steps=1, coefficients=(0.0, factor, 0.0) if order == 1 else (0.0, 0.0, factor))
        off, bound = _ortho.within(y.t() if m > n else y, want, error, dt)
        assert off <= bound, (order, off, bound, want.norm().item())


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", _ortho.SIZES)
def test_what_is_handed_on(m, n, dt):
    """Three steps of (1.5, 0, 0), 1.5^3 X_0: P is 1.5 I to the bit, so an entry is off by what it is held to three times, by the
    roundings of three products of one term each (what each leaves out, 2^-24, and two sums), and by X_0's factor and the result's
    rounding: 3 (2^-23 + 4 u) + 2 u + 3 u, under 2^-19.9 of itself and 2^-35 of one each time, multiplied by up to 1.5^3."""
    x = make(m, n, dt)
    want = 1.5**3 * _ortho.start(x)
    y = fg.orthogonalize(x, steps=3, coefficients=(1.5, 0.0, 0.0))
    off = ((y.t() if m > n else y).double() - want).abs()
    half = 0 if dt is torch.float32 else 2.0**-8
    assert (off <= (2.0**-19.9 + half) * want.abs() + (1.5**3 + 1.5**2 + 1.5) * 2.0**-35).all()
