"""Orthogonalisation where what lies between its products passes 64: what it reaches is NaN, and nothing else is touched.

diag(1, 0.01, 0.01, ...) with coefficients (1, 1, 100): P = I + A + 100 A^2 has 102 / |x|^2 and 100 / |x|^4 more in its corner,
past 64, and 1.0001 elsewhere.  In the last step P multiplies nothing but X: row 0 of y (of tall matrices column 0) is NaN, the
others are right, to a rounding of X_0, of P and of the result and what three products leave out, 2^-21 of themselves."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu


def corner(m, n, dtype):
    x = torch.zeros((m, n), dtype=torch.float32)
    x.diagonal().fill_(0.01)
    x[0, 0] = 1
    return x.cuda().to(dtype)


SIZES = [(2, 2), (64, 70), (70, 64), (128, 128), (300, 700), (700, 300), (1100, 1100), (1500, 2500), (2500, 1500)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", SIZES)
def test_in_the_last_step(m, n, dt):
    x = corner(m, n, dt)
    y = fg.orthogonalize(x, steps=1, coefficients=(1.0, 1.0, 100.0))
    z = x.double() / (x.double().norm() + 1e-7)
    want = z + z**3 + 100 * z**5  # of a diagonal matrix
    if m > n:
        y, want = y.t(), want.t()
    assert torch.isnan(y[0]).all()
    half = 2.0**-24 if dt is torch.float32 else 2.0**-8
    assert ((y[1:].double() - want[1:]).abs() <= (2.0**-21 + half) * want[1:].abs()).all()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("coef", [(1.0, 1.0, 100.0), (20.0, 0.0, 0.0)])  # P passes in the first step; A in the second
@pytest.mark.parametrize("m,n", SIZES)
def test_before_the_last_step(m, n, coef, dt):
    assert torch.isnan(fg.orthogonalize(corner(m, n, dt), steps=3, coefficients=coef)).all()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_a_result_may_be_larger(dt):
    """y itself is not held between products: (50, 20, 0) of a 1 x 1 matrix, P = 70 past the bound, and (30, 20, 10), 60, not."""
    x = torch.ones((1, 1), dtype=dt, device="cuda")
    assert torch.isnan(fg.orthogonalize(x, steps=1, eps=0.0, coefficients=(50.0, 20.0, 0.0))).all()
    assert fg.orthogonalize(x, steps=1, eps=0.0, coefficients=(30.0, 20.0, 10.0)).item() == 60.0
