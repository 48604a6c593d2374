"""Orthogonalised updates in bfloat16: the same numbers as in float32, rounded once, whatever the singular values are.

Against 64 bits: a result is off by its rounding, |bf16(want) - want|, and by what the steps leave of it, e, which moves that
rounding by at most itself again: |y - want| <= |bf16(want) - want| + 2 e.  e: a step's X takes some six roundings of 2^-23 of
their value at most, as root mean squares 2^-23 sqrt(6 / 3), times about 3.44: 2^-20.8 |X|.  What reaches a direction whose
singular value is still small grows by 3.4445 a step, as that value itself does, and stops growing with it at about one; updates
rounded to bfloat16 have none below 2^-9 / sqrt(n), which arrives within five steps, so no more than (3.4445^5 - 1) / 2.4445 =
198 of 2^-20.8: 1.1e-4 of the norm.  3e-4 is allowed for."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)


def rnd(seed, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def make(kind, m, n):
    x = rnd(1, m, n)
    if kind.startswith("rank"):  # a small batch's gradient
        r = int(kind[4:])
        x = rnd(2, m, r) @ rnd(3, r, n)
    elif kind == "sparse":
        x = x * (rnd(4, m, n).abs() > 2.33)  # one in fifty
    elif kind == "few rows":  # all but four units without a gradient
        x[4:] = 0
    elif kind == "orthogonal":
        s = min(m, n)
        q, v = torch.linalg.qr(rnd(5, m, s).double().cpu())[0], torch.linalg.qr(rnd(6, n, s).double().cpu())[0]
        x = (q @ v.t()).cuda()
    elif kind == "rows of many sizes":
        x = x * torch.exp(2 * rnd(7, m, 1))
    return x.bfloat16()


KINDS = ["normal", "rank1", "rank4", "rank16", "sparse", "few rows", "orthogonal", "rows of many sizes"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n", [(32, 32), (64, 64), (96, 400), (400, 96), (256, 700), (700, 256)])
@pytest.mark.parametrize("steps", [1, 2, 4, 5, 6, 7, 8, 12])
def test_error_beside_the_rounding(kind, m, n, steps):
    x = make(kind, m, n)
    y = fg.orthogonalize(x, steps=steps).double()
    z = x.double() / (x.double().norm() + 1e-7)
    z = z.t().contiguous() if m > n else z
    a, b, c = COEF
    for _ in range(steps):
        g = z @ z.t().contiguous()
        z = a * z + (b * g + c * (g @ g)) @ z
    z = z.t() if m > n else z
    bound = (z.bfloat16().double() - z).norm() + 2 * 3e-4 * z.norm()
    assert (y - z).norm() <= bound, ((y - z).norm() / z.norm(), bound / z.norm())


@pytest.mark.parametrize("m,n", [(1, 1), (7, 300), (64, 64), (96, 400), (400, 96), (500, 700), (700, 500), (2110, 1317),
                                 (1030, 4099), (8200, 1032), (3004, 2000)])
@pytest.mark.parametrize("steps,coef", [(1, COEF), (5, COEF), (8, COEF), (4, (2.0, -1.5, 0.5))])
def test_the_float32_result_rounded(m, n, steps, coef):
    x = rnd(m + n, m, n).bfloat16()
    want = fg.orthogonalize(x.float(), steps=steps, coefficients=coef)
    assert torch.equal(fg.orthogonalize(x, steps=steps, coefficients=coef), want.bfloat16())
