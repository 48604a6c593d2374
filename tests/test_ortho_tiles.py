"""Which kernels the orthogonalisation's products take, on the CPU: the sizes that are tested against 64 bits take all of them,
and the bound of those tests would show a lost plane."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

from . import _ortho  # noqa: E402

tile = fg.lib.fgpu_orthogonalize_tile


def kernels(m, n):
    return {(product, m > n, tile(m, n, product)) for product in range(3)}


def test_every_kernel_is_tested():
    """Over sides of 1 to 16384, a sixth of an octave apart."""
    sides = sorted({int(round(2**(i / 6))) for i in range(85)})
    reached = set().union(*(kernels(m, n) for m in sides for n in sides))
    tested = set().union(*(kernels(m, n) for m, n in _ortho.SIZES))
    assert reached <= tested, sorted(reached - tested)


def test_refused():
    assert tile(0, 5, 0) == tile(5, 0, 0) == tile(-1, 5, 0) == tile((1 << 16) + 1, 5, 0) == -1
    assert tile(5, 5, 3) == tile(5, 5, -1) == -1


def planes(v):
    h = (v * 1024).half().double() / 1024
    return h, ((v - h) * 1024).half().double() / 1024


@pytest.mark.parametrize("m,n", [(70, 200), (300, 400), (500, 500)])
@pytest.mark.parametrize("order", [1, 2])
@pytest.mark.parametrize("lost", ["none", "X in A", "A in A^2", "P", "X"])
def test_a_lost_plane_shows(m, n, order, lost):
    """The products of one step as the kernels form them, in 64 bits, with one plane left out of one operand of one product."""
    g = torch.Generator().manual_seed(m + n)
    x0 = _ortho.start(torch.randn((m, n), generator=g))
    factor = float(m)**order

    def times(p, q, lose):
        (ph, pl), (qh, ql) = p, q
        return ph @ qh + ph @ ql + (0 if lose else pl @ qh)

    x = planes(x0)
    a = planes(times(x, [v.t() for v in x], lost == "X in A"))
    if order == 2:
        s = times(a, a, lost == "A in A^2")
    elif lost == "A in A^2":
        return
    p = planes(factor * (s if order == 2 else sum(a)))
    y = times(p, x, lost == "P") if lost != "X" else p[0] @ x[0] + p[1] @ x[0]
    off, bound = _ortho.within(y, *_ortho.step_of_gram(x0, order, factor), torch.float32)
    assert (off <= bound) == (lost == "none"), (off, bound)
