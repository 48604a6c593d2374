"""What a query head keeps between calls: its 8-bit copies, its moments."""
import pytest

torch = pytest.importorskip("torch")

from fusiongpu_amd.query_head import QueryHead  # noqa: E402

pytestmark = pytest.mark.gpu


def batch(rows=20, dim=64, n=50):
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    return (torch.randn((rows, dim), generator=g, device="cuda"), torch.randn((n, dim), generator=g, device="cuda"),
            torch.arange(rows, device="cuda"))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_8_bit_head_is_the_head_as_it_was(dtype, gated):
    """Steps that the head takes afterwards do not reach it."""
    head = QueryHead(64, 32, 64, dtype=dtype, gated=gated)
    x, cand, t = batch()
    small = head.int8()
    before = small(x)
    for matrix_lr in (None, 0.01):
        head.train_step(x, cand, t, lr=0.1, matrix_lr=matrix_lr)
        assert torch.equal(small(x), before)
    assert not torch.equal(head.int8()(x), before)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adam_after_orthogonalised_steps(dtype):
    """Two steps with matrix_lr, one without, one with, two without: each Adam step moves the weights by both moments of all
    gradients so far, to a rounding of the rate."""
    head = QueryHead(48, 32, 64, dtype=dtype, gated=True)
    x, cand, t = batch(dim=48)[0], batch()[1], batch()[2]
    moments = {n: (torch.zeros_like(p), torch.zeros_like(p)) for n, p in head.params.items()}
    for step, matrix_lr in enumerate((0.01, 0.01, None, 0.01, None, None), 1):
        _, grads = head.loss(x, cand, t)
        before = {n: p.clone() for n, p in head.params.items()}
        head.train_step(x, cand, t, lr=1e-2, matrix_lr=matrix_lr)
        rate = 1e-2 * (1 - 0.98**step)**0.5 / (1 - 0.9**step)
        for n in QueryHead.NAMES:
            m, v = moments[n]
            g = grads[n].float()
            m.lerp_(g, 1 - 0.9)
            v.lerp_(g * g, 1 - 0.98)
            if matrix_lr is None or before[n].dim() == 1:
                want = before[n] - rate * m / (v.sqrt() + 1e-8)
                assert (head.params[n] - want).abs().max() <= 2.0**-22 * want.abs().max(), (step, n)
