"""What a query head keeps between calls: its 8-bit copies."""
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
