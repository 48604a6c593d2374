"""The query head's targets: those outside the candidates leave their row without a loss, whatever integer type they have."""
import pytest

torch = pytest.importorskip("torch")

from fusiongpu_amd.query_head import QueryHead  # noqa: E402

pytestmark = pytest.mark.gpu


def test_targets_beyond_int32_are_no_targets():
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    head = QueryHead(64, 96, 32, dtype=torch.float32)
    x = torch.randn((6, 64), generator=g, device="cuda")
    cand = torch.randn((20, 32), generator=g, device="cuda")
    none = torch.tensor([0, -1, 19, -1, -1, 7], device="cuda")
    far = torch.tensor([0, 20, 19, (1 << 32) + 3, -(1 << 40) + 5, 7], device="cuda")
    want, wgrads = head.loss(x, cand, none.to(torch.int32))
    for t in (none, far):
        loss, grads = head.loss(x, cand, t)
        assert torch.equal(loss, want) and all(torch.equal(grads[n], wgrads[n]) for n in QueryHead.NAMES)
