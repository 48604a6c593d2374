"""8-bit layers give a row the same bits whatever batch it comes in: sums of whole numbers are exact, and every kernel (up to
16 rows; some hundred; tiles of 64, 128 and 256) takes the same steps after them."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu


def rnd(seed, *shape, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("k,n", [(400, 200), (77, 131), (512, 1040)])
def test_a_row_in_any_batch(k, n, bias, act, dt):
    rows = (1, 16, 17, 300, 2500, 9000, 20000)
    x, r = rnd(1, rows[-1], k, dtype=dt), rnd(2, rows[-1], n, dtype=dt)
    b = rnd(3, 2 * n, dtype=dt) if bias else None
    q, xs = fg.quantize_rows(x)
    w, ws = fg.quantize_rows(rnd(4, 2 * n, k, scale=k**-0.5))
    half = (w[:n].contiguous(), ws[:n].contiguous(), None if b is None else b[:n].contiguous())
    for f in (lambda x, m, **kw: fg.linear_int8(x, *half, r[:m], act=act, **kw),
              lambda x, m, **kw: fg.linear_int8(x, *half, act=act, **kw),
              lambda x, m, **kw: fg.gated_linear_int8(x, w, ws, b, act=act, **kw)):
        every = f(x, rows[-1])
        for m in rows:
            got = f(x[:m], m)
            assert torch.equal(got, every[:m]), (m, (got != every[:m]).float().mean().item())
            assert torch.equal(f(q[:m], m, x_scale=xs[:m], dtype=dt), every[:m]), m
