"""The query head's products on every tile they have, in every form, against the definitions in 64 bits.

Which tile a size takes is asked for and compared, so that a rule that changes leaves no kernel without its test.  Sizes are
odd, or whole 16-byte rows (operands read as they are), never whole tiles."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402
from tests.test_gpu_head import check_linear, check_linear_grads, check_loss, loss_inputs, rnd  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
PAIR = 1024


def tile(m, k, n, dt, product):
    return fg.lib.fgpu_linear_tile(m, k, n, int(dt == "bf16"), product)


FORWARD = [("f32", 64, 163, 1285, 156), ("f32", 128, 1089, 153, 5507), ("f32", 256, 6591, 153, 1860), ("f32", 64, 174, 1416, 152),
           ("f32", 128, 2694, 152, 2280), ("f32", 256, 769, 144, 15312), ("f32", 256, 8200, 136, 8200),
           ("bf16", 64, 160, 1076, 150), ("bf16", 128, 1796, 263, 1706), ("bf16", 256, 4298, 150, 2403), ("bf16", 64, 153, 264, 144),
           ("bf16", 128, 1594, 264, 1936), ("bf16", 256, 3339, 152, 3088), ("bf16", 128, 4097, 1032, 4104),
           ("bf16", 128, 8200, 136, 8200), ("bf16", 256, 9001, 152, 8200)]


@pytest.mark.parametrize("dt,want,m,k,n", FORWARD)
@pytest.mark.parametrize("act,bias,residual,save", [("gelu", True, False, True), ("silu", True, True, False), ("relu", False, True, True),
                                                   ("none", True, True, True), ("none", False, False, False)])
def test_forward(dt, want, m, k, n, act, bias, residual, save):
    """The last two sizes of bfloat16 and the last of float32 have results of more than 2^28 bytes (with a kept
    pre-activation), which are stored past the caches."""
    assert tile(m, k, n, dt, 0) == want
    check_linear(m, k, n, dt, act, bias, residual, save)


BACKWARD = [("f32", 256, 64, 5585, 2246, 151), ("f32", 64, 128, 152, 4610, 3433), ("f32", 64, 256, 154, 2249, 5442),
            ("f32", PAIR + 64, PAIR + 64, 155, 162, 1810), ("f32", 128, 64, 1356, 11257, 153), ("f32", 256, 64, 5171, 2376, 152),
            ("f32", 64, 128, 153, 4984, 3144), ("f32", 64, 256, 160, 3400, 3632), ("f32", 128, 64, 1622, 9448, 152),
            ("f32", PAIR + 128, PAIR + 128, 67, 8728, 2232), ("bf16", 128, 64, 1203, 4291, 158), ("bf16", 64, 128, 151, 3876, 1290),
            ("bf16", 64, 256, 158, 4925, 2122), ("bf16", PAIR + 64, PAIR + 64, 2924, 167, 162),
            ("bf16", PAIR + 128, PAIR + 128, 265, 10091, 279), ("bf16", 256, 64, 1634, 6277, 153), ("bf16", 128, 64, 787, 6344, 144),
            ("bf16", 64, 128, 155, 4840, 1040), ("bf16", 64, 256, 152, 5704, 1808), ("bf16", PAIR + 128, PAIR + 128, 258, 10632, 272),
            ("bf16", 256, 64, 1312, 7760, 152), ("bf16", 256, 256, 4097, 1032, 4104)]


@pytest.mark.parametrize("dt,want_x,want_w,m,k,n", BACKWARD)
@pytest.mark.parametrize("act", ["gelu", "silu", "none"])
def test_backward(dt, want_x, want_w, m, k, n, act):
    assert (tile(m, k, n, dt, 1), tile(m, k, n, dt, 2)) == (want_x, want_w)
    t = TYPES[dt]
    dy, x, w = rnd(1, m, n, dtype=t), rnd(2, m, k, dtype=t), rnd(3, n, k, scale=k**-0.5, dtype=t)
    pre = rnd(4, m, n, scale=1.5, dtype=t) if act != "none" else None
    dx, dw, db = fg.linear_backward(dy, x, w, pre, act=act)
    check_linear_grads(dy, x, w, pre, act, dt, dx, dw, db)
    for only in ("x", "weight", "bias"):
        one = fg.linear_backward(dy, x, w, pre, act=act, want=(only,))
        at = ("x", "weight", "bias").index(only)
        assert torch.equal(one[at], (dx, dw, db)[at]) and all(o is None for i, o in enumerate(one) if i != at)


def test_backward_streamed():
    """An input gradient of more than 2^28 bytes."""
    m, k, n = 16390, 8208, 136
    dy, x, w = (rnd(i, *s, dtype=torch.bfloat16) for i, s in enumerate(((m, n), (m, k), (n, k))))
    check_linear_grads(dy, x, w, None, "none", "bf16", *fg.linear_backward(dy, x, w))


# The loss above 128 dims.  (11600, 11601) in bfloat16 and (6701, 6702) in float32: score gradients of more than 2^28 bytes.
LOSS = [(64, 300, 1500, 200), (128, 1500, 2201, 136), (128, 2301, 2203, 203), (256, 3301, 4100, 200), (256, 6701, 6702, 136),
        (256, 5003, 3001, 131), (256, 11600, 11601, 137)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("want,nq,nc,dim", LOSS)
def test_loss(want, nq, nc, dim, dt):
    assert fg.lib.fgpu_contrastive_loss_tile(nq, nc, dim, int(dt == "bf16")) == want
    q, c, t, scale, bias, ids = loss_inputs(nq, nc, dim, dt)
    check_loss(q, c, t, scale, None, None, dt)
    t[::5], t[3], t[nq - 1] = -1, nc + 7, nc - 1
    bias[::7], bias[4] = -torch.inf, torch.finfo(torch.float32).min
    bias[nc - 1] = 0
    check_loss(q, c, t, scale, bias, ids, dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [40, 64, 90, 96, 121, 128])
@pytest.mark.parametrize("nq,nc", [(1021, 1030), (3001, 30011)])
def test_loss_up_to_128_dims(nq, nc, dim, dt):
    """The shape for few pairs and the one for many, for 64, 96 and 128 dims, whole and odd."""
    q, c, t, scale, bias, ids = loss_inputs(nq, nc, dim, dt)
    t[::5], t[3], t[nq - 1] = -1, nc + 7, nc - 1
    bias[::7], bias[4] = -torch.inf, torch.finfo(torch.float32).min
    bias[nc - 1] = 0
    check_loss(q, c, t, scale, bias, ids, dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nc,dim", [(3301, 4100, 200), (1500, 2201, 136)])
def test_loss_masked_places_may_hold_anything(nq, nc, dim, dt):
    """Infinities and NaN in masked candidates and in rows without a target reach no result, on the large tiles too."""
    q, c, t, scale, bias, ids = loss_inputs(nq, nc, dim, dt)
    hide = torch.zeros(nc, dtype=torch.bool, device="cuda")
    hide[[0, 63, 64, 255, 256, 1000, nc - 1]] = True
    bias[hide] = -torch.inf
    t[hide[t.long()]] = 5
    t[[0, 300, nq - 1]] = -1
    clean = check_loss(q, c, t, scale, bias, ids, dt)
    c[hide] = torch.nan
    c[0] = torch.inf
    q[[0, nq - 1]], q[300] = torch.nan, -torch.inf
    loss, lse = fg.contrastive_loss(q, c, t, scale, bias=bias, ids=ids)
    got = fg.contrastive_loss_backward(rnd(99, nq), q, c, t, lse, scale, bias=bias, ids=ids)
    keep = t >= 0
    for a, b in zip((loss, lse[keep], *got), (clean[0], clean[1][keep], *clean[2:])):
        assert torch.equal(a, b)


def least_workspace(q, c, t, lse, scale, bias, ids, full):
    """The smallest workspace the backward call takes, in steps of 2 KB: its chunks are then 256 columns."""
    low, high = 0, full
    while high - low > 2048:
        mid = (low + high) // 2
        try:
            fg.contrastive_loss_backward(torch.zeros_like(lse), q, c, t, lse, scale, bias=bias, ids=ids,
                                         workspace=torch.empty(mid, dtype=torch.uint8, device="cuda"))
            high = mid
        except fg.FgpuError as e:
            assert "256 columns" in str(e)
            low = mid
    return high


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nc,dim", [(300, 2900, 200), (6000, 9001, 136), (300, 2900, 72)])
def test_loss_gradients_in_chunks_down_to_the_least(nq, nc, dim, dt):
    """Chunks of 256 columns, of some thousand (on 256 x 256 tiles at 6000 queries) and of all: each within the bounds."""
    q, c, t, scale, bias, ids = loss_inputs(nq, nc, dim, dt)
    bias[::11] = -torch.inf
    t[::9] = -1
    full = fg.lib.fgpu_contrastive_loss_backward_workspace_bytes(nq, nc, dim, int(dt == "bf16"))
    _, lse = fg.contrastive_loss(q, c, t, scale, bias=bias, ids=ids)
    least = least_workspace(q, c, t, lse, scale, bias, ids, full)
    assert least < 0.9 * full
    for size in (least, (least + full) // 2, full):
        check_loss(q, c, t, scale, bias, ids, dt, workspace=torch.empty(size, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nc,dim", [(300, 900, 72), (300, 900, 200), (1500, 2201, 136), (1501, 30011, 128)])
def test_loss_gradients_of_some(nq, nc, dim, dt):
    """Each gradient alone, as C callers may ask, has the bits it has among the others."""
    q, c, t, scale, bias, ids = loss_inputs(nq, nc, dim, dt)
    bias[::7], t[::9] = -torch.inf, -1
    t[5:9] = t[4]
    code, dl = int(dt == "bf16"), rnd(99, nq)
    _, lse = fg.contrastive_loss(q, c, t, scale, bias=bias, ids=ids)
    full = fg.contrastive_loss_backward(dl, q, c, t, lse, scale, bias=bias, ids=ids)
    size = fg.lib.fgpu_contrastive_loss_backward_workspace_bytes(nq, nc, dim, code)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    for some in ((0,), (1,), (2,), (0, 2), (1, 2), (0, 1), ()):
        out = [torch.full_like(g, 7) if i in some else None for i, g in enumerate(full)]
        assert fg.lib.fgpu_contrastive_loss_backward(dl.data_ptr(), q.data_ptr(), c.data_ptr(), t.data_ptr(), lse.data_ptr(),
                                                     bias.data_ptr(), ids.data_ptr(), nq, nc, dim, code, scale,
                                                     *(None if o is None else o.data_ptr() for o in out), ws.data_ptr(), size,
                                                     fg._stream()) == 0
        assert all(o is None or torch.equal(o, g) for o, g in zip(out, full))


@pytest.mark.parametrize("nq,nc,dim", [(5000, 3, 200), (3000, 10, 136), (9000, 300, 130), (130, 20, 200), (64, 15, 700), (9, 2, 1000)])
def test_loss_of_few_candidates(nq, nc, dim):
    """Many rows with one target, as a classifier has."""
    q, c, t, scale, bias, _ = loss_inputs(nq, nc, dim, "bf16")
    check_loss(q, c, t, scale, bias, None, "bf16")
    check_loss(q, c, torch.full_like(t, nc - 1), scale, bias, None, "bf16")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nc,dim", [(1500, 2201, 136), (3301, 4100, 200)])
def test_loss_captured_and_replayed(nq, nc, dim, dt):
    """Above 128 dims: replays on changing inputs and targets, with eager calls between, are the eager results."""
    q, c, t, scale, bias, ids = loss_inputs(nq, nc, dim, dt)
    dl = rnd(99, nq)

    def step():
        loss, lse = fg.contrastive_loss(q, c, t, scale, bias=bias, ids=ids)
        return [loss, lse, *fg.contrastive_loss_backward(dl, q, c, t, lse, scale, bias=bias, ids=ids)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        q.copy_(rnd(100 + k, nq, dim, dtype=q.dtype))
        t.copy_(t.roll(7 + k))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
