"""The gated query head end to end: its gradients against autograd in 64 bits, orthogonalised steps, 8-bit serving, and all of
them in one captured graph."""
import math

import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402
from fusiongpu_amd.query_head import QueryHead, demo  # noqa: E402

pytestmark = pytest.mark.gpu


def forward64(p, x, skip):
    def norm(v, g, b):
        d = v - v.mean(1, keepdim=True)
        return d / torch.sqrt(d.square().mean(1, keepdim=True) + 1e-5) * g + b

    a = norm(x.double(), p["in_gain"], p["in_offset"])
    gate, up = (a @ p["w1"].t() + p["b1"]).chunk(2, 1)
    z = gate * torch.sigmoid(gate) * up @ p["w2"].t() + p["b2"] + (x.double() if skip else 0)
    return norm(z, p["out_gain"], p["out_offset"])


def make(in_dim, dim, hidden=100, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    head = QueryHead(in_dim, hidden, dim, dtype=dtype, seed=1, gated=True)
    for n, p in head.params.items():  # away from ones and zeros
        p += 0.1 * torch.randn(p.shape, generator=g, device="cuda") * (1 if p.dim() == 1 else 0)
    head._cast()
    x = torch.randn((77, in_dim), generator=g, device="cuda")
    cand = torch.randn((300, dim), generator=g, device="cuda")
    t = torch.randperm(300, generator=g, device="cuda")[:77]
    return head, x, cand, t


@pytest.mark.parametrize("in_dim,dim", [(100, 96), (128, 128)])
def test_gradients_against_autograd(in_dim, dim):
    """float32: each operator is exact to about 1e-6 of its result, and six of them follow one another."""
    head, x, cand, t = make(in_dim, dim)
    loss, grads = head.loss(x, cand, t, scale=0.1)
    p = {n: v.double().requires_grad_() for n, v in head.params.items()}
    e = forward64(p, x, in_dim == dim)
    s = -0.05 * (e[:, None] - cand.double()[None]).square().sum(2)
    want = (torch.logsumexp(s, 1) - s[torch.arange(77, device="cuda"), t]).mean()
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    for n in QueryHead.NAMES:
        assert (grads[n].double() - p[n].grad).norm() <= 2e-5 * p[n].grad.norm(), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_step_with_matrix_lr_moves_the_weights_by_orthogonal_updates(dtype):
    head, x, cand, t = make(100, 96, dtype=dtype)
    before = {n: p.clone() for n, p in head.params.items()}
    _, grads = head.loss(x, cand, t, scale=0.1)
    head.train_step(x, cand, t, scale=0.1, matrix_lr=0.01)
    for n in ("w1", "w2"):
        rows, cols = before[n].shape
        m = torch.zeros_like(before[n]).lerp_(grads[n].float(), 1 - 0.9)
        want = before[n] - 0.01 * max(1, rows / cols)**0.5 * fg.orthogonalize(m.to(dtype)).float()
        assert torch.equal(head.params[n], want), n
    assert not torch.equal(head.params["b1"], before["b1"])


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("in_dim,dim", [(768, 128), (128, 128)])
def test_int8_head(in_dim, dim, gated):
    """Rounding to 8 bits is off by half a step of max / 127 an element.  A dot product of n terms of a row and a column,
    whose largest elements are about 3.5 of their root mean square, is then off by about 3.5 / 127 / sqrt(12) sqrt(2) of what
    its terms' root sum of squares is: 1.1 % a layer, two layers; five times that, and bfloat16's own, bounds every row."""
    head = QueryHead(in_dim, 512, dim, gated=gated)
    x = torch.randn((300, in_dim), device="cuda")
    full, small = head(x).float(), head.int8()(x).float()
    off = (full - small).norm(dim=1) / full.norm(dim=1)
    assert off.max() <= 0.12
    assert head.int8()(x[:0]).shape == (0, dim)
    one = head.int8()(x[7:8]).float()
    assert (one - small[7:8]).norm() <= 0.03 * one.norm()  # both rounded the same way, bfloat16 between the layers


def test_searches_on_another_stream():
    base = torch.from_numpy(fg.gen_gmm(4000, 128, 16, seed=5, sig_lo=0.2)).cuda()
    index = fg.Index.from_arrays(128, 32, *fg.build_ivfpq(base, 32, 32, kmeans_iters=4, init_mode=1, pq_iters=3))
    head = QueryHead(256, 128, 128, gated=True)
    x = torch.randn((40, 256), device="cuda")
    small = head.int8()
    for h in (head, small):
        ids, d = h.search(index, x, 8, 5)
        wids, wd = index.search(h(x).float(), 8, 5)
        assert torch.equal(ids, wids) and torch.equal(d, wd)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        sids, _ = h.search(index, x, 8, 5, stream=side)
        side.synchronize()
        assert torch.equal(sids, wids)
    index.close()


def test_captured_and_replayed():
    """The gated head, its gradients, an orthogonalised update of each weight and the 8-bit head in one graph, replayed on
    changing inputs with eager calls between."""
    head, x, cand, t = make(100, 96, dtype=torch.bfloat16)
    small = head.int8()

    def every():
        loss, grads = head.loss(x, cand, t, scale=0.1)
        return [loss, head(x), small(x), fg.orthogonalize(grads["w1"]), fg.orthogonalize(grads["w2"])] + list(grads.values())

    every()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = every()
    g = torch.Generator(device="cuda")
    for k in range(3):
        g.manual_seed(50 + k)
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        assert all(torch.equal(a, b) for a, b in zip(got, every()))


@pytest.mark.parametrize("gated,matrix_lr", [(True, None), (True, 0.02), (False, 0.02)])
def test_demo_runs(gated, matrix_lr):
    said = []
    before, after = demo(n=3000, steps=3, batch=256, gated=gated, matrix_lr=matrix_lr, log=said.append)
    assert 0 <= before <= 1 and 0 <= after <= 1 and math.isfinite(before + after) and "8-bit" in said[-1]
