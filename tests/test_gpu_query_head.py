"""The query head end to end: its gradients against autograd in 64 bits, training, and the search behind it."""
import math

import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402
from fusiongpu_amd.query_head import QueryHead, demo  # noqa: E402

pytestmark = pytest.mark.gpu


def loss64(params, x, cand, targets, scale, ids, skip):
    """The head and its loss in float64 by autograd."""
    p = {n: v.double().requires_grad_() for n, v in params.items()}

    def norm(v, g, b):
        d = v - v.mean(1, keepdim=True)
        return d / torch.sqrt(d.square().mean(1, keepdim=True) + 1e-5) * g + b

    a = norm(x.double(), p["in_gain"], p["in_offset"])
    z1 = a @ p["w1"].t() + p["b1"]
    h = z1 * torch.special.erfc(-z1 / math.sqrt(2)) / 2
    z = h @ p["w2"].t() + p["b2"] + (x.double() if skip else 0)
    e = norm(z, p["out_gain"], p["out_offset"])
    s = -0.5 * scale * torch.cdist(e, cand.double()).square()
    at = targets.long()
    same = ids[None, :] == ids[at][:, None]
    same[torch.arange(at.numel(), device="cuda"), at] = False
    s = s.masked_fill(same, -math.inf)
    loss = (torch.logsumexp(s, 1) - s[torch.arange(at.numel(), device="cuda"), at]).mean()
    loss.backward()
    return loss.detach(), {n: v.grad for n, v in p.items()}


@pytest.mark.parametrize("in_dim,dim", [(100, 96), (128, 128)])
def test_gradients_against_autograd(in_dim, dim):
    """float32: each operator is exact to about 1e-6 of its result, and six of them follow one another."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    head = QueryHead(in_dim, 200, dim, dtype=torch.float32, seed=1)
    for n, p in head.params.items():  # away from ones and zeros
        p += 0.1 * torch.randn(p.shape, generator=g, device="cuda") * (1 if p.dim() == 1 else 0)
    head._cast()
    x = torch.randn((77, in_dim), generator=g, device="cuda")
    cand = torch.randn((300, dim), generator=g, device="cuda")
    t = torch.randperm(300, generator=g, device="cuda")[:77]
    ids = torch.randint(250, (300,), generator=g, device="cuda", dtype=torch.int32)
    loss, grads = head.loss(x, cand, t, scale=0.1, ids=ids)
    want, wgrads = loss64(head.params, x, cand, t, 0.1, ids, in_dim == dim)
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    for n in QueryHead.NAMES:
        assert (grads[n].double() - wgrads[n]).norm() <= 2e-5 * wgrads[n].norm(), n


def test_embeddings_of_one_and_of_many_agree():
    """A query's embedding does not depend on the batch it comes in, beyond rounding to bfloat16."""
    head = QueryHead(768, 1024, 128)
    x = torch.randn((300, 768), device="cuda")
    many = head(x).float()
    one = torch.cat([head(x[i:i + 1]) for i in (0, 17, 299)]).float()
    assert (many[[0, 17, 299]] - one).abs().max() <= 2.0**-4  # layer norm's values reach 4: four units of the last place
    assert many.shape == (300, 128) and head(x[:0]).shape == (0, 128)


def test_trains_and_searches():
    before, after = demo(n=5000, steps=120, batch=512, log=None)
    assert before < 0.05 and after > 0.5


def test_search_is_the_index_search_of_the_embeddings():
    base = torch.from_numpy(fg.gen_gmm(4000, 128, 16, seed=5, sig_lo=0.2)).cuda()
    index = fg.Index.from_arrays(128, 32, *fg.build_ivfpq(base, 32, 32, kmeans_iters=4, init_mode=1, pq_iters=3))
    head = QueryHead(256, 128, 128)
    x = torch.randn((40, 256), device="cuda")
    ids, d = head.search(index, x, 8, 5)
    wids, wd = index.search(head(x).float(), 8, 5)
    assert torch.equal(ids, wids) and torch.equal(d, wd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    sids, _ = head.search(index, x, 8, 5, stream=side)
    side.synchronize()
    assert torch.equal(sids, wids)
    index.close()
