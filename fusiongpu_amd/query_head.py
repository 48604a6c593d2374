"""A query head: the small trained map from an encoder's hidden states to an index's space, and its training.

    x [rows][in_dim] -> layer norm -> linear + gelu -> linear (+ x where the widths agree) -> layer norm -> [rows][dim]

The forward pass serves (one query or a batch, straight into Index.search); train_step takes hidden states of questions,
the index's vectors that answer them and any further candidates, and moves the parameters by the softmax contrastive
loss under the index's own L2 metric.  Every heavy step is a call of this package's kernels (linear, layer_norm,
contrastive_loss and their backward calls); the parameter update is elementwise torch.

    python -m fusiongpu_amd.query_head     # trains a head on synthetic data and searches with it
"""
from __future__ import annotations

import math

import torch

import fusiongpu_amd as fg


class QueryHead:
    """Parameters in float32, computed in `dtype` (torch.bfloat16 or torch.float32)."""

    NAMES = ("in_gain", "in_offset", "w1", "b1", "w2", "b2", "out_gain", "out_offset")

    def __init__(self, in_dim: int, hidden: int, dim: int, dtype=torch.bfloat16, seed: int = 0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def normal(*shape, scale):
            return torch.randn(shape, generator=g, device="cuda") * scale

        one, zero = (lambda n: torch.ones(n, device="cuda")), (lambda n: torch.zeros(n, device="cuda"))
        self.dtype, self.skip, self.steps = dtype, in_dim == dim, 0
        self.params = dict(in_gain=one(in_dim), in_offset=zero(in_dim), w1=normal(hidden, in_dim, scale=in_dim**-0.5),
                           b1=zero(hidden), w2=normal(dim, hidden, scale=hidden**-0.5), b2=zero(dim), out_gain=one(dim),
                           out_offset=zero(dim))
        self._moments = {n: (torch.zeros_like(p), torch.zeros_like(p)) for n, p in self.params.items()}
        self._cast()

    def _cast(self):
        """The parameters in the compute type: laid out once a step, not once a call."""
        self._c = {n: p.to(self.dtype) for n, p in self.params.items()}

    def __call__(self, x, stream=None):
        """Embeddings [rows][dim] in the head's type."""
        with torch.cuda.stream(stream):  # None: the current one
            return self._forward(x, False)[0]

    def _forward(self, x, keep):
        c, x = self._c, x.to(self.dtype)
        a, am, ar = fg.layer_norm(x, c["in_gain"], c["in_offset"])
        h = fg.linear(a, c["w1"], c["b1"], act="gelu", save_pre=keep)
        h, pre = h if keep else (h, None)
        z = fg.linear(h, c["w2"], c["b2"], residual=x if self.skip else None)
        e, zm, zr = fg.layer_norm(z, c["out_gain"], c["out_offset"])
        return e, (x, a, am, ar, h, pre, z, zm, zr) if keep else None

    def _backward(self, de, kept):
        c = self._c
        x, a, am, ar, h, pre, z, zm, zr = kept
        g = {}
        dz, g["out_gain"], g["out_offset"] = fg.layer_norm_backward(de, z, c["out_gain"], zm, zr)
        dh, g["w2"], g["b2"] = fg.linear_backward(dz, h, c["w2"])
        da, g["w1"], g["b1"] = fg.linear_backward(dh, a, c["w1"], pre, act="gelu")
        # the hidden states are the encoder's: their own gradient is not wanted
        _, g["in_gain"], g["in_offset"] = fg.layer_norm_backward(da, x, c["in_gain"], am, ar, want=("gamma", "beta"))
        return g

    def loss(self, x, candidates, targets, scale: float = 1.0, ids=None, grads: bool = True):
        """(mean loss over the rows with a target, gradients by parameter name): targets [rows] index the candidates
        [n][dim] (outside [0, n): no target), whose softmax is that of -scale |q - c|^2 / 2; ids [n] name their documents."""
        cand = candidates.to(self.dtype)
        bias = cand.float().square().sum(1) * (-0.5 * scale)
        live = (targets >= 0) & (targets < cand.shape[0])
        targets = torch.where(live, targets, -1).to(torch.int32)  # before the type's range could wrap one into the candidates
        live = live.float()
        weight = live / live.sum().clamp(min=1)
        e, kept = self._forward(x, grads)
        loss, lse = fg.contrastive_loss(e, cand, targets, scale, bias=bias, ids=ids)
        mean = (loss * weight).sum()
        if not grads:
            return mean, None
        de, _, _ = fg.contrastive_loss_backward(weight, e, cand, targets, lse, scale, bias=bias, ids=ids,
                                                candidate_grads=False)
        return mean, self._backward(de, kept)

    def train_step(self, x, candidates, targets, scale: float = 1.0, ids=None, lr: float = 1e-3, betas=(0.9, 0.98),
                   eps: float = 1e-8):
        """One Adam step on the contrastive loss; returns the mean loss before it (a device scalar)."""
        mean, grads = self.loss(x, candidates, targets, scale, ids)
        self.steps += 1
        rate = lr * math.sqrt(1 - betas[1]**self.steps) / (1 - betas[0]**self.steps)
        for n in self.NAMES:
            g, (m, v) = grads[n].float(), self._moments[n]
            m.lerp_(g, 1 - betas[0])
            v.lerp_(g * g, 1 - betas[1])
            self.params[n] -= rate * m / (v.sqrt() + eps)
        self._cast()
        return mean

    def search(self, index, x, nprobe: int, k: int, stream=None):
        """index.search of the rows' embeddings: (ids, dists)."""
        with torch.cuda.stream(stream):
            return index.search(self(x).float(), nprobe, k)


def demo(n=20000, dim=128, in_dim=768, hidden=1024, steps=300, batch=2048, seed=0, log=print):
    """Hidden states are a fixed random nonlinear view of the answering base vector, plus noise; returns recall@1 of the
    searched index before and after training."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    base = torch.from_numpy(fg.gen_gmm(n, dim, 64, seed=seed + 1, sig_lo=0.3)).cuda()
    view = torch.randn((dim, in_dim), generator=g, device="cuda") / dim**0.5

    def states(rows):
        return torch.tanh(base[rows] @ view) + 0.1 * torch.randn((rows.numel(), in_dim), generator=g, device="cuda")

    index = fg.Index.from_arrays(dim, 32, *fg.build_ivfpq(base, 64, 32, kmeans_iters=8, init_mode=1, pq_iters=6))
    head = QueryHead(in_dim, hidden, dim, seed=seed)
    test = torch.randperm(n, generator=g, device="cuda")[:1000]
    xs = states(test)

    def recall():
        ids, _ = head.search(index, xs, 16, 1)
        return (ids[:, 0].long() == test).float().mean().item()

    before = recall()
    for s in range(steps):
        rows = torch.randint(n, (2 * batch,), generator=g, device="cuda")  # the second half are negatives alone
        t = torch.arange(batch, device="cuda", dtype=torch.int32)
        loss = head.train_step(states(rows[:batch]), base[rows], t, scale=1.0, ids=rows.to(torch.int32), lr=2e-3)
        if log and (s + 1) % 100 == 0:
            log(f"step {s + 1}: loss {loss.item():.3f}")
    after = recall()
    if log:
        log(f"recall@1 of the searched index: {before:.3f} before, {after:.3f} after")
    index.close()
    return before, after


if __name__ == "__main__":
    demo()
