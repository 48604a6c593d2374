"""The operators of a query head (the trained map from an encoder's hidden state to the index's space) as measured cases.

Each case is one call of the library's public entry points, or the two calls of a loss and its gradient: the linear layer
with bias, activation and residual in its epilogue, layer norm, and the softmax contrastive loss of queries against
candidate vectors, forward and backward.  `own` says whether run() makes the library's calls or computes the same in
elementary torch operations in float32.  Inputs come from a seed.
"""
import math

import torch

own = False
DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # One interactive query through one layer of the head: nothing but latency.
        dict(name="linear_one", op="linear", rows=1, k=1024, n=1024, dtype="bf16", act="gelu", bias=True, residual=False,
             save=False),
        # The search pipeline's default batch of 128 queries through the head's widening layer.
        dict(name="linear_b128", op="linear", rows=128, k=768, n=2048, dtype="bf16", act="gelu", bias=True, residual=False,
             save=False),
        # C1's 1000 queries in the index's own type, nothing round, with a skip connection.
        dict(name="linear_ragged_f32", op="linear", rows=1000, k=385, n=771, dtype="f32", act="silu", bias=True,
             residual=True, save=False),
        # The head's widening layer over a training batch, the pre-activation kept for the backward pass.
        dict(name="linear_train", op="linear", rows=65536, k=1024, n=4096, dtype="bf16", act="gelu", bias=True,
             residual=False, save=True),
        # Its gradients over a smaller training batch.
        dict(name="linear_bwd", op="linear_bwd", rows=16384, k=1024, n=4096, dtype="bf16", act="gelu"),
        # Gradients of a layer into the index's 96 dims, in float32, over an odd number of rows.
        dict(name="linear_bwd_f32", op="linear_bwd", rows=4099, k=771, n=96, dtype="f32", act="relu"),
        # The layer norm in front of the head for one interactive query.
        dict(name="norm_one", op="norm", rows=1, dim=1024, dtype="bf16"),
        # A base's embeddings normalised before an index is built over them: odd rows, odd dims, float32.
        dict(name="norm_rows_f32", op="norm", rows=100_003, dim=771, dtype="f32"),
        # The training batch's layer norm gradients.
        dict(name="norm_bwd", op="norm_bwd", rows=65536, dim=1024, dtype="bf16"),
        # In-batch negatives: every query against every query's document, in the index's 128 dims.
        dict(name="contrast_inbatch", op="contrast", nq=1024, nc=1024, dim=128, dtype="bf16", fixed=False, dups=0.02,
             masked=0.0, ignored=0.0),
        # C1's 1000 queries against its whole base (fixed candidates, the index's L2 metric through the bias), float32.
        dict(name="contrast_base_f32", op="contrast", nq=1000, nc=100_000, dim=128, dtype="f32", fixed=True, dups=0.0,
             masked=0.001, ignored=0.01),
        # A large training step against its documents and their mined hard negatives, wide embeddings.
        dict(name="contrast_hard", op="contrast", nq=8192, nc=65536, dim=768, dtype="bf16", fixed=False, dups=0.01,
             masked=0.001, ignored=0.01),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):  # two in three are multiples of 8, as layer widths are
        w = log(lo, hi)
        return w if rng.random() < 1 / 3 else max(8, w // 8 * 8)

    op = rng.choice(["linear", "linear", "linear_bwd", "linear_bwd", "norm", "norm_bwd", "contrast", "contrast"])
    c = dict(op=op, dtype=rng.choice(["f32", "bf16", "bf16"]))
    small = 4 if c["dtype"] == "f32" else 1
    if op == "linear":
        c.update(rows=log(1, 65536 // small), k=width(64, 2048), n=width(64, 2048),
                 act=rng.choice(["none", "relu", "gelu", "silu"]), bias=rng.random() < 0.8, residual=rng.random() < 0.4,
                 save=rng.random() < 0.4)
    elif op == "linear_bwd":
        c.update(rows=log(16, 32768 // small), k=width(64, 2048), n=width(64, 2048),
                 act=rng.choice(["none", "relu", "gelu", "silu"]))
    elif op in ("norm", "norm_bwd"):
        c.update(rows=log(1, 131072 // small), dim=width(64, 4096))
    else:
        fixed = rng.random() < 0.4
        nq = log(32, 8192 // small)
        c.update(nq=nq, nc=max(nq, log(256, 65536 // small)), dim=rng.choice([96, 128, 128, width(64, 1024)]), fixed=fixed,
                 dups=rng.choice([0.0, 0.01, 0.05]), masked=rng.choice([0.0, 0.001, 0.02]),
                 ignored=rng.choice([0.0, 0.01, 0.2]))
    return c


# ---- inputs -------------------------------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1009 + 17)
    t, op = DTYPES[case["dtype"]], case["op"]
    s = dict(case=dict(case))
    if op in ("linear", "linear_bwd"):
        m, k, n = case["rows"], case["k"], case["n"]
        # Normalised activations and weights of a trained layer's scale: pre-activations of about unit size.
        s["x"], s["w"] = _normal(g, m, k).to(t), (_normal(g, n, k) / math.sqrt(k)).to(t)
        if op == "linear":
            s["b"] = (_normal(g, n) * 0.1).to(t) if case["bias"] else None
            s["r"] = _normal(g, m, n).to(t) if case["residual"] else None
        else:
            s["dy"] = (_normal(g, m, n) * 1e-2).to(t)
            s["pre"] = _normal(g, m, n).to(t) if case["act"] != "none" else None
    elif op in ("norm", "norm_bwd"):
        r, d = case["rows"], case["dim"]
        # Hidden states: rows of different scale and offset, a few dims far larger than the rest.
        x = _normal(g, r, d) * (0.5 + 2 * torch.rand((r, 1), generator=g, device=DEV)) + 0.3 * _normal(g, r, 1)
        x *= torch.where(torch.rand((d,), generator=g, device=DEV) < 0.005, 8.0, 1.0)
        s["x"] = x.to(t)
        s["g"], s["b"] = (1 + 0.2 * _normal(g, d)).to(t), (0.1 * _normal(g, d)).to(t)
        if op == "norm_bwd":
            s["dy"] = (_normal(g, r, d) * 1e-2).to(t)
            v = s["x"].float()
            s["mean"] = v.mean(1)
            s["rstd"] = torch.rsqrt((v - s["mean"][:, None]).square().mean(1) + 1e-5)
    else:
        nq, nc, d = case["nq"], case["nc"], case["dim"]
        c = _normal(g, nc, d)
        c *= (1 + 0.05 * _normal(g, nc, 1)) / c.norm(dim=1, keepdim=True)
        tgt = torch.randperm(nc, generator=g, device=DEV)[:nq] if case["fixed"] else torch.arange(nq, device=DEV)
        q = 0.35 * c[tgt] + 0.65 * _normal(g, nq, d) / math.sqrt(d)  # half trained: neither sure nor blind
        q /= q.norm(dim=1, keepdim=True)
        ids = torch.randint(1 << 30, (nc,), generator=g, device=DEV, dtype=torch.int32)
        dup = torch.rand((nc,), generator=g, device=DEV) < case["dups"]  # copies of other candidates' documents
        ids = torch.where(dup, ids[torch.randint(nc, (nc,), generator=g, device=DEV)], ids)
        s["q"], s["c"] = q.to(t), c.to(t)
        s["scale"] = 20.0
        bias = -0.5 * s["scale"] * s["c"].float().square().sum(1)  # the L2 metric
        hide = torch.rand((nc,), generator=g, device=DEV) < case["masked"]
        hide[tgt] = False
        s["bias"] = torch.where(hide, -math.inf, bias)
        skip = torch.rand((nq,), generator=g, device=DEV) < case["ignored"]
        s["tgt"] = torch.where(skip, -1, tgt).to(torch.int32)
        s["ids"] = ids
        s["dloss"] = torch.full((nq,), 1.0 / nq, device=DEV)
    return s


# ---- the library's calls ------------------------------------------------------------------------------------------
def _run_own(s):
    import fusiongpu_amd as fg

    c = s["case"]
    if c["op"] == "linear":
        r = fg.linear(s["x"], s["w"], s["b"], s["r"], act=c["act"], save_pre=c["save"])
        return dict(y=r[0], pre=r[1]) if c["save"] else dict(y=r)
    if c["op"] == "linear_bwd":
        dx, dw, db = fg.linear_backward(s["dy"], s["x"], s["w"], s["pre"], act=c["act"])
        return dict(dx=dx, dw=dw, db=db)
    if c["op"] == "norm":
        y, mean, rstd = fg.layer_norm(s["x"], s["g"], s["b"], eps=1e-5)
        return dict(y=y, mean=mean, rstd=rstd)
    if c["op"] == "norm_bwd":
        dx, dg, db = fg.layer_norm_backward(s["dy"], s["x"], s["g"], s["mean"], s["rstd"])
        return dict(dx=dx, dg=dg, db=db)
    loss, lse = fg.contrastive_loss(s["q"], s["c"], s["tgt"], s["scale"], bias=s["bias"], ids=s["ids"])
    dq, dc, dbias = fg.contrastive_loss_backward(s["dloss"], s["q"], s["c"], s["tgt"], lse, s["scale"], bias=s["bias"],
                                                 ids=s["ids"], candidate_grads=not c["fixed"])
    out = dict(loss=loss, lse=lse, dq=dq)
    return out if c["fixed"] else dict(out, dc=dc, dbias=dbias)


# ---- the plain form -----------------------------------------------------------------------------------------------
def _phi(z):
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))


def _act(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: z * _phi(z),
            "silu": lambda: z * torch.sigmoid(z)}[act]()


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return _phi(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    sg = torch.sigmoid(z)
    return sg * (1 + z * (1 - sg))


def _run_plain(s):
    c = s["case"]
    t = DTYPES[c["dtype"]]
    if c["op"] == "linear":
        z = s["x"].float() @ s["w"].float().t()
        if s["b"] is not None:
            z = z + s["b"].float()
        y = _act(z, c["act"])
        if s["r"] is not None:
            y = y + s["r"].float()
        return dict(y=y.to(t), pre=z.to(t)) if c["save"] else dict(y=y.to(t))
    if c["op"] == "linear_bwd":
        dz = s["dy"].float()
        if c["act"] != "none":
            dz = dz * _act_grad(s["pre"].float(), c["act"])
        return dict(dx=(dz @ s["w"].float()).to(t), dw=(dz.t() @ s["x"].float()).to(t), db=dz.sum(0).to(t))
    if c["op"] == "norm":
        x = s["x"].float()
        mean = x.mean(1)
        h = x - mean[:, None]
        rstd = torch.rsqrt(h.square().mean(1) + 1e-5)
        return dict(y=(h * rstd[:, None] * s["g"].float() + s["b"].float()).to(t), mean=mean, rstd=rstd)
    if c["op"] == "norm_bwd":
        dy = s["dy"].float()
        h = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        u = dy * s["g"].float()
        dx = (u - u.mean(1, keepdim=True) - h * (u * h).mean(1, keepdim=True)) * s["rstd"][:, None]
        return dict(dx=dx.to(t), dg=(dy * h).sum(0).to(t), db=dy.sum(0).to(t))
    q, cand, tgt = s["q"].float(), s["c"].float(), s["tgt"].long()
    live = tgt >= 0
    tc = tgt.clamp(min=0)[:, None]
    sc = s["scale"] * (q @ cand.t()) + s["bias"]
    other = torch.arange(c["nc"], device=DEV) != tc
    sc = sc.masked_fill((s["ids"] == s["ids"][tc]) & other & live[:, None], -math.inf)
    top = sc.amax(1, keepdim=True)
    e = torch.exp(sc - top)
    z = e.sum(1, keepdim=True)
    lse = (top + torch.log(z))[:, 0]
    loss = torch.where(live, lse - sc.gather(1, tc)[:, 0], 0.0)
    gr = (e / z - (~other).float()) * (s["dloss"] * live)[:, None]
    out = dict(loss=loss, lse=lse, dq=(s["scale"] * (gr @ cand)).to(t))
    if c["fixed"]:
        return out
    return dict(out, dc=(s["scale"] * (gr.t() @ q)).to(t), dbias=gr.sum(0))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    e, op = DTYPES[case["dtype"]].itemsize, case["op"]
    if op == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return dict(bytes=e * (m * k + n * k + n * case["bias"] + m * n * (1 + case["residual"] + case["save"])),
                    flops=2 * m * n * k)
    if op == "linear_bwd":
        m, k, n = case["rows"], case["k"], case["n"]
        return dict(bytes=e * (2 * m * k + 2 * n * k + n + m * n * (1 + (case["act"] != "none"))), flops=4 * m * n * k)
    if op == "norm":
        return dict(bytes=e * (2 * case["rows"] + 2) * case["dim"] + 8 * case["rows"], flops=8 * case["rows"] * case["dim"])
    if op == "norm_bwd":
        return dict(bytes=e * (3 * case["rows"] + 3) * case["dim"] + 8 * case["rows"], flops=12 * case["rows"] * case["dim"])
    # The scores, and each gradient's product; the scores need not be computed twice.
    nq, nc, d = case["nq"], case["nc"], case["dim"]
    return dict(bytes=e * d * (2 * nq + nc * (1 if case["fixed"] else 2)) + 16 * nq + 8 * nc + 4 * nc * (not case["fixed"]),
                flops=(4 if case["fixed"] else 6) * nq * nc * d)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    f = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    if op == "linear":
        pre = torch.mm(f["x"], f["w"].t().contiguous())
        if f["b"] is not None:
            pre += f["b"][None]
        y = pre
        if case["act"] == "relu":
            y = torch.where(pre > 0, pre, 0.0)
        elif case["act"] == "gelu":
            y = pre * torch.special.erfc(-pre / math.sqrt(2.0)) / 2
        elif case["act"] == "silu":
            y = pre / (1 + torch.exp(-pre))
        if f["r"] is not None:
            y = y + f["r"]
        return dict(y=y, pre=pre) if case["save"] else dict(y=y)
    if op == "linear_bwd":
        dz, p = f["dy"], f["pre"]
        if case["act"] == "relu":
            dz = torch.where(p > 0, dz, 0.0)
        elif case["act"] == "gelu":
            dz = dz * (torch.special.erfc(-p / math.sqrt(2.0)) / 2 + p * torch.exp(-p * p / 2) / math.sqrt(2 * math.pi))
        elif case["act"] == "silu":
            en = torch.exp(-p)
            dz = dz * (1 / (1 + en) + p * en / (1 + en) ** 2)
        return dict(dx=torch.mm(dz, f["w"]), dw=torch.mm(dz.t().contiguous(), f["x"]), db=dz.sum(dim=0))
    if op == "norm":
        var, mean = torch.var_mean(f["x"], dim=1, correction=0)
        rstd = 1 / torch.sqrt(var + 1e-5)
        return dict(y=torch.addcmul(f["b"], (f["x"] - mean[:, None]) * rstd[:, None], f["g"]), mean=mean, rstd=rstd)
    if op == "norm_bwd":
        x, rs, d = f["x"], f["rstd"][:, None], case["dim"]
        h = (x - f["mean"][:, None]) * rs
        gu = f["dy"] * f["g"]
        dx = rs / d * (d * gu - gu.sum(1, keepdim=True) - h * (h * gu).sum(1, keepdim=True))
        return dict(dx=dx, dg=torch.einsum("rd,rd->d", f["dy"], h), db=f["dy"].sum(dim=0))
    q, c, nq, nc = f["q"], f["c"], case["nq"], case["nc"]
    loss, lse = torch.zeros(nq, dtype=torch.float64, device=DEV), torch.zeros(nq, dtype=torch.float64, device=DEV)
    dq, dc, dbias = torch.zeros_like(q), torch.zeros_like(c), torch.zeros(nc, dtype=torch.float64, device=DEV)
    for b in range(0, nq, 2048):
        t = s["tgt"][b:b + 2048].long()
        rows = torch.arange(t.numel(), device=DEV)
        live, at = t >= 0, t.clamp(min=0)
        sc = torch.addmm(f["bias"], q[b:b + 2048], c.t().contiguous(), alpha=s["scale"])
        same = s["ids"][None, :] == s["ids"][at][:, None]
        same[rows, at] = False
        same[~live] = False
        sc[same] = -math.inf
        lse[b:b + 2048] = torch.logsumexp(sc, dim=1)
        loss[b:b + 2048] = torch.where(live, lse[b:b + 2048] - sc[rows, at], 0.0)
        gr = torch.softmax(sc, dim=1)
        gr[rows, at] -= 1
        gr *= torch.where(live, f["dloss"][b:b + 2048], 0.0)[:, None]
        dq[b:b + 2048] = s["scale"] * torch.mm(gr, c)
        dc += s["scale"] * torch.mm(gr.t().contiguous(), q[b:b + 2048])
        dbias += gr.sum(dim=0)
    out = dict(loss=loss, lse=lse, dq=dq)
    return out if case["fixed"] else dict(out, dc=dc, dbias=dbias)
