"""A gated block of the query head as measured cases: trained, its updates orthogonalised, and served in 8-bit integers.

Each case is one call of the library's public entry points: the gated layer act(x Wg^T + bg) (x Wu^T + bu) and its
gradients, the orthogonalisation of a weight's update by Newton-Schulz products, the rounding of rows to 8-bit integers
with a scale each, and the linear and the gated layer on such weights.  `own` says whether run() makes the library's calls
or computes the same in elementary torch operations in float32.  Inputs come from a seed.
"""
import math

import torch

own = False
DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def listed():
    return [
        # One interactive query through the gated layer: nothing but latency.
        dict(name="gated_one", op="gated", rows=1, k=1024, n=2048, dtype="bf16", act="silu", bias=True, save=False),
        # C1's 1000 queries in the index's own type, nothing round.
        dict(name="gated_ragged_f32", op="gated", rows=1000, k=385, n=771, dtype="f32", act="gelu", bias=True, save=False),
        # A training batch through the gated layer, both pre-activations kept for the backward pass.
        dict(name="gated_train", op="gated", rows=65536, k=1024, n=4096, dtype="bf16", act="silu", bias=True, save=True),
        # Its gradients over a smaller training batch.
        dict(name="gated_bwd", op="gated_bwd", rows=16384, k=1024, n=4096, dtype="bf16", act="silu"),
        # Gradients of a narrow gated layer in float32, over an odd number of rows.
        dict(name="gated_bwd_f32", op="gated_bwd", rows=4099, k=771, n=96, dtype="f32", act="gelu"),
        # One interactive query through a linear layer with 8-bit weights: a quarter of a float32 layer's bytes.
        dict(name="int8_one", op="int8", rows=1, k=1024, n=4096, dtype="bf16", act="gelu", bias=True, residual=False,
             gated=False),
        # C1's 1000 queries in float32 through a linear layer with a skip connection, nothing round.
        dict(name="int8_ragged_f32", op="int8", rows=1000, k=385, n=771, dtype="f32", act="silu", bias=True, residual=True,
             gated=False),
        # A base's embeddings through the gated layer before an index is built over them.
        dict(name="int8_base", op="int8", rows=65536, k=1024, n=4096, dtype="bf16", act="silu", bias=True, residual=False,
             gated=True),
        # A trained layer's float32 weight, laid out once for serving.
        dict(name="quantize_weight_f32", op="quantize", rows=771, dim=385, dtype="f32"),
        # A base's hidden states.
        dict(name="quantize_base", op="quantize", rows=100_003, dim=1024, dtype="bf16"),
        # The update of the layer into the index's 128 dims, in float32: short products, one after the other.
        dict(name="ortho_small_f32", op="ortho", rows=128, cols=771, dtype="f32", steps=5),
        # The update of the gated layer's stacked weight, far taller than wide.
        dict(name="ortho_train", op="ortho", rows=8192, cols=1024, dtype="bf16", steps=5),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):  # two in three are multiples of 8, as layer widths are
        w = log(lo, hi)
        return w if rng.random() < 1 / 3 else max(8, w // 8 * 8)

    op = rng.choice(["gated", "gated", "gated_bwd", "gated_bwd", "int8", "int8", "int8", "quantize", "ortho", "ortho"])
    c = dict(op=op, dtype=rng.choice(["f32", "bf16", "bf16"]))
    small = 4 if c["dtype"] == "f32" else 1
    if op == "gated":
        c.update(rows=log(1, 65536 // small), k=width(64, 2048), n=width(64, 2048),
                 act=rng.choice(["none", "relu", "gelu", "silu", "silu"]), bias=rng.random() < 0.5, save=rng.random() < 0.5)
    elif op == "gated_bwd":
        c.update(rows=log(16, 32768 // small), k=width(64, 2048), n=width(64, 2048),
                 act=rng.choice(["none", "relu", "gelu", "silu", "silu"]))
    elif op == "int8":
        gated = rng.random() < 0.4
        c.update(rows=log(1, 65536), k=width(64, 2048), n=width(64, 2048), act=rng.choice(["none", "relu", "gelu", "silu"]),
                 bias=rng.random() < 0.7, residual=not gated and rng.random() < 0.4, gated=gated)
    elif op == "quantize":
        c.update(rows=log(1, 131072), dim=width(64, 4096))
    else:
        c.update(rows=width(32, 4096), cols=width(32, 2048), steps=rng.choice([5, 5, 6]))
    return c


# ---- 8-bit rows -----------------------------------------------------------------------------------------------------
def _row(dim):  # a row's bytes: whole groups of 16, zeros behind the values
    return (dim + 15) // 16 * 16


def _codes(x):
    """(whole numbers [rows][dim], scales [rows]): x 127 / amax to the nearest, in 64 bits, where the borders between two
    numbers are what they are."""
    top = x.float().abs().amax(1)
    safe = torch.where(top > 0, top, 1.0).double()[:, None]
    return torch.round(x.double() * 127 / safe), top / 127


# ---- inputs -------------------------------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _hidden(gen, rows, dim):
    """Hidden states: rows of different scale, a few dims far larger than the rest."""
    x = _normal(gen, rows, dim) * (0.5 + 2 * torch.rand((rows, 1), generator=gen, device=DEV))
    return x * torch.where(torch.rand((dim,), generator=gen, device=DEV) < 0.005, 8.0, 1.0)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1009 + 29)
    t, op = DTYPES[case["dtype"]], case["op"]
    s = dict(case=dict(case))
    if op in ("gated", "gated_bwd"):
        m, k, n = case["rows"], case["k"], case["n"]
        # Normalised activations and weights of a trained layer's scale: pre-activations of about unit size.
        s["x"], s["w"] = _normal(g, m, k).to(t), (_normal(g, 2 * n, k) / math.sqrt(k)).to(t)
        if op == "gated":
            s["b"] = (_normal(g, 2 * n) * 0.1).to(t) if case["bias"] else None
        else:
            s["dh"], s["pre"] = (_normal(g, m, n) * 1e-2).to(t), _normal(g, m, 2 * n).to(t)
    elif op == "int8":
        m, k, n = case["rows"], case["k"], case["n"] * (2 if case["gated"] else 1)
        s["x"] = _hidden(g, m, k).to(t)
        q, s["ws"] = _codes(_normal(g, n, k) / math.sqrt(k))
        s["w"] = torch.zeros((n, _row(k)), dtype=torch.int8, device=DEV)
        s["w"][:, :k] = q
        s["b"] = (_normal(g, n) * 0.1).to(t) if case["bias"] else None
        s["r"] = _normal(g, m, n).to(t) if case["residual"] else None
    elif op == "quantize":
        s["x"] = _hidden(g, case["rows"], case["dim"]).to(t)
    else:
        # Momentum of a weight: a few strong directions, ever weaker, over the noise of its batches.
        m, n = case["rows"], case["cols"]
        r = max(1, min(m, n) // 8)
        strong = _normal(g, m, r) / torch.arange(1, r + 1, device=DEV)
        s["x"] = (1e-3 * (_normal(g, m, n) + strong @ _normal(g, r, n))).to(t)
    return s


# ---- the library's calls ------------------------------------------------------------------------------------------
def _run_own(s):
    import fusiongpu_amd as fg

    c = s["case"]
    if c["op"] == "gated":
        r = fg.gated_linear(s["x"], s["w"], s["b"], act=c["act"], save_pre=c["save"])
        return dict(h=r[0], pre=r[1]) if c["save"] else dict(h=r)
    if c["op"] == "gated_bwd":
        dx, dw, db = fg.gated_linear_backward(s["dh"], s["x"], s["w"], s["pre"], act=c["act"])
        return dict(dx=dx, dw=dw, db=db)
    if c["op"] == "int8":
        if c["gated"]:
            return dict(y=fg.gated_linear_int8(s["x"], s["w"], s["ws"], s["b"], act=c["act"]))
        return dict(y=fg.linear_int8(s["x"], s["w"], s["ws"], s["b"], s["r"], act=c["act"]))
    if c["op"] == "quantize":
        q, scale = fg.quantize_rows(s["x"])
        return dict(x=q[:, :c["dim"]] * scale[:, None], scale=scale)
    return dict(y=fg.orthogonalize(s["x"], steps=c["steps"], coefficients=COEFFICIENTS))


# ---- the plain form -----------------------------------------------------------------------------------------------
def _phi(z):
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))


def _act(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: z * _phi(z),
            "silu": lambda: z * torch.sigmoid(z)}[act]()


def _act_grad(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return _phi(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    sg = torch.sigmoid(z)
    return sg * (1 + z * (1 - sg))


def _step(x, tall):
    """One Newton-Schulz step; the square products are those of the shorter side."""
    a, b, c = COEFFICIENTS
    g = x.t() @ x if tall else x @ x.t()
    p = b * g + c * (g @ g)
    return a * x + (x @ p if tall else p @ x)


def _run_plain(s):
    c = s["case"]
    t, n = DTYPES[c["dtype"]], c.get("n")
    if c["op"] == "gated":
        z = s["x"].float() @ s["w"].float().t()
        if s["b"] is not None:
            z = z + s["b"].float()
        h = (_act(z[:, :n], c["act"]) * z[:, n:]).to(t)
        return dict(h=h, pre=z.to(t)) if c["save"] else dict(h=h)
    if c["op"] == "gated_bwd":
        dh, g, u = s["dh"].float(), s["pre"][:, :n].float(), s["pre"][:, n:].float()
        dz = torch.cat([dh * u * _act_grad(g, c["act"]), dh * _act(g, c["act"])], 1)
        return dict(dx=(dz @ s["w"].float()).to(t), dw=(dz.t() @ s["x"].float()).to(t), db=dz.sum(0).to(t))
    if c["op"] == "int8":
        q, scale = _codes(s["x"])
        y = (q.float() @ s["w"][:, :c["k"]].float().t()) * scale[:, None] * s["ws"]
        if s["b"] is not None:
            y = y + s["b"].float()
        y = _act(y[:, :n], c["act"]) * y[:, n:] if c["gated"] else _act(y, c["act"])
        if s["r"] is not None:
            y = y + s["r"].float()
        return dict(y=y.to(t))
    if c["op"] == "quantize":
        q, scale = _codes(s["x"])
        return dict(x=q.float() * scale[:, None], scale=scale)
    x = s["x"].float()
    x = x / (x.norm() + 1e-7)
    for _ in range(c["steps"]):
        x = _step(x, c["rows"] > c["cols"])
    return dict(y=x.to(t))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    e, op = DTYPES[case["dtype"]].itemsize, case["op"]
    if op == "gated":
        m, k, n = case["rows"], case["k"], case["n"]
        return dict(bytes=e * (m * k + 2 * n * k + 2 * n * case["bias"] + m * n * (1 + 2 * case["save"])),
                    flops=4 * m * n * k)
    if op == "gated_bwd":
        m, k, n = case["rows"], case["k"], case["n"]
        return dict(bytes=e * (2 * m * k + 4 * n * k + 2 * n + 3 * m * n), flops=8 * m * n * k)
    if op == "int8":
        m, k, n, both = case["rows"], case["k"], case["n"], 1 + case["gated"]
        return dict(bytes=e * (m * k + m * n * (1 + case["residual"]) + both * n * case["bias"]) + both * n * (k + 4),
                    flops=2 * both * m * n * k)
    if op == "quantize":
        m, d = case["rows"], case["dim"]
        return dict(bytes=m * d * (e + 1) + 4 * m, flops=3 * m * d)
    # Of the two square products half, as they are symmetric.
    s, l = sorted((case["rows"], case["cols"]))
    return dict(bytes=2 * e * s * l, flops=case["steps"] * (s * s * l + s * s * s + 2 * s * s * l))


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _act64(p, act):
    """(value, slope)"""
    if act == "relu":
        on = (p > 0).double()
        return p * on, on
    if act == "gelu":
        cdf = torch.special.erfc(-p / math.sqrt(2.0)) / 2
        return p * cdf, cdf + p * torch.exp(-p * p / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        en = torch.exp(-p)
        return p / (1 + en), 1 / (1 + en) + p * en / (1 + en) ** 2
    return p, torch.ones_like(p)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    f = {k: v.double() if torch.is_tensor(v) else v for k, v in s.items()}
    if op == "gated":
        gate, up = torch.mm(f["x"], f["w"].t().contiguous()).chunk(2, dim=1)
        if f["b"] is not None:
            bg, bu = f["b"].chunk(2)
            gate, up = gate + bg, up + bu
        h = _act64(gate, case["act"])[0] * up
        return dict(h=h, pre=torch.cat([gate, up], dim=1)) if case["save"] else dict(h=h)
    if op == "gated_bwd":
        gate, up = f["pre"].chunk(2, dim=1)
        value, slope = _act64(gate, case["act"])
        dg, du = f["dh"] * up * slope, f["dh"] * value
        wg, wu = f["w"].chunk(2, dim=0)
        xs = f["x"]
        return dict(dx=torch.mm(dg, wg) + torch.mm(du, wu),
                    dw=torch.cat([torch.mm(dg.t().contiguous(), xs), torch.mm(du.t().contiguous(), xs)]),
                    db=torch.cat([dg.sum(dim=0), du.sum(dim=0)]))
    if op in ("int8", "quantize"):
        amax = f["x"].abs().max(dim=1, keepdim=True).values
        unit = torch.where(amax > 0, amax, 1.0)
        near = torch.round(f["x"] * 127.0 / unit)
        if op == "quantize":
            return dict(x=near * (amax / 127.0), scale=(amax / 127.0)[:, 0])
        z = torch.mm(near, f["w"][:, :case["k"]].t().contiguous()) * (amax / 127.0) * f["ws"][None]
        if f["b"] is not None:
            z += f["b"][None]
        if case["gated"]:
            gate, up = z.chunk(2, dim=1)
            return dict(y=_act64(gate, case["act"])[0] * up)
        y = _act64(z, case["act"])[0]
        return dict(y=y if f["r"] is None else y + f["r"])
    x = f["x"] / (torch.linalg.vector_norm(f["x"]) + 1e-7)
    flip = case["rows"] > case["cols"]
    x = x.t().contiguous() if flip else x
    a, b, c = COEFFICIENTS
    for _ in range(case["steps"]):
        gram = torch.mm(x, x.t().contiguous())
        x = a * x + torch.mm(torch.addmm(gram, gram, gram, beta=b, alpha=c), x)
    return dict(y=x.t().contiguous() if flip else x)
