"""The query head's operators against their definitions in 64 bits.

Bounds are derived, not fitted.  u = 2^-24.  A float32 sum of n products is off by at most (n + c) u times the sum of
their magnitudes (c for the products, the split float32 operands' dropped terms and what follows the sum); a result in
bfloat16 adds half a unit of its last place, at most 2^-8 of the result (eight significant bits).  Where bfloat16 operands are made inside a call (dz, the
score gradient), each term carries another 2^-8.
"""
import math

import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0**-24
LOWEST = torch.finfo(torch.float32).min
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def rnd(seed, *shape, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def within(got, want, bound, what):
    """|got - want| <= bound + half a last place of got's type, element by element."""
    got = got.double()
    off = (got - want).abs() - (bound + HALF_OF[what[1]] * (want.abs() + bound))
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 1e-37, f"{what}: {worst} over the bound at {torch.argmax(off).item()}"


HALF_OF = {"f32": 2 * U, "bf16": 2.0**-8}


def phi(z):
    return torch.special.erfc(-z * math.sqrt(0.5)) / 2


def act64(z, act):
    return {"none": z, "relu": z.clamp(min=0), "gelu": z * phi(z), "silu": z * torch.sigmoid(z)}[act]


def slope64(z, act):
    s = torch.sigmoid(z)
    return {"none": torch.ones_like(z), "relu": (z > 0).double(),
            "gelu": phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), "silu": s * (1 + z * (1 - s))}[act]


# ---- linear ---------------------------------------------------------------------------------------------------------
# One row and one of everything, sizes around a tile (64, 128, 256) and around 8 and 16, odd strides, k split, wide and tall.
LINEAR = [(1, 1, 1), (1, 64, 64), (1, 1000, 33), (2, 8, 1030), (3, 7, 5), (5, 129, 2), (8, 1024, 512), (16, 100, 17),
          (17, 512, 64), (31, 4096, 24), (33, 65, 63), (64, 64, 64), (65, 72, 130), (127, 8, 129), (200, 100, 77),
          (300, 513, 257), (257, 2056, 255), (1000, 385, 771), (2048, 256, 520), (16390, 64, 1028)]


def check_linear(m, k, n, dt, act, bias, residual, save, seed=0, x=None):
    t = TYPES[dt]
    x = rnd(seed + 1, m, k, dtype=t) if x is None else x
    w = rnd(seed + 2, n, k, scale=1 / math.sqrt(k), dtype=t)
    b = rnd(seed + 3, n, dtype=t) if bias else None
    r = rnd(seed + 4, m, n, dtype=t) if residual else None
    got = fg.linear(x, w, b, r, act=act, save_pre=save)
    y, pre = got if save else (got, None)
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if bias:
        z, mag = z + b.double(), mag + b.double().abs()
    zb = (k + 12) * U * mag
    if save:
        assert pre.dtype == t
        within(pre, z, zb, ("pre", dt, m, k, n))
    # slopes of the activations are at most 1.13; their own error: 1.5e-7 of z for the normal distribution's tail and a
    # few roundings of the value
    want = act64(z, act)
    yb = 1.13 * zb + (2e-7 * z.abs() + 8 * U * want.abs() if act != "none" else 0)
    if residual:
        want = want + r.double()
        yb = yb + 2 * U * (want.abs() + r.double().abs())
    assert y.dtype == t and y.shape == (m, n)
    within(y, want, yb, ("y", dt, m, k, n, act))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", LINEAR)
def test_linear(m, k, n, dt):
    check_linear(m, k, n, dt, "gelu", True, False, True)
    check_linear(m, k, n, dt, "none", False, True, False, seed=10)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("m", [1, 9, 150])
def test_linear_activations(act, dt, m):
    check_linear(m, 96, 128, dt, act, True, True, True)


@pytest.mark.parametrize("act", ["gelu", "silu", "relu"])
def test_activation_far_out(act):
    """Large pre-activations of both signs: finite, and exactly zero or z where the activation is."""
    z = torch.tensor([[-3e38, -1e4, -90.0, -40.0, -13.0, 0.0, 13.0, 40.0, 90.0, 1e4, 3e38]], device="cuda")
    y = fg.linear(torch.ones((1, 1), device="cuda"), torch.zeros((11, 1), device="cuda"), bias=z[0], act=act)
    want = act64(z.double(), act)
    assert torch.isfinite(y).all()
    assert (y.double() - want).abs().le(1e-6 + 8 * U * want.abs()).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (5, 9, 3), (64, 64, 64), (65, 130, 72), (100, 77, 100), (300, 257, 513),
                                   (1000, 385, 96), (4099, 100, 64), (520, 1028, 2056), (16385, 72, 128)])
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_backward(m, k, n, dt, act):
    t = TYPES[dt]
    dy, x, w = rnd(1, m, n, dtype=t), rnd(2, m, k, dtype=t), rnd(3, n, k, scale=1 / math.sqrt(k), dtype=t)
    pre = rnd(4, m, n, scale=1.5, dtype=t) if act != "none" else None
    dx, dw, db = fg.linear_backward(dy, x, w, pre, act=act)
    check_linear_grads(dy, x, w, pre, act, dt, dx, dw, db)


def check_linear_grads(dy, x, w, pre, act, dt, dx, dw, db):
    (m, n), k = dy.shape, x.shape[1]
    d, x, w = dy.double(), x.double(), w.double()
    dz, dze = d, torch.zeros_like(d)
    if act != "none":
        z = pre.double()
        dz = d * slope64(z, act)
        dze = d.abs() * (4e-7 * (1 + z.abs()) + 8 * U)  # the slope's error
    one = dze + (2.0**-8 * dz.abs() if dt == "bf16" and act != "none" else 0)  # dz as an operand
    within(dx, dz @ w, one @ w.abs() + (n + 12) * U * (dz.abs() @ w.abs()), ("dx", dt, m, k, n, act))
    within(dw, dz.t() @ x, one.t() @ x.abs() + (m + 12) * U * (dz.abs().t() @ x.abs()), ("dw", dt, m, k, n, act))
    within(db, dz.sum(0), dze.sum(0) + (m + 4) * U * dz.abs().sum(0), ("db", dt, m, k, n, act))


@pytest.mark.parametrize("want", [("x",), ("weight",), ("bias",), ("x", "bias"), ()])
def test_linear_backward_of_some(want):
    dy, x, w, pre = rnd(1, 70, 50), rnd(2, 70, 30), rnd(3, 50, 30), rnd(4, 70, 50)
    full = dict(zip(("x", "weight", "bias"), fg.linear_backward(dy, x, w, pre, act="silu")))
    some = dict(zip(("x", "weight", "bias"), fg.linear_backward(dy, x, w, pre, act="silu", want=want)))
    for name, v in some.items():
        assert (v is None) == (name not in want)
        assert v is None or torch.equal(v, full[name])


@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
def test_linear_gradient_against_differences(act):
    """d/de of sum(dy * linear(x + e v)) by central differences of the forward pass.  Third derivatives of the
    activations are below 2, so the difference's own error is e^2 / 3 |dy| |v|^3; the rounding of y adds u / e."""
    m, k, n, e = 37, 45, 51, 2.0**-7
    x, w, b, dy = rnd(1, m, k), rnd(2, n, k, scale=1 / math.sqrt(k)), rnd(3, n), rnd(4, m, n)
    _, pre = fg.linear(x, w, b, act=act, save_pre=True)
    grads = fg.linear_backward(dy, x, w, pre, act=act)
    for i, (p, g) in enumerate(zip((x, w, b), grads)):
        v = rnd(10 + i, *p.shape)
        args = [x, w, b]

        def at(s):
            args[i] = p + s * v
            return (dy.double() * fg.linear(*args, act=act).double()).sum()

        diff = ((at(e) - at(-e)) / (2 * e)).item()
        dzv = [lambda: v.double() @ w.double().t(), lambda: x.double() @ v.double().t(), lambda: v.double().expand(m, n)][i]()
        bound = (dy.double().abs() * (e * e / 3 * dzv.abs()**3 + 200 * U / e * (1 + pre.double().abs()))).sum().item()
        assert abs(diff - (g.double() * v.double()).sum().item()) <= bound


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_linear_views(dt):
    """Strided, transposed and unaligned views, as a caller slices them, against their contiguous copies."""
    t = TYPES[dt]
    big = rnd(1, 70, 200, dtype=t)
    for x in (big[:, 3:99], big[1::2, :96], big.t()[:96, 5:].t(), big.reshape(-1)[1:1 + 60 * 96].view(60, 96)):
        w = rnd(2, 50, 97, dtype=t)[:, 1:]
        assert torch.equal(fg.linear(x, w), fg.linear(x.contiguous().clone(), w.contiguous().clone()))


def test_linear_in_place_residual_and_numpy():
    x, w, r = rnd(1, 33, 40), rnd(2, 24, 40), rnd(3, 33, 24)
    want = fg.linear(x, w, residual=r)
    assert torch.equal(fg.linear(x, w, residual=r, out=r), want) and torch.equal(r, want)
    assert torch.equal(fg.linear(x.cpu().numpy(), w.cpu().numpy()), fg.linear(x, w))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_linear_no_rows(dt):
    t = TYPES[dt]
    x, w = torch.empty((0, 16), dtype=t, device="cuda"), rnd(1, 8, 16, dtype=t)
    assert fg.linear(x, w).shape == (0, 8)
    dx, dw, db = fg.linear_backward(torch.empty((0, 8), dtype=t, device="cuda"), x, w)
    assert dx.shape == (0, 16) and not dw.any() and not db.any() and dw.shape == (8, 16)


def test_linear_not_finite():
    """A row that is not finite makes its own results so, and no others."""
    for dt in TYPES:
        x, w = rnd(1, 70, 64, dtype=TYPES[dt]), rnd(2, 40, 64, dtype=TYPES[dt])
        x[3, 5], x[8, 0], x[69, 63] = math.nan, math.inf, -math.inf
        y = fg.linear(x, w)
        bad = torch.zeros(70, dtype=torch.bool, device="cuda")
        bad[[3, 8, 69]] = True
        assert not torch.isfinite(y[bad]).any() and torch.isfinite(y[~bad]).all()


def test_linear_float32_range():
    """Values near the ends of float32's range, where a rounded split would overflow."""
    x = torch.tensor([[3.4028235e38, 0.0], [1e-38, 3e38], [1e-30, 1e-35]], device="cuda")
    w = torch.tensor([[1.0, 0.0], [0.5, 2.0**-100], [2.0**60, 1.0]], device="cuda")
    y, want = fg.linear(x, w[:2]), x.double() @ w[:2].double().t()
    assert (y.double() - want).abs().le(1e-6 * want.abs() + 2.0**-126).all()
    y, want = fg.linear(x[2:], w), x[2:].double() @ w.double().t()
    assert (y.double() - want).abs().le(1e-6 * want.abs() + 2.0**-126).all()


def test_linear_offsets_past_32_bits():
    """An input and an output of more than 2^32 bytes: the last rows agree with the same rows alone."""
    m = (1 << 21) + 77
    x = torch.empty((m, 1040), dtype=torch.bfloat16, device="cuda")
    for i in range(0, m, 1 << 19):
        x[i:i + (1 << 19)] = rnd(i, min(1 << 19, m - i), 1040, dtype=torch.bfloat16)
    w = rnd(2, 1048, 1040, scale=1 / 32, dtype=torch.bfloat16)
    y = fg.linear(x, w)
    for a, b in ((0, 300), (m - 5000, m)):
        want = x[a:b].double() @ w.double().t()
        within(y[a:b], want, 1052 * U * (x[a:b].double().abs() @ w.double().abs().t()), ("y", "bf16"))
    _, dw, _ = fg.linear_backward(y, x, w, want=("weight",))
    want, mag = torch.zeros((1048, 1040), dtype=torch.float64, device="cuda"), 0
    for i in range(0, m, 1 << 18):
        yd, xd = y[i:i + (1 << 18)].double(), x[i:i + (1 << 18)].double()
        want += yd.t() @ xd
        mag = mag + yd.abs().t() @ xd.abs()
    # a float32 sum of 2^21 terms: rounding errors of random sign, so the square root of the worst case's count (times 8)
    within(dw, want, 8 * math.sqrt(m) * U * mag, ("dw", "bf16"))


# ---- layer norm -----------------------------------------------------------------------------------------------------
NORM = [(1, 1), (1, 5), (2, 63), (3, 256), (7, 257), (4, 300), (5, 512), (100, 771), (9, 1024), (33, 1025), (50, 2048),
        (6, 2049), (9, 4097), (5, 16384), (5000, 96), (20011, 130)]
# Depth of a row's sums: at most 16 in a lane, 6 across the wave, 16 across the waves.
DEPTH = 48


def norm64(x, g, b, eps):
    x = x.double()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1 / torch.sqrt(d.square().mean(1) + eps)
    y = d * rstd[:, None]
    if g is not None:
        y = y * g.double()
    if b is not None:
        y = y + b.double()
    return y, mean, rstd, d


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim", NORM)
def test_layer_norm(rows, dim, dt):
    t = TYPES[dt]
    x = (rnd(1, rows, dim) * 3 + rnd(2, rows, 1) * 10).to(t)
    g, b = rnd(3, dim, dtype=t), rnd(4, dim, dtype=t)
    for ga, be in ((g, b), (None, None), (g, None)):
        y, mean, rstd = fg.layer_norm(x, ga, be, eps=1e-5)
        wy, wm, wr, d = norm64(x, ga, be, 1e-5)
        me = (DEPTH * U * x.double().abs().mean(1))  # the mean's error
        within(mean, wm, me, ("mean", "f32"))
        # variance: each difference is off by the mean's error and a rounding; the errors' first order sums to nothing
        # worse than twice their size times the mean difference
        var = d.square().mean(1) + 1e-5
        ve = 2 * (me[:, None] + U * d.abs()).mul(d.abs()).mean(1) + me**2 + DEPTH * U * var
        rrel = 0.5 * ve / var + 3 * U
        within(rstd, wr, rrel * wr * 1.01, ("rstd", "f32"))
        ga = 1.0 if ga is None else ga.double().abs()
        be = 0.0 if be is None else be.double().abs()
        h = d.abs() * wr[:, None]
        yb = ga * (me[:, None] * wr[:, None] + h * (rrel[:, None] * 1.01 + 4 * U)) * 1.01 + 2 * U * be
        within(y, wy, yb, ("y", dt, rows, dim))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim", NORM)
def test_layer_norm_backward(rows, dim, dt):
    t = TYPES[dt]
    x, dy, g = (rnd(1, rows, dim) * 3 + 1).to(t), rnd(2, rows, dim, dtype=t), rnd(3, dim, dtype=t)
    _, wm, wr, _ = norm64(x, None, None, 1e-5)
    mean, rstd = wm.float(), wr.float()  # inputs of the call: the definition takes the same
    for ga in (g, None):
        dx, dg, db = fg.layer_norm_backward(dy, x, ga, mean, rstd)
        d, rs = dy.double(), rstd.double()[:, None]
        h = (x.double() - mean.double()[:, None]) * rs
        he = 3 * U * h.abs()
        u = d if ga is None else d * ga.double()
        m1, m2 = u.mean(1, keepdim=True), (u * h).mean(1, keepdim=True)
        want = rs * (u - m1 - h * m2)
        e1 = (DEPTH + 4) * U * u.abs().mean(1, keepdim=True)
        e2 = (DEPTH + 8) * U * (u * h).abs().mean(1, keepdim=True)
        bound = rs * (e1 + h.abs() * e2 + he * m2.abs() + 8 * U * (u.abs() + m1.abs() + (h * m2).abs()))
        within(dx, want, bound, ("dx", dt, rows, dim))
        within(dg, (d * h).sum(0), (rows + 8) * U * (d * h).abs().sum(0), ("dgamma", dt, rows, dim))
        within(db, d.sum(0), (rows + 4) * U * d.abs().sum(0), ("dbeta", dt, rows, dim))


def test_layer_norm_gradient_against_differences():
    rows, dim, e = 11, 70, 2.0**-8
    x, g, b, dy = rnd(1, rows, dim) * 2, 1 + rnd(2, dim) / 4, rnd(3, dim), rnd(4, rows, dim)
    _, mean, rstd = fg.layer_norm(x, g, b)
    for i, (p, gr) in enumerate(zip((x, g, b), fg.layer_norm_backward(dy, x, g, mean, rstd))):
        v, args = rnd(10 + i, *p.shape), [x, g, b]

        def at(s):
            args[i] = p + s * v
            return (dy.double() * fg.layer_norm(*args)[0].double()).sum()

        diff = ((at(e) - at(-e)) / (2 * e)).item()
        # y's third derivative along v is of the size of (|v| rstd)^3 |g|; its roundings add u / e
        size = (dy.abs() * g.abs()).double().sum().item()
        assert abs(diff - (gr.double() * v.double()).sum().item()) <= size * (8 * e * e + 64 * U / e)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_layer_norm_edges(dt):
    t = TYPES[dt]
    x = torch.full((5, 100), 7.0, dtype=t, device="cuda")  # no variance: h = 0 whatever eps
    x[1] = 0
    y, mean, rstd = fg.layer_norm(x, eps=1e-5)
    assert not y.any() and torch.equal(mean, x[:, 0].float())
    assert torch.allclose(rstd, torch.full_like(rstd, 1e-5**-0.5), rtol=1e-6, atol=0)
    x[2, 3] = math.nan
    x[3, 4] = math.inf
    y, _, _ = fg.layer_norm(x)
    assert torch.isnan(y[2:4]).all() and not y[[0, 1, 4]].any()
    big = rnd(1, 3, 64, scale=1e15)  # squares of 1e30 stay inside float32
    assert torch.isfinite(fg.layer_norm(big)[0]).all()
    z = torch.empty((0, 100), dtype=t, device="cuda")
    y, mean, rstd = fg.layer_norm(z)
    assert y.shape == (0, 100) and mean.shape == (0,)
    dx, dg, db = fg.layer_norm_backward(z, z, None, mean, rstd)
    assert dx.shape == (0, 100) and not dg.any() and not db.any()


def test_layer_norm_in_place_and_views():
    x, g = rnd(1, 40, 301), rnd(2, 301)
    y, mean, rstd = fg.layer_norm(x, g)
    v = x.clone()
    assert torch.equal(fg.layer_norm(v, g, out=v)[0], y) and torch.equal(v, y)
    assert torch.equal(fg.layer_norm(rnd(1, 40, 301).t().contiguous().t(), g)[0], y)
    wide = rnd(3, 40, 305)
    assert torch.equal(fg.layer_norm(wide[:, 2:303], g)[0], fg.layer_norm(wide[:, 2:303].clone(), g)[0])
    dx = fg.layer_norm_backward(y, x, g, mean, rstd, want=("x",))
    assert dx[1] is None and dx[2] is None and torch.equal(dx[0], fg.layer_norm_backward(y, x, g, mean, rstd)[0])


def test_layer_norm_offsets_past_32_bits():
    m = 2_800_001
    x = torch.empty((m, 771), dtype=torch.bfloat16, device="cuda")
    for i in range(0, m, 1 << 19):
        x[i:i + (1 << 19)] = rnd(i, min(1 << 19, m - i), 771, dtype=torch.bfloat16)
    y, mean, rstd = fg.layer_norm(x)
    a = m - 3000
    assert torch.equal(y[a:], fg.layer_norm(x[a:].clone())[0])
    dx, _, _ = fg.layer_norm_backward(y, x, None, mean, rstd, want=("x",))
    assert torch.equal(dx[a:], fg.layer_norm_backward(y[a:].clone(), x[a:].clone(), None, mean[a:], rstd[a:], want=("x",))[0])


# ---- contrastive loss -------------------------------------------------------------------------------------------------
LOSS = [(1, 1, 1), (1, 2, 3), (3, 64, 8), (5, 9, 17), (64, 64, 64), (65, 63, 96), (100, 333, 128), (130, 1000, 100),
        (257, 513, 40), (1024, 1024, 128), (700, 20001, 72), (4100, 8190, 64), (40, 3000, 1030),
        (129, 700, 129), (300, 1500, 200), (257, 66, 33)]


def scores64(q, c, t, scale, bias, ids):
    """(scores with -inf where left out, live rows, bound on a score's error)."""
    nq, nc = q.shape[0], c.shape[0]
    hide = torch.zeros(nc, dtype=torch.bool, device="cuda") if bias is None else bias <= -2.0**126
    cd = torch.where(hide[:, None], 0.0, c.double())
    s = scale * (q.double() @ cd.t())
    err = (q.shape[1] + 14) * U * abs(scale) * (q.double().abs() @ cd.abs().t()) + 4 * U * s.abs()
    if bias is not None:
        bd = torch.where(hide, 0.0, bias.double())
        s = s + bd
        err = err + 4 * U * (s.abs() + bd.abs())
    live = (t >= 0) & (t < nc)
    at = torch.where(live, t, 0).long()
    out = hide[None, :].expand(nq, nc).clone()
    if ids is not None:
        same = (ids[None, :] == ids[at][:, None]) & live[:, None]
        same[torch.arange(nq, device="cuda"), at] = False
        out |= same
    return s.masked_fill(out, -math.inf), live, at, hide, cd, err


def check_loss(q, c, t, scale, bias, ids, dt, dloss=None, workspace=None):
    nq, nc = q.shape[0], c.shape[0]
    t = t.to(torch.int32)
    loss, lse = fg.contrastive_loss(q, c, t, scale, bias=bias, ids=ids)
    s, live, at, hide, cd, err = scores64(q, c, t, scale, bias, ids)
    rows = torch.arange(nq, device="cuda")
    wl = torch.logsumexp(s, 1)
    top = torch.where(torch.isfinite(s), err, 0.0).amax(1)  # a score's error in this row
    # the sums: at most nc / 16 + 64 deep; exponentials and logarithms to a few last places of a number up to |s| log2 e
    big = torch.where(torch.isfinite(s), s.abs(), 0.0).amax(1)
    le = top + (nc / 16 + 96) * U + 8 * U * big
    some = torch.isfinite(wl)
    assert torch.equal(torch.isneginf(lse), ~some)
    within(lse[some], wl[some], le[some], ("lse", "f32"))
    st = s[rows, at]
    w_loss = torch.where(live & some, wl - st, 0.0)
    fin = torch.isfinite(w_loss)
    assert torch.equal(torch.isposinf(loss), ~fin)
    within(loss[fin], w_loss[fin], torch.where(live & some, le + top + 4 * U * big, 0.0)[fin], ("loss", "f32"))
    # gradients: P off by the factor exp(error of s - lse), G rounded to bf16 for the products
    dloss = rnd(99, nq) if dloss is None else dloss
    grad = live & some & ~hide[at]
    p = torch.where(grad[:, None], torch.exp(s - torch.where(some, wl, 0.0)[:, None]), 0.0)
    hot = torch.zeros_like(p)
    hot[rows, at] = grad.double()
    gw = dloss.double().abs()[:, None] * grad.double()[:, None]
    g = torch.where(grad, dloss.double(), 0.0)[:, None] * (p - hot)
    ge = gw * (p * (2 * (top + le)[:, None] + 16 * U) + 2 * U * hot)
    ge = torch.where(grad[:, None], ge, 0.0)
    gr = ge + (2.0**-8 * g.abs() if dt == "bf16" else 0)
    qd = torch.where(grad[:, None], q.double(), 0.0)
    dq, dc, db = fg.contrastive_loss_backward(dloss, q, c, t, lse, scale, bias=bias, ids=ids, workspace=workspace)
    a = abs(scale)
    within(dq, scale * (g @ cd), a * (gr @ cd.abs() + (nc + 12) * U * (g.abs() @ cd.abs())), ("dq", dt, nq, nc))
    within(dc, scale * (g.t() @ qd), a * (gr.t() @ qd.abs() + (nq + 12) * U * (g.abs().t() @ qd.abs())), ("dc", dt, nq, nc))
    within(db, g.sum(0), ge.sum(0) + (nq + 4) * U * g.abs().sum(0), ("dbias", "f32", nq, nc))
    only, none_c, none_b = fg.contrastive_loss_backward(dloss, q, c, t, lse, scale, bias=bias, ids=ids, candidate_grads=False,
                                                        workspace=workspace)
    assert none_c is None and none_b is None and torch.equal(only, dq)
    return loss, lse, dq, dc, db


def loss_inputs(nq, nc, dim, dt, seed=1):
    q, c = rnd(seed, nq, dim, dtype=TYPES[dt]), rnd(seed + 1, nc, dim, dtype=TYPES[dt])
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 2)
    t = torch.randint(nc, (nq,), generator=g, device="cuda", dtype=torch.int32)
    ids = torch.randint(max(1, nc // 2), (nc,), generator=g, device="cuda", dtype=torch.int32)
    bias = rnd(seed + 3, nc)
    return q, c, t, 2.0 / math.sqrt(dim), bias, ids


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("nq,nc,dim", LOSS)
def test_contrastive_loss(nq, nc, dim, dt):
    q, c, t, scale, bias, ids = loss_inputs(nq, nc, dim, dt)
    check_loss(q, c, t, scale, None, None, dt)
    if nq > 3:
        t[::5] = -1
        t[3] = nc + 7
    if nc > 8:
        bias[::7] = -math.inf
        bias[4] = LOWEST
    check_loss(q, c, t, scale, bias, ids, dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_contrastive_loss_masked_places_may_hold_anything(dt):
    """Infinities and NaN in masked candidates and in rows without a target reach no result."""
    q, c, t, scale, bias, ids = loss_inputs(130, 300, 96, dt)
    bias[10:20], bias[299] = -math.inf, LOWEST
    t[t == 299] = 0
    t = torch.where((t >= 10) & (t < 20), 0, t)
    t[[5, 129]] = -1
    clean = check_loss(q, c, t, scale, bias, ids, dt)
    c[10:15], c[15:20], c[299] = math.nan, math.inf, -math.inf
    q2 = q.clone()
    q2[5], q2[129] = math.nan, math.inf
    loss, lse = fg.contrastive_loss(q2, c, t, scale, bias=bias, ids=ids)
    dq, dc, db = fg.contrastive_loss_backward(rnd(99, 130), q2, c, t, lse, scale, bias=bias, ids=ids)
    keep = t >= 0
    for got, want in ((loss, clean[0]), (lse[keep], clean[1][keep]), (dq, clean[2]), (dc, clean[3]), (db, clean[4])):
        assert torch.equal(got, want)
    assert not dq[5].any() and not dc[10:20].any() and not db[10:20].any()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("low", [-math.inf, LOWEST, torch.finfo(torch.bfloat16).min])
def test_contrastive_loss_nothing_left(dt, low):
    """Every candidate masked: lse -inf, loss 0, no gradient.  A masked target among others: infinite loss, no gradient."""
    q, c, t, scale, bias, _ = loss_inputs(70, 90, 40, dt)
    check_loss(q, c, t, scale, torch.full_like(bias, low), None, dt)
    bias[t[0].item()] = low
    loss, _, dq, _, _ = check_loss(q, c, t, scale, bias, None, dt)
    assert torch.isposinf(loss[0]) and not dq[0].any()
    alone = torch.zeros(90, dtype=torch.int32, device="cuda")  # every candidate a copy of the target: it alone is left
    loss, lse, dq, dc, db = check_loss(q, c, t, scale, None, alone, dt)
    assert loss.abs().max() <= 1e-5 and db.abs().max() <= 1e-4


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_contrastive_loss_far_scores(dt):
    """Scores of +-1e4, where an exponential without the running maximum would overflow."""
    q, c, t, _, bias, ids = loss_inputs(90, 200, 64, dt)
    loss, lse = fg.contrastive_loss(q, c, t, 600.0, bias=bias, ids=ids)
    s, live, at, _, _, err = scores64(q, c, t, 600.0, bias, ids)
    wl = torch.logsumexp(s, 1)
    e = torch.where(torch.isfinite(s), err, 0.0).amax(1) + 32 * U * wl.abs() + 1e-5
    within(lse, wl, e, ("lse", "f32"))
    assert torch.isfinite(loss).all()
    for g in fg.contrastive_loss_backward(rnd(9, 90), q, c, t, lse, 600.0, bias=bias, ids=ids):
        assert torch.isfinite(g).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_contrastive_loss_l2_metric(dt):
    """bias = -scale |c|^2 / 2 makes the softmax that of -scale |q - c|^2 / 2."""
    q, c, t, _, _, _ = loss_inputs(50, 400, 96, dt)
    scale = 0.2
    bias = -0.5 * scale * c.float().square().sum(1)
    loss, lse, *_ = check_loss(q, c, t, scale, bias, None, dt)
    d = -0.5 * scale * (q.double()[:, None] - c.double()[None]).square().sum(2)
    want = torch.logsumexp(d, 1) - d[torch.arange(50, device="cuda"), t.long()]
    assert (loss.double() - want).abs().max() <= 1e-4


def test_contrastive_gradient_against_differences():
    nq, nc, dim, e = 30, 77, 33, 2.0**-6
    q, c, t, scale, bias, ids = loss_inputs(nq, nc, dim, "f32")
    t[::9] = -1
    dloss = rnd(50, nq)
    _, lse = fg.contrastive_loss(q, c, t, scale, bias=bias, ids=ids)
    grads = fg.contrastive_loss_backward(dloss, q, c, t, lse, scale, bias=bias, ids=ids)
    for i, (p, g) in enumerate(zip((q, c, bias), grads)):
        v, args = rnd(60 + i, *p.shape), [q, c, bias]

        def at(s):
            args[i] = p + s * v
            return (dloss.double() * fg.contrastive_loss(args[0], args[1], t, scale, bias=args[2], ids=ids)[0].double()).sum()

        diff = ((at(e) - at(-e)) / (2 * e)).item()
        # along v a score moves by at most `move`; a log-sum-exp's third derivative is below the cube of its scores' moves
        move = [lambda: scale * (v.double() @ c.double().t()).abs().amax(1), lambda: scale * (q.double() @ v.double().t()).abs().amax(1),
                lambda: v.double().abs().max().expand(nq)][i]()
        bound = (dloss.double().abs() * (e * e / 6 * (2 * move)**3 + 512 * U / e)).sum().item()
        assert abs(diff - (g.double() * v.double()).sum().item()) <= bound


@pytest.mark.parametrize("dim", [72, 200])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_contrastive_backward_in_chunks(dt, dim):
    """A workspace too small for all columns (up to 128 dims: for all splits): the same gradients from column chunks, down
    to 256 columns."""
    q, c, t, scale, bias, ids = loss_inputs(300, 2900, dim, dt)
    full = fg.lib.fgpu_contrastive_loss_backward_workspace_bytes(300, 2900, dim, int(dt == "bf16"))
    seen = []
    for part in (0.8, 0.65, 0.6):
        ws = torch.empty(int(full * part), dtype=torch.uint8, device="cuda")
        seen.append(check_loss(q, c, t, scale, bias, ids, dt, workspace=ws))
    with pytest.raises(fg.FgpuError, match="256 columns"):
        check_loss(q, c, t, scale, bias, ids, dt, workspace=torch.empty(4096, dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_contrastive_no_queries(dt):
    q = torch.empty((0, 24), dtype=TYPES[dt], device="cuda")
    c, t = rnd(1, 40, 24, dtype=TYPES[dt]), torch.empty(0, dtype=torch.int32, device="cuda")
    loss, lse = fg.contrastive_loss(q, c, t)
    assert loss.shape == (0,) and lse.shape == (0,)
    dq, dc, db = fg.contrastive_loss_backward(loss, q, c, t, lse)
    assert dq.shape == (0, 24) and not dc.any() and not db.any()


# ---- streams, graphs, repeatability ---------------------------------------------------------------------------------
def everything(s):
    """Every operator once, on the inputs of `s`."""
    y, pre = fg.linear(s["x"], s["w"], s["b"], act="gelu", save_pre=True)
    grads = fg.linear_backward(s["dy"], s["x"], s["w"], pre, act="gelu")
    n, mean, rstd = fg.layer_norm(y, s["g"], s["be"])
    ngrads = fg.layer_norm_backward(s["dy"], y, s["g"], mean, rstd)
    loss, lse = fg.contrastive_loss(n, s["c"], s["t"], 0.1, bias=s["bias"], ids=s["ids"])
    lgrads = fg.contrastive_loss_backward(s["dl"], n, s["c"], s["t"], lse, 0.1, bias=s["bias"], ids=s["ids"])
    return [y, pre, *grads, n, mean, rstd, *ngrads, loss, lse, *lgrads]


def inputs(dt, rows=300, k=520, n=104, nc=2000):
    t = TYPES[dt]
    s = dict(x=rnd(1, rows, k, dtype=t), w=rnd(2, n, k, scale=0.05, dtype=t), b=rnd(3, n, dtype=t), dy=rnd(4, rows, n, dtype=t),
             g=rnd(5, n, dtype=t), be=rnd(6, n, dtype=t), c=rnd(7, nc, n, dtype=t), bias=rnd(8, nc), dl=rnd(9, rows))
    s["t"] = torch.arange(rows, device="cuda", dtype=torch.int32) * 6
    s["ids"] = torch.arange(nc, device="cuda", dtype=torch.int32) // 2
    return s


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [4, 300])
def test_same_bits_every_time_on_any_stream(dt, rows):
    s = inputs(dt, rows)
    want = everything(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = everything(s)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = fg.linear(s["x"], s["w"], s["b"], act="gelu", stream=side)
    side.synchronize()
    assert torch.equal(got, want[0])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_captured_and_replayed(dt):
    """One graph of every operator, replayed on changing inputs with eager calls between."""
    s = inputs(dt)
    everything(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = everything(s)
    for k in range(4):
        s["x"].copy_(rnd(100 + k, *s["x"].shape, dtype=s["x"].dtype))
        s["dy"].copy_(rnd(200 + k, *s["dy"].shape, dtype=s["dy"].dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        assert all(torch.equal(a, b) for a, b in zip(got, everything(s)))
