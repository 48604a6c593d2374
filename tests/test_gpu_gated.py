"""The gated layer and its gradients against their definitions in 64 bits.

u = 2^-24, half a last place of float32 at most.  A float32 sum of n products is off by at most (n + c) u times the sum of
their magnitudes (c: the products, what split float32 operands leave out, the bias); a value of a product of two factors by
each factor's error times the other.  A result in bfloat16 adds 2^-8 of itself; a bfloat16 operand made inside a call, 2^-8 of
each term."""
import math

import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": U, "bf16": 2.0**-8}
ACTS = ["none", "relu", "gelu", "silu"]


def rnd(seed, *shape, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def within(got, want, bound, dt, what):
    off = (got.double() - want).abs() - (bound + HALF[dt] * (want.abs() + bound))
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 1e-37, f"{what}: {worst} over the bound at {torch.argmax(off).item()}"


def value_slope(z, act):
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        phi = torch.special.erfc(-z * math.sqrt(0.5)) / 2
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


# One of everything, sizes around the kernels' columns (8, 16, 32), k steps and tiles (64, 128, 256), odd strides.
SIZES = [(1, 1, 1), (1, 1024, 2048), (1, 1000, 33), (2, 8, 1030), (3, 7, 5), (5, 129, 2), (16, 100, 17), (17, 512, 64),
         (31, 4096, 24), (33, 65, 63), (64, 64, 32), (65, 72, 130), (127, 8, 129), (300, 513, 257), (257, 2056, 255),
         (1000, 385, 771), (2048, 256, 520), (16390, 64, 516), (40000, 24, 40), (9000, 136, 1100)]


def check_gated(m, k, n, dt, act, bias, save, seed=0, **kw):
    t = TYPES[dt]
    x, w = rnd(seed + 1, m, k, dtype=t), rnd(seed + 2, 2 * n, k, scale=1 / math.sqrt(k), dtype=t)
    b = rnd(seed + 3, 2 * n, dtype=t) if bias else None
    got = fg.gated_linear(x, w, b, act=act, save_pre=save, **kw)
    h, pre = got if save else (got, None)
    z = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if bias:
        z, mag = z + b.double(), mag + b.double().abs()
    zb = (k + 12) * U * mag
    if save:
        assert pre.dtype == t and pre.shape == (m, 2 * n)
        within(pre, z, zb, dt, ("pre", m, k, n, act))
    value, _ = value_slope(z[:, :n], act)
    u = z[:, n:]
    # slopes are at most 1.13; the activation's own error as in the linear layer's tests, of bfloat16 results 7.2e-7 of z
    vb = 1.13 * zb[:, :n] + ((2e-7 if dt == "f32" else 8e-7) * z[:, :n].abs() + 8 * U * value.abs() if act != "none" else 0)
    bound = vb * u.abs() + value.abs() * zb[:, n:] + vb * zb[:, n:] + 2 * U * (value * u).abs()
    assert h.dtype == t and h.shape == (m, n)
    within(h, value * u, bound, dt, ("h", m, k, n, act))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_gated(m, k, n, dt):
    check_gated(m, k, n, dt, "silu", True, True)
    check_gated(m, k, n, dt, "gelu", False, False, seed=10)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [1, 20, 150])
def test_activations(act, dt, m):
    check_gated(m, 96, 136, dt, act, True, True)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
def test_every_tile(act, dt):
    """A size that takes each kernel, with rows and columns that end inside a tile and a k that ends inside a step."""
    seen = set()
    sizes = [(15, 200, 70), (70, 200, 100), (1500, 200, 999), (2500, 72, 700), (5000, 328, 1030), (20000, 72, 1030), (3000, 520, 1000),
             (960, 643, 577), (4555, 291, 1556)]
    for m, k, n in sizes:
        seen.add(fg.lib.fgpu_gated_linear_tile(m, k, n, int(dt == "bf16")))
        check_gated(m, k, n, dt, act, True, True, seed=m)
    split = 2048  # planes formed on the way: 64 and 128 wide
    assert seen >= ({0, 256, split + 64, split + 128} if dt == "f32" else {0, 64, 128, 256}), seen


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (5, 9, 3), (64, 64, 64), (65, 130, 72), (100, 77, 101), (300, 257, 513),
                                   (1000, 385, 98), (4099, 100, 64), (520, 1028, 1030), (16385, 72, 128), (3, 5, 1)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_backward(m, k, n, dt, act):
    t = TYPES[dt]
    dh, x, w = rnd(1, m, n, dtype=t), rnd(2, m, k, dtype=t), rnd(3, 2 * n, k, scale=1 / math.sqrt(k), dtype=t)
    pre = rnd(4, m, 2 * n, scale=1.5, dtype=t)
    check_grads(dh, x, w, pre, act, dt, *fg.gated_linear_backward(dh, x, w, pre, act=act))


def check_grads(dh, x, w, pre, act, dt, dx, dw, db):
    (m, n), k = dh.shape, x.shape[1]
    d, x, w, g, u = dh.double(), x.double(), w.double(), pre[:, :n].double(), pre[:, n:].double()
    value, slope = value_slope(g, act)
    dz = torch.cat([d * u * slope, d * value], 1)
    # the slope's and the value's own errors (bfloat16's shorter polynomial: 7.2e-7 of the tail), two or three roundings
    e = 4e-7 if dt == "f32" else 1e-6
    dze = torch.cat([(d * u).abs() * (e * (1 + g.abs()) + 8 * U), d.abs() * (e * g.abs() + 8 * U * value.abs())], 1)
    one = dze + (2.0**-8 * dz.abs() if dt == "bf16" else 0)
    within(dx, dz @ w, one @ w.abs() + (2 * n + 12) * U * (dz.abs() @ w.abs()), dt, ("dx", m, k, n, act))
    within(dw, dz.t() @ x, one.t() @ x.abs() + (m + 12) * U * (dz.abs().t() @ x.abs()), dt, ("dw", m, k, n, act))
    within(db, dz.sum(0), dze.sum(0) + (m + 4) * U * dz.abs().sum(0), dt, ("db", m, k, n, act))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n", [7, 8, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257])
def test_backward_of_narrow_layers(n, dt):
    """Every count of rows a wave takes at once, of rows that do not divide by it."""
    t = TYPES[dt]
    dh, x, w = rnd(1, 715, n, dtype=t), rnd(2, 715, 41, dtype=t), rnd(3, 2 * n, 41, scale=0.2, dtype=t)
    pre = rnd(4, 715, 2 * n, dtype=t)
    check_grads(dh, x, w, pre, "silu", dt, *fg.gated_linear_backward(dh, x, w, pre, act="silu"))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
def test_backward_activations(act, dt):
    t = TYPES[dt]
    dh, x, w = rnd(1, 90, 50, dtype=t), rnd(2, 90, 40, dtype=t), rnd(3, 100, 40, scale=0.2, dtype=t)
    pre = rnd(4, 90, 100, dtype=t)
    check_grads(dh, x, w, pre, act, dt, *fg.gated_linear_backward(dh, x, w, pre, act=act))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("want", [("x",), ("weight",), ("bias",), ("x", "bias"), ()])
@pytest.mark.parametrize("m", [30, 3000])
def test_backward_of_some(want, dt, m):
    """What is not asked for does not change the bits of what is."""
    t = TYPES[dt]
    dh, x, w, pre = rnd(1, m, 51, dtype=t), rnd(2, m, 30, dtype=t), rnd(3, 102, 30, dtype=t), rnd(4, m, 102, dtype=t)
    every = dict(zip(("x", "weight", "bias"), fg.gated_linear_backward(dh, x, w, pre)))
    some = dict(zip(("x", "weight", "bias"), fg.gated_linear_backward(dh, x, w, pre, want=want)))
    for name in every:
        assert (some[name] is None) if name not in want else torch.equal(some[name], every[name])


@pytest.mark.parametrize("act", ["silu", "gelu", "none"])
def test_gradient_against_differences(act):
    """sum(h c) in float32, by central differences of the layer itself along random directions.  f's rounding: each h is good
    to about 60 u of its magnitude, its sum over 40 x 12 elements of size one to 480 60 u = 2e-3 at most; over 2 step that is
    1e-1 of a unit for step 1e-2; the third derivative's part is of the order of step^2."""
    m, k, n, step = 40, 24, 12, 1e-2
    x, w, b = rnd(1, m, k), rnd(2, 2 * n, k, scale=k**-0.5), rnd(3, 2 * n)
    c = rnd(4, m, n)
    _, pre = fg.gated_linear(x, w, b, act=act, save_pre=True)
    grads = fg.gated_linear_backward(c, x, w, pre, act=act)

    def f(x, w, b):
        return (fg.gated_linear(x, w, b, act=act).double() * c.double()).sum()

    for i, (p, g) in enumerate(zip((x, w, b), grads)):
        d = rnd(10 + i, *p.shape)
        d /= d.norm()
        args = [[x, w, b], [x, w, b]]
        args[0][i], args[1][i] = p + step * d, p - step * d
        diff = (f(*args[0]) - f(*args[1])) / (2 * step)
        assert abs(diff - (g.double() * d.double()).sum()) <= 0.1 + 1e-2 * g.double().norm()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_views_and_alignment(dt):
    """Rows of a wider matrix, a transposed weight, arrays off 16 bytes: the same bits as from plain copies."""
    t = TYPES[dt]
    wide, wt = rnd(1, 50, 100, dtype=t), rnd(2, 72, 66, dtype=t)
    x, w, b = wide[:, 13:85], wt.t(), rnd(3, 67, dtype=t)[1:]
    pre_in, dh = rnd(4, 50 * 66 + 1, dtype=t)[1:].view(50, 66), rnd(5, 50 * 33 + 1, dtype=t)[1:].view(50, 33)
    c = [a.clone(memory_format=torch.contiguous_format) for a in (x, w, b, pre_in, dh)]
    assert torch.equal(fg.gated_linear(x, w, b), fg.gated_linear(c[0], c[1], c[2]))
    for p, q in zip(fg.gated_linear_backward(dh, x, w, pre_in), fg.gated_linear_backward(c[4], c[0], c[1], c[3])):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_no_rows(dt):
    t = TYPES[dt]
    x, w = torch.zeros((0, 24), dtype=t, device="cuda"), rnd(1, 20, 24, dtype=t)
    h, pre = fg.gated_linear(x, w, save_pre=True)
    assert h.shape == (0, 10) and pre.shape == (0, 20)
    dx, dw, db = fg.gated_linear_backward(h, x, w, pre)
    assert dx.shape == (0, 24) and torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(db))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", [(3, 40, 20), (300, 72, 100)])
def test_not_finite(m, k, n, dt):
    """A row that holds NaN or infinity spoils itself alone; the other rows keep their bits."""
    t = TYPES[dt]
    x, w = rnd(1, m, k, dtype=t), rnd(2, 2 * n, k, dtype=t)
    clean = fg.gated_linear(x, w)
    y = x.clone()
    y[1, 3], y[2, 5] = math.nan, math.inf
    h = fg.gated_linear(y, w)
    assert torch.isnan(h[1]).all() and not torch.isfinite(h[2]).any()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(h[keep], clean[keep])


@pytest.mark.parametrize("m,k,n", [(5, 40, 20), (300, 72, 99), (3000, 40, 99)])
def test_writes_nothing_beside_its_outputs(m, k, n):
    """Outputs in the middle of larger arrays, whose surroundings stay."""
    x, w = rnd(1, m, k, dtype=torch.bfloat16), rnd(2, 2 * n, k, dtype=torch.bfloat16)
    hold = torch.full((m * n + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = hold[32:32 + m * n].view(m, n)
    fg.gated_linear(x, w, out=out)
    assert torch.equal(out, fg.gated_linear(x, w))
    assert (hold[:32] == 7).all() and (hold[32 + m * n:] == 7).all()


def test_offsets_past_32_bits():
    """More than 2^32 bytes of x, of h and of what is kept: the last rows agree with the same rows alone."""
    m, k, n = (1 << 20) + 77, 2056, 1032
    x, w = torch.empty((m, k), dtype=torch.bfloat16, device="cuda"), rnd(1, 2 * n, k, scale=0.02, dtype=torch.bfloat16)
    x[:-300].fill_(0.5)
    x[-300:] = rnd(2, 300, k, dtype=torch.bfloat16)
    h, pre = fg.gated_linear(x, w, save_pre=True)
    h1, pre1 = fg.gated_linear(x[-300:].contiguous(), w, save_pre=True)
    # the sums' order may differ between tiles: two roundings to bfloat16 and k u apart
    assert ((h[-300:].double() - h1.double()).abs() <= 2.0**-7 * h1.double().abs() + 1e-3).all()
    assert ((pre[-300:].double() - pre1.double()).abs() <= 2.0**-7 * pre1.double().abs() + 1e-3).all()
    assert torch.equal(h[0], h[5000]) and torch.equal(pre[0], pre[(1 << 20) - 300])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 77, 3000])
def test_same_bits_on_another_stream_and_replayed(dt, m):
    """One graph of a forward and a backward call, replayed on changing inputs with eager calls between."""
    t = TYPES[dt]
    x, w, b = rnd(1, m, 100, dtype=t), rnd(2, 140, 100, scale=0.1, dtype=t), rnd(3, 140, dtype=t)
    dh = rnd(4, m, 70, dtype=t)

    def both():
        h, pre = fg.gated_linear(x, w, b, save_pre=True)
        return (h, pre) + fg.gated_linear_backward(dh, x, w, pre)

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(3):
        x.copy_(rnd(100 + k, m, 100, dtype=t))
        dh.copy_(rnd(200 + k, m, 70, dtype=t))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        assert all(torch.equal(p, q) for p, q in zip(got, both()))
