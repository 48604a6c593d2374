"""Rows as 8-bit integers and the layers on weights held so, against their definitions in 64 bits.

The whole numbers are compared exactly: x 127 is exact in 64 bits, and its quotient by the row's maximum is a tie of two
whole numbers only where it is one exactly, as quotients of 31 by 24 bits lie 2^-33 apart.  The products' sums are exact, so a
layer is off by the roundings that follow them: the sum to float32, two scales, the bias (5 u of each, u = 2^-24), the
activation's own error as in the linear layer's tests, and half a last place of the result."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": U, "bf16": 2.0**-8}


def rnd(seed, *shape, scale=1.0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def codes(x):
    x = x.double().cpu()
    top = x.abs().amax(1)
    q = torch.round(x * 127 / torch.where(top > 0, top, 1.0)[:, None])
    return q, (top.float() / 127)


def check_quantize(x):
    q, scale = fg.quantize_rows(x)
    want, ws = codes(x)
    dim = x.shape[1]
    assert q.dtype == torch.int8 and q.shape == (x.shape[0], fg.int8_row(dim))
    assert torch.equal(scale.cpu(), ws)
    assert torch.equal(q[:, :dim].cpu().double(), want)
    assert (q[:, dim:] == 0).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 7), (3, 8), (5, 15), (4, 16), (9, 17), (130, 100), (7, 511), (6, 513),
                                      (2050, 520), (2500, 2048), (100, 2049), (3, 8192), (2, 8200), (2, 65536), (1, 20001),
                                      (33000, 24)])
def test_quantize(rows, dim, dt):
    x = rnd(rows + dim, rows, dim, dtype=TYPES[dt])
    x *= torch.where(rnd(1, rows, 1).abs() < 0.3, 1e-3, 50.0).to(x.dtype)
    check_quantize(x)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_quantize_at_the_borders(dt):
    """Values that lie on the border between two whole numbers, and the nearest numbers to it on both sides."""
    t = TYPES[dt]
    rows = []
    for top in (1.0, 127.0, 254.0, 3.0, 0.7, 1.9921875):
        top = torch.tensor(top).to(t).double().item()
        border = (torch.arange(-127, 127).double() + 0.5) * top / 127
        mid = border.to(t)
        step = torch.int32 if dt == "f32" else torch.int16
        up, down = (mid.view(step) + 1).view(t), (mid.view(step) - 1).view(t)
        rows.append(torch.cat([mid, up, down, torch.tensor([top, -top]).to(t)]))
    x = torch.stack(rows)
    assert (x[2].double() * 127 / 254 % 1 == 0.5).any()  # exact ties among them
    check_quantize(x.cuda())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_quantize_range(dt):
    """Rows near both ends of the type, rows of zeros, and values far below the row's largest."""
    t = TYPES[dt]
    base = rnd(1, 8, 40)
    scale = torch.tensor([3e38, 1e30, 1e-30, 1e-37, 2e-38, 1e-39, 1.0, 1.0], device="cuda")[:, None]
    x = (base / base.abs().amax(1, keepdim=True) * scale).to(t)
    x[6] = 0
    x[7, 1:] *= 1e-30
    x[7, 3] = -0.0
    check_quantize(x)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_quantize_not_finite(dt):
    x = rnd(1, 5, 30, dtype=TYPES[dt])
    want, ws = codes(x)
    x[1, 4], x[2, 0], x[3, 29] = math.nan, math.inf, -math.inf
    if dt == "f32":  # a NaN that carries something in its low bits
        x.view(torch.int32)[1, 5] = 0x7FC12345
    q, scale = fg.quantize_rows(x)
    assert torch.isnan(scale[1:4]).all() and (q[1:4] == 0).all()
    assert torch.equal(q[[0, 4], :30].cpu().double(), want[[0, 4]]) and torch.equal(scale[[0, 4]].cpu(), ws[[0, 4]])


def act64(z, act):
    phi = torch.special.erfc(-z * math.sqrt(0.5)) / 2
    return {"none": z, "relu": z.clamp(min=0), "gelu": z * phi, "silu": z * torch.sigmoid(z)}[act]


def check_layer(m, k, n, dt, act, bias, residual, gated, given, seed=0):
    """given: x comes as 8-bit integers already."""
    t = TYPES[dt]
    out = 2 * n if gated else n
    x = rnd(seed + 1, m, k, dtype=t)
    w, ws = fg.quantize_rows(rnd(seed + 2, out, k, scale=1 / math.sqrt(k), dtype=t))
    b = rnd(seed + 3, out, dtype=t) if bias else None
    r = rnd(seed + 4, m, n, dtype=t) if residual else None
    q, xs = fg.quantize_rows(x)
    kw = dict(x_scale=xs, dtype=t) if given else {}
    a = q if given else x
    y = fg.gated_linear_int8(a, w, ws, b, act=act, **kw) if gated else fg.linear_int8(a, w, ws, b, r, act=act, **kw)
    z = (q.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    zb = 4 * U * z.abs()
    if bias:
        z = z + b.double()
        zb = zb + U * z.abs()
    f = 2e-7 if dt == "f32" else 8e-7
    if gated:
        g, u = z[:, :n], z[:, n:]
        v = act64(g, act)
        vb = 1.13 * zb[:, :n] + (f * g.abs() + 8 * U * v.abs() if act != "none" else 0)
        want = v * u
        bound = vb * u.abs() + v.abs() * zb[:, n:] + 2 * U * want.abs()
    else:
        want = act64(z, act)
        bound = 1.13 * zb + (f * z.abs() + 8 * U * want.abs() if act != "none" else 0)
        if residual:
            want = want + r.double()
            bound = bound + 2 * U * (want.abs() + r.double().abs())
    assert y.dtype == t and y.shape == (m, n)
    off = (y.double() - want).abs() - (bound + HALF[dt] * (want.abs() + bound))
    assert off.max().item() <= 1e-37, (m, k, n, dt, act, gated, given, off.max().item())


SIZES = [(1, 1, 1), (1, 1024, 4096), (1, 1000, 33), (2, 8, 1030), (16, 100, 17), (16, 4100, 40), (17, 100, 17), (33, 65, 63),
         (64, 64, 64), (127, 15, 129), (300, 513, 257), (257, 2056, 255), (1000, 385, 771), (2050, 1024, 520), (16390, 64, 516),
         (40000, 24, 40), (3, 30000, 5), (3000, 1040, 1000), (3000, 1040, 2000), (5000, 656, 1030), (5000, 656, 2060),
         (200, 512, 800), (260, 500, 1000)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_layers(m, k, n, dt):
    check_layer(m, k, n, dt, "none", True, True, False, False)
    check_layer(m, k, n, dt, "silu", True, False, True, False, seed=10)
    check_layer(m, k, n, dt, "gelu", False, False, False, True, seed=20)
    check_layer(m, k, n, dt, "none", False, False, True, True, seed=30)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("m,n", [(9, 100), (150, 100), (3000, 700), (9000, 1030)])
def test_activations(act, m, n, dt):
    check_layer(m, 96, n, dt, act, True, True, False, False)
    check_layer(m, 96, n, dt, act, True, False, True, False)


@pytest.mark.parametrize("m", [5, 100])
def test_largest_sums_are_exact(m):
    """2^16 products of 127 127 and of 128 128 in one sum, which 32 bits hold."""
    k = 1 << 16
    for v in (127, -128):
        x = torch.full((m, k), v, dtype=torch.int8, device="cuda")
        w = torch.full((40, k), v, dtype=torch.int8, device="cuda")
        one = torch.ones(40, device="cuda")
        y = fg.linear_int8(x, w, one, x_scale=one[:1].expand(m).contiguous(), dtype=torch.float32)
        assert (y == float(v * v * k)).all()


@pytest.mark.parametrize("m", [5, 100])
@pytest.mark.parametrize("gated", [False, True])
def test_what_lies_behind_a_row_is_not_read_from_x(m, gated):
    """Weights that hold something behind their rows' values: x's zeros there keep it out."""
    x = rnd(1, m, 40, dtype=torch.bfloat16)
    w, ws = fg.quantize_rows(rnd(2, 48, 40))
    f = fg.gated_linear_int8 if gated else fg.linear_int8
    want = f(x, w, ws)
    w[:, 40:] = 99
    assert torch.equal(f(x, w, ws), want)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m", [3, 100])
def test_a_row_that_is_not_finite_spoils_itself_alone(m, dt):
    x = rnd(1, m, 40, dtype=TYPES[dt])
    w, ws = fg.quantize_rows(rnd(2, 50, 40))
    clean = fg.linear_int8(x, w, ws)
    x[1, 7] = math.inf
    x[2] = 0
    y = fg.linear_int8(x, w, ws)
    assert torch.isnan(y[1]).all() and (y[2] == 0).all() and torch.equal(y[0], clean[0])
    assert torch.equal(y[3:], clean[3:])


def test_views_and_numpy():
    x, w = rnd(1, 20, 100)[:, 11:77], rnd(2, 66, 30).t()
    q, s = fg.quantize_rows(w)
    qc, sc = fg.quantize_rows(w.clone(memory_format=torch.contiguous_format))
    assert torch.equal(q, qc) and torch.equal(s, sc)
    y = fg.linear_int8(x, q, s)
    assert torch.equal(y, fg.linear_int8(x.contiguous(), q, s))
    assert torch.equal(y, fg.linear_int8(x.cpu().numpy(), q.cpu().numpy(), s.cpu().numpy().astype(np.float32)))
    out = torch.empty_like(y)
    assert fg.linear_int8(x, q, s, out=out) is out and torch.equal(out, y)
    r = rnd(3, 20, 30)
    want = fg.linear_int8(x, q, s, residual=r)
    assert torch.equal(fg.linear_int8(x, q, s, residual=r, out=r), want)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_no_rows(dt):
    x = torch.zeros((0, 24), dtype=TYPES[dt], device="cuda")
    q, s = fg.quantize_rows(x)
    assert q.shape == (0, 32) and s.shape == (0,)
    w, ws = fg.quantize_rows(rnd(1, 20, 24))
    assert fg.linear_int8(x, w, ws).shape == (0, 20) and fg.gated_linear_int8(x, w, ws).shape == (0, 10)


def test_offsets_past_32_bits():
    m, k, n = (1 << 20) + 77, 4112, 24
    x = torch.empty((m, k), dtype=torch.bfloat16, device="cuda")
    x[:-300].fill_(0.5)
    x[-300:] = rnd(2, 300, k, dtype=torch.bfloat16)
    w, ws = fg.quantize_rows(rnd(1, n, k, scale=0.02))
    y, tail = fg.linear_int8(x, w, ws, dtype=torch.bfloat16), fg.linear_int8(x[-300:].contiguous(), w, ws)
    assert torch.equal(y[-300:], tail) and torch.equal(y[0], y[-301])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 77, 3000])
def test_same_bits_on_another_stream_and_replayed(dt, m):
    t = TYPES[dt]
    x, w0, b = rnd(1, m, 100, dtype=t), rnd(2, 140, 100, scale=0.1, dtype=t), rnd(3, 140, dtype=t)

    def every():
        w, ws = fg.quantize_rows(w0)
        return w, ws, fg.linear_int8(x, w, ws, b, act="gelu"), fg.gated_linear_int8(x, w, ws, b)

    first = every()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = every()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = every()
    for k in range(3):
        x.copy_(rnd(100 + k, m, 100, dtype=t))
        w0.copy_(rnd(200 + k, 140, 100, scale=0.1, dtype=t))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        assert all(torch.equal(p, q) for p, q in zip(got, every()))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,n", [(700, 600, 200), (2049, 640, 1111), (6000, 528, 2120), (9001, 1040, 2304)])
def test_residual_in_place_of_every_tile(m, k, n, dt):
    """Rows and columns that end inside a tile and inside a wave's 64 columns, the residual where the result goes."""
    t = TYPES[dt]
    x, r, b = rnd(1, m, k, dtype=t), rnd(2, m, n, dtype=t), rnd(4, n, dtype=t)
    q, s = fg.quantize_rows(rnd(3, n, k, scale=1 / math.sqrt(k)))
    check_layer(m, k, n, dt, "gelu", True, True, False, False)
    want = fg.linear_int8(x, q, s, b, r, act="gelu")
    hold = torch.full((m * n + 64,), 7.0, dtype=t, device="cuda")
    y = hold[32:32 + m * n].view(m, n)
    y.copy_(r)
    assert torch.equal(fg.linear_int8(x, q, s, b, y, act="gelu", out=y), want)
    assert (hold[:32] == 7).all() and (hold[-32:] == 7).all()
