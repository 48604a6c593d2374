"""The refusals of the gated layer, the 8-bit layers and the orthogonalisation, on the CPU: every bad argument is turned
down before anything reaches the device."""
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

L = fg.lib
ARG, UNSUPPORTED, WORKSPACE = 1, 2, 6
P = 1 << 20  # stands for a 16-byte-aligned device pointer: refused calls never read it
F32, BF16 = 0, 1
INF = float("inf")


def gated(x=P, w=P, b=None, rows=4, k=8, n=8, dt=F32, act=3, h=P, pre=None, ws=P, wsb=1 << 40):
    return L.fgpu_gated_linear(x, w, b, rows, k, n, dt, act, h, pre, ws, wsb, None)


def gated_bwd(dh=P, x=P, w=P, pre=P, rows=4, k=8, n=8, dt=F32, act=3, dx=P, dw=P, db=P, ws=P, wsb=1 << 40):
    return L.fgpu_gated_linear_backward(dh, x, w, pre, rows, k, n, dt, act, dx, dw, db, ws, wsb, None)


def quantize(x=P, rows=4, dim=8, dt=F32, q=P, scale=P):
    return L.fgpu_quantize_rows(x, rows, dim, dt, q, scale, None)


def int8(x=P, xs=None, w=P, wsc=P, rows=4, k=8, n=8, dt=F32, act=0, y=P, ws=P, wsb=1 << 40):
    return L.fgpu_linear_int8(x, xs, w, wsc, None, None, rows, k, n, dt, act, y, ws, wsb, None)


def gated_int8(x=P, xs=None, w=P, wsc=P, rows=4, k=8, n=8, dt=F32, act=0, h=P, ws=P, wsb=1 << 40):
    return L.fgpu_gated_linear_int8(x, xs, w, wsc, None, rows, k, n, dt, act, h, ws, wsb, None)


def ortho(x=P, rows=8, cols=8, dt=F32, steps=5, a=3.0, b=-4.0, c=2.0, eps=1e-7, y=P, ws=P, wsb=1 << 40):
    return L.fgpu_orthogonalize(x, rows, cols, dt, steps, a, b, c, eps, y, ws, wsb, None)


ALL = [gated, gated_bwd, quantize, int8, gated_int8, ortho]


@pytest.mark.parametrize("f,args,want", [(f, a, w) for f in ALL for a, w in [
    (dict(dt=2), ARG), (dict(dt=-1), ARG), (dict(rows=-1), ARG), (dict(x=None), ARG)]] + [
    (f, a, w) for f in (gated, gated_bwd, int8, gated_int8) for a, w in [
        (dict(act=4), ARG), (dict(act=-1), ARG), (dict(k=0), ARG), (dict(n=0), ARG), (dict(w=None), ARG), (dict(x=P + 4), ARG),
        (dict(w=P + 8), ARG), (dict(ws=P + 4), ARG), (dict(k=(1 << 16) + 1), UNSUPPORTED),
        (dict(rows=(1 << 30) + 1), UNSUPPORTED)]] + [
    (gated, dict(h=None), ARG), (gated, dict(n=(1 << 15) + 1), UNSUPPORTED), (gated, dict(n=1 << 30), UNSUPPORTED),
    (gated, dict(rows=1 << 16, k=1023, n=1024, dt=BF16, wsb=0), WORKSPACE),
    (gated, dict(rows=1 << 16, k=1024, n=1024, dt=F32, ws=None), WORKSPACE),
    (gated_bwd, dict(dh=None), ARG), (gated_bwd, dict(pre=None), ARG), (gated_bwd, dict(n=(1 << 15) + 1), UNSUPPORTED),
    (gated_bwd, dict(rows=1 << 16, k=1024, n=1024, dt=BF16, wsb=0), WORKSPACE),
    (quantize, dict(dim=0), ARG), (quantize, dict(q=None), ARG), (quantize, dict(scale=None), ARG), (quantize, dict(q=P + 8), ARG),
    (quantize, dict(dim=(1 << 16) + 1), UNSUPPORTED), (quantize, dict(rows=(1 << 30) + 1), UNSUPPORTED),
    (int8, dict(wsc=None), ARG), (int8, dict(y=None), ARG), (int8, dict(n=(1 << 16) + 1), UNSUPPORTED),
    (int8, dict(rows=1 << 12, k=1024, wsb=0), WORKSPACE), (int8, dict(rows=1 << 12, k=1024, ws=None), WORKSPACE),
    (gated_int8, dict(wsc=None), ARG), (gated_int8, dict(h=None), ARG), (gated_int8, dict(n=(1 << 15) + 1), UNSUPPORTED),
    (gated_int8, dict(n=(1 << 31) - 1), UNSUPPORTED), (gated_int8, dict(rows=1 << 12, k=1024, wsb=0), WORKSPACE),
    (ortho, dict(cols=-1), ARG), (ortho, dict(steps=0), ARG), (ortho, dict(steps=65), ARG), (ortho, dict(eps=-1.0), ARG),
    (ortho, dict(eps=INF), ARG), (ortho, dict(a=INF), ARG), (ortho, dict(b=float("nan")), ARG), (ortho, dict(c=-INF), ARG),
    (ortho, dict(y=None), ARG), (ortho, dict(ws=P + 8), ARG), (ortho, dict(wsb=0), WORKSPACE), (ortho, dict(ws=None), WORKSPACE),
    (ortho, dict(rows=(1 << 16) + 1), UNSUPPORTED), (ortho, dict(cols=1 << 33), UNSUPPORTED),
])
def test_refused_with_its_status(f, args, want):
    assert f(**args) == want
    assert L.fgpu_last_error()


def test_no_rows_is_no_work():
    assert gated(rows=0, x=None, h=None) == 0
    assert quantize(rows=0, x=None, q=None) == 0
    assert int8(rows=0, x=None, y=None) == 0
    assert gated_int8(rows=0, x=None, h=None) == 0
    assert ortho(rows=0, x=None, y=None) == 0 and ortho(cols=0, x=None, y=None) == 0


def test_workspace_sizes():
    # a smaller workspace than asked for is refused, one of that size would be taken
    for f, size, args in [
            (gated, L.fgpu_gated_linear_workspace_bytes(5000, 1023, 512, BF16), dict(rows=5000, k=1023, n=512, dt=BF16)),
            (gated_bwd, L.fgpu_gated_linear_backward_workspace_bytes(5000, 100, 30, F32), dict(rows=5000, k=100, n=30)),
            (int8, L.fgpu_linear_int8_workspace_bytes(5000, 1000, 30, F32, 0), dict(rows=5000, k=1000, n=30)),
            (gated_int8, L.fgpu_gated_linear_int8_workspace_bytes(5000, 1000, 30, BF16, 0), dict(rows=5000, k=1000, n=30, dt=BF16)),
            (ortho, L.fgpu_orthogonalize_workspace_bytes(1000, 30, F32), dict(rows=1000, cols=30))]:
        assert size > 0 and f(**args, wsb=size - 1) == WORKSPACE
    assert L.fgpu_gated_linear_workspace_bytes(1 << 16, 1024, 4096, BF16) == 0
    assert L.fgpu_linear_int8_workspace_bytes(16, 1024, 4096, BF16, 0) == 0
    assert L.fgpu_linear_int8_workspace_bytes(1 << 16, 1024, 4096, BF16, 1) == 0
    assert L.fgpu_linear_int8_workspace_bytes(4, 8, 8, 9, 0) == 0
    assert L.fgpu_gated_linear_tile(0, 8, 8, BF16) == -1


@pytest.fixture
def host(monkeypatch):
    """The Python mirror's checks without a device: tensors stay where they are and no call goes out."""
    def no_call(*a):
        raise AssertionError("a refused call reached the library")
    for name in ("fgpu_gated_linear", "fgpu_gated_linear_backward", "fgpu_quantize_rows", "fgpu_linear_int8",
                 "fgpu_gated_linear_int8", "fgpu_orthogonalize"):
        monkeypatch.setattr(fg.lib, name, no_call)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(fg, "_device_now", lambda: -1)
    monkeypatch.setattr(fg, "_stream", lambda: None)


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


I8, B16 = torch.int8, torch.bfloat16


@pytest.mark.parametrize("call,error", [
    (lambda: fg.gated_linear(t(2, 8), t(4, 8), act="tanh"), ValueError),
    (lambda: fg.gated_linear(t(2, 8), t(5, 8)), ValueError),
    (lambda: fg.gated_linear(t(2, 8), t(4, 7)), ValueError),
    (lambda: fg.gated_linear(t(2, 8), t(4, 8, dtype=B16)), TypeError),
    (lambda: fg.gated_linear(t(2, 8), t(4, 8), bias=t(2)), ValueError),
    (lambda: fg.gated_linear(t(2, 8), t(4, 8), out=t(2, 4)), ValueError),
    (lambda: fg.gated_linear_backward(t(2, 2), t(2, 8), t(4, 8), t(2, 2)), ValueError),
    (lambda: fg.gated_linear_backward(t(2, 2), t(2, 8), t(4, 8), None), TypeError),
    (lambda: fg.gated_linear_backward(t(2, 2), t(3, 8), t(4, 8), t(2, 4)), ValueError),
    (lambda: fg.gated_linear_backward(t(2, 2), t(2, 8), t(2, 8), t(2, 4)), ValueError),
    (lambda: fg.gated_linear_backward(t(2, 2), t(2, 8), t(4, 8), t(2, 4), want=("gate",)), ValueError),
    (lambda: fg.quantize_rows(t(8)), ValueError),
    (lambda: fg.quantize_rows(t(2, 8, dtype=torch.int32)), TypeError),
    (lambda: fg.linear_int8(t(2, 8), t(4, 8, dtype=I8), t(4)), ValueError),
    (lambda: fg.linear_int8(t(2, 8), t(4, 16), t(4)), TypeError),
    (lambda: fg.linear_int8(t(2, 8), t(4, 16, dtype=I8), t(3)), ValueError),
    (lambda: fg.linear_int8(t(2, 8), t(4, 16, dtype=I8), t(4), bias=t(4, dtype=B16)), TypeError),
    (lambda: fg.linear_int8(t(2, 8), t(4, 16, dtype=I8), t(4), residual=t(2, 5)), ValueError),
    (lambda: fg.linear_int8(t(2, 8), t(4, 16, dtype=I8), t(4), dtype=B16), TypeError),
    (lambda: fg.linear_int8(t(2, 8, dtype=I8), t(4, 16, dtype=I8), t(4), x_scale=t(2)), ValueError),
    (lambda: fg.linear_int8(t(2, 16, dtype=I8), t(4, 16, dtype=I8), t(4)), TypeError),
    (lambda: fg.linear_int8(t(2, 16, dtype=I8), t(4, 16, dtype=I8), t(4), x_scale=t(3)), ValueError),
    (lambda: fg.linear_int8(t(2, 16, dtype=I8), t(4, 16, dtype=I8), t(4), x_scale=t(2), dtype=torch.float16), TypeError),
    (lambda: fg.linear_int8(t(2, 8), t(4, 16, dtype=I8), t(4), out=t(2, 4, dtype=B16)), ValueError),
    (lambda: fg.gated_linear_int8(t(2, 8), t(5, 16, dtype=I8), t(5)), ValueError),
    (lambda: fg.gated_linear_int8(t(2, 8), t(4, 16, dtype=I8), t(4), bias=t(2)), ValueError),
    (lambda: fg.gated_linear_int8(t(2, 8), t(4, 16, dtype=I8), t(4), act="swish"), ValueError),
    (lambda: fg.orthogonalize(t(8)), ValueError),
    (lambda: fg.orthogonalize(t(2, 8), coefficients=(1.0, 2.0)), ValueError),
    (lambda: fg.orthogonalize(t(2, 8), out=t(8, 2)), ValueError),
])
def test_python_refusals(host, call, error):
    with pytest.raises(error):
        call()


def test_tensors_of_another_device_are_refused(host, monkeypatch):
    monkeypatch.setattr(fg, "_device_now", lambda: 1)
    w8, s = t(4, 16, dtype=I8), t(4)
    for call in (lambda: fg.gated_linear(t(2, 8), t(4, 8)), lambda: fg.gated_linear_backward(t(2, 2), t(2, 8), t(4, 8), t(2, 4)),
                 lambda: fg.quantize_rows(t(2, 8)), lambda: fg.linear_int8(t(2, 8), w8, s),
                 lambda: fg.gated_linear_int8(t(2, 8), w8, s), lambda: fg.orthogonalize(t(2, 8))):
        with pytest.raises(ValueError, match="current device"):
            call()


def test_row_bytes():
    assert [fg.int8_row(d) for d in (1, 15, 16, 17, 1024)] == [16, 16, 16, 32, 1024]
