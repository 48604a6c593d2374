"""The query head's refusals, on the CPU: every bad argument is turned down before anything reaches the device."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import fusiongpu_amd as fg  # noqa: E402

L = fg.lib
ARG, UNSUPPORTED, WORKSPACE = 1, 2, 6
P = 1 << 20  # stands for a 16-byte-aligned device pointer: refused calls never read it
F32, BF16 = 0, 1


def linear(x=P, w=P, b=None, r=None, rows=4, k=8, n=8, dt=F32, act=0, y=P, pre=None, ws=P, wsb=1 << 30):
    return L.fgpu_linear(x, w, b, r, rows, k, n, dt, act, y, pre, ws, wsb, None)


def linear_bwd(dy=P, x=P, w=P, pre=None, rows=4, k=8, n=8, dt=F32, act=0, dx=P, dw=P, db=P, ws=P, wsb=1 << 30):
    return L.fgpu_linear_backward(dy, x, w, pre, rows, k, n, dt, act, dx, dw, db, ws, wsb, None)


def norm(x=P, rows=4, dim=8, dt=F32, eps=1e-5, y=P):
    return L.fgpu_layer_norm(x, None, None, rows, dim, dt, eps, y, None, None, None)


def norm_bwd(dy=P, x=P, mean=P, rstd=P, rows=4, dim=8, dt=F32, dg=P, ws=P, wsb=1 << 30):
    return L.fgpu_layer_norm_backward(dy, x, None, mean, rstd, rows, dim, dt, P, dg, None, ws, wsb, None)


def loss(q=P, c=P, t=P, nq=4, nc=8, dim=8, dt=F32, out=P, lse=P, ws=P, wsb=1 << 30):
    return L.fgpu_contrastive_loss(q, c, t, None, None, nq, nc, dim, dt, 1.0, out, lse, ws, wsb, None)


def loss_bwd(g=P, q=P, c=P, t=P, lse=P, nq=4, nc=8, dim=8, dt=F32, ws=P, wsb=1 << 30):
    return L.fgpu_contrastive_loss_backward(g, q, c, t, lse, None, None, nq, nc, dim, dt, 1.0, P, P, P, ws, wsb, None)


@pytest.mark.parametrize("f,args,want", [
    (linear, dict(dt=2), ARG), (linear, dict(act=4), ARG), (linear, dict(act=-1), ARG), (linear, dict(rows=-1), ARG),
    (linear, dict(k=0), ARG), (linear, dict(n=0), ARG), (linear, dict(x=None), ARG), (linear, dict(w=None), ARG),
    (linear, dict(y=None), ARG), (linear, dict(x=P + 4), ARG), (linear, dict(w=P + 8), ARG), (linear, dict(ws=P + 4), ARG),
    (linear, dict(rows=1 << 16, k=1023, n=1024, dt=BF16, wsb=0), WORKSPACE), (linear, dict(k=(1 << 16) + 1), UNSUPPORTED), (linear, dict(rows=(1 << 30) + 1), UNSUPPORTED),
    (linear_bwd, dict(dt=-1), ARG), (linear_bwd, dict(act=2), ARG), (linear_bwd, dict(dy=None), ARG),
    (linear_bwd, dict(w=None), ARG), (linear_bwd, dict(x=None), ARG), (linear_bwd, dict(dy=P + 2), ARG),
    (linear_bwd, dict(rows=1 << 16, k=1024, n=1024, dt=BF16, wsb=0), WORKSPACE), (linear_bwd, dict(n=0), ARG), (linear_bwd, dict(n=1 << 17), UNSUPPORTED),
    (norm, dict(dt=7), ARG), (norm, dict(dim=0), ARG), (norm, dict(eps=-1.0), ARG), (norm, dict(eps=float("nan")), ARG),
    (norm, dict(x=None), ARG), (norm, dict(y=None), ARG), (norm, dict(rows=-2), ARG), (norm, dict(dim=16385), UNSUPPORTED),
    (norm_bwd, dict(mean=None), ARG), (norm_bwd, dict(rstd=None), ARG), (norm_bwd, dict(dy=None), ARG),
    (norm_bwd, dict(wsb=0), WORKSPACE), (norm_bwd, dict(dt=3), ARG),
    (loss, dict(dt=2), ARG), (loss, dict(nc=0), ARG), (loss, dict(dim=0), ARG), (loss, dict(nq=-1), ARG), (loss, dict(q=None), ARG),
    (loss, dict(t=None), ARG), (loss, dict(lse=None), ARG), (loss, dict(c=P + 8), ARG), (loss, dict(wsb=0), WORKSPACE),
    (loss, dict(nq=(1 << 20) + 1), UNSUPPORTED), (loss, dict(dim=1 << 17), UNSUPPORTED),
    (loss_bwd, dict(g=None), ARG), (loss_bwd, dict(lse=None), ARG), (loss_bwd, dict(q=P + 4), ARG),
    (loss_bwd, dict(wsb=0), WORKSPACE), (loss_bwd, dict(nc=0), ARG),
])
def test_refused_with_its_status(f, args, want):
    assert f(**args) == want
    assert L.fgpu_last_error()


@pytest.mark.parametrize("f", [linear, norm])
def test_no_rows_is_no_work(f):
    assert f(rows=0, x=None, y=None) == 0


def test_no_queries_is_no_work():
    assert loss(nq=0, q=None, c=None, t=None) == 0


def test_workspace_sizes():
    # bf16 rows of whole 16-byte groups enter the product as they are; others, and float32, are copied.
    assert L.fgpu_linear_workspace_bytes(0, 8, 8, BF16) == 0
    assert L.fgpu_linear_workspace_bytes(1 << 16, 1024, 4096, BF16) == 0
    assert L.fgpu_linear_workspace_bytes(1 << 16, 1023, 4096, BF16) >= (1 << 16) * 1024 * 2
    assert L.fgpu_linear_workspace_bytes(1 << 16, 1024, 4096, F32) >= (1 << 16) * 1024 * 6
    assert L.fgpu_linear_workspace_bytes(4, 8, 8, 9) == 0
    # above 128 dims the score gradient is held whole up to 2^31 elements, in column chunks beyond; up to 128, not at all
    whole = L.fgpu_contrastive_loss_backward_workspace_bytes(4096, 65536, 256, BF16)
    assert whole >= 4096 * 65536 * 2
    assert L.fgpu_contrastive_loss_backward_workspace_bytes(1 << 16, 1 << 20, 136, BF16) < (1 << 33)
    assert L.fgpu_contrastive_loss_backward_workspace_bytes(4096, 65536, 128, BF16) < whole // 4


@pytest.fixture
def host(monkeypatch):
    """The Python mirror's checks without a device: tensors stay where they are and no call goes out."""
    def no_call(*a):
        raise AssertionError("a refused call reached the library")
    for name in ("fgpu_linear", "fgpu_linear_backward", "fgpu_layer_norm", "fgpu_layer_norm_backward", "fgpu_contrastive_loss",
                 "fgpu_contrastive_loss_backward"):
        monkeypatch.setattr(fg.lib, name, no_call)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(fg, "_stream", lambda: None)


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call,error", [
    (lambda: fg.linear(t(2, 8), t(4, 8), act="tanh"), ValueError),
    (lambda: fg.linear(t(2, 8), t(4, 7)), ValueError),
    (lambda: fg.linear(t(2, 8), t(4, 8, dtype=torch.bfloat16)), TypeError),
    (lambda: fg.linear(t(2, 8, dtype=torch.bfloat16), t(4, 8)), TypeError),
    (lambda: fg.linear(t(8), t(4, 8)), ValueError),
    (lambda: fg.linear(t(2, 8, dtype=torch.int32), t(4, 8)), TypeError),
    (lambda: fg.linear(t(2, 8), t(4, 8), bias=t(3)), ValueError),
    (lambda: fg.linear(t(2, 8), t(4, 8), residual=t(2, 3)), ValueError),
    (lambda: fg.linear(t(2, 8), [[0.0] * 8]), TypeError),
    (lambda: fg.linear(t(2, 8), t(4, 8), out=t(2, 5)), ValueError),
    (lambda: fg.linear_backward(t(2, 4), t(2, 8), t(4, 8), act="gelu"), ValueError),
    (lambda: fg.linear_backward(t(2, 4), t(3, 8), t(4, 8)), ValueError),
    (lambda: fg.linear_backward(t(2, 4), t(2, 8), t(4, 8), want=("w",)), ValueError),
    (lambda: fg.layer_norm(t(2, 8), gamma=t(7)), ValueError),
    (lambda: fg.layer_norm(t(2, 8), gamma=t(8, dtype=torch.bfloat16)), TypeError),
    (lambda: fg.layer_norm_backward(t(2, 8), t(2, 8), None, t(3), t(2)), ValueError),
    (lambda: fg.layer_norm_backward(t(2, 8), t(2, 8), None, t(2), t(2), want=("y",)), ValueError),
    (lambda: fg.contrastive_loss(t(2, 8), t(4, 9), np.zeros(2, np.int32)), ValueError),
    (lambda: fg.contrastive_loss(t(2, 8), t(4, 8), np.zeros(3, np.int32)), ValueError),
    (lambda: fg.contrastive_loss(t(2, 8), t(4, 8), np.zeros(2, np.int32), bias=t(5)), ValueError),
    (lambda: fg.contrastive_loss(t(2, 8), t(4, 8), np.zeros(2, np.float32)), TypeError),
    (lambda: fg.contrastive_loss(t(2, 8), t(4, 8), np.full(2, 1 << 40)), ValueError),
    (lambda: fg.contrastive_loss_backward(t(3), t(2, 8), t(4, 8), np.zeros(2, np.int32), t(2)), ValueError),
])
def test_python_refusals(host, call, error):
    with pytest.raises(error):
        call()


def test_header_constants_match():
    assert fg.ACTIVATIONS == dict(none=0, relu=1, gelu=2, silu=3)
    assert ctypes.c_float(-2.0**126).value == np.float32(-8.507059173023462e37)
