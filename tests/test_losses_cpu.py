"""Host-side checks of the loss operators that need no GPU: refusals of the
Python functions and of the C ABI, workspace sizes, and empty calls."""

import ctypes

import pytest
import torch

from pytorch_opt_b200 import _lib, losses

BF16, F16, F32, F64 = 1, 2, 0, 3
P = ctypes.c_void_p(256)  # never followed: every call below is refused or empty


def test_losses_refuse_cpu_tensors():
    h, w = torch.randn(4, 8), torch.randn(16, 8)
    i, t = torch.zeros(4, 2, dtype=torch.long), torch.zeros(4, 2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        losses.linear_cross_entropy(h, w, torch.zeros(4, dtype=torch.long))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        losses.linear_distillation(h, w, i, t)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        losses.distillation(torch.randn(4, 16), i, t)
    with pytest.raises(RuntimeError, match="expected a tensor"):
        losses.linear_cross_entropy(h.tolist(), w, None)


def _head(lib, dtype=BF16, T=4, D=8, V=16, teacher=None, tdt=F32, top=1, smoothing=0.0, z_loss=0.0, temp=1.0, mean=1,
          row_grad=None, h_ld=8, w_ld=8, index_ld=1, t_ld=8, dh=None, dw=None, ws=P, ws_bytes=1 << 30, hidden=P,
          weight=P, index=P, rows=P):
    return lib.po_linear_loss(hidden, h_ld, weight, w_ld, dtype, T, D, V, index, index_ld, teacher, t_ld, tdt, top,
                              -100, smoothing, z_loss, temp, mean, row_grad, rows, P, dh, D, dw, D, 0, ws, ws_bytes,
                              None)


@pytest.mark.parametrize("bad, word", [
    (dict(dtype=F64), "dtype"), (dict(T=-1), "size"), (dict(D=0), "size"), (dict(V=0), "size"),
    (dict(T=1 << 30), "too large"), (dict(top=2), "top"), (dict(teacher=P, top=1025), "top"),
    (dict(teacher=P, top=0), "top"), (dict(teacher=P, tdt=F64), "teacher dtype"),
    (dict(teacher=P, temp=0.0), "temperature"), (dict(teacher=P, temp=float("nan")), "temperature"),
    (dict(temp=2.0), "temperature"), (dict(smoothing=-0.1), "smoothing"), (dict(smoothing=1.5), "smoothing"),
    (dict(z_loss=float("inf")), "z_loss"), (dict(teacher=P, smoothing=0.1), "smoothing"),
    (dict(row_grad=P, dh=P), "row_grad"), (dict(row_grad=P, mean=0), "row_grad"), (dict(h_ld=7), "pitch"),
    (dict(w_ld=7), "pitch"), (dict(index_ld=0), "pitch"), (dict(teacher=P, top=9, index_ld=9), "pitch"),
    (dict(hidden=None), "null"), (dict(weight=None), "null"), (dict(index=None), "null"), (dict(rows=None), "null"),
])
def test_linear_loss_abi_refuses(bad, word):
    lib = _lib.load()
    assert _head(lib, **bad) == 1
    assert word in _lib.last_error()


def test_linear_loss_abi_refuses_small_workspace():
    lib = _lib.load()
    assert _head(lib, ws=None) == 3
    need = lib.po_linear_loss_workspace_bytes(P, 8, BF16, 4, 8, 16, 1, 0, 0, 0)
    assert _head(lib, ws_bytes=need // 4) == 3
    assert "workspace" in _lib.last_error()


@pytest.mark.parametrize("bad, word", [
    (dict(dtype=F64), "dtype"), (dict(tdt=F64), "teacher dtype"), (dict(T=-1), "size"), (dict(V=0), "size"),
    (dict(top=0), "top"), (dict(top=1025), "top"), (dict(temp=-1.0), "temperature"), (dict(ld=15), "pitch"),
    (dict(index_ld=1), "pitch"), (dict(t_ld=1), "pitch"), (dict(row_grad=P, dz=P), "row_grad"),
    (dict(row_grad=P, mean=0), "row_grad"), (dict(logits=None), "null"), (dict(index=None), "null"),
])
def test_distill_abi_refuses(bad, word):
    lib = _lib.load()
    a = dict(dtype=BF16, T=4, V=16, top=2, tdt=F32, temp=1.0, mean=1, row_grad=None, ld=16, index_ld=2, t_ld=2, dz=None,
             logits=P, index=P)
    a.update(bad)
    rc = lib.po_distill_logits(a["logits"], a["ld"], a["dtype"], a["T"], a["V"], a["index"], a["index_ld"], P, a["t_ld"],
                               a["tdt"], a["top"], a["temp"], a["mean"], a["row_grad"], P, P, a["dz"], 16, P, 8, None)
    assert rc == 1
    assert word in _lib.last_error()


def test_scale_abi_refuses():
    lib = _lib.load()
    assert lib.po_scale_inplace(P, 4, None, 0, F64, P, None) == 1
    assert lib.po_scale_inplace(P, -4, None, 0, F32, P, None) == 1
    assert lib.po_scale_inplace(P, 4, P, -4, F32, P, None) == 1
    assert lib.po_scale_inplace(None, 4, None, 0, F32, P, None) == 1
    assert lib.po_scale_inplace(P, 4, None, 0, F32, None, None) == 1
    assert lib.po_scale_inplace(None, 0, None, 0, F32, None, None) == 0


def test_workspace_follows_what_is_asked():
    lib = _lib.load()
    size = lambda dtype=BF16, T=4096, D=1024, V=50257, top=1, dh=1, dw=1, chunk=0, ld=1024: (  # noqa: E731
        lib.po_linear_loss_workspace_bytes(P, ld, dtype, T, D, V, top, dh, dw, chunk))
    logits = 4096 * 50257 * 2
    assert size(dh=0, dw=0) < logits // 4  # losses alone never hold the logits
    assert logits < size() < 2 * logits
    assert size(chunk=512, dw=0) < logits // 4  # a chunk of rows bounds what gradients hold
    assert size(dtype=F32) > size()
    assert size(ld=1025) > size(dh=1, dw=1) + 50257 * 1024  # a pitch that TMA does not take: staged copy
    assert lib.po_linear_loss_workspace_bytes(P, 8, BF16, 0, 8, 8, 1, 1, 1, 0) == 0
    assert lib.po_distill_logits_workspace_bytes(0) == 0
