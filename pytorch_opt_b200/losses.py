"""Losses of language-model training over a large vocabulary, with their gradients.

Three functions of CUDA tensors (bf16, fp16 or fp32), differentiable by
``torch.autograd``; the kernels are those of ``po_linear_loss`` and
``po_distill_logits`` (``include/pytorch_opt_b200.h``):

* ``linear_cross_entropy(hidden, weight, target)`` — softmax cross entropy of
  ``hidden @ weight.T`` without that product as a tensor: per-token losses
  leave two numbers a row and 256 columns, gradients the scaled exponentials
  of one chunk of rows in 16 bits while the call runs;
* ``linear_distillation(hidden, weight, teacher_index, teacher_logits)`` — the
  divergence of the same product's softmax from a teacher's top logits;
* ``distillation(logits, teacher_index, teacher_logits)`` — the same for
  student logits that are there already.

Rows that count for nothing (``ignore_index``, no teacher's entry) have loss
and gradient 0, are left out of the mean, and cost no product. With a scalar
reduction the gradients are made together with the loss (the softmax is not
computed a second time) whenever an input requires grad (fp16 ones by powers of
two, so that neither a loss scale nor a division of the sum comes too late); with
``reduction="none"`` they are made in the backward pass from the upstream
gradient of each row. Derivatives are first order and reverse mode only: a dual
tensor of forward mode is refused. Errors are ``RuntimeError`` as in ``native``;
there is no CPU path.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_REDUCTIONS = ("mean", "sum", "none")
MAX_TOP = 1024
_MEAN_SCALED, _SUM_SCALED = 2, 3  # PO_MEAN_SCALED, PO_SUM_SCALED


def _check_tensors(name: str, first, *others) -> None:
    if not isinstance(first, torch.Tensor):
        raise RuntimeError(f"{name}: expected a tensor, got {type(first).__name__}")
    at = first.device
    if at.type != "cuda":
        raise RuntimeError("pytorch_opt_b200 runs on CUDA tensors only (there is no CPU path)")
    for t in others:
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(f"{name}: expected a tensor, got {type(t).__name__}")
        if t.device != at:
            raise RuntimeError("pytorch_opt_b200 runs on CUDA tensors only, all on the same device")


def _check_reduction(name: str, reduction: str) -> None:
    if reduction not in _REDUCTIONS:
        raise RuntimeError(f"{name}: reduction must be mean|sum|none, got {reduction}")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """The tensor as rows of its last axis, each contiguous (a copy only if they are not)."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if not x.is_contiguous():
        rows, cols = x.shape
        if cols > 1 and x.stride(1) != 1 or rows > 1 and x.stride(0) < cols:
            x = x.contiguous()
    return x


def _pitch(x: torch.Tensor) -> int:
    """Elements from one row to the next."""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


@functools.lru_cache(maxsize=512)
def _workspace_bytes(aligned: bool, *args) -> int:
    # Of the weight's address the workspace depends only on whether TMA takes it.
    return (_lib.load().po_linear_loss_workspace_bytes(16 if aligned else 2, *args) + 15) // 16 * 16


def _linear_loss(hidden, weight, index, teacher, ignore_index, smoothing, z_loss, temperature, mean, scalar, row_grad,
                 want_dh, want_dw, chunk_rows):
    """One call of po_linear_loss: (per-row losses or None, scalar loss or None, dhidden, dweight, unscale).

    ``unscale`` (or None): the factors that dhidden and dweight are still to be multiplied by.
    """
    tokens, dim = hidden.shape
    vocab, top = weight.shape[0], index.shape[1]
    dev, dtype = hidden.device, hidden.dtype
    code, w_ptr, w_ld = _lib.DTYPE_CODE[dtype], weight.data_ptr(), _pitch(weight)
    unscale = None
    with _lib.on_device(dev):
        nbytes = _workspace_bytes(w_ptr % 16 == 0, w_ld, code, tokens, dim, vocab, top, want_dh, want_dw, chunk_rows)
        if scalar:  # the per-row losses are the call's own: 4 bytes a row at the end of its workspace
            loss = torch.empty((), dtype=torch.float32, device=dev)
            ws = _lib.workspace(nbytes + 4 * tokens, dev)
            losses, rows_ptr = None, ws.data_ptr() + nbytes
            if dtype is torch.float16 and (want_dh or want_dw) and tokens:
                mean, rows = _MEAN_SCALED if mean else _SUM_SCALED, torch.empty(tokens + 2, dtype=torch.float32, device=dev)
                rows_ptr, unscale = rows.data_ptr(), rows[tokens:]
        else:
            loss, losses = None, torch.empty(tokens, dtype=torch.float32, device=dev)
            ws, rows_ptr = _lib.workspace(nbytes, dev), losses.data_ptr()
        dh = hidden.new_empty((tokens, dim)) if want_dh else None
        dw = weight.new_empty((vocab, dim)) if want_dw else None
        if teacher is None:
            t_ptr, t_ld, t_code = None, 0, 0
        else:
            t_ptr, t_ld, t_code = teacher.data_ptr(), _pitch(teacher), _lib.DTYPE_CODE[teacher.dtype]
        status = _lib.load().po_linear_loss(
            hidden.data_ptr(), _pitch(hidden), w_ptr, w_ld, code, tokens, dim, vocab, index.data_ptr(), _pitch(index),
            t_ptr, t_ld, t_code, top, ignore_index, smoothing, z_loss, temperature, mean,
            None if row_grad is None else row_grad.data_ptr(), rows_ptr, loss.data_ptr() if scalar else None,
            dh.data_ptr() if want_dh else None, dim, dw.data_ptr() if want_dw else None, dim, chunk_rows,
            ws.data_ptr(), nbytes, _lib.stream_ptr(dev))
        if status:
            _lib.check(status, "po_linear_loss")
    return losses, loss, dh, dw, unscale


def _distill_logits(logits, index, teacher, temperature, mean, scalar, row_grad, want_grad):
    """One call of po_distill_logits: (per-row losses or None, scalar loss or None, dlogits, unscale), as above."""
    tokens, vocab = logits.shape
    dev, dtype = logits.device, logits.dtype
    with _lib.on_device(dev):
        lib = _lib.load()
        dz = logits.new_empty((tokens, vocab)) if want_grad else None
        unscale = None
        if scalar:
            nbytes = (lib.po_distill_logits_workspace_bytes(tokens) + 15) // 16 * 16
            loss, losses = torch.empty((), dtype=torch.float32, device=dev), None
            ws = _lib.workspace(nbytes + 4 * tokens, dev)
            rows_ptr = ws.data_ptr() + nbytes
            if dtype is torch.float16 and want_grad and tokens:
                mean, rows = _MEAN_SCALED if mean else _SUM_SCALED, torch.empty(tokens + 1, dtype=torch.float32, device=dev)
                rows_ptr, unscale = rows.data_ptr(), rows[tokens:]
        else:
            nbytes, ws, loss = 0, None, None
            losses = torch.empty(tokens, dtype=torch.float32, device=dev)
            rows_ptr = losses.data_ptr()
        status = lib.po_distill_logits(
            logits.data_ptr(), _pitch(logits), _lib.DTYPE_CODE[dtype], tokens, vocab, index.data_ptr(), _pitch(index),
            teacher.data_ptr(), _pitch(teacher), _lib.DTYPE_CODE[teacher.dtype], index.shape[1], temperature, mean,
            None if row_grad is None else row_grad.data_ptr(), rows_ptr, loss.data_ptr() if scalar else None,
            dz.data_ptr() if want_grad else None, vocab, ws.data_ptr() if scalar else None, nbytes,
            _lib.stream_ptr(dev))
        if status:
            _lib.check(status, "po_distill_logits")
    return losses, loss, dz, unscale


def _upstream(up: torch.Tensor) -> torch.Tensor:
    return up if up.dtype == torch.float32 and up.is_contiguous() else up.float().contiguous()


def _scale(factor: torch.Tensor, *grads) -> None:
    """Gradients times a device scalar, in place; a factor of 1 (``loss.backward()``) moves no data."""
    have = [g for g in grads if g is not None]
    if not have:
        return
    x, y = have[0], have[1] if len(have) > 1 else None
    dev = factor.device
    with _lib.on_device(dev):
        _lib.check(_lib.load().po_scale_inplace(x.data_ptr(), x.numel(), None if y is None else y.data_ptr(),
                                                0 if y is None else y.numel(), _lib.DTYPE_CODE[x.dtype],
                                                factor.data_ptr(), _lib.stream_ptr(dev)), "po_scale_inplace")


def _chain(up: torch.Tensor, unscale, *grads) -> None:
    """Stored gradients to those of the upstream factor: fp16 ones each have a factor of their own."""
    if unscale is None:
        _scale(up, *grads)
    else:
        for factor, g in zip((up * unscale).unbind(), grads):
            _scale(factor, g)


def _records(*tensors) -> bool:
    """Whether the call goes through autograd's function: where it would be recorded, and inside a dual level, where
    a tensor may carry a tangent without requires_grad (also under no_grad): the function refuses those."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                return True
    return False


class _LinearLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, index, teacher, opts):
        reduction, chunk_rows, *terms = opts
        scalar = reduction != "none"
        want = ctx.needs_input_grad[:2] if scalar else (False, False)
        losses, loss, dh, dw, unscale = _linear_loss(hidden, weight, index, teacher, *terms, reduction == "mean", scalar, None,
                                            *want, chunk_rows)
        ctx.opts = opts
        if scalar:
            ctx.grads, ctx.unscale = (dh, dw), unscale
            return loss
        ctx.save_for_backward(hidden, weight, index, teacher)
        return losses

    @staticmethod
    def backward(ctx, up):
        return _LinearLoss._once(ctx, up) if torch.is_grad_enabled() else _LinearLoss._backward(ctx, up)

    @staticmethod
    def _backward(ctx, up):
        reduction, chunk_rows, *terms = ctx.opts
        up = _upstream(up)
        if reduction != "none":
            if ctx.grads is None:
                raise RuntimeError("the gradients of this loss were handed out already: one backward pass per loss")
            (dh, dw), ctx.grads = ctx.grads, None
            _chain(up, ctx.unscale, dh, dw)
            return dh, dw, None, None, None
        hidden, weight, index, teacher = ctx.saved_tensors
        _, _, dh, dw, _ = _linear_loss(hidden, weight, index, teacher, *terms, False, False, up, *ctx.needs_input_grad[:2],
                                    chunk_rows)
        return dh, dw, None, None, None

    _once = staticmethod(torch.autograd.function.once_differentiable(_backward))  # under create_graph


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, index, teacher, reduction, temperature):
        scalar = reduction != "none"
        losses, loss, dz, unscale = _distill_logits(logits, index, teacher, temperature, reduction == "mean", scalar, None,
                                           scalar and ctx.needs_input_grad[0])
        ctx.scalar, ctx.temperature = scalar, temperature
        if scalar:
            ctx.grad, ctx.unscale = dz, unscale
            return loss
        ctx.save_for_backward(logits, index, teacher)
        return losses

    @staticmethod
    def backward(ctx, up):
        return _Distillation._once(ctx, up) if torch.is_grad_enabled() else _Distillation._backward(ctx, up)

    @staticmethod
    def _backward(ctx, up):
        up = _upstream(up)
        if ctx.scalar:
            if ctx.grad is None:
                raise RuntimeError("the gradient of this loss was handed out already: one backward pass per loss")
            dz, ctx.grad = ctx.grad, None
            _chain(up, ctx.unscale, dz)
            return dz, None, None, None, None
        logits, index, teacher = ctx.saved_tensors
        return _distill_logits(logits, index, teacher, ctx.temperature, False, False, up, True)[2], None, None, None, None

    _once = staticmethod(torch.autograd.function.once_differentiable(_backward))  # under create_graph


def _head_loss(hidden, weight, index, teacher, reduction, chunk_rows, *terms):
    lead = hidden.shape[:-1]
    rows, head = _rows(hidden), _rows(weight)
    if _records(hidden, weight):
        out = _LinearLoss.apply(rows, head, index, teacher, (reduction, chunk_rows, *terms))
    else:
        each, scalar, *_ = _linear_loss(rows, head, index, teacher, *terms, reduction == "mean", reduction != "none",
                                          None, False, False, chunk_rows)
        out = each if scalar is None else scalar
    return out.reshape(lead) if reduction == "none" and len(lead) != 1 else out


def _check_head(name: str, hidden: torch.Tensor, weight: torch.Tensor) -> None:
    if hidden.dtype not in _DTYPES or weight.dtype != hidden.dtype:
        raise RuntimeError(f"{name}: hidden and weight must both be bf16, fp16 or fp32, got {hidden.dtype} and "
                           f"{weight.dtype}")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or not weight.numel():
        raise RuntimeError(f"{name}: expects hidden (..., dim) and weight (vocab, dim), got {tuple(hidden.shape)} and "
                           f"{tuple(weight.shape)}")


def _check_teacher(name: str, lead, index: torch.Tensor, teacher: torch.Tensor, temperature: float):
    if index.dtype != torch.int64 and index.dtype != torch.int32:
        raise RuntimeError(f"{name}: teacher_index must be int64 or int32, got {index.dtype}")
    if teacher.dtype not in _DTYPES:
        raise RuntimeError(f"{name}: teacher_logits must be fp32, bf16 or fp16, got {teacher.dtype}")
    if index.dim() < 1 or index.shape != teacher.shape or index.shape[:-1] != lead:
        raise RuntimeError(f"{name}: teacher_index and teacher_logits must be (..., top) over the same tokens, got "
                           f"{tuple(index.shape)} and {tuple(teacher.shape)} for {tuple(lead)}")
    if not 1 <= index.shape[-1] <= MAX_TOP:
        raise RuntimeError(f"{name}: 1 to {MAX_TOP} entries a token, got {index.shape[-1]}")
    if not 2.0**-60 <= temperature <= 2.0**60:  # its square and its reciprocal are fp32 numbers
        raise RuntimeError(f"{name}: temperature must be 2^-60 to 2^60, got {temperature}")
    return _rows(index.long()), _rows(teacher.detach() if teacher.requires_grad else teacher)


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, *, ignore_index: int = -100,
                         label_smoothing: float = 0.0, z_loss: float = 0.0, reduction: str = "mean",
                         chunk_rows: int = 0) -> torch.Tensor:
    """Softmax cross entropy of the logits ``hidden @ weight.T`` (fp32 result).

    ``hidden`` (..., dim), ``weight`` (vocab, dim), ``target`` (...) of indices.
    A token's loss is ``lse(z) - (1 - s) z_y - s mean(z) + z_loss lse(z)^2``
    with s = ``label_smoothing``. Tokens with ``target == ignore_index`` count
    for nothing; "mean" divides by the others (0 if there are none). A target
    outside the vocabulary makes its loss NaN and its gradient 0.
    ``chunk_rows``: tokens whose exponentials may lie in the workspace at once
    while gradients are made (0: as many as fit 2 GiB).
    """
    name = "linear_cross_entropy"
    _check_tensors(name, hidden, weight, target)
    _check_reduction(name, reduction)
    _check_head(name, hidden, weight)
    if target.dtype not in (torch.int64, torch.int32) or target.shape != hidden.shape[:-1]:
        raise RuntimeError(f"{name}: target must be int64 or int32 of shape {tuple(hidden.shape[:-1])}, got "
                           f"{target.dtype} {tuple(target.shape)}")
    if not 0.0 <= label_smoothing <= 1.0 or not abs(z_loss) < float("inf"):
        raise RuntimeError(f"{name}: label_smoothing must be in [0, 1] and z_loss finite")
    if chunk_rows < 0:
        raise RuntimeError(f"{name}: chunk_rows must not be negative")
    return _head_loss(hidden, weight, _rows(target.long().reshape(-1, 1)), None, reduction, int(chunk_rows),
                      int(ignore_index), float(label_smoothing), float(z_loss), 1.0)


def linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_index: torch.Tensor,
                        teacher_logits: torch.Tensor, *, temperature: float = 1.0, reduction: str = "mean",
                        chunk_rows: int = 0) -> torch.Tensor:
    """Divergence of ``softmax(hidden @ weight.T / a)`` from a teacher's top logits (fp32 result).

    ``teacher_index`` and ``teacher_logits`` (..., top): where a token's index
    is negative there is no entry. With q the softmax of the entries' logits
    divided by a = ``temperature``, a token's loss is ``a^2 sum_k q_k (log q_k
    - log p_k)``, p the student's softmax over the whole vocabulary. Tokens
    without an entry count for nothing. An index past the vocabulary makes its
    token's loss NaN and its gradient 0. ``chunk_rows`` as in
    ``linear_cross_entropy``.
    """
    name = "linear_distillation"
    _check_tensors(name, hidden, weight, teacher_index, teacher_logits)
    _check_reduction(name, reduction)
    _check_head(name, hidden, weight)
    if chunk_rows < 0:
        raise RuntimeError(f"{name}: chunk_rows must not be negative")
    lead = hidden.shape[:-1]
    index, teacher = _check_teacher(name, lead, teacher_index, teacher_logits, temperature)
    return _head_loss(hidden, weight, index, teacher, reduction, int(chunk_rows), 0, 0.0, 0.0, float(temperature))


def distillation(logits: torch.Tensor, teacher_index: torch.Tensor, teacher_logits: torch.Tensor, *,
                 temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """``linear_distillation`` for student logits (..., vocab) that are there already (fp32 result)."""
    name = "distillation"
    _check_tensors(name, logits, teacher_index, teacher_logits)
    _check_reduction(name, reduction)
    if logits.dtype not in _DTYPES or logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError(f"{name}: logits must be (..., vocab) of bf16, fp16 or fp32, got {logits.dtype} "
                           f"{tuple(logits.shape)}")
    lead = logits.shape[:-1]
    index, teacher = _check_teacher(name, lead, teacher_index, teacher_logits, temperature)
    rows = _rows(logits)
    if _records(logits):
        out = _Distillation.apply(rows, index, teacher, reduction, float(temperature))
    else:
        each, mean, *_ = _distill_logits(rows, index, teacher, float(temperature), reduction == "mean",
                                        reduction != "none", None, False)
        out = each if mean is None else mean
    return out.reshape(lead) if reduction == "none" and len(lead) != 1 else out
