"""Sparse teachers: the largest logits of each teacher row, and the
distillation loss from them, with HIP kernels.

A teacher stage that hands on ``top_logits`` instead of its logits sends
``k * 6 + 4`` bytes a row in 16-bit types where the logits are ``2 * classes``;
``top_distil_loss_fn`` is the ``loss_fn`` plug-in on that side of the pipeline
(tspipe/gpu_task.py:178-179).
"""
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _lib
from ._vocab import floats_of, host_for, mask_of, ptr, recorded, rows_of, same_device, temperature_of
from .losses import _once, _scale_saved_grad

MAX_ENTRIES = 256  # entries a row may keep


class TopLogits(NamedTuple):
    values: Tensor      # [..., k], the logits' type, largest first
    indices: Tensor     # [..., k], int32
    logsumexp: Tensor   # [...], fp32, of logits / temperature


def top_logits(logits: Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The ``k`` largest logits of each row (last dimension), largest first and
    equal ones by their place, with the log-sum-exp of ``logits / temperature``;
    all detached.  ``1 <= k <= min(classes, 256)``."""
    t = temperature_of(temperature, "top_logits")
    k = int(k)
    host = host_for(logits)
    if host is not None and logits.dim() > 0 and 1 <= k <= min(int(logits.shape[-1]), MAX_ENTRIES):
        out = host[0].vocab_top(logits, k, t, host[1])
        if out is not None:
            return TopLogits(*out)
    r = rows_of(logits, "top_logits")
    if not 1 <= k <= min(r.V, MAX_ENTRIES):
        raise ValueError(f"top_logits keeps 1 to {min(r.V, MAX_ENTRIES)} of {r.V} classes, asked for {k}")
    dev = logits.device
    shape = logits.shape[:-1]
    values = torch.empty(shape + (k,), dtype=logits.dtype, device=dev)
    indices = torch.empty(shape + (k,), dtype=torch.int32, device=dev)
    lse = torch.empty(shape, dtype=torch.float32, device=dev)
    with _lib.on_device(dev):
        status = _lib.lib().ts_top_logits(*r.geometry, k, t, values.data_ptr(), indices.data_ptr(), lse.data_ptr(),
                                          r.code, _lib.current_stream_ptr(dev))
    _lib.check(status, "ts_top_logits")
    return TopLogits(values, indices, lse)


class _TopDistilFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, s_logits: Tensor, t_values: Tensor, t_indices: Tensor, t_logsumexp: Optional[Tensor],
                row_mask: Optional[Tensor], T: float, weight: float):
        what = "top_logits_distil_loss"
        r = rows_of(s_logits, what)
        same_device(s_logits.device, t_values=t_values, t_indices=t_indices, t_logsumexp=t_logsumexp, row_mask=row_mask)
        shape = s_logits.shape[:-1]
        if t_values.dim() < 1 or t_values.shape[:-1] != shape or t_indices.shape != t_values.shape:
            raise ValueError(f"teacher entries of shapes {tuple(t_values.shape)} and {tuple(t_indices.shape)} for "
                             f"rows of shape {tuple(shape)}")
        k = int(t_values.shape[-1])
        if not 1 <= k <= MAX_ENTRIES:
            raise ValueError(f"1 to {MAX_ENTRIES} teacher entries a row, got {k}")
        if t_indices.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"teacher indices are int32 or int64, got {t_indices.dtype}")
        vals = t_values.detach().contiguous()
        v_code = _lib.dtype_code(vals.dtype)
        idx = t_indices.detach()
        if idx.dtype == torch.int64:
            idx = idx.clamp(-1, 2 ** 31 - 1).to(torch.int32)  # what is out of range stays so
        idx = idx.contiguous()
        lse = None if t_logsumexp is None else floats_of(t_logsumexp, shape, "t_logsumexp")
        mask = mask_of(row_mask, shape, what)
        dev = s_logits.device
        lib = _lib.lib()
        ws = torch.empty(lib.ts_top_distil_workspace_bytes(r.count, k), dtype=torch.uint8, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        grad = torch.empty(s_logits.shape, dtype=s_logits.dtype, device=dev) if ctx.needs_input_grad[0] else None
        with _lib.on_device(dev):
            status = lib.ts_top_distil_fwd_bwd(*r.geometry, vals.data_ptr(), v_code, idx.data_ptr(), ptr(lse), k,
                                               ptr(mask), T, weight, ws.data_ptr(), loss.data_ptr(), ptr(grad), r.code,
                                               _lib.current_stream_ptr(dev))
        _lib.check(status, "ts_top_distil_fwd_bwd")
        ctx.grad, ctx.dims, ctx.backward_done = grad, (r.count, r.V), False
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output: Tensor):
        if not ctx.needs_input_grad[0]:
            return (None,) * 7
        _once(ctx)
        grad, ctx.grad = ctx.grad, None  # autograd can adopt it as .grad
        return (_scale_saved_grad(grad, grad_output, *ctx.dims),) + (None,) * 6


def top_logits_distil_loss(s_logits: Tensor, t_values: Tensor, t_indices: Tensor, T: float, weight: float = 1.0,
                           row_mask: Optional[Tensor] = None, t_logsumexp: Optional[Tensor] = None) -> Tensor:
    """``kd_soft_target_loss`` against a teacher of which each row's largest
    logits are known (``t_values``, ``t_indices``, ``[..., k]``): ``weight * T^2``
    times the mean over the rows of ``row_mask`` of ``sum p (log p - log q)``,
    ``q`` the student's ``softmax(s_logits / T)`` over all classes.

    Without ``t_logsumexp`` the teacher's probabilities are normalised over the
    kept entries.  With it (of the teacher's ``logits / T``, as ``top_logits``
    returns it) they are the full softmax's, and all other classes form one
    more outcome: what the teacher leaves to them against what the student
    does (up to 2^20 classes).  What is left over by no more than
    ``t_logsumexp``'s error, 4e-6 and a rounding, is nothing where the student
    leaves them less than e^-69 (a vocabulary masked to fewer tokens than
    entries), and an infinite loss if more is left where it leaves them nothing.

    Entries with an index outside the classes are absent and those of value
    -inf weigh nothing; a token named twice counts with both its entries.  Up
    to 256 entries a row; the teacher's type may differ from the student's."""
    T = temperature_of(T, "top_logits_distil_loss")
    host = host_for(s_logits, t_values, t_indices, t_logsumexp, row_mask)
    if host is not None:
        out = host[0].vocab_top_distil(s_logits, t_values, t_indices, t_logsumexp, row_mask, T, float(weight), host[1])
        if out is not None:
            return out
    return _TopDistilFn.apply(recorded(s_logits), t_values, t_indices, t_logsumexp, row_mask, T, float(weight))


def top_distil_loss_fn(student_outputs, teacher_outputs, labels, tspipe_args, params, epoch: int) -> Tensor:
    """``loss_fn`` plug-in: the distillation term of ``distil_loss_fn``
    (benchmarks/distilbert/distiller.py:719-740) from a sparse teacher.
    ``teacher_outputs`` holds ``top_values``, ``top_indices`` and
    ``top_logsumexp`` (a teacher that ran ``top_logits`` itself, at
    ``params.temperature``) or ``logits``, of which the ``params.top_k`` largest
    are taken here.  ``params`` further carries ``alpha_ce``,
    ``restrict_ce_to_mask`` and optionally ``top_tail`` (default true: the other
    classes as one outcome)."""
    lm_labels, attention_mask = labels
    mask = (lm_labels > -1) if params.restrict_ce_to_mask else attention_mask
    if "top_values" in teacher_outputs:
        top = TopLogits(teacher_outputs["top_values"], teacher_outputs["top_indices"], teacher_outputs["top_logsumexp"])
    else:
        top = top_logits(teacher_outputs["logits"], params.top_k, params.temperature)
    tail = getattr(params, "top_tail", True)
    return top_logits_distil_loss(student_outputs["logits"], top.values, top.indices, params.temperature,
                                  weight=params.alpha_ce, row_mask=mask, t_logsumexp=top.logsumexp if tail else None)
