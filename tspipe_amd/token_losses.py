"""Post-training losses on the log probabilities of sampled tokens, with fused
forward+backward HIP kernels: token log probabilities, a preference loss over
pairs of answers, and a clipped policy loss with a KL term.

The frozen or momentum teacher of the pipeline is the reference model here: its
log probabilities come from ``token_log_probs``, and ``preference_loss_fn`` /
``policy_loss_fn`` are ``loss_fn`` plug-ins (tspipe/gpu_task.py:178-179) that
take the student's and the teacher's logits.

The losses are returned in fp32 and, like those of ``losses``, keep one
gradient buffer, so that backward can run once per forward; ``weight`` scales
loss and gradient before the gradient is rounded to the logits' type (a half
precision gradient's loss scale belongs there).
"""
from typing import Optional

import torch
from torch import Tensor

from . import _lib
from ._vocab import floats_of, host_for, labels_of, mask_of, ptr, recorded, rows_of, same_device, temperature_of
from .losses import _once, _scale_saved_grad


class _TokenLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, labels: Tensor, row_mask: Optional[Tensor], temperature: float, ignore_index: int):
        r = rows_of(logits, "token_log_probs")
        same_device(logits.device, labels=labels, row_mask=row_mask)
        shape = logits.shape[:-1]
        lab = labels_of(labels, shape, "token_log_probs")
        mask = mask_of(row_mask, shape, "token_log_probs")
        dev = logits.device
        out = torch.empty(shape, dtype=torch.float32, device=dev)
        need = ctx.needs_input_grad[0]
        stats = torch.empty((r.count, 2), dtype=torch.float32, device=dev) if need else None
        with _lib.on_device(dev):
            status = _lib.lib().ts_token_logp_fwd(*r.geometry, lab.data_ptr(), ptr(mask), ignore_index, temperature,
                                                  out.data_ptr(), ptr(stats), r.code, _lib.current_stream_ptr(dev))
        _lib.check(status, "ts_token_logp_fwd")
        if need:
            ctx.save_for_backward(logits, lab, mask, stats)
            ctx.args = (temperature, ignore_index)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output: Tensor):
        logits, lab, mask, stats = ctx.saved_tensors
        temperature, ignore_index = ctx.args
        r = rows_of(logits, "token_log_probs")
        dev = logits.device
        g = grad_output.detach().to(torch.float32).contiguous()
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        with _lib.on_device(dev):
            status = _lib.lib().ts_token_logp_bwd(*r.geometry, lab.data_ptr(), ptr(mask), ignore_index, temperature,
                                                  stats.data_ptr(), g.data_ptr(), grad.data_ptr(), r.code,
                                                  _lib.current_stream_ptr(dev))
        _lib.check(status, "ts_token_logp_bwd")
        return grad, None, None, None, None


def token_log_probs(logits: Tensor, labels: Tensor, temperature: float = 1.0, ignore_index: int = -100,
                    row_mask: Optional[Tensor] = None) -> Tensor:
    """``log_softmax(logits / temperature)`` at ``labels``, fp32, in the shape
    of ``labels`` (``logits.shape[:-1]``).  Rows whose label is ``ignore_index``
    or outside the classes, or whose ``row_mask`` entry is 0, are not read: 0,
    with a zero gradient."""
    temperature, ignore_index = temperature_of(temperature, "token_log_probs"), int(ignore_index)
    host = host_for(logits, labels, row_mask)
    if host is not None:
        out = host[0].vocab_log_probs(logits, labels, row_mask, temperature, ignore_index, host[1])
        if out is not None:
            return out
    return _TokenLogProbsFn.apply(recorded(logits), labels, row_mask, temperature, ignore_index)


_PREFERENCE_KINDS = {"sigmoid": 0, "hinge": 1, "ipo": 2}


class _PreferenceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, labels: Tensor, ref: Tensor, row_mask: Optional[Tensor], beta: float, kind: int,
                smoothing: float, average: bool, weight: float, ignore_index: int):
        r = rows_of(logits, "preference_loss")
        same_device(logits.device, labels=labels, ref_log_probs=ref, row_mask=row_mask)
        shape = logits.shape[:-1]
        lab = labels_of(labels, shape, "preference_loss")
        mask = mask_of(row_mask, shape, "preference_loss")
        per_token = ref.dim() == 2
        ref = floats_of(ref, shape if per_token else shape[:1], "ref_log_probs")
        dev = logits.device
        lib = _lib.lib()
        ws = torch.empty(lib.ts_token_loss_workspace_bytes(r.n_seq, r.seq_len), dtype=torch.uint8, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        rewards = torch.empty(shape[:1], dtype=torch.float32, device=dev)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if ctx.needs_input_grad[0] else None
        with _lib.on_device(dev):
            status = lib.ts_preference_fwd_bwd(*r.geometry, lab.data_ptr(), ptr(mask), ignore_index, ref.data_ptr(),
                                               1 if per_token else 0, beta, kind, smoothing, 1 if average else 0,
                                               weight, ws.data_ptr(), loss.data_ptr(), rewards.data_ptr(), ptr(grad),
                                               r.code, _lib.current_stream_ptr(dev))
        _lib.check(status, "ts_preference_fwd_bwd")
        ctx.grad, ctx.dims, ctx.backward_done = grad, (r.count, r.V), False
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output: Tensor, _):
        return (_take_grad(ctx, grad_output),) + (None,) * 9


def _take_grad(ctx, grad_output: Tensor) -> Optional[Tensor]:
    """The gradient the forward pass left, scaled; the context lets go of it,
    so that autograd can adopt it as .grad instead of copying."""
    if not ctx.needs_input_grad[0]:
        return None
    _once(ctx)
    grad, ctx.grad = ctx.grad, None
    return _scale_saved_grad(grad, grad_output, *ctx.dims)


def preference_loss(logits: Tensor, labels: Tensor, ref_log_probs: Tensor, beta: float = 0.1,
                    loss_type: str = "sigmoid", label_smoothing: float = 0.0, length_average: bool = False,
                    weight: float = 1.0, ignore_index: int = -100, row_mask: Optional[Tensor] = None,
                    return_rewards: bool = False):
    """Preference loss over pairs of answers, mean over the pairs.

    ``logits`` is ``[2 pairs, tokens, classes]``, answer ``2i`` preferred to
    answer ``2i + 1`` (neighbours, so that a scatter along dim 0 keeps pairs
    together); ``labels`` are the tokens scored at each position, ``ignore_index``
    on prompts and padding.  ``ref_log_probs`` are the reference model's, per
    token (``labels.shape``) or summed per answer (``[2 pairs]``).  With ``R`` an
    answer's sum of ``log p - ref`` (its mean with ``length_average``, for which
    a per-answer reference has to be a mean as well) and ``h`` the difference
    within the pair:

    * ``"sigmoid"``: ``-(1 - s) log sigmoid(beta h) - s log sigmoid(-beta h)``, ``s`` the label smoothing,
    * ``"hinge"``: ``max(0, 1 - beta h)``,
    * ``"ipo"``: ``(h - 1 / (2 beta))^2``.

    With ``return_rewards`` also returns ``beta * R`` per answer, detached.  An
    answer without a token that counts has ``R = 0`` before a per-answer reference."""
    if logits.dim() != 3:
        raise ValueError(f"preference_loss expects [2 * pairs, tokens, classes] logits, got {tuple(logits.shape)}")
    if logits.shape[0] % 2:
        raise ValueError(f"preference_loss expects pairs of neighbouring answers, got {logits.shape[0]} answers")
    if loss_type not in _PREFERENCE_KINDS:
        raise ValueError(f"loss_type {loss_type!r}: one of {sorted(_PREFERENCE_KINDS)}")
    if not beta > 0:
        raise ValueError(f"preference_loss needs a positive beta, got {beta}")
    if not 0 <= label_smoothing <= 1 or (label_smoothing and loss_type != "sigmoid"):
        raise ValueError(f"label_smoothing {label_smoothing} with loss_type {loss_type!r}")
    kind = _PREFERENCE_KINDS[loss_type]
    host, out = host_for(logits, labels, ref_log_probs, row_mask), None
    if host is not None:
        out = host[0].vocab_preference(logits, labels, ref_log_probs, row_mask,
                                       (float(beta), float(label_smoothing), float(weight)),
                                       (kind, 1 if length_average else 0, int(ignore_index)), host[1])
    if out is None:
        out = _PreferenceFn.apply(recorded(logits), labels, ref_log_probs, row_mask, float(beta), kind,
                                  float(label_smoothing), bool(length_average), float(weight), int(ignore_index))
    loss, rewards = out
    return (loss, rewards) if return_rewards else loss


class _PolicyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, labels: Tensor, old: Tensor, adv: Tensor, ref: Optional[Tensor],
                row_mask: Optional[Tensor], kl_weight: float, clip_lo: float, clip_hi: float, temperature: float,
                per_seq: bool, weight: float, ignore_index: int):
        r = rows_of(logits, "clipped_policy_loss")
        same_device(logits.device, labels=labels, old_log_probs=old, advantages=adv, ref_log_probs=ref,
                    row_mask=row_mask)
        shape = logits.shape[:-1]
        lab = labels_of(labels, shape, "clipped_policy_loss")
        mask = mask_of(row_mask, shape, "clipped_policy_loss")
        old = floats_of(old, shape, "old_log_probs")
        ref = None if ref is None else floats_of(ref, shape, "ref_log_probs")
        adv_per_seq = adv.dim() == 1
        adv = floats_of(adv, shape[:1] if adv_per_seq else shape, "advantages")
        dev = logits.device
        lib = _lib.lib()
        ws = torch.empty(lib.ts_token_loss_workspace_bytes(r.n_seq, r.seq_len), dtype=torch.uint8, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        logp = torch.empty(shape, dtype=torch.float32, device=dev)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if ctx.needs_input_grad[0] else None
        with _lib.on_device(dev):
            status = lib.ts_policy_fwd_bwd(*r.geometry, lab.data_ptr(), ptr(mask), ignore_index, temperature,
                                           old.data_ptr(), ptr(ref), adv.data_ptr(), 1 if adv_per_seq else 0,
                                           kl_weight, clip_lo, clip_hi, 1 if per_seq else 0, weight, ws.data_ptr(),
                                           loss.data_ptr(), logp.data_ptr(), ptr(grad), r.code,
                                           _lib.current_stream_ptr(dev))
        _lib.check(status, "ts_policy_fwd_bwd")
        ctx.grad, ctx.dims, ctx.backward_done = grad, (r.count, r.V), False
        ctx.mark_non_differentiable(logp)
        return loss, logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output: Tensor, _):
        return (_take_grad(ctx, grad_output),) + (None,) * 12


def clipped_policy_loss(logits: Tensor, labels: Tensor, old_log_probs: Tensor, advantages: Tensor,
                        ref_log_probs: Optional[Tensor] = None, kl_weight: float = 0.0, clip_low: float = 0.2,
                        clip_high: float = 0.2, temperature: float = 1.0, reduction: str = "token",
                        weight: float = 1.0, ignore_index: int = -100, row_mask: Optional[Tensor] = None,
                        return_log_probs: bool = False):
    """Clipped policy loss on sampled answers.

    ``logits`` is ``[answers, tokens, classes]``; ``labels`` are the sampled
    tokens, ``ignore_index`` on prompts and padding; ``old_log_probs`` are the
    sampling policy's (``labels.shape``), ``advantages`` per token or per answer
    (``[answers]``).  With ``r = exp(log p - old)`` a token's term is
    ``-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_weight (exp(d) - d - 1)``,
    ``d = ref - log p``.  ``reduction="token"`` is the mean over all tokens that
    count, ``"sequence"`` the mean over the answers that have such tokens of
    each one's mean.  With ``return_log_probs`` also returns ``log p`` per token,
    detached."""
    if logits.dim() != 3:
        raise ValueError(f"clipped_policy_loss expects [answers, tokens, classes] logits, got {tuple(logits.shape)}")
    if reduction not in ("token", "sequence"):
        raise ValueError(f"reduction {reduction!r}: 'token' or 'sequence'")
    if kl_weight != 0 and ref_log_probs is None:
        raise ValueError("a KL term needs ref_log_probs")
    if not (clip_low >= 0 and clip_high >= 0):
        raise ValueError(f"clipping range [1 - {clip_low}, 1 + {clip_high}]")
    temperature = temperature_of(temperature, "clipped_policy_loss")
    numbers = (float(kl_weight), 1.0 - float(clip_low), 1.0 + float(clip_high), temperature)
    host, out = host_for(logits, labels, old_log_probs, advantages, ref_log_probs, row_mask), None
    if host is not None:
        out = host[0].vocab_policy(logits, labels, old_log_probs, advantages, ref_log_probs, row_mask,
                                   (*numbers, float(weight)), (1 if reduction == "sequence" else 0, int(ignore_index)),
                                   host[1])
    if out is None:
        out = _PolicyFn.apply(recorded(logits), labels, old_log_probs, advantages, ref_log_probs, row_mask, *numbers,
                              reduction == "sequence", float(weight), int(ignore_index))
    loss, logp = out
    return (loss, logp) if return_log_probs else loss


# ---------------------------------------------------------------------------
# loss_fn plug-ins
# ---------------------------------------------------------------------------

def _next_tokens(tokens: Tensor, answer_mask: Tensor) -> Tensor:
    """What the logits at each position of a causal model are scored against:
    the token at the next one where that belongs to the answer, else -100 (the
    shift of benchmarks/distilbert/distiller.py:745-749)."""
    shifted = torch.full_like(tokens, -100, dtype=torch.int64)
    shifted[..., :-1] = tokens[..., 1:].masked_fill(answer_mask[..., 1:] == 0, -100)
    return shifted


def preference_loss_fn(student_outputs, teacher_outputs, labels, tspipe_args, params, epoch: int) -> Tensor:
    """``loss_fn`` plug-in: ``preference_loss`` of a causal student against the
    frozen teacher.  ``labels`` is ``(tokens, answer_mask)``, both ``[2 pairs,
    tokens]``; ``params`` carries ``beta`` and optionally ``preference_type``,
    ``label_smoothing``, ``length_average`` and ``weight`` (a half precision
    gradient's loss scale)."""
    targets = _next_tokens(*labels)
    with torch.no_grad():
        ref = token_log_probs(teacher_outputs["logits"].detach(), targets)
    return preference_loss(student_outputs["logits"], targets, ref, beta=params.beta,
                           loss_type=getattr(params, "preference_type", "sigmoid"),
                           label_smoothing=getattr(params, "label_smoothing", 0.0),
                           length_average=getattr(params, "length_average", False),
                           weight=getattr(params, "weight", 1.0))


def policy_loss_fn(student_outputs, teacher_outputs, labels, tspipe_args, params, epoch: int) -> Tensor:
    """``loss_fn`` plug-in: ``clipped_policy_loss`` of a causal student with the
    teacher as the reference of the KL term.  ``labels`` is ``(tokens,
    answer_mask, old_log_probs, advantages)``, ``old_log_probs`` at the position
    whose logits gave them; ``params`` carries ``kl_weight``, ``clip_low``,
    ``clip_high`` and optionally ``temperature``, ``reduction`` and ``weight`` (a
    half precision gradient's loss scale)."""
    tokens, answer_mask, old, adv = labels
    targets = _next_tokens(tokens, answer_mask)
    temperature = getattr(params, "temperature", 1.0)
    ref = None
    if params.kl_weight != 0:
        with torch.no_grad():
            ref = token_log_probs(teacher_outputs["logits"].detach(), targets, temperature)
    return clipped_policy_loss(student_outputs["logits"], targets, old, adv, ref, params.kl_weight, params.clip_low,
                               params.clip_high, temperature, getattr(params, "reduction", "token"),
                               weight=getattr(params, "weight", 1.0))
