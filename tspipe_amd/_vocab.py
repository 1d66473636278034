"""Argument handling shared by the losses on rows of vocabulary logits."""
import math
from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _lib


_HOST_NODE = True   # tests switch this off to reach the Python autograd.Functions


def host_for(*tensors):
    """The C++ host helper and the current stream's handle when it may take a
    call on these tensors (plain device tensors, None allowed), else None: the
    same entry points on the same arguments, so the same bits, without the
    interpreter's share of the host time.  Its functions return None for calls
    that are not plain, and the Python function takes those."""
    host = _lib.host_helper() if _HOST_NODE else None
    if host is None or not hasattr(host, "vocab_top"):
        return None
    for t in tensors:
        if t is not None and type(t) is not Tensor:
            return None
    if not tensors[0].is_cuda:
        return None
    return host, _lib.current_stream_ptr(tensors[0].device)


class Rows(NamedTuple):
    """Logits as the kernels take them: ``n_seq`` sequences of ``seq_len``
    tokens, strides in elements; ``x`` keeps the memory alive."""
    x: Tensor
    n_seq: int
    seq_len: int
    V: int
    ld_seq: int
    ld_tok: int
    code: int

    @property
    def geometry(self):
        return self.x.data_ptr(), self.n_seq, self.seq_len, self.V, self.ld_seq, self.ld_tok

    @property
    def count(self) -> int:
        return self.n_seq * self.seq_len


def rows_of(logits: Tensor, what: str) -> Rows:
    """Slices and other strided views are read where they lie; only a last
    dimension that is not dense is copied."""
    if not isinstance(logits, Tensor):
        raise TypeError(f"{what}: expected a tensor of logits")
    if not logits.is_cuda:
        raise TypeError("tspipe_amd losses run on device tensors only (no host fallback)")
    code = _lib.dtype_code(logits.dtype)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: expected [..., classes] logits, got shape {tuple(logits.shape)}")
    x = logits.detach()
    V = int(x.shape[-1])
    if V > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    if x.dim() == 1:
        x = x[None]
    elif x.dim() > 3:
        x = x.reshape(math.prod(x.shape[:-2]), x.shape[-2], V)  # (-1 is ambiguous where there is nothing)
        if V > 1 and x.stride(-1) != 1:
            x = x.contiguous()
    if x.dim() == 2:
        return Rows(x, 1, int(x.shape[0]), V, 0, x.stride(0), code)
    return Rows(x, int(x.shape[0]), int(x.shape[1]), V, x.stride(0), x.stride(1), code)


def recorded(logits: Tensor) -> Tensor:
    """The logits as an autograd function should see them: without gradient
    mode nothing is recorded, so no gradient buffer is wanted either."""
    if not torch.is_grad_enabled():
        return logits.detach()
    if logits.requires_grad and logits.is_leaf and logits.is_cuda:
        host = _lib.host_helper()
        if host is not None and hasattr(host, "check_capture"):
            host.check_capture(logits, _lib.current_stream_ptr(logits.device))
    return logits


def same_device(device, **tensors: Optional[Tensor]) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} lies on {t.device}, the logits on {device}")


def labels_of(labels: Tensor, shape, what: str) -> Tensor:
    if labels.dtype.is_floating_point or labels.dtype.is_complex or labels.dtype == torch.bool:
        raise TypeError(f"{what}: labels are integers, got {labels.dtype}")
    if tuple(labels.shape) != tuple(shape):
        raise ValueError(f"{what}: labels of shape {tuple(labels.shape)} for rows of shape {tuple(shape)}")
    return labels.detach().to(torch.int64).contiguous()


def mask_of(row_mask: Optional[Tensor], shape, what: str) -> Optional[Tensor]:
    if row_mask is None:
        return None
    if row_mask.numel() != torch.Size(shape).numel():
        raise ValueError(f"{what}: row mask has {row_mask.numel()} entries for rows of shape {tuple(shape)}")
    m = row_mask.detach().reshape(-1)
    if m.dtype != torch.bool:
        m = m != 0
    return m.contiguous().view(torch.uint8)


def floats_of(t: Tensor, shape, name: str) -> Tensor:
    if not t.dtype.is_floating_point:
        raise TypeError(f"{name} must be floating point, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t.detach().to(torch.float32).contiguous()


def temperature_of(temperature: float, what: str) -> float:
    t = float(temperature)
    if not 1e-30 <= t <= 1e30:
        raise ValueError(f"{what} needs a positive temperature, got {temperature}")
    return t


def ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()
