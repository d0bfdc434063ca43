"""A teacher's top logits and the distillation loss from them, on the HIP kernels
of libmtp_glora_amd.so.

``StableSoftCrossEntropy`` reads whole teacher rows. Where a teacher is stored or
sent, its k largest logits a row do: ``top_logits`` takes them from the teacher's
logits, ``top_logits_cross_entropy`` is the loss against them, with the sum over
rows that the sampler's loss returns (mtp_glora/core/loss.py:294), and
``top_logits_loss_and_grad`` gives loss and gradient in one pass over the student's
logits.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .ops import _dev, _stream, dtype_code

MAX_TOP = 1024          # most logits kept of a row
MAX_VOCAB = 1 << 20     # longest row that is put in order
MAX_CE_VOCAB = 1 << 30  # longest row of the loss
INT32_MAX = (1 << 31) - 1


class TopLogits(NamedTuple):
    values: torch.Tensor   # [..., k], the logits' dtype, in order
    ids: torch.Tensor      # [..., k] int32
    lse: torch.Tensor      # [...] fp32


def row_view(name: str, t: torch.Tensor) -> torch.Tensor:
    """[..., V] as [rows, V] with contiguous columns (a copy only if needed)."""
    _dev(name, t)
    if t.dim() < 1 or t.shape[-1] == 0:
        raise ValueError(f"{name}: expected [..., V] with V > 0, got {tuple(t.shape)}")
    if max(t.shape[-1], t.shape[:-1].numel()) > INT32_MAX:
        raise ValueError(f"{name}: {tuple(t.shape)} has more than {INT32_MAX} rows or columns")
    v = t.detach().reshape(-1, t.shape[-1])
    if v.stride(1) != 1 or (v.shape[0] > 1 and v.stride(0) < v.shape[1]):
        v = v.contiguous()
    return v


def row_stride(v: torch.Tensor) -> int:
    return max(v.stride(0), v.shape[1])   # one row may carry any stride


def _like(name: str, t: torch.Tensor, lead, device) -> None:
    _dev(name, t)
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the logits on {device}")
    if tuple(t.shape[:len(lead)]) != tuple(lead):
        raise ValueError(f"{name}: leading shape {tuple(t.shape)} does not fit the logits' {tuple(lead)}")


def _temperature(t) -> float:
    t = float(t)
    if not 2.0 ** -60 <= t <= 2.0 ** 60:
        raise ValueError(f"temperature must be within 2^-60 to 2^60 (got {t})")
    return t


def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The k largest logits of each row of ``logits`` [..., V], in order (value
    descending, the lower id first among equals; NaN below -inf), their ids, and
    the row's log-sum-exp of logits / temperature. k <= 1024, V <= 1 048 576. No
    gradient: a teacher's logits."""
    k = int(k)
    temperature = _temperature(temperature)
    r = _lib.native("top_logits", logits, k, temperature)
    if r is not None:
        return TopLogits(*r)
    x = row_view("logits", logits)
    N, V = x.shape
    code = dtype_code(x.dtype)
    if not 1 <= k <= min(V, MAX_TOP):
        raise ValueError(f"k must be 1 to {min(V, MAX_TOP)} (got {k})")
    if V > MAX_VOCAB:
        raise ValueError(f"{V} columns; at most {MAX_VOCAB}")
    lead = logits.shape[:-1]
    values = torch.empty(*lead, k, device=x.device, dtype=x.dtype)
    ids = torch.empty(*lead, k, device=x.device, dtype=torch.int32)
    lse = torch.empty(lead, device=x.device, dtype=torch.float32)
    if N:
        with torch.cuda.device(x.device):
            _lib.call("mga_top_logits", x.data_ptr(), row_stride(x), N, V, code, k, temperature, values.data_ptr(),
                      ids.data_ptr(), lse.data_ptr(), _stream(x))
    return TopLogits(values, ids, lse)


class _Teacher(NamedTuple):
    values: torch.Tensor
    ids: torch.Tensor
    lse: torch.Tensor | None


def _student(t: torch.Tensor) -> torch.Tensor:
    x = row_view("student", t)
    if x.shape[1] > MAX_CE_VOCAB:
        raise ValueError(f"{x.shape[1]} columns; at most {MAX_CE_VOCAB}")
    return x


def _teacher(student: torch.Tensor, values: torch.Tensor, ids: torch.Tensor, lse) -> _Teacher:
    lead = student.shape[:-1]
    _like("values", values, lead, student.device)
    _like("ids", ids, lead, student.device)
    if values.shape != ids.shape or values.dim() != student.dim():
        raise ValueError(f"values {tuple(values.shape)} and ids {tuple(ids.shape)} must both be [..., k]")
    if not 1 <= values.shape[-1] <= MAX_TOP:
        raise ValueError(f"k must be 1 to {MAX_TOP} (got {values.shape[-1]})")
    dtype_code(values.dtype)
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids: int32 or int64 required (got {ids.dtype})")
    if lse is not None:
        _like("lse", lse, lead, student.device)
        if lse.shape != lead:
            raise ValueError(f"lse: shape {tuple(lse.shape)}, expected {tuple(lead)}")
        if lse.dtype != torch.float32:
            raise TypeError(f"lse: float32 required (got {lse.dtype})")
        lse = lse.detach().reshape(-1).contiguous()
    return _Teacher(row_view("values", values), row_view("ids", ids), lse)


def _common(x: torch.Tensor, t: _Teacher):
    return (x.data_ptr(), row_stride(x), t.values.data_ptr(), row_stride(t.values), dtype_code(t.values.dtype),
            t.ids.data_ptr(), row_stride(t.ids), int(t.ids.dtype == torch.int64),
            t.lse.data_ptr() if t.lse is not None else None, x.shape[0], x.shape[1], t.ids.shape[1])


class TopLogitsCrossEntropy(torch.autograd.Function):
    """``apply(student, values, ids, lse, temperature)``; see top_logits_cross_entropy."""

    @classmethod
    def apply(cls, student, *args):
        _lib.check_capture("top_logits_cross_entropy", student)
        return super().apply(student, *args)

    @staticmethod
    def forward(ctx, student, values, ids, lse, temperature):
        x = _student(student)
        code = dtype_code(x.dtype)
        t = _teacher(student, values, ids, lse)
        N, V = x.shape
        opts = dict(device=x.device, dtype=torch.float32)
        total = torch.zeros((), **opts) if N == 0 else torch.empty((), **opts)
        stats, q = torch.empty(3, N, **opts), torch.empty(N, t.ids.shape[1], **opts)
        if N:
            loss = torch.empty(N, **opts)
            ws = torch.empty(int(_lib.load().mga_top_logits_ce_workspace_floats(N, V)), **opts)
            with torch.cuda.device(x.device):
                _lib.call("mga_top_logits_ce_fwd", *_common(x, t), temperature, code, q.data_ptr(), stats.data_ptr(),
                          loss.data_ptr(), total.data_ptr(), ws.data_ptr(), _stream(x))
        ctx.save_for_backward(x, t.ids, q, stats)
        ctx.meta = (temperature, student.shape)
        return total

    @staticmethod
    def backward(ctx, grad_output):
        x, ids, q, stats = ctx.saved_tensors
        temperature, shape = ctx.meta
        N, V = x.shape
        grad = torch.empty(N, V, device=x.device, dtype=x.dtype)
        if N:
            go = grad_output.detach().reshape(1).to(device=x.device, dtype=torch.float32).contiguous()
            with torch.cuda.device(x.device):
                _lib.call("mga_top_logits_ce_bwd", x.data_ptr(), row_stride(x), ids.data_ptr(), row_stride(ids),
                          int(ids.dtype == torch.int64), q.data_ptr(), stats.data_ptr(), N, V, ids.shape[1],
                          temperature, dtype_code(x.dtype), go.data_ptr(), grad.data_ptr(), V, _stream(x))
        return _lib.once("top_logits_cross_entropy", grad.view(shape)), None, None, None, None


def top_logits_cross_entropy(student: torch.Tensor, values: torch.Tensor, ids: torch.Tensor,
                             lse: torch.Tensor | None = None, temperature: float = 1.0) -> torch.Tensor:
    """Sum over the rows of ``student`` [..., V] of

        temperature^2 * sum_k q_k (logsumexp(y) - y[ids_k]),   y = student / temperature

    with q the teacher's probabilities of the kept logits ``values`` [..., k] at
    ``ids`` [..., k]: exp(values / temperature - lse) if the row's log-sum-exp
    ``lse`` [...] is given (of logits / temperature, as top_logits returns it;
    what was not kept then carries the rest), else renormalised over the kept. An
    id outside [0, V) is padding; a row with no entry left has loss and gradient
    zero. ``values`` may have another dtype than the student. Differentiable in
    ``student``, once; the teacher gets no gradient. With k = V kept and temperature 1
    this is StableSoftCrossEntropy. k <= 1024, V <= 2^30. Under graph capture refused
    while an eager graph of the same leaf lives; top_logits_loss_and_grad needs no
    graph."""
    temperature = _temperature(temperature)
    r = _lib.native("top_logits_ce", student, values, ids, lse, temperature)
    return r if r is not None else TopLogitsCrossEntropy.apply(student, values, ids, lse, temperature)


def top_logits_loss_and_grad(student: torch.Tensor, values: torch.Tensor, ids: torch.Tensor,
                             lse: torch.Tensor | None = None, temperature: float = 1.0, scale: float = 1.0):
    """(loss, grad): top_logits_cross_entropy and ``scale`` times its gradient for
    ``student``, in the student's dtype and shape, in one pass over the rows. For a
    training step whose loss scale is known:

        loss, grad = top_logits_loss_and_grad(logits, values, ids, lse, scale=1 / chunks)
        logits.backward(grad)

    ``loss`` is not scaled and carries no graph."""
    temperature, scale = _temperature(temperature), float(scale)
    r = _lib.native("top_logits_step", student, values, ids, lse, temperature, scale)
    if r is not None:
        return r
    x = _student(student)
    code = dtype_code(x.dtype)
    t = _teacher(student, values, ids, lse)
    N, V = x.shape
    opts = dict(device=x.device, dtype=torch.float32)
    grad = torch.empty(N, V, device=x.device, dtype=x.dtype)
    if N == 0:
        return torch.zeros((), **opts), grad.view(student.shape)
    loss, total = torch.empty(N, **opts), torch.empty((), **opts)
    ws = torch.empty(int(_lib.load().mga_top_logits_ce_step_workspace_floats(N, V, t.ids.shape[1])), **opts)
    with torch.cuda.device(x.device):
        _lib.call("mga_top_logits_ce_step", *_common(x, t), temperature, scale, code, loss.data_ptr(), total.data_ptr(),
                  grad.data_ptr(), V, ws.data_ptr(), _stream(x))
    return total, grad.view(student.shape)
