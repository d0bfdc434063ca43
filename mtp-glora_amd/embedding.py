"""Scaled embedding lookup with its gradient by sorted tokens, on the HIP kernels
of libmtp_glora_amd.so.

The embedding is where an MTP chunk begins (Qwen3Model.forward,
mtp_glora/models/modeling_qwen3.py:436), and D of every 1 + D of a chunk's
tokens can be the one ``<mask>`` token that resize_token_embeddings added: its row
has to be learned, and its gradient is a sum over hundreds to thousands of rows.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib
from .distill import INT32_MAX
from .ops import _dev, _stream, dtype_code


def _check(ids: torch.Tensor, device) -> torch.Tensor:
    _dev("ids", ids)
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids: int32 or int64 required (got {ids.dtype})")
    if ids.device != device:
        raise ValueError(f"ids are on {ids.device}, the table on {device}")
    if ids.numel() > INT32_MAX:
        raise ValueError(f"{ids.numel()} ids; at most {INT32_MAX}")
    return ids.detach().reshape(-1).contiguous()


def _rows2(t: torch.Tensor, width: int) -> torch.Tensor:
    v = t.detach().reshape(-1, width)
    if v.stride(1) != 1 or (v.shape[0] > 1 and v.stride(0) < width):
        v = v.contiguous()
    return v


def _stride0(v: torch.Tensor) -> int:
    return max(v.stride(0), v.shape[1])


def embedding_grad(grad_out: torch.Tensor, ids: torch.Tensor, num_embeddings: int, scale: float = 1.0,
                   padding_idx: int | None = None, out: torch.Tensor | None = None,
                   accumulate: bool = False) -> torch.Tensor:
    """Gradient [num_embeddings, H] of scaled_embedding for its table:
    row v is scale times the sum of ``grad_out`` [..., H] over the tokens with id v,
    added in fp32 in a fixed order; ids equal to ``padding_idx`` or
    outside the table count nowhere. ``out`` (the gradients' dtype or fp32) receives
    it; with ``accumulate`` the sums are added to ``out``, whose other rows are
    neither read nor written: the chunks of a sequence can share one buffer. At most
    2^26 ids."""
    _dev("grad_out", grad_out)
    if grad_out.dim() < 1 or grad_out.shape[:-1] != ids.shape:
        raise ValueError(f"grad_out {tuple(grad_out.shape)} does not fit ids {tuple(ids.shape)}")
    code, H, V = dtype_code(grad_out.dtype), grad_out.shape[-1], int(num_embeddings)
    i = _check(ids, grad_out.device)
    if not (0 < V <= INT32_MAX and 0 < H <= INT32_MAX):
        raise ValueError(f"bad table size [{V}, {H}]")
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    if out is None:
        out = torch.empty(V, H, device=grad_out.device, dtype=grad_out.dtype)
    else:
        _dev("out", out)
        if tuple(out.shape) != (V, H) or out.device != grad_out.device:
            raise ValueError(f"out: expected [{V}, {H}] on {grad_out.device}, got {tuple(out.shape)} on {out.device}")
        if out.dtype not in (grad_out.dtype, torch.float32):
            raise TypeError(f"out: {grad_out.dtype} or float32 required (got {out.dtype})")
        if out.stride(1) != 1 or (V > 1 and out.stride(0) < H):
            raise ValueError("out: rows must be contiguous and must not overlap")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out must not require a gradient")
        torch.autograd.graph.increment_version(out)   # a graph that saved it sees the write
    dy = _rows2(grad_out, H)
    n = i.numel()
    nb = int(_lib.load().mga_embedding_workspace_bytes(n, H))
    ws = torch.empty(nb, device=dy.device, dtype=torch.uint8)
    pad = -1 if padding_idx is None else int(padding_idx)
    with torch.cuda.device(dy.device):
        _lib.call("mga_embedding_bwd", dy.data_ptr() if n else None, _stride0(dy), i.data_ptr() if n else None,
                  int(i.dtype == torch.int64), n, float(scale), pad, V, H, code, out.data_ptr(), _stride0(out),
                  dtype_code(out.dtype), int(accumulate), ws.data_ptr() if n else None, nb, _stream(dy))
    return out


def _lookup(ids: torch.Tensor, weight: torch.Tensor, scale: float) -> torch.Tensor:
    i = _check(ids, weight.device)
    w = _rows2(weight, weight.shape[1])
    out = torch.empty(*ids.shape, w.shape[1], device=w.device, dtype=w.dtype)
    if out.numel():
        with torch.cuda.device(w.device):
            _lib.call("mga_embedding_fwd", i.data_ptr(), int(i.dtype == torch.int64), i.numel(), w.data_ptr(),
                      _stride0(w), w.shape[0], w.shape[1], scale, dtype_code(w.dtype), out.data_ptr(), w.shape[1],
                      _stream(w))
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.meta = (weight.shape[0], scale, padding_idx)
        return _lookup(ids, weight, scale)

    @staticmethod
    def backward(ctx, grad_out):
        (ids,), (V, scale, padding_idx) = ctx.saved_tensors, ctx.meta
        grad = embedding_grad(grad_out, ids, V, scale, padding_idx)
        return None, _lib.once("scaled_embedding", grad) if grad_out.requires_grad else grad, None, None


def scaled_embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                     padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[ids]`` [..., H] for ids [...] (int32 or int64) of a table
    ``weight`` [V, H], rounded once to its dtype; zeros for an id outside the
    table. Differentiable in ``weight``, once (a dense gradient, embedding_grad);
    ``padding_idx`` is looked up like any other id and has no gradient. Under graph
    capture refused while an eager graph of the same leaf lives (its backward would
    join the default stream); embedding_grad needs no graph."""
    _dev("weight", weight)
    if weight.dim() != 2 or weight.numel() == 0 or max(weight.shape) > INT32_MAX:
        raise ValueError(f"weight: expected [V, H], got {tuple(weight.shape)}")
    dtype_code(weight.dtype)
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise ValueError(f"padding_idx {padding_idx} outside a table of {weight.shape[0]} rows")
        padding_idx = int(padding_idx) % weight.shape[0]
    r = _lib.native("embedding", ids, weight, float(scale), -1 if padding_idx is None else padding_idx)
    if r is not None:
        return r
    _lib.check_capture("scaled_embedding", weight)
    return _Embedding.apply(ids, weight, float(scale), padding_idx)


class ScaledEmbedding(nn.Embedding):
    """``nn.Embedding`` whose lookup is multiplied by ``scale``, by the HIP kernels:
    the same parameter and state-dict key."""

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: int | None = None, scale: float = 1.0,
                 device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx, device=device, dtype=dtype)
        self.scale = float(scale)

    @classmethod
    def wrap(cls, base: nn.Embedding, scale: float = 1.0) -> "ScaledEmbedding":
        """The layer of ``base``'s own parameter (shared, not copied), in its place: with
        its hooks (shared too: their handles remove them here), training flag and other
        attributes. A layer whose class or instance has a ``forward`` of its own, or
        whose weight is no plain parameter, is refused."""
        if base.max_norm is not None or base.scale_grad_by_freq or base.sparse:
            raise NotImplementedError("max_norm, scale_grad_by_freq and sparse gradients are not supported")
        if type(base).forward is not nn.Embedding.forward or "forward" in vars(base):
            raise NotImplementedError(f"{type(base).__name__} has a forward of its own")
        if not isinstance(base._parameters.get("weight"), nn.Parameter):
            raise NotImplementedError("the weight is not a parameter of the layer itself")
        m = cls.__new__(cls)
        nn.Module.__init__(m)
        vars(m).update(vars(base))
        for own in ("_parameters", "_buffers", "_modules", "_non_persistent_buffers_set"):
            vars(m)[own] = vars(base)[own].copy()
        vars(m).pop("_compiled_call_impl", None)   # the base's own forward, compiled
        m.scale = float(scale)
        return m

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        return scaled_embedding(input, self.weight, self.scale, self.padding_idx)
