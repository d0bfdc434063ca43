"""A paged 8-bit KV cache for several sequences, and the attention of new tokens over
it, on the HIP kernels of libmtp_glora_amd.so: the decoding side of the model that
``StreamingKVCache`` and ``mtp_attention`` train.

A decoding step takes each sequence's new tokens (an accepted token and its drafted
mask tokens, a prompt, or a part of one) as rows packed one behind the other:

    pages = cache.pages(layer)
    q = paged_append(k, v, pages, table, cu_tokens, lengths, query=q, cos=cos, sin=sin)
    o = paged_attention(q, pages, table, cu_tokens, lengths, scaling)

``table`` [B, W] (int32) holds each sequence's pages in order, ``cu_tokens`` [B + 1]
(int32) bounds its new tokens among the rows, ``lengths`` [B] (int32) counts its
tokens in the cache. All three stay on the device and nothing is read back, so a step can
be captured in a graph and replayed with other lengths: a batch of fewer tokens than
rows ends at cu_tokens[B], a sequence without new tokens takes none. Rejected drafts are
dropped by not adding them to ``lengths``: the next append overwrites them. The scale of
their page does not shrink again, so that a page in which a large value was dropped holds
its other values by fewer bits until it is begun anew. Which pages a
sequence gets is the caller's to say; no two may write to one page, any may read it.

Neither call computes a gradient; operands that ask for one, in reverse or forward mode, are refused.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .distill import row_stride
from .ops import _dev, _stream, dtype_code, no_tangent

PAGE_SIZES = (16, 32, 64, 128)
CODE_DTYPE = torch.float8_e4m3fn


class KVPages(NamedTuple):
    k: torch.Tensor         # [num_pages, Hkv, page_size, D] e4m3
    v: torch.Tensor         # [num_pages, Hkv, D, page_size] e4m3
    k_scale: torch.Tensor   # [num_pages, Hkv] fp32 powers of two
    v_scale: torch.Tensor


def _pages(pages) -> KVPages:
    p = KVPages(*pages)
    for name, t in zip(KVPages._fields, p):
        _dev(name, t)
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.device != p.k.device:
            raise ValueError(f"{name} is on {t.device}, k on {p.k.device}")
    if p.k.dim() != 4 or p.v.dim() != 4:
        raise ValueError(f"pages: expected k [pages, Hkv, page_size, D] and v [pages, Hkv, D, page_size], got "
                         f"{tuple(p.k.shape)} and {tuple(p.v.shape)}")
    n, h, ps, d = p.k.shape
    if tuple(p.v.shape) != (n, h, d, ps):
        raise ValueError(f"v: expected [{n}, {h}, {d}, {ps}], got {tuple(p.v.shape)}")
    if ps not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES} (got {ps})")
    for name, t, shape, dtype in (("k", p.k, (n, h, ps, d), CODE_DTYPE), ("v", p.v, (n, h, d, ps), CODE_DTYPE),
                                  ("k_scale", p.k_scale, (n, h), torch.float32),
                                  ("v_scale", p.v_scale, (n, h), torch.float32)):
        if t.dtype != dtype:
            raise TypeError(f"{name}: {dtype} required (got {t.dtype})")
        if tuple(t.shape) != shape:
            raise ValueError(f"{name}: expected {list(shape)}, got {tuple(t.shape)}")
    return p


def _batch(table, cu_tokens, lengths, device):
    for name, t in (("block_table", table), ("cu_tokens", cu_tokens), ("lengths", lengths)):
        _dev(name, t)
        if t.dtype != torch.int32:
            raise TypeError(f"{name}: int32 required (got {t.dtype})")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, the pages on {device}")
    if table.dim() != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError(f"block_table: expected [sequences, pages], got {tuple(table.shape)}")
    B = table.shape[0]
    if tuple(cu_tokens.shape) != (B + 1,) or tuple(lengths.shape) != (B,):
        raise ValueError(f"{B} sequences need cu_tokens [{B + 1}] and lengths [{B}], got {tuple(cu_tokens.shape)} and "
                         f"{tuple(lengths.shape)}")
    if table.stride(1) != 1 or table.stride(0) < table.shape[1]:
        table = table.contiguous()
    return table, cu_tokens.contiguous(), lengths.contiguous()


def _heads3(name: str, t: torch.Tensor, D: int, device) -> torch.Tensor:
    _dev(name, t)
    if t.dim() != 3 or t.shape[2] != D:
        raise ValueError(f"{name}: expected [tokens, heads, {D}], got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the pages on {device}")
    t = t.detach()
    return t if t.stride(2) == 1 and t.stride(0) >= 0 and t.stride(1) >= 0 else t.contiguous()


def _no_grad(fn: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{fn} computes no gradient; call it under torch.no_grad()")


def paged_append(key: torch.Tensor, value: torch.Tensor, pages, block_table: torch.Tensor, cu_tokens: torch.Tensor,
                 lengths: torch.Tensor, query: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                 sin: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor | None:
    """Store the new tokens' ``key`` and ``value`` [T, Hkv, D] in ``pages`` (KVPages) at
    the positions behind their sequences' ``lengths``, and return ``query`` [T, Hq, D]
    prepared like the keys (None without a query).

    Keys and queries are normalised where ``k_weight`` / ``q_weight`` [D] are given (RMS
    norm) and rotated where ``cos`` / ``sin`` [T, D] are (the rotary tables of each
    token, in the model's dtype or fp32), keys in fp64 and queries in fp32, with one rounding at the
    end, unlike ``qk_norm_rope``, which rounds after every op as the reference's ops do. Keys and
    values are stored in e4m3, under a power-of-two scale for each page and head that
    grows with the values the page takes; an append at a page's row 0 begins it anew.
    NaN and infinities are stored as NaN. A position without a page is not
    stored. Rows of the result behind the last sequence's tokens are zeros."""
    _no_grad("paged_append", key, value, query, q_weight, k_weight, cos, sin, *pages)
    r = _lib.native("paged_append", key, value, *pages, block_table, cu_tokens, lengths, query, cos, sin, q_weight,
                    k_weight, eps)
    if r is not None:
        return r[0] if query is not None else None
    no_tangent("paged_append", key, value, query, q_weight, k_weight, cos, sin, *pages)
    p = _pages(pages)
    table, cu, lens = _batch(block_table, cu_tokens, lengths, p.k.device)
    n, Hkv, ps, D = p.k.shape
    k, v = _heads3("key", key, D, p.k.device), _heads3("value", value, D, p.k.device)
    T = k.shape[0]
    if k.shape[1] != Hkv or v.shape != k.shape:
        raise ValueError(f"key {tuple(key.shape)} and value {tuple(value.shape)} do not fit pages of {Hkv} heads of {D}")
    code = dtype_code(k.dtype)
    q = qo = None
    if query is not None:
        q = _heads3("query", query, D, p.k.device)
        if q.shape[0] != T:
            raise ValueError(f"query: {q.shape[0]} rows, {T} keys")
        qo = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    for name, t in (("value", v), ("query", q), ("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None and t.dtype != k.dtype:
            raise TypeError(f"{name} dtype {t.dtype} != key dtype {k.dtype}")
    weights = []
    for name, t in (("q_weight", q_weight), ("k_weight", k_weight)):
        if t is not None:
            _dev(name, t)
            if tuple(t.shape) != (D,) or t.device != p.k.device:
                raise ValueError(f"{name}: expected [{D}] on {p.k.device}, got {tuple(t.shape)} on {t.device}")
            t = t.detach().contiguous()
        weights.append(t)
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if cos is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            _dev(name, t)
            if tuple(t.shape) != (T, D) or t.device != p.k.device:
                raise ValueError(f"{name}: expected [{T}, {D}] on {p.k.device}, got {tuple(t.shape)} on {t.device}")
            if t.dtype not in (k.dtype, torch.float32) or t.dtype != cos.dtype:
                raise TypeError(f"{name}: {k.dtype} or float32 required, cos and sin alike (got {t.dtype})")
        cos, sin = cos.detach(), sin.detach()
        if cos.stride(1) != 1 or cos.stride() != sin.stride() or cos.stride(0) < 0:
            cos, sin = cos.contiguous(), sin.contiguous()
    for t in p:
        torch.autograd.graph.increment_version(t)   # a graph that saved them sees the write
    if T == 0:
        return qo
    ptr = lambda t: t.data_ptr() if t is not None else None   # noqa: E731
    st = lambda t: (t.stride(0), t.stride(1)) if t is not None else (0, 0)   # noqa: E731
    with torch.cuda.device(p.k.device):
        _lib.call("mga_paged_append", ptr(k), *st(k), ptr(v), *st(v), ptr(q), *st(q), ptr(weights[0]), ptr(weights[1]),
                  ptr(cos), ptr(sin), cos.stride(0) if cos is not None else 0,
                  int(cos is not None and cos.dtype == torch.float32), float(eps), T, table.shape[0],
                  q.shape[1] if q is not None else 0, Hkv, D, code, ptr(p.k), ptr(p.v), ptr(p.k_scale), ptr(p.v_scale), n,
                  ps, ptr(table), row_stride(table), table.shape[1], ptr(cu), ptr(lens), ptr(qo), *st(qo), _stream(p.k))
    return qo


def paged_attention(query: torch.Tensor, pages, block_table: torch.Tensor, cu_tokens: torch.Tensor,
                    lengths: torch.Tensor, scaling: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention [T, Hq, D] of the new tokens' ``query`` over their sequences in
    ``pages`` (KVPages): token i of a sequence sees positions 0 .. lengths + i, its own
    included, so append first, with the same table, cu_tokens and lengths. Query head h
    reads KV head h // (Hq / Hkv). Positions without a page are masked; a row that sees
    nothing is zeros. Scores, sums and outputs in fp32; the probabilities are held to 16 bits (fp32
    queries: 24; bf16 queries in a batch of prompts, which takes another form by its average number of new
    tokens: 8, as the output). ``out`` (``query`` itself, or
    rows that do not overlap it) receives the result; its rows
    behind the last sequence's tokens stay as they are, in a tensor made here they are
    zeros. Hq / Hkv <= 32, at most 4096 sequences."""
    _no_grad("paged_attention", query, *pages)
    r = _lib.native("paged_attention", query, *pages, block_table, cu_tokens, lengths, scaling, out)
    if r is not None:
        return r
    no_tangent("paged_attention", query, out, *pages)
    p = _pages(pages)
    table, cu, lens = _batch(block_table, cu_tokens, lengths, p.k.device)
    n, Hkv, ps, D = p.k.shape
    q = _heads3("query", query, D, p.k.device)
    code, eb = dtype_code(q.dtype), q.element_size()
    if q.data_ptr() % 16 or q.stride(0) * eb % 16 or q.stride(1) * eb % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    T, Hq = q.shape[0], q.shape[1]
    if Hq == 0 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads for {Hkv} KV heads")
    fresh = out is None
    if fresh:
        out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    else:
        _dev("out", out)
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device:
            raise ValueError(f"out: expected {tuple(q.shape)} {q.dtype} on {q.device}, got {tuple(out.shape)} {out.dtype} "
                             f"on {out.device}")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out must not require a gradient")
        if out.data_ptr() % 16 or out.stride(2) != 1 or any(s * eb % 16 or s < D for s in out.stride()[:2]):
            raise ValueError("out: rows must be contiguous, 16-byte aligned and must not overlap")
        torch.autograd.graph.increment_version(out)
    if T == 0:
        return out
    with torch.cuda.device(p.k.device):
        nb = int(_lib.load().mga_paged_attn_workspace_bytes(T, table.shape[0], Hq, Hkv, D, ps, table.shape[1], code))
        ws = torch.empty(nb, device=q.device, dtype=torch.uint8)
        _lib.call("mga_paged_attn", q.data_ptr(), q.stride(0), q.stride(1), p.k.data_ptr(), p.v.data_ptr(),
                  p.k_scale.data_ptr(), p.v_scale.data_ptr(), n, ps, table.data_ptr(), row_stride(table), table.shape[1],
                  cu.data_ptr(), lens.data_ptr(), T, table.shape[0], Hq, Hkv, D, code, float(scaling), out.data_ptr(),
                  out.stride(0), out.stride(1), int(fresh), ws.data_ptr() if nb else None, nb, _stream(q))
    return out


class PagedKVCache:
    """The pages of every layer, and the batch that the layers of a step share.

    ``begin(block_table, cu_tokens, lengths)`` sets the batch; then each layer calls
    ``append`` and ``attend`` (``qwen3_attention_forward`` does, when it is given this
    as past_key_value). Freeing, sharing and handing out pages is the caller's."""

    def __init__(self, num_pages: int, num_layers: int, num_kv_heads: int, head_dim: int, page_size: int = 64,
                 device="cuda"):
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} (got {page_size})")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128 (got {head_dim})")
        if min(num_pages, num_layers, num_kv_heads) < 1:
            raise ValueError(f"bad sizes: {num_pages} pages, {num_layers} layers, {num_kv_heads} heads")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError(f"PagedKVCache lives in GPU memory; got device {device}")
        self.num_pages, self.page_size, self.num_layers = int(num_pages), int(page_size), int(num_layers)
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        code = lambda s: torch.zeros(s, dtype=torch.uint8, device=device).view(CODE_DTYPE)   # noqa: E731
        scale = lambda: torch.ones(shape[:2], dtype=torch.float32, device=device)   # noqa: E731
        self._layers = [KVPages(code(shape), code((*shape[:2], head_dim, page_size)), scale(), scale())
                        for _ in range(num_layers)]
        self._batch = None

    def pages(self, layer_idx: int) -> KVPages:
        return self._layers[layer_idx]

    def begin(self, block_table: torch.Tensor, cu_tokens: torch.Tensor, lengths: torch.Tensor) -> None:
        """The batch of the appends and attentions that follow. The tensors are held, not
        copied, if they are contiguous (a table's rows may lie apart): what is written to
        them later, counts; a graph that begins outside its capture needs them so."""
        self._batch = _batch(block_table, cu_tokens, lengths, self._layers[0].k.device)

    def _step(self):
        if self._batch is None:
            raise RuntimeError("PagedKVCache: begin a batch first")
        return self._batch

    def append(self, layer_idx: int, key, value, **prepare):
        """``paged_append`` to a layer's pages."""
        return paged_append(key, value, self._layers[layer_idx], *self._step(), **prepare)

    def attend(self, layer_idx: int, query, scaling: float, out=None):
        """``paged_attention`` over a layer's pages."""
        return paged_attention(query, self._layers[layer_idx], *self._step(), scaling, out=out)

    def dequantized(self, layer_idx: int, block_table_row: torch.Tensor, length: int):
        """Keys and values [Hkv, length, D] (fp32) that a layer holds of a sequence, zeros at
        positions without a page, by elementary operations: for inspection, and to hand a prefix to
        another cache."""
        p, n = self._layers[layer_idx], int(length)
        if block_table_row.dim() != 1 or not 0 <= n <= block_table_row.shape[0] * self.page_size:
            raise ValueError(f"{n} tokens in a table row {tuple(block_table_row.shape)} of pages of {self.page_size}")
        ids = block_table_row.to(p.k.device).long()[:-(-n // self.page_size)]
        there = (ids >= 0) & (ids < self.num_pages)
        ids, there = torch.where(there, ids, 0), there[:, None, None, None]
        read = lambda c, s: torch.where(   # noqa: E731
            there, c.view(torch.uint8)[ids].view(CODE_DTYPE).float() * s[ids][..., None, None], 0.0)
        k, v = read(p.k, p.k_scale), read(p.v, p.v_scale).transpose(2, 3)
        return tuple(t.transpose(0, 1).flatten(1, 2)[:, :n] for t in (k, v))
