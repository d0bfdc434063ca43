"""Token sampling from rows of logits, and the penalties, biases and masks before it, on
the HIP kernels of libmtp_glora_amd.so."""
from __future__ import annotations

import torch

from . import _lib
from .ops import _dev, _stream, dtype_code, no_tangent
from .distill import INT32_MAX, MAX_VOCAB, row_stride, row_view


def _setting(name: str, v, rows: int, device, dtype):
    """(tensor with one value a row, None) or (None, number)."""
    if not isinstance(v, torch.Tensor):
        return None, (int(v) if dtype == torch.int32 else float(v))
    _dev(name, v)
    if v.device != device:
        raise ValueError(f"{name} is on {v.device}, the logits on {device}")
    if v.is_floating_point() != (dtype == torch.float32) or v.is_complex() or v.dtype == torch.bool:
        raise TypeError(f"{name}: expected {'whole numbers' if dtype == torch.int32 else 'floating point'}, "
                        f"got {v.dtype}")
    if v.numel() not in (1, rows):
        raise ValueError(f"{name}: {v.numel()} values for {rows} rows")
    if v.dtype == torch.int64:
        v = v.clamp(-1, MAX_VOCAB)   # past the columns is past the columns
    return v.detach().reshape(-1).to(dtype).expand(rows).contiguous(), None


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0) -> torch.Tensor:
    """One token id (int64) for each row of ``logits`` [..., V], drawn with the
    given numbers ``uniform`` [...] (fp32, in [0, 1)).

    In the order of the logits (descending, the lower id first among equals) and
    with w = exp((x - max) / temperature): ``top_k`` keeps the first k tokens (0:
    all), ``top_p`` of those the shortest leading run that holds at least top_p of
    their weight (1: all), ``min_p`` the tokens with w >= min_p (above 1: as 1). With
    +inf among the logits those have w = 1 and all others 0. The token is the first,
    by ascending id, at which the running sum of the kept weights exceeds uniform
    times their total. ``temperature`` 0 takes the largest logit, the lowest id among
    equals. Each setting is a number or a tensor with one value a row and is taken
    in fp32 (top_k: int32). -inf and NaN logits are never drawn; a row with nothing
    else gives -1. Sums are exact: the same inputs give the same tokens on every
    call. V <= 1 048 576."""
    given = ((temperature, float), (top_k, int), (top_p, float), (min_p, float))
    r = _lib.native("sample", logits, uniform, *(v if isinstance(v, torch.Tensor) else None for v, _ in given),
                    *(0 if isinstance(v, torch.Tensor) else number(v) for v, number in given))
    if r is not None:
        return r
    _dev("logits", logits)
    lead = logits.shape[:-1]
    rows = lead.numel()
    settings = [_setting(n, v, rows, logits.device, dt)
                for n, v, dt in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                                 ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32))]
    _dev("uniform", uniform)
    if uniform.dtype != torch.float32:
        raise TypeError(f"uniform: float32 required (got {uniform.dtype})")
    if uniform.device != logits.device:
        raise ValueError(f"uniform is on {uniform.device}, the logits on {logits.device}")
    if uniform.shape != lead:
        raise ValueError(f"uniform: shape {tuple(uniform.shape)}, expected {tuple(lead)}")
    x = row_view("logits", logits)
    code = dtype_code(x.dtype)
    if x.shape[1] > MAX_VOCAB:
        raise ValueError(f"{x.shape[1]} columns; at most {MAX_VOCAB}")
    u = uniform.detach().contiguous()
    token = torch.empty(lead, device=x.device, dtype=torch.int64)
    if rows:
        args = [a for t, v in settings for a in (t.data_ptr() if t is not None else None, v if v is not None else 0)]
        args[3] = max(-1, min(args[3], MAX_VOCAB))
        with torch.cuda.device(x.device):
            _lib.call("mga_sample", x.data_ptr(), row_stride(x), rows, x.shape[1], code, u.data_ptr(), *args,
                      token.data_ptr(), _stream(x))
    return token


def _row_list(name: str, t: torch.Tensor, lead, device, dtypes, shared: bool = True):
    """([rows or 1, n] view with contiguous entries, row stride, 0 where one row is shared)."""
    _dev(name, t)
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: {' or '.join(str(d) for d in dtypes)} required (got {t.dtype})")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the logits on {device}")
    if t.dim() < 1 or (tuple(t.shape[:-1]) != tuple(lead) and not (shared and t.dim() == 1)):
        raise ValueError(f"{name}: expected {list(lead)} rows{' or one' if shared else ''}, got {tuple(t.shape)}")
    n = t.shape[-1]
    if n > INT32_MAX:
        raise ValueError(f"{name}: {n} entries; at most {INT32_MAX}")
    v = t.detach().reshape(-1, n) if n else t.detach()
    if n and (v.stride(1) != 1 or (v.shape[0] > 1 and v.stride(0) != 0 and v.stride(0) < n)):
        v = v.contiguous()
    return v, 0 if n == 0 or v.shape[0] == 1 else v.stride(0)


def _row_counts(name: str, t, lead, device):
    if t is None:
        return None
    _dev(name, t)
    if t.dtype != torch.int32:
        raise TypeError(f"{name}: int32 required (got {t.dtype})")
    if t.device != device or tuple(t.shape) != tuple(lead):
        raise ValueError(f"{name}: expected {list(lead)} on {device}, got {tuple(t.shape)} on {t.device}")
    return t.contiguous()


def adjust_logits(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, lengths: torch.Tensor | None = None,
                  prompt_lengths: torch.Tensor | None = None, repetition=1.0, frequency=0.0, presence=0.0,
                  bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                  allowed: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows of ``logits`` [..., V] shaped before ``sample_tokens``, in fp32 and rounded
    once to their dtype.

    ``tokens`` [..., L] (int32 or int64) are each row's tokens, the prompt's first;
    ``lengths`` [...] (int32; all) says how many count, ``prompt_lengths`` [...] (int32; 0) how
    many of those are the prompt's. A token seen in prompt or output has its logit divided by
    ``repetition`` if positive, else multiplied by it; one of the output loses
    ``frequency`` times its count there and ``presence`` once. Each of the three is a number or
    a tensor with one value a row; a repetition that is not positive is refused as a
    number and counts as 1 in a tensor. ``bias`` [..., K] or [K] (fp32) is added at
    ``bias_ids`` (int32 or int64), equal ids one after the other. ``allowed`` [..., ceil(V / 32)] or [ceil(V / 32)]
    (int32) holds a bit for each token, token v's at bit v % 32 of word v // 32; where it is
    0 the result is -inf. Ids outside [0, V) (padding) do not count. ``out`` may be ``logits``.
    V <= 2^30. No gradient."""
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad
                                       for t in (logits, bias, repetition, frequency, presence)):
        raise NotImplementedError("adjust_logits computes no gradient; call it under torch.no_grad()")
    given = (repetition, frequency, presence)
    r = _lib.native("adjust_logits", logits, tokens, lengths, prompt_lengths,
                    *(v if isinstance(v, torch.Tensor) else None for v in given),
                    *(0.0 if isinstance(v, torch.Tensor) else float(v) for v in given), bias_ids, bias, allowed, out)
    if r is not None:
        return r
    no_tangent("adjust_logits", logits, bias, *given, out)
    _dev("logits", logits)
    lead, V, dev = logits.shape[:-1], logits.shape[-1] if logits.dim() else 0, logits.device
    x = row_view("logits", logits)
    code, rows = dtype_code(x.dtype), x.shape[0]
    held = [_setting(n, v, rows, dev, torch.float32)
            for n, v in (("repetition", repetition), ("frequency", frequency), ("presence", presence))]
    ints = (torch.int32, torch.int64)
    tok = bid = bval = ok = None
    trs = brs = vrs = ars = 0
    if tokens is not None:
        tok, trs = _row_list("tokens", tokens, lead, dev, ints, shared=False)
    elif lengths is not None or prompt_lengths is not None:
        raise ValueError("lengths and prompt_lengths need tokens")
    lens, prompts = _row_counts("lengths", lengths, lead, dev), _row_counts("prompt_lengths", prompt_lengths, lead, dev)
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias come together")
    if bias is not None:
        bid, brs = _row_list("bias_ids", bias_ids, lead, dev, ints)
        bval, vrs = _row_list("bias", bias, lead, dev, (torch.float32,))
        if bid.shape[-1] != bval.shape[-1]:
            raise ValueError(f"{bid.shape[-1]} bias_ids and {bval.shape[-1]} biases")
    if allowed is not None:
        ok, ars = _row_list("allowed", allowed, lead, dev, (torch.int32,))
        if ok.shape[-1] != -(-V // 32):
            raise ValueError(f"allowed: {-(-V // 32)} words a row for {V} columns (got {ok.shape[-1]})")
    if out is None:
        out = torch.empty(logits.shape, device=dev, dtype=x.dtype)
    else:
        _dev("out", out)
        if out.shape != logits.shape or out.dtype != x.dtype or out.device != dev:
            raise ValueError(f"out: expected {tuple(logits.shape)} {x.dtype} on {dev}, got {tuple(out.shape)} {out.dtype} "
                             f"on {out.device}")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out must not require a gradient")
    if rows == 0:
        return out
    o = out.detach().view(-1, V) if out.is_contiguous() else out.detach().reshape(-1, V)
    if o.data_ptr() != out.data_ptr() or o.stride(1) != 1 or (rows > 1 and o.stride(0) < V):
        raise ValueError("out: rows must be contiguous and must not overlap")
    torch.autograd.graph.increment_version(out)   # a graph that saved it sees the write
    ptr = lambda t: t.data_ptr() if t is not None and t.numel() else None   # noqa: E731
    n = lambda t: t.shape[-1] if t is not None else 0   # noqa: E731
    wide = lambda t: int(t is not None and t.dtype == torch.int64)   # noqa: E731
    with torch.cuda.device(dev):
        _lib.call("mga_adjust_logits", x.data_ptr(), row_stride(x), rows, V, code, ptr(tok), wide(tok), trs, n(tok),
                  ptr(lens), ptr(prompts), *(a for t, v in held for a in (ptr(t), v if v is not None else 1.0)), ptr(bid),
                  wide(bid), brs, ptr(bval), vrs, n(bid), ptr(ok), ars, o.data_ptr(), row_stride(o), _stream(x))
    return out
