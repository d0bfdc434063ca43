"""Token sampling from rows of logits, on the HIP kernel of libmtp_glora_amd.so."""
from __future__ import annotations

import torch

from . import _lib
from .ops import _dev, _stream, dtype_code
from .distill import MAX_VOCAB, row_stride, row_view


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
