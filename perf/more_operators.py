"""The operators of a decoding step over a paged 8-bit cache, timed: appending new
keys and values with their rotation, attention of the new tokens over the cache,
and the penalties, biases and masks of the logits.

A case is a dict of plain values. ``prepare`` makes what the program has in hand
before the call, ``run`` is one pass: in elementary torch operations where
``own`` is false, by the framework's calls where it is true. ``exact`` gives the
same outputs in 64 bits. Kinds:

* ``append`` - a ragged batch of new tokens: q and k are normalised (where the
  model does so) and rotated, k and v stored in 8 bits (e4m3) in the pages of
  their sequences, with one power-of-two scale a page and head: the least at which
  no value that the page has taken passes 448. Where a page's scale grows, the
  rows that it holds from before are rounded again. Outputs: the rotated q, and
  codes and scales of the cache.
* ``attend`` - each new token against its sequence's cache, itself included.
* ``logits`` - repetition, frequency and presence penalties by the tokens of a
  row's history, added biases, and a bit mask of the allowed tokens.

Key pages are [page, head, row, channel], value pages [page, head, channel, row].
"""
import importlib
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
EPS = 1e-6
QWEN3_VOCAB = 151936
LLAMA_VOCAB = 128256


def listed():
    big = dict(hq=32, hkv=8, dim=128)
    small = dict(hq=4, hkv=2, dim=64)     # the decoder of the end-to-end tests
    return [
        # a token each for a batch of sequences
        dict(name="append_tokens", kind="append", batch=64, new_lo=1, new_hi=1, len_lo=16, len_hi=8192, page=64,
             norm=True, dtype="bf16", plan=1, **big),
        # a small fp32 model's drafts, sequences that only begin among them: launches and latency
        dict(name="append_drafts_small", kind="append", batch=5, new_lo=1, new_hi=9, len_lo=0, len_hi=300, page=16,
             norm=False, dtype="fp32", plan=2, **small),
        # prompts, some of them behind a part that is cached already
        dict(name="append_prompts", kind="append", batch=3, new_lo=1200, new_hi=2048, len_lo=0, len_hi=4096, page=64,
             norm=True, dtype="bf16", plan=3, **big),
        # one token of one sequence: latency
        dict(name="attend_one", kind="attend", batch=1, new_lo=1, new_hi=1, len_lo=1000, len_hi=1000, page=64,
             dtype="bf16", plan=4, **big),
        # a token each for a batch of sequences of very different lengths
        dict(name="attend_tokens", kind="attend", batch=64, new_lo=1, new_hi=1, len_lo=64, len_hi=16384, page=64,
             dtype="bf16", plan=5, **big),
        # an accepted token and four drafted ones
        dict(name="attend_drafts", kind="attend", batch=16, new_lo=5, new_hi=5, len_lo=500, len_hi=8192, page=32,
             dtype="fp16", plan=6, **big),
        # few long sequences
        dict(name="attend_long", kind="attend", batch=2, new_lo=1, new_hi=5, len_lo=100000, len_hi=131072, page=64,
             dtype="bf16", plan=7, **big),
        # prompts, most of them behind a part that is cached already
        dict(name="attend_prompts", kind="attend", batch=4, new_lo=1024, new_hi=4096, len_lo=0, len_hi=16384, page=64,
             dtype="bf16", plan=51, **big),
        # the small fp32 model
        dict(name="attend_drafts_small", kind="attend", batch=5, new_lo=1, new_hi=9, len_lo=0, len_hi=300, page=16,
             dtype="fp32", plan=9, **small),
        # one row: latency
        dict(name="logits_one", kind="logits", rows=1, vocab=QWEN3_VOCAB, history=700, bias=0, mask=False, dtype="bf16"),
        # the rows of a batch of drafts under a grammar, a few tokens biased
        dict(name="logits_drafts", kind="logits", rows=80, vocab=QWEN3_VOCAB, history=2048, bias=8, mask=True,
             dtype="bf16"),
        # long histories and many biases, fp32 logits of an odd vocabulary
        dict(name="logits_batch", kind="logits", rows=256, vocab=32003, history=4096, bias=300, mask=False,
             dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "logits"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "logits":
        vocab = rng.choice([QWEN3_VOCAB, LLAMA_VOCAB, 32003, _log_int(rng, 700, 150000)])
        return dict(kind=kind, rows=_log_int(rng, 1, 40 if dtype == "fp32" else 80), vocab=vocab,
                    history=_log_int(rng, 1, 4096), bias=rng.choice([0, 0, 8, 300]), mask=rng.random() < 0.5,
                    dtype=dtype)
    hq, hkv, dim = rng.choice([(32, 8, 128), (32, 8, 128), (16, 8, 128), (4, 2, 64), (14, 2, 64), (8, 8, 64)])
    if rng.random() < 0.3:     # prompts
        batch, lo, hi, most = rng.randint(1, 3), 17, _log_int(rng, 64, 1500), _log_int(rng, 100, 8192)
    else:
        batch, lo = _log_int(rng, 1, 64), 1
        hi, most = rng.choice([1, 1, 5, 9]), _log_int(rng, 100, 16384)
    case = dict(kind=kind, batch=batch, new_lo=lo, new_hi=hi, len_lo=rng.choice([0, 16]), len_hi=most,
                page=rng.choice([16, 32, 64, 64, 128]), dtype=dtype, plan=rng.randint(1, 1 << 30), hq=hq, hkv=hkv, dim=dim)
    if kind == "append":
        case["norm"] = rng.random() < 0.5
    return case


def _plan(case):
    """New tokens and cached tokens of each sequence: the case's own, for any seed."""
    r = random.Random(case["plan"])
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    lo = max(case["len_lo"], 1)
    cached = [_log_int(r, lo, max(case["len_hi"], lo)) for _ in range(case["batch"])]
    if case["len_lo"] == 0:
        cached[0] = 0
    return new, cached


# ---- inputs ------------------------------------------------------------------

def _pow2(e):
    return ((e.int() + 127) << 23).view(torch.float32)


def _scale_of(amax):
    """The least power of two, 2^-100 to 2^119, of which 448 hold amax."""
    m, e = torch.frexp(amax)
    return _pow2(torch.where(amax > 0, e - 9 + (m > 0.875), -100).clamp(-100, 119))


def _pool(pages, case, spread, g, dev):
    """Codes [page, head, row, channel] and scales [page, head] of a cache in use."""
    x = torch.randn(pages, case["hkv"], case["page"], case["dim"], generator=g, device=dev)
    x *= torch.exp(0.5 * torch.randn(case["hkv"], 1, case["dim"], generator=g, device=dev))
    x *= torch.exp(spread * torch.randn(pages, 1, 1, 1, generator=g, device=dev))
    s = _scale_of(x.abs().amax((2, 3)))
    return (x / s[..., None, None]).to(E4M3), s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = dict(case=case)
    if case["kind"] == "logits":
        n, v, h = case["rows"], case["vocab"], case["history"]
        x = torch.randn(n, v, generator=g, device=dev).mul_(2.5)
        ids = (torch.rand(n, h, generator=g, device=dev).pow_(5) * v).long().clamp_(max=v - 1)
        # a row's own tokens stand out of it
        x.scatter_add_(1, ids, torch.rand(n, h, generator=g, device=dev) * 2)
        st["logits"], st["tokens"] = x.to(dt), ids
        st["lengths"] = (h * (0.5 + 0.5 * torch.rand(n, generator=g, device=dev))).int().clamp_(min=1)
        st["prompts"] = (st["lengths"] * torch.rand(n, generator=g, device=dev)).int()
        st["repetition"] = 1.0 + 0.3 * torch.rand(n, generator=g, device=dev)
        st["frequency"] = torch.rand(n, generator=g, device=dev) * 0.5
        st["presence"] = torch.rand(n, generator=g, device=dev)
        st["bias_ids"] = st["bias"] = st["allowed"] = None
        if case["bias"]:
            st["bias_ids"] = torch.randint(v, (n, case["bias"]), generator=g, device=dev, dtype=torch.int32)
            st["bias"] = torch.randn(n, case["bias"], generator=g, device=dev) * 4
        if case["mask"]:   # some rows may go on with nearly anything, some with few tokens
            words = -(-v // 32)
            few = torch.rand(n, 1, generator=g, device=dev) < 0.5
            bits = torch.randint(-2 ** 31, 2 ** 31, (2, n, words), generator=g, device=dev).int()
            rare = torch.rand(n, words, generator=g, device=dev) < 0.02
            st["allowed"] = torch.where(few, torch.where(rare, bits[0] & bits[1], 0), bits[0] | bits[1])
        return st
    new, cached = _plan(case)
    b, p, t = case["batch"], case["page"], sum(new)
    need = [-(-(n + c) // p) for n, c in zip(new, cached)]
    pages = sum(need) + 3
    st["k"], st["k_scale"] = _pool(pages, case, 0.3, g, dev)
    codes, st["v_scale"] = _pool(pages, case, 0.3, g, dev)
    st["v"] = codes.view(torch.uint8).transpose(2, 3).contiguous().view(E4M3)
    # each sequence's pages, in any order; -1 behind them
    order = torch.randperm(pages, generator=g, device=dev).int()
    table = torch.full((b, max(need)), -1, dtype=torch.int32, device=dev)
    at = torch.arange(max(need), device=dev)[None]
    n_pages = torch.tensor(need, device=dev)
    first = torch.cumsum(n_pages, 0) - n_pages
    st["table"] = torch.where(at < n_pages[:, None], order[(first[:, None] + at).clamp(max=pages - 1)], table)
    st["cu"] = torch.tensor([0] + new, device=dev).cumsum(0).int()
    st["lengths"] = torch.tensor(cached, device=dev, dtype=torch.int32)
    st["most"] = max(new)
    if case["kind"] == "attend":
        st["q"] = (torch.randn(t, case["hq"], case["dim"], generator=g, device=dev) * 1.2).to(dt)
        return st
    # one projection's output, q, k and v beside each other in each row
    x = torch.randn(t, case["hq"] + 2 * case["hkv"], case["dim"], generator=g, device=dev)
    x *= torch.exp(0.5 * torch.randn(x.shape[1:], generator=g, device=dev))
    st["qkv"] = x.to(dt)
    st["q_weight"] = st["k_weight"] = None
    if case["norm"]:
        st["q_weight"], st["k_weight"] = (1 + 0.2 * torch.randn(2, case["dim"], generator=g, device=dev)).to(dt)
    pos = torch.cat([torch.arange(c, c + n, device=dev) for n, c in zip(new, cached)]).double()
    angle = pos[:, None] * (1e6 ** (-torch.arange(0, case["dim"], 2, device=dev).double() / case["dim"]))[None]
    angle = torch.cat([angle, angle], -1)
    st["cos"], st["sin"] = torch.cos(angle).to(dt), torch.sin(angle).to(dt)
    return st


# ---- one pass ----------------------------------------------------------------

def _framework():
    return importlib.import_module("mtp-glora_amd")


def _places(st, tokens):
    """Sequence, position, page and row of each new token."""
    cu, p = st["cu"].long(), st["case"]["page"]
    at = torch.arange(tokens, device=cu.device)
    seq = torch.searchsorted(cu[1:], at, right=True)
    pos = st["lengths"].long()[seq] + at - cu[seq]
    return seq, pos, st["table"][seq, pos // p].long(), pos % p


def _rotated(x, weight, st):
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    a, b = x.chunk(2, -1)
    return x * st["cos"].float()[:, None] + torch.cat([-b, a], -1) * st["sin"].float()[:, None]


def _store(codes, scale, x, page, row, old_page, old_rows):
    """x [token, head, channel] into codes [page, head, row, channel], a view, and their scales."""
    amax = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
    touched = torch.zeros_like(scale[:, :1]).index_fill_(0, page, 1.0) > 0
    kept = torch.zeros_like(scale[:, :1]).index_put_((old_page,), (old_rows > 0).float()[:, None]) > 0
    grown = torch.where(touched, torch.maximum(_scale_of(amax), torch.where(kept, scale, 0.0)), scale)
    bytes_ = codes.view(torch.uint8)
    before = bytes_[old_page]
    ratio = (scale / grown)[old_page][:, :, None, None]
    again = (before.view(E4M3).float() * ratio).to(E4M3).view(torch.uint8)
    stays = torch.arange(codes.shape[2], device=x.device)[None] < old_rows[:, None]
    bytes_[old_page] = torch.where(stays[:, None, :, None], again, before)
    bytes_[page, :, row] = (x / grown[page][..., None]).to(E4M3).view(torch.uint8)
    scale.copy_(grown)


def _plain_append(st):
    c = st["case"]
    q, k, v = st["qkv"].float().split([c["hq"], c["hkv"], c["hkv"]], 1)
    q, k = _rotated(q, st["q_weight"], st), _rotated(k, st["k_weight"], st)
    seq, pos, page, row = _places(st, len(q))
    cached = st["lengths"].long()
    old_page = st["table"].gather(1, (cached // c["page"])[:, None])[:, 0].long()
    _store(st["k"], st["k_scale"], k, page, row, old_page, cached % c["page"])
    _store(st["v"].transpose(2, 3), st["v_scale"], v, page, row, old_page, cached % c["page"])
    return q.to(st["qkv"].dtype), st["k"], st["v"], st["k_scale"], st["v_scale"]


def _plain_attend(st):
    c, q = st["case"], st["q"]
    table = st["table"].long().clamp(min=0)
    b, hkv, dim, group = len(table), c["hkv"], c["dim"], c["hq"] // c["hkv"]
    k = st["k"].view(torch.uint8)[table].view(E4M3).float() * st["k_scale"][table][..., None, None]
    v = st["v"].view(torch.uint8)[table].view(E4M3).float() * st["v_scale"][table][..., None, None]
    k = k.permute(0, 2, 4, 1, 3).reshape(b, hkv, dim, -1)
    v = v.permute(0, 2, 1, 4, 3).reshape(b, hkv, -1, dim)
    cu, most = st["cu"].long(), st["most"]
    each = torch.arange(most, device=q.device)
    x = q.float()[(cu[:-1, None] + each).clamp(max=len(q) - 1)]
    x = x.reshape(b, most, hkv, group, dim).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * most, dim)
    s = torch.matmul(x, k).mul_(dim ** -0.5).view(b, hkv, group, most, -1)
    last = st["lengths"].long()[:, None] + each
    s.masked_fill_(torch.arange(s.shape[-1], device=q.device) > last[:, None, None, :, None], float("-inf"))
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    s /= s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(b, hkv, group * most, -1), v).view(b, c["hq"], most, dim)
    seq = torch.searchsorted(cu[1:], torch.arange(len(q), device=q.device), right=True)
    return o[seq, :, torch.arange(len(q), device=q.device) - cu[seq]].to(q.dtype)


def _plain_logits(st):
    x, ids = st["logits"].float(), st["tokens"]
    at = torch.arange(ids.shape[1], device=x.device)[None]
    inside = at < st["lengths"][:, None]
    seen = torch.zeros_like(x).scatter_add_(1, ids, inside.float()) > 0
    count = torch.zeros_like(x).scatter_add_(1, ids, (inside & (at >= st["prompts"][:, None])).float())
    r = st["repetition"][:, None]
    y = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    y = y - st["frequency"][:, None] * count - st["presence"][:, None] * (count > 0)
    if st["bias"] is not None:
        y.scatter_add_(1, st["bias_ids"].long(), st["bias"])
    if st["allowed"] is not None:
        col = torch.arange(x.shape[1], device=x.device)
        y = torch.where((st["allowed"][:, col // 32] >> (col % 32)) & 1 > 0, y, float("-inf"))
    return y.to(st["logits"].dtype)


def run(st):
    c = st["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "logits": _plain_logits}[c["kind"]](st)
    mga = _framework()
    if c["kind"] == "logits":
        return mga.adjust_logits(st["logits"], st["tokens"], lengths=st["lengths"], prompt_lengths=st["prompts"],
                                 repetition=st["repetition"], frequency=st["frequency"], presence=st["presence"],
                                 bias_ids=st["bias_ids"], bias=st["bias"], allowed=st["allowed"])
    pages = (st["k"], st["v"], st["k_scale"], st["v_scale"])
    if c["kind"] == "attend":
        return mga.paged_attention(st["q"], pages, st["table"], st["cu"], st["lengths"], scaling=c["dim"] ** -0.5)
    q, k, v = st["qkv"].split([c["hq"], c["hkv"], c["hkv"]], 1)
    q = mga.paged_append(k, v, pages, st["table"], st["cu"], st["lengths"], query=q, cos=st["cos"], sin=st["sin"],
                         q_weight=st["q_weight"], k_weight=st["k_weight"], eps=EPS)
    return (q, *pages)


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    eb = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "logits":
        n, v = case["rows"], case["vocab"]
        other = case["history"] * 8 + case["bias"] * 8 + (v // 8 if case["mask"] else 0) + 20
        return dict(bytes=n * (2 * v * eb + other), flops=4 * n * v)
    new, cached = _plan(case)
    t, hq, hkv, d = sum(new), case["hq"], case["hkv"], case["dim"]
    if case["kind"] == "append":
        return dict(bytes=t * d * ((2 * hq + 2 * hkv + 2) * eb + 2 * hkv), flops=t * d * (hq + 2 * hkv) * 8)
    seen = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, cached))
    return dict(bytes=2 * t * hq * d * eb + 2 * hkv * d * sum(n + c for n, c in zip(new, cached)), flops=4 * hq * d * seen)


# ---- the same in 64 bits -----------------------------------------------------

def _round_e4m3(x):
    """The nearest of e4m3's numbers, the even one of two as near."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_store(codes, scale, x, table, lengths, new, page):
    """codes [page, head, row, channel] and scale in 64 bits, one page of a sequence after the other."""
    t = 0
    for b, n in enumerate(new):
        at, end = lengths[b], lengths[b] + n
        while at < end:
            stop = min(end, (at // page + 1) * page)
            which, r0, r1 = table[b][at // page], at % page, at % page + stop - at
            rows = x[t:t + stop - at].transpose(0, 1)
            t, at = t + stop - at, stop
            top = rows.abs().amax((1, 2))
            need = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(-100, 119))
            was = scale[which]
            now = torch.maximum(was, need) if r0 else need
            codes[which][:, :r0] = _round_e4m3(codes[which][:, :r0] * (was / now)[:, None, None])
            codes[which][:, r0:r1] = _round_e4m3(rows / now[:, None, None])
            scale[which] = now


def _exact_append(case, st):
    new, cached = _plan(case)
    x = st["qkv"].double()
    q, k, v = x[:, :case["hq"]], x[:, case["hq"]:case["hq"] + case["hkv"]], x[:, case["hq"] + case["hkv"]:]
    half = case["dim"] // 2
    cos, sin = st["cos"].double()[:, None, :half], st["sin"].double()[:, None, :half]

    def turned(y, w):
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * w.double()
        z = torch.complex(y[..., :half], y[..., half:]) * torch.complex(cos, sin)
        return torch.cat([z.real, z.imag], -1)

    table = st["table"].tolist()
    codes, ks, vs = st["k"].double(), st["k_scale"].double(), st["v_scale"].double()
    _exact_store(codes, ks, turned(k, st["k_weight"]), table, cached, new, case["page"])
    values = st["v"].double().transpose(2, 3).contiguous()
    _exact_store(values, vs, v, table, cached, new, case["page"])
    return turned(q, st["q_weight"]), codes, values.transpose(2, 3).contiguous(), ks, vs


def _exact_attend(case, st):
    new, cached = _plan(case)
    group, t, out = case["hq"] // case["hkv"], 0, []
    for b, (n, c) in enumerate(zip(new, cached)):
        which = st["table"][b, :-(-(n + c) // case["page"])].long()
        k = st["k"].view(torch.uint8)[which].view(E4M3).double() * st["k_scale"][which].double()[..., None, None]
        v = st["v"].view(torch.uint8)[which].view(E4M3).double() * st["v_scale"][which].double()[..., None, None]
        k = k.transpose(0, 1).flatten(1, 2)[:, :n + c]
        v = v.permute(1, 2, 0, 3).flatten(2, 3)[:, :, :n + c]
        masked = torch.arange(n + c, device=k.device)[None] > (c + torch.arange(n, device=k.device))[:, None]
        heads = [None] * case["hq"]
        for h in range(case["hq"]):
            s = (k[h // group] @ st["q"][t:t + n, h].double().T).T * case["dim"] ** -0.5
            p = torch.softmax(s.masked_fill(masked, float("-inf")), -1)
            heads[h] = (v[h // group] @ p.T).T
        out.append(torch.stack(heads, 1))
        t += n
    return torch.cat(out)


def _exact_logits(case, st):
    y = st["logits"].double()
    size = case["vocab"]
    for r in range(case["rows"]):
        n, m = int(st["lengths"][r]), int(st["prompts"][r])
        seen = torch.bincount(st["tokens"][r, :n], minlength=size)
        count = torch.bincount(st["tokens"][r, m:n], minlength=size)
        factor = torch.where(seen > 0, st["repetition"][r].double(), 1.0)
        y[r] = torch.where(y[r] > 0, y[r] / factor, y[r] * factor)
        y[r] -= count * st["frequency"][r].double() + (count > 0) * st["presence"][r].double()
        if st["bias"] is not None:
            y[r].index_add_(0, st["bias_ids"][r].long(), st["bias"][r].double())
        if st["allowed"] is not None:
            bit = torch.ones(32, dtype=torch.int32, device=y.device) << torch.arange(32, device=y.device).int()
            y[r].masked_fill_(((st["allowed"][r][:, None] & bit) == 0).flatten()[:size], float("-inf"))
    return y


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logits": _exact_logits}[case["kind"]](case, st)
