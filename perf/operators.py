"""The vocabulary's operators of a chunked MTP training run, timed: a teacher's
top logits, the distillation loss from them, token sampling, and the scaled
embedding with its gradient.

A case is a dict of plain values. ``prepare`` makes what the program has in
hand before the call, ``run`` is one pass: in elementary torch operations where
``own`` is false, by the framework's calls where it is true. ``exact`` gives the
same outputs in 64 bits. Kinds:

* ``top_logits`` - the k largest logits of each teacher row, their ids (lowest
  first among equals) and the row's log-sum-exp.
* ``distill`` - the cross-entropy against a teacher's top logits. mode
  ``forward``: the loss; ``train``: loss and ``backward()``; ``fused``: loss and
  scaled gradient in one call.
* ``sample`` - a token per row from given uniform numbers, with temperature,
  top-k, top-p and min-p per row.
* ``embed`` - the scaled lookup of a chunk's tokens. mode ``forward``, or
  ``train``: lookup and the weight's gradient.
"""
import importlib
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
QWEN3_VOCAB = 151936
LLAMA_VOCAB = 128256


def listed():
    return [
        # the teacher's side of an ordinary chunk: 256 x 4 drafted positions
        dict(name="top_logits_ordinary", kind="top_logits", rows=1024, vocab=QWEN3_VOCAB, k=64, tau=1.0, dtype="bf16"),
        # a short last chunk of an fp32 run with a vocabulary of odd size
        dict(name="top_logits_ragged", kind="top_logits", rows=77, vocab=32003, k=20, tau=2.0, dtype="fp32"),
        # the loss and its gradient over an ordinary chunk, the loss scale known
        dict(name="distill_fused", kind="distill", mode="fused", rows=1024, vocab=QWEN3_VOCAB, k=64, lse=True, tau=1.0,
             pad=0.0, dtype="bf16"),
        # the same through autograd, for the few rows of a short chunk, some of
        # them padding, the teacher renormalised over what was kept of it
        dict(name="distill_train_few", kind="distill", mode="train", rows=52, vocab=QWEN3_VOCAB, k=32, lse=False,
             tau=2.0, pad=0.1, dtype="bf16"),
        # an evaluation pass of an fp16 run
        dict(name="distill_eval_fp16", kind="distill", mode="forward", rows=333, vocab=LLAMA_VOCAB, k=128, lse=True,
             tau=1.0, pad=0.0, dtype="fp16"),
        # one drafted token: latency
        dict(name="sample_one", kind="sample", rows=1, vocab=QWEN3_VOCAB, mix="nucleus", dtype="bf16"),
        # a batch of drafts, each row with its own settings, greedy ones among them
        dict(name="sample_mixed", kind="sample", rows=256, vocab=QWEN3_VOCAB, mix="mixed", dtype="bf16"),
        # fp32 logits by temperature alone: every token stays in
        dict(name="sample_temperature", kind="sample", rows=96, vocab=32003, mix="temperature", dtype="fp32"),
        # an ordinary chunk's tokens, 1024 of 5120 the mask token
        dict(name="embed_lookup", kind="embed", mode="forward", n_reg=4096, anchors=256, draft=4, pad=0,
             vocab=QWEN3_VOCAB, hidden=4096, scale=1.0, dtype="bf16"),
        # the small fp32 decoder of the end-to-end tests: launches and latency
        dict(name="embed_train_small", kind="embed", mode="train", n_reg=256, anchors=16, draft=4, pad=3, vocab=1024,
             hidden=256, scale=16.0, dtype="fp32"),
        # lookup and gradient of a dense MTP chunk: two of three tokens are the mask
        dict(name="embed_train_dense", kind="embed", mode="train", n_reg=2048, anchors=1024, draft=4, pad=0,
             vocab=32003, hidden=2560, scale=50.596443, dtype="fp16"),
        # the ordinary chunk against the whole vocabulary: the gradient's
        # 1.2 GB are the work
        dict(name="embed_train_ordinary", kind="embed", mode="train", n_reg=4096, anchors=256, draft=4, pad=0,
             vocab=QWEN3_VOCAB, hidden=4096, scale=1.0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["top_logits", "distill", "distill", "sample", "sample", "embed", "embed"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = rng.choice([QWEN3_VOCAB, QWEN3_VOCAB, LLAMA_VOCAB, 32003, _log_int(rng, 700, 150000)])
    most = 512 if dtype == "fp32" else 1024
    if kind == "top_logits":
        return dict(kind=kind, rows=_log_int(rng, 1, most), vocab=vocab, k=_log_int(rng, 1, 256),
                    tau=rng.choice([1.0, 1.0, 0.5, 2.0]), dtype=dtype)
    if kind == "distill":
        return dict(kind=kind, mode=rng.choice(["forward", "train", "fused", "fused"]), rows=_log_int(rng, 1, most),
                    vocab=vocab, k=_log_int(rng, 4, 256), lse=rng.random() < 0.5, tau=rng.choice([1.0, 1.0, 0.5, 2.0]),
                    pad=rng.choice([0.0, 0.0, 0.1]), dtype=dtype)
    if kind == "sample":
        return dict(kind=kind, rows=_log_int(rng, 1, 256), vocab=vocab,
                    mix=rng.choice(["nucleus", "mixed", "mixed", "temperature"]), dtype=dtype)
    draft = rng.choice([2, 4, 4, 8])
    n_reg = _log_int(rng, 16, 4096)
    return dict(kind=kind, mode=rng.choice(["forward", "train", "train"]), n_reg=n_reg,
                anchors=max(1, int(n_reg * rng.uniform(0.03, 0.5) / draft)), draft=draft, pad=rng.choice([0, 0, 7]),
                vocab=min(vocab, 130000) if dtype != "fp32" else min(vocab, 60000),
                hidden=rng.choice([256, 1000, 2560, 4096]), scale=rng.choice([1.0, 1.0, 16.0]), dtype=dtype)


# ---- inputs ------------------------------------------------------------------

def _logits(rows, vocab, g, dev):
    """Rows as a language model's head gives them: a broad bulk and some hundred
    tokens that stand out of it, the first of them far."""
    x = torch.randn(rows, vocab, generator=g, device=dev).mul_(2.0)
    n = min(vocab, 200)
    at = torch.randint(vocab, (rows, n), generator=g, device=dev)
    up = torch.rand(rows, n, generator=g, device=dev).pow_(4).mul_(12.0)
    return x.scatter_add_(1, at, up)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = dict(case=case)
    if case["kind"] == "top_logits":
        st["logits"] = _logits(case["rows"], case["vocab"], g, dev).to(dt)[None]
    elif case["kind"] == "distill":
        n, v, k = case["rows"], case["vocab"], min(case["k"], case["vocab"])
        x = _logits(n, v, g, dev)
        # the student has learned part of what the teacher says
        st["student"] = (x * 0.8 + torch.randn(n, v, generator=g, device=dev) * 0.6).to(dt)[None]
        values, ids = torch.topk(x, k, dim=-1)
        ids = ids.to(torch.int32)
        if case["pad"]:
            # padded rows, and rows of which fewer than k logits were kept
            dead = torch.rand(n, 1, generator=g, device=dev) < case["pad"]
            short = torch.arange(k, device=dev) >= k - (torch.rand(n, 1, generator=g, device=dev) < 0.3).int() * (k // 3)
            ids = torch.where(dead | short, -1, ids)
        st["values"], st["ids"] = values.to(dt)[None], ids[None]
        st["lse"] = torch.logsumexp(x / case["tau"], -1)[None] if case["lse"] else None
        st["scale"] = 0.125    # one of eight chunks
    elif case["kind"] == "sample":
        n, v = case["rows"], case["vocab"]
        x = _logits(n, v, g, dev)
        if case["dtype"] == "fp32":    # a vocabulary of which a part is masked out
            x[:, torch.randint(v, (v // 8,), generator=g, device=dev)] = float("-inf")
            x[:, 0] = 0.0
        st["logits"] = x.to(dt)
        st["u"] = torch.rand(n, generator=g, device=dev)
        one = torch.ones(n, device=dev)
        pick = torch.randint(6, (n,), generator=g, device=dev)
        if case["mix"] == "nucleus":
            st["temperature"], st["top_k"], st["top_p"], st["min_p"] = one * 0.7, one.int() * 50, one * 0.9, one * 0.0
        elif case["mix"] == "temperature":
            st["temperature"], st["top_k"], st["top_p"], st["min_p"] = one * 1.0, one.int() * 0, one * 1.0, one * 0.0
        else:    # greedy; top-p; top-k; min-p; top-k and top-p; temperature alone
            st["temperature"] = torch.tensor([0.0, 0.8, 1.0, 1.2, 0.6, 0.9], device=dev)[pick]
            st["top_k"] = torch.tensor([0, 0, 40, 0, 200, 0], device=dev, dtype=torch.int32)[pick]
            st["top_p"] = torch.tensor([1.0, 0.95, 1.0, 1.0, 0.8, 1.0], device=dev)[pick]
            st["min_p"] = torch.tensor([0.0, 0.0, 0.0, 0.05, 0.0, 0.0], device=dev)[pick]
    else:
        v, h, n_reg = case["vocab"], case["hidden"], case["n_reg"]
        st["weight"] = (torch.randn(v, h, generator=g, device=dev) * 0.02).to(dt)
        # regular tokens by a heavy-tailed frequency; after each anchor, draft mask tokens; padding at the end
        ids = (torch.rand(n_reg, generator=g, device=dev).pow_(6) * (v - 1)).long().clamp_(max=v - 2)
        at = torch.sort(torch.randperm(n_reg, generator=g, device=dev)[:case["anchors"]]).values
        count = torch.zeros(n_reg, dtype=torch.long, device=dev).index_fill_(0, at, case["draft"])
        end = torch.cumsum(count + 1, 0)
        out = torch.full((int(end[-1]) + case["pad"],), v - 1, dtype=torch.long, device=dev)
        out[end - count - 1] = ids
        if case["pad"]:
            out[-case["pad"]:] = 0
        st["ids"] = out[None]
        st["grad_out"] = (torch.randn(1, out.numel(), h, generator=g, device=dev) * 0.1).to(dt)
    return st


# ---- one pass ----------------------------------------------------------------

def _framework():
    return importlib.import_module("mtp-glora_amd")


def _plain_top_logits(x, k, tau):
    xf = x.float()
    values, ids = torch.sort(xf, dim=-1, descending=True, stable=True)
    y = xf / tau
    m = y.amax(-1, keepdim=True)
    lse = torch.log(torch.exp(y - m).sum(-1)) + m[..., 0]
    return values[..., :k].to(x.dtype), ids[..., :k].int(), lse


def _plain_distill(st):
    """Loss and scale x its gradient, in 32 bits."""
    c, ids = st["case"], st["ids"].long()
    tau = c["tau"]
    x = st["student"]
    y = x.float() / tau
    s = st["values"].float() / tau
    valid = ids >= 0
    s = torch.where(valid, s, float("-inf"))
    if st["lse"] is not None:
        q = torch.exp(s - st["lse"][..., None])
    else:
        top = s.amax(-1, keepdim=True).clamp_(min=-3e38)
        q = torch.exp(s - top)
        q = q / q.sum(-1, keepdim=True).clamp_(min=1e-30)
    at = ids.clamp(min=0)
    m = y.amax(-1, keepdim=True)
    e = torch.exp(y - m)
    z = e.sum(-1, keepdim=True)
    lse = (torch.log(z) + m)[..., 0]
    total = q.sum(-1)
    loss = tau * tau * (total * lse - (q * torch.gather(y, -1, at)).sum(-1)).sum()
    if c["mode"] == "forward":
        return loss
    factor = tau * (st["scale"] if c["mode"] == "fused" else 1.0)
    grad = e * (total[..., None] / z)
    grad.scatter_add_(-1, at, -q)
    return loss, (grad * factor).to(x.dtype)


def _plain_sample(st):
    """In 64 bits: the borders between tokens are nearer to each other than sums
    in 32 bits are right."""
    x = st["logits"].double()
    t, k = st["temperature"].double()[:, None], st["top_k"].long()[:, None]
    p, m = st["top_p"].double()[:, None], st["min_p"].double()[:, None]
    greedy = t == 0
    t = torch.where(greedy, 1.0, t)
    top = x.amax(-1, keepdim=True)
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)
    ws = torch.exp((xs - top) / t)
    rank = torch.arange(x.shape[-1], device=x.device)[None]
    keep = (k <= 0) | (rank < k)
    cum = torch.cumsum(torch.where(keep, ws, 0.0), -1)
    before = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], -1)
    keep &= (p >= 1) | (before < p * cum[:, -1:])
    keep &= ws >= m
    w = torch.zeros_like(x).scatter_(1, order, torch.where(keep, ws, 0.0))
    cum = torch.cumsum(w, -1)
    token = (cum > st["u"].double()[:, None] * cum[:, -1:]).int().argmax(-1)
    return torch.where(greedy[:, 0], order[:, 0], token)


def _plain_embed(st):
    c, w, ids, dy = st["case"], st["weight"], st["ids"], st["grad_out"]
    out = (w[ids].float() * c["scale"]).to(w.dtype)
    if c["mode"] == "forward":
        return out
    dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    dw.index_add_(0, ids.reshape(-1), dy.reshape(-1, w.shape[1]).float())
    return out, (dw * c["scale"]).to(w.dtype)


def run(st):
    c = st["case"]
    if not own:
        if c["kind"] == "top_logits":
            return _plain_top_logits(st["logits"], min(c["k"], c["vocab"]), c["tau"])
        if c["kind"] == "distill":
            return _plain_distill(st)
        return _plain_sample(st) if c["kind"] == "sample" else _plain_embed(st)
    mga = _framework()
    if c["kind"] == "top_logits":
        return tuple(mga.top_logits(st["logits"], min(c["k"], c["vocab"]), temperature=c["tau"]))
    if c["kind"] == "distill":
        args = (st["values"], st["ids"], st["lse"], c["tau"])
        if c["mode"] == "forward":
            return mga.top_logits_cross_entropy(st["student"], *args)
        if c["mode"] == "fused":
            return mga.top_logits_loss_and_grad(st["student"], *args, scale=st["scale"])
        x = st["student"].detach().requires_grad_()
        loss = mga.top_logits_cross_entropy(x, *args)
        loss.backward()
        return loss.detach(), x.grad
    if c["kind"] == "sample":
        return mga.sample_tokens(st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])
    if c["mode"] == "forward":
        return mga.scaled_embedding(st["ids"], st["weight"], c["scale"])
    w = st["weight"].detach().requires_grad_()
    out = mga.scaled_embedding(st["ids"], w, c["scale"])
    out.backward(st["grad_out"])
    return out.detach(), w.grad


# ---- what a pass cannot do without -------------------------------------------

def _tokens(c):
    return c["n_reg"] + c["anchors"] * c["draft"] + c["pad"]


def work(case):
    eb = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "embed":
        n, h = _tokens(case), case["hidden"]
        lookup = n * 8 + min(n, case["vocab"]) * h * eb + n * h * eb
        if case["mode"] == "forward":
            return dict(bytes=lookup, flops=n * h)
        return dict(bytes=lookup + n * h * eb + case["vocab"] * h * eb, flops=3 * n * h)
    n, v = case["rows"], case["vocab"]
    if case["kind"] == "top_logits":
        return dict(bytes=n * (v * eb + case["k"] * (eb + 4) + 4), flops=4 * n * v)
    if case["kind"] == "sample":
        return dict(bytes=n * (v * eb + 28), flops=4 * n * v)
    small = n * (case["k"] * (eb + 4) + 4)
    if case["mode"] == "forward":
        return dict(bytes=n * v * eb + small, flops=4 * n * v)
    return dict(bytes=2 * n * v * eb + small, flops=6 * n * v)


# ---- the same in 64 bits -----------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "top_logits":
        x = st["logits"][0]
        n, v = x.shape
        # one whole number a logit: its place among the values, then the lower index
        b = x.float().contiguous().view(torch.int32).long()
        b = torch.where(b < 0, -(b & 0x7FFFFFFF), b)
        comp = (b << 20) + ((1 << 20) - 1 - torch.arange(v, device=x.device))
        ids = ((1 << 20) - 1) - (torch.topk(comp, min(case["k"], v), -1).values & ((1 << 20) - 1))
        return (torch.gather(x, 1, ids)[None].double(), ids.int()[None],
                torch.logsumexp(x.double() / case["tau"], -1)[None])
    if case["kind"] == "distill":
        return _exact_distill(case, st)
    if case["kind"] == "sample":
        return _exact_sample(st)
    ids, w, dy = st["ids"][0], st["weight"], st["grad_out"][0]
    out = torch.index_select(w, 0, ids).double()[None] * case["scale"]
    if case["mode"] == "forward":
        return out
    # the tokens in sorted order, differences of their running sums
    order = torch.argsort(ids, stable=True)
    found, count = torch.unique_consecutive(ids[order], return_counts=True)
    run_ = torch.cumsum(dy[order].double(), 0)
    end = torch.cumsum(count, 0) - 1
    sums = run_[end]
    sums = torch.cat([sums[:1], sums[1:] - sums[:-1]])
    dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    dw[found] = sums * case["scale"]
    return out, dw


def _exact_distill(case, st):
    x = st["student"][0].double()
    n, v = x.shape
    tau, ids = case["tau"], st["ids"][0].long()
    logp = torch.log_softmax(x / tau, -1)
    # the teacher's row laid out over the whole vocabulary, one column behind it for what is padding
    t = torch.zeros(n, v + 1, dtype=torch.float64, device=x.device)
    s = torch.where(ids >= 0, st["values"][0].double() / tau, float("-inf"))
    norm = st["lse"][0].double() if case["lse"] else torch.logsumexp(s, -1)
    q = torch.where(torch.isfinite(norm)[:, None], torch.exp(s - norm[:, None]), 0.0)
    t.scatter_(1, torch.where(ids >= 0, ids, v), q)
    t = t[:, :v]
    loss = -tau * tau * (t * logp).sum()
    if case["mode"] == "forward":
        return loss
    factor = tau * (st["scale"] if case["mode"] == "fused" else 1.0)
    return loss, (factor * (torch.exp(logp) * t.sum(-1, keepdim=True) - t))[None]


def _exact_sample(st):
    x = st["logits"].double().cpu().numpy()
    p = {k: st[k].double().cpu().numpy() for k in ("u", "temperature", "top_k", "top_p", "min_p")}
    out = np.empty(len(x), np.int64)
    for r, row in enumerate(x):
        if p["temperature"][r] == 0:
            out[r] = int(np.argmax(row))
            continue
        w = np.exp((row - row.max()) / p["temperature"][r])
        # only what the thresholds can leave in is put in order
        order = np.argsort(-row, kind="stable")
        if p["top_k"][r] > 0:
            order = order[:int(p["top_k"][r])]
        if p["top_p"][r] < 1:
            c = np.cumsum(w[order].astype(np.longdouble))
            order = order[:int(np.searchsorted(c, p["top_p"][r] * c[-1])) + 1]
        order = np.sort(order[w[order] >= p["min_p"][r]])
        c = np.cumsum(w[order].astype(np.longdouble))
        out[r] = order[min(len(order) - 1, int(np.searchsorted(c, p["u"][r] * c[-1], side="right")))]
    return torch.from_numpy(out).to(st["logits"].device)
