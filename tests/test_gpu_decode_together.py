"""A decoding step as it is used: a Qwen3-style decoder over the paged cache (prompts, then
drafts of which some are dropped), its logits through adjust_logits and sample_tokens; steps in
captured graphs whose batches change between replays; other streams.

The decoder's reference runs in float64 on the keys and values that the cache holds
after each append, so that it differs from the fp32 model by fp32 arithmetic alone: logits
max-abs 1e-5, mean-abs 1e-6, as of the streaming cache's end-to-end test (the same
model, the same depth). The cache's contents are checked against the reference's own keys
and values: each code is the nearest to its value, half a step of e4m3 (2^-4 of the value,
2^-10 of the scale below the normal range), once more where a page's scale grew later, beside the fp32 model's
1e-5."""
import numpy as np
import pytest
import torch

from oracle import vocab as vo

pytestmark = pytest.mark.gpu

transformers = pytest.importorskip("transformers")
from transformers import Qwen3Config, Qwen3ForCausalLM  # noqa: E402

VOCAB, LAYERS, D, PS = 1024, 2, 64, 16


def decoder(dev):
    cfg = Qwen3Config(vocab_size=VOCAB, hidden_size=256, intermediate_size=512, num_hidden_layers=LAYERS,
                      num_attention_heads=4, num_key_value_heads=2, head_dim=D, max_position_embeddings=4096)
    torch.manual_seed(7)
    return Qwen3ForCausalLM(cfg).eval().to(dev)


def forward(model, ids, pos, attention):
    """Logits of packed tokens; attention(layer, x, (cos, sin)) is the self-attention's output."""
    m = model.model
    h = m.embed_tokens(ids[None])
    pe = m.rotary_emb(h, pos[None])
    for i, layer in enumerate(m.layers):
        h = h + attention(i, layer.self_attn, layer.input_layernorm(h), pe)
        h = h + layer.mlp(layer.post_attention_layernorm(h))
    return model.lm_head(m.norm(h))[0]


def reference_attention(cache, new, cached, table, checks):
    def attend(i, attn, x, pe):
        T = x.shape[1]
        cos, sin = (t[0][:, None] for t in pe)
        turn = lambda y: y * cos + torch.cat([-y[..., D // 2:], y[..., :D // 2]], -1) * sin   # noqa: E731
        q = turn(attn.q_norm(attn.q_proj(x).view(T, -1, D)))
        k = turn(attn.k_norm(attn.k_proj(x).view(T, -1, D)))
        v = attn.v_proj(x).view(T, -1, D)
        out, at = [], 0
        for b, (n, c) in enumerate(zip(new, cached)):
            if n == 0:
                continue
            kd, vd = (t.double().cpu() for t in cache.dequantized(i, table[b], c + n))
            checks.append((i, b, c, k[at:at + n].transpose(0, 1), v[at:at + n].transpose(0, 1), kd, vd))
            kk, vv = kd.repeat_interleave(2, 0), vd.repeat_interleave(2, 0)
            s = q[at:at + n].transpose(0, 1) @ kk.transpose(1, 2) * D ** -0.5
            masked = torch.arange(c + n)[None] > (c + torch.arange(n))[:, None]
            out.append((torch.softmax(s.masked_fill(masked, float("-inf")), -1) @ vv).transpose(0, 1))
            at += n
        return attn.o_proj(torch.cat(out).reshape(1, T, -1))
    return attend


@torch.no_grad()
def test_rollout(mga, dev):
    model = decoder(dev)
    exact = decoder("cpu").double()
    g = torch.Generator().manual_seed(3)
    cached = [0, 0, 0]
    cache = mga.PagedKVCache(24, LAYERS, 2, D, page_size=PS, device=dev)
    pages = torch.randperm(24, generator=g).view(3, 8).int()
    history = [[], [], []]
    steps = [[21, 5, 40], [5, 5, 5], [3, 0, 5], [1, 1, 1], [5, 12, 5]]
    keeps = [[21, 5, 40], [2, 5, 1], [3, 0, 2], [1, 1, 1], [0, 0, 0]]   # of a step's tokens, those that stay
    fed = [torch.randint(VOCAB, (n,), generator=g).tolist() for n in steps[0]]
    for new, keep in zip(steps, keeps):
        fed = [(f + torch.randint(VOCAB, (n,), generator=g).tolist())[:n] for f, n in zip(fed, new)]
        ids = torch.tensor([t for f in fed for t in f])
        pos = torch.cat([torch.arange(c, c + n) for c, n in zip(cached, new)])
        cu = torch.tensor([0] + new).cumsum(0).int()
        cache.begin(pages.to(dev), cu.to(dev), torch.tensor(cached, dtype=torch.int32, device=dev))
        logits = forward(model, ids.to(dev), pos.to(dev), lambda i, attn, x, pe: mga.qwen3_attention_forward(
            attn, x, pe, None, past_key_value=cache)[0])
        checks = []
        want = forward(exact, ids, pos, reference_attention(cache, new, cached, pages, checks))
        err = (logits.double().cpu() - want).abs()
        assert err.max() <= 1e-5 and err.mean() <= 1e-6, (float(err.max()), float(err.mean()))
        for i, b, c, k, v, kd, vd in checks:
            p = cache.pages(i)
            for x, got, scale in ((k, kd, p.k_scale), (v, vd, p.v_scale)):
                s = scale[pages[b].long().to(dev)].double().cpu().repeat_interleave(PS, 0)[c:c + x.shape[1]].t()[..., None]
                assert ((got[:, c:] - x).abs() <= x.abs() * 2.0 ** -4 + s * 2.0 ** -10 + 1e-5).all()
        # a token for each sequence from its last row, its history penalised, half the vocabulary allowed
        last = [int(cu[b + 1]) - 1 for b in range(3) if new[b]]
        who = [b for b in range(3) if new[b]]
        for b, f, kp in zip(range(3), fed, keep):
            history[b] += f[:kp]
        L = max(len(history[b]) for b in who) + 2
        tokens = torch.full((len(who), L), -1)
        for r, b in enumerate(who):
            tokens[r, :len(history[b])] = torch.tensor(history[b])
        lens = torch.tensor([len(history[b]) for b in who], dtype=torch.int32)
        allowed = torch.randint(-2 ** 31, 2 ** 31, (VOCAB // 32,), generator=g).int()
        u = torch.rand(len(who), generator=g)
        shaped = mga.adjust_logits(logits[last], tokens.to(dev), lengths=lens.to(dev), repetition=1.2, frequency=0.1,
                                   presence=0.2, allowed=allowed.to(dev))
        drawn = mga.sample_tokens(shaped, u.to(dev), 0.8, 50, 0.95)
        ref, mag = vo.adjust(logits[last].double().cpu().numpy(), tokens.numpy(), lens.numpy(), None, 1.2, 0.1, 0.2,
                             allowed=allowed.numpy())
        got = shaped.double().cpu().numpy()
        with np.errstate(invalid="ignore"):
            assert ((np.abs(got - ref) <= 5 * 2.0 ** -24 * mag) | (got == ref)).all()
        for r, b in enumerate(who):
            assert int(drawn[r]) == vo.sample_row(got[r], float(u[r]), float(np.float32(0.8)), 50, float(np.float32(0.95)), 0.0)
            fed[b] = [int(drawn[r])]
        cached = [c + kp for c, kp in zip(cached, keep)]


class Step:
    """One layer's step on buffers that stay, with the batch in them."""

    def __init__(self, mga, dev, dtype, B, T, W, Hq=8, Hkv=2, V=3001, ps=32, dim=128):
        self.mga, self.dev, self.dtype, self.shape = mga, dev, dtype, (B, T, W, Hq, Hkv, V, ps, dim)
        n = B * W
        e4m3 = torch.float8_e4m3fn
        z = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=dev).view(e4m3)   # noqa: E731
        self.pages = z(n, Hkv, ps, dim), z(n, Hkv, dim, ps), torch.ones(n, Hkv, device=dev), torch.ones(n, Hkv, device=dev)
        i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)   # noqa: E731
        self.table, self.cu, self.len = i(B, W), i(B + 1), i(B)
        self.table.copy_(torch.randperm(n, device=dev).view(B, W))
        self.qkv = torch.zeros(T, Hq + 2 * Hkv, dim, dtype=dtype, device=dev)
        self.cos, self.sin = torch.zeros(2, T, dim, dtype=dtype, device=dev)
        self.head = torch.randn(V, Hq * dim, device=dev).to(dtype) * 0.05
        self.tokens, self.lens, self.u = torch.zeros(T, 40, dtype=torch.long, device=dev), i(T), torch.zeros(T, device=dev)

    def fill(self, seed, new, cached):
        B, T, W, Hq, Hkv, V, ps, dim = self.shape
        g = torch.Generator(device=self.dev).manual_seed(seed)
        self.cu.copy_(torch.tensor([0] + new).cumsum(0).int())
        self.len.copy_(torch.tensor(cached).int())
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=g, device=self.dev))
        a = torch.rand(T, dim, generator=g, device=self.dev) * 6
        self.cos.copy_(a.cos())
        self.sin.copy_(a.sin())
        self.tokens.copy_(torch.randint(V, self.tokens.shape, generator=g, device=self.dev))
        self.lens.copy_(torch.randint(41, (T,), generator=g, device=self.dev))
        self.u.copy_(torch.rand(T, generator=g, device=self.dev))
        for t in self.pages[:2]:
            c = torch.randint(0, 0x60, t.shape, generator=g, device=self.dev, dtype=torch.uint8)
            t.view(torch.uint8).copy_(c)
        for t in self.pages[2:]:
            t.copy_(torch.exp2(torch.randint(-8, -4, t.shape, generator=g, device=self.dev).float()))

    def run(self):
        B, T, W, Hq, Hkv, V, ps, dim = self.shape
        q, k, v = self.qkv.split([Hq, Hkv, Hkv], 1)
        q = self.mga.paged_append(k, v, self.pages, self.table, self.cu, self.len, query=q, cos=self.cos, sin=self.sin)
        o = self.mga.paged_attention(q, self.pages, self.table, self.cu, self.len, dim ** -0.5)
        logits = (o.view(T, -1).float() @ self.head.float().t()).to(self.dtype)
        shaped = self.mga.adjust_logits(logits, self.tokens, lengths=self.lens, repetition=1.1, frequency=0.2)
        return q, o, shaped, self.mga.sample_tokens(shaped, self.u, 0.9, 40)

    def state(self):
        return [t.view(torch.uint8).clone() if t.dtype == torch.float8_e4m3fn else t.clone() for t in self.pages]


BATCHES = [([3, 1, 4], [0, 900, 31]), ([1, 1, 1], [5000, 2, 64]), ([2, 0, 6], [33, 7, 0]), ([0, 0, 1], [1, 2, 3]),
           ([4, 2, 2], [100, 1000, 2000])]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("W", [200, 24])     # equal shares; a workgroup a tile
def test_captured_steps(mga, dev, dtype, W):
    """Two graphs, replayed in turn with other batches, eager work between; every replay against the eager step."""
    steps = [Step(mga, dev, dtype, 3, 8, W), Step(mga, dev, dtype, 3, 8, W)]
    graphs, outs = [], []
    for s in steps:
        s.fill(0, *BATCHES[0])
        s.run()
    torch.cuda.synchronize()
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(s.run())
        graphs.append(graph)
    for i, (new, cached) in enumerate(BATCHES):
        cached = [min(c, W * 32 - n) for c, n in zip(cached, new)]
        for s in steps:
            s.fill(10 + i, new, cached)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] + s.state() for o, s in zip(outs, steps)]
        for s, have in zip(steps, got):
            s.fill(10 + i, new, cached)
            want = list(s.run()) + s.state()
            torch.cuda.synchronize()
            for a, b in zip(have, want):
                assert torch.equal(a, b)
            assert not have[1][sum(new):].any()


def test_captured_prompts(mga, dev):
    step = Step(mga, dev, torch.bfloat16, 4, 2200, 60, Hq=16, Hkv=8, V=50, ps=64)
    step.fill(0, [900, 700, 100, 500], [0, 64, 1000, 3])
    step.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step.run()
    for i, (new, cached) in enumerate([([900, 700, 100, 500], [0, 64, 1000, 3]), ([1, 2000, 0, 150], [3000, 0, 5, 77])]):
        step.fill(i, new, cached)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out] + step.state()
        step.fill(i, new, cached)
        for a, b in zip(got, list(step.run()) + step.state()):
            assert torch.equal(a, b)


def test_other_streams(mga, dev):
    """A step on a stream of its own, beside another one's, gives what it gives on the default stream."""
    steps = [Step(mga, dev, torch.bfloat16, 3, 8, 200) for _ in range(2)]
    want = []
    for i, s in enumerate(steps):
        s.fill(i, *BATCHES[i])
        want.append([t.clone() for t in s.run()] + s.state())
        s.fill(i, *BATCHES[i])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = []
    for _ in range(3):
        got = []
        for s, st in zip(steps, streams):
            with torch.cuda.stream(st):
                got.append(s.run())
    torch.cuda.synchronize()
    for s, a, b in zip(steps, got, want):
        for x, y in zip(list(a) + s.state(), b):
            assert torch.equal(x, y)


def test_adapter_refusals(mga, dev):
    model = decoder(dev)
    attn = model.model.layers[0].self_attn
    cache = mga.PagedKVCache(4, LAYERS, 2, D, page_size=PS, device=dev)
    cache.begin(torch.arange(4, dtype=torch.int32, device=dev)[None], torch.tensor([0, 3], dtype=torch.int32, device=dev),
                torch.zeros(1, dtype=torch.int32, device=dev))
    x = torch.randn(2, 3, 256, device=dev)
    pe = model.model.rotary_emb(x, torch.arange(3, device=dev)[None])
    with torch.no_grad(), pytest.raises(ValueError, match="packed"):
        mga.qwen3_attention_forward(attn, x, pe, None, past_key_value=cache)
    with pytest.raises(NotImplementedError, match="no_grad"):
        mga.qwen3_attention_forward(attn, x[:1], pe, None, past_key_value=cache)
