"""Attention over the paged 8-bit cache in each of its forms, at both head sizes, against the
float64 oracle: which form a batch takes is asserted by the rule that chooses it
(csrc/mga_paged_attn.hip: shape_of), so that a batch cannot leave the form it was made for.
Tolerances: test_gpu_paged.py. The exact values of these larger batches come from a dense form in
float64, which a test on the CPU compares with the oracle."""
import types

import numpy as np
import pytest
import torch

import test_gpu_paged as base
from oracle import paged as po
from test_gpu_paged import DTYPES, PARTS, Pool, attend, queries


def dense(q, k, v, pool, scale):
    """q [T, Hq, D]; k, v [pages, Hkv, page_size, D] in value, float64: out and sum p |v| [T, Hq, D], NaN in out
    alone, a sequence at a time."""
    cu, lens = pool.cu.tolist(), pool.len.tolist()
    Hkv, D = k.shape[1], k.shape[3]
    G = q.shape[1] // Hkv
    out, weight = torch.zeros_like(q), torch.zeros_like(q)
    for b, (first, end) in enumerate(zip(cu, cu[1:])):
        n, L = end - first, min(lens[b] + end - first, pool.table.shape[1] * pool.ps)
        if n == 0:
            continue
        ids = pool.table[b].long()
        there = ((ids >= 0) & (ids < len(k))).repeat_interleave(pool.ps)[:L]
        of = lambda t: t[ids.clamp(0, len(k) - 1)].transpose(0, 1).reshape(Hkv, -1, D)[:, :L]   # noqa: E731, B023
        kk, vv = of(k), of(v)
        at = torch.arange(L, device=q.device)
        sees = (at[None] <= lens[b] + torch.arange(n, device=q.device)[:, None]) & there[None]
        x = q[first:end].reshape(n, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * n, D).contiguous()
        s = (x @ kk.transpose(1, 2).contiguous()) * scale
        s = s.masked_fill(~sees.repeat(G, 1), float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True)).masked_fill(~sees.any(-1).repeat(G)[:, None], 0.0)
        p = p / p.sum(-1, keepdim=True).masked_fill(~sees.any(-1).repeat(G)[:, None], 1.0)
        bad = vv.isnan()
        vv = vv.masked_fill(bad, 0.0)
        o = (p @ vv).masked_fill((sees.repeat(G, 1).double()[None] @ bad.double()) > 0, float("nan"))
        for to, t in ((out, o), (weight, p @ vv.abs())):
            to[first:end] = t.view(Hkv, G, n, D).permute(2, 0, 1, 3).reshape(n, Hkv * G, D)
    return out, weight


def check_attention(got, q, pool, scale):
    k, v = (torch.as_tensor(t, device=q.device) for t in pool.kv())
    qd = q[:pool.T].double()
    want, weight = dense(qd, k, v, pool, scale)
    D, n = q.shape[2], int((pool.len + pool.cu.diff()).max())
    kmax = float(k.square().sum(-1).sqrt().nan_to_num(0.0).max())
    qmax = float(qd.square().sum(-1).sqrt().max())
    es = 2 * (D + 16) * 2.0 ** -24 * qmax * kmax * scale + 2.0 ** -20 + n * 2.0 ** -24
    ep = 2.0 ** (-8 * PARTS[q.dtype])
    info = torch.finfo(q.dtype)
    bound = (ep + es) * weight.nan_to_num(float("inf")) + info.eps / 2 * want.abs() + info.tiny
    g = got[:pool.T].double()
    assert torch.equal(g.isnan(), want.isnan())
    off = ((g - want).abs() / bound).nan_to_num(0.0).max()
    assert off <= 1, f"{float(off)} of the bound"
    return want.cpu().numpy()


def test_dense_form_against_the_oracle():
    dev = torch.device("cpu")
    for new, cached, ps in (([3, 0, 40], [20, 5, 0], 16), ([1, 70], [130, 31], 32)):
        pool = Pool(dev, new, cached, 2, 64, ps, seed=1, width=6)
        t0 = pool.table.clone()
        pool.table[0, 1] = -1
        pool.table[len(new) - 1, 0] = pool.n
        pool.v[t0[len(new) - 1, 1], 1, 5, 3] = 0x7f
        pool.k[t0[0, 0], 0, 2, 7] = 0xff
        q = queries(pool, 6, 64, torch.float32, dev)
        k, v = pool.kv()
        with np.errstate(all="ignore"):
            want, weight = po.attend(q.double().numpy(), k, v, pool.cu.numpy(), pool.len.numpy(), pool.table.numpy(), ps, 0.1)
        got, w = dense(q.double(), torch.tensor(k), torch.tensor(v), pool, 0.1)
        assert np.isnan(want).any() and not np.isnan(want).all()
        assert np.allclose(got.numpy(), want, rtol=1e-12, atol=1e-14, equal_nan=True)
        assert np.allclose(np.where(np.isnan(weight), 0, w.numpy()), np.nan_to_num(weight), rtol=1e-12, atol=1e-14)


def form(pool_T, B, Hq, Hkv, keys):
    """(form, 16-row tiles a wave, waves of the join a row) for sequences of up to ``keys`` keys."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    G = Hq // Hkv
    rows = -(-pool_T * G // B)

    def shift(most_rows, most):
        return max(s for s in range(most + 1) if s == 0 or (1 << s) * G <= most_rows)

    if rows >= 64 and ((pool_T >> shift(128, 7)) + B) * Hkv >= cus:
        return "prompts", 0, 0
    NT = 1 if rows <= 16 and G <= 16 else 2
    if keys <= 1024:
        return "tiles", NT, 0
    tm = shift(16 * NT, 6)
    tiles = ((pool_T >> tm) + B) * Hkv
    return "shares", NT, 1 if tiles * min(1 << tm, -(-pool_T // B)) * G >= 8 * cus else 4


def form_of(pool, Hq):
    return form(pool.T, len(pool.len), Hq, pool.k.shape[1], pool.table.shape[1] * pool.ps)


# ---- prompts ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,ps", [(64, 16), (128, 32), (64, 64), (128, 64), (64, 128), (128, 128)])
def test_prompts_with_holes_and_nan(mga, dev, dtype, D, ps):
    """Missing pages, NaN that some rows see, garbage behind the sequences' ends."""
    new, cached = [900, 40, 700, 633], [0, 77, 190, 3]
    pool = Pool(dev, new, cached, 8, D, ps, seed=6, scales=(-6, 0))
    t0 = pool.table.cpu()
    pool.v[t0[0, 130 // ps], 0, 3, 130 % ps] = 0x7f    # position 130: the later rows of the first sequence
    pool.v[t0[0, 899 // ps], 7, D - 1, 899 % ps] = 0xff
    pool.k[t0[2, 400 // ps], 5, 400 % ps, 5] = 0xff    # a key of the third
    for b in range(4):                                  # behind the ends
        end = new[b] + cached[b]
        if end % ps:
            pool.v[t0[b, end // ps], :, :, end % ps:] = 0x7f
            pool.k[t0[b, end // ps], :, end % ps:] = 0xff
    pool.table[3, 100 // ps] = -1
    pool.table[2, 0] = pool.n
    assert form_of(pool, 16) == ("prompts", 0, 0)
    q = queries(pool, 16, D, dtype, dev, extra=2)
    got = attend(mga, pool, q)
    want = check_attention(got, q, pool, D ** -0.5)
    nan = np.isnan(want)
    assert nan[130:900, 0:2, 3].all() and not nan[:130].any() and nan[899, 14, D - 1] and not nan[898, 14, D - 1]
    assert nan[940 + 210:940 + 700, 10].all() and not nan[940 + 700:].any()
    assert not got[pool.T:].any()
    pool.table[3, :] = -1
    assert not attend(mga, pool, q)[1640:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
def test_prompts_over_pages_never_written(mga, dev, dtype, ps, monkeypatch):
    """Anything in the scales of pages that hold no token, and of page 0 where a page is missing."""
    new, cached = [1000, 1000], [33, 300]
    assert form(2000, 2, 16, 8, 1400) == ("prompts", 0, 0)
    monkeypatch.setattr(base, "check_attention", check_attention)
    base.test_attention_of_pages_never_written(mga, dev, dtype, ps, 16, new, cached)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_of_small_queries(mga, dev, dtype, monkeypatch):
    assert form(2200, 2, 16, 4, 3000) == ("prompts", 0, 0)
    monkeypatch.setattr(base, "check_attention", check_attention)
    base.test_attention_small_queries(mga, dev, dtype, [1500, 700], [300, 0])


@pytest.mark.gpu
def test_prompts_in_place(mga, dev):
    assert form(2300, 2, 16, 8, 3000) == ("prompts", 0, 0)
    base.test_attention_in_place(mga, dev, [1300, 1000], [90, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D,ps", [(8, 8, 64, 64), (64, 8, 128, 16), (33, 3, 64, 32), (64, 2, 64, 128)])
def test_prompts_of_head_groups(mga, dev, dtype, Hq, Hkv, D, ps):
    """Groups of 1, 8, 11 (tiles of 8 tokens in 88 of 128 rows) and 32 query heads, rows behind the last sequence."""
    new, cached = {(8, 8): ([700, 1, 1600, 300, 1500], [0, 60, 500, 77, 0]), (64, 8): ([300, 1, 250], [0, 60, 500]),
                   (33, 3): ([500, 2, 700], [0, 60, 100]), (64, 2): ([200, 350], [100, 0])}[Hq, Hkv]
    pool = Pool(dev, new, cached, Hkv, D, ps, seed=3)
    assert form_of(pool, Hq) == ("prompts", 0, 0)
    q = queries(pool, Hq, D, dtype, dev, extra=3)
    got = attend(mga, pool, q)
    assert not got[pool.T:].any()
    check_attention(got, q, pool, D ** -0.5)


# ---- equal shares ----------------------------------------------------------------------

SHARES = [([1, 1, 1], [3000, 20, 1500], 1, 4),                       # a token each
          ([1] * 70, [(37 * i) % 1900 for i in range(70)], 1, 1),
          ([2, 3, 0, 1], [1999, 0, 70, 2500], 1, 4),
          ([5, 5, 9], [2000, 64, 1200], 2, 4),                       # drafts
          ([5] * 24, [(97 * i) % 1800 for i in range(24)], 2, 1),
          ([40], [2900], 2, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("case", range(len(SHARES)))
def test_shares(mga, dev, dtype, D, ps, case):
    new, cached, NT, waves = SHARES[case]
    Hkv = 8 if waves == 1 else 2
    pool = Pool(dev, new, cached, Hkv, D, ps, seed=case, width=3300 // ps)
    assert form_of(pool, 4 * Hkv) == ("shares", NT, waves)
    q = queries(pool, 4 * Hkv, D, dtype, dev)
    check_attention(attend(mga, pool, q), q, pool, D ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps", [32, 64])
@pytest.mark.parametrize("new", [[1, 1, 1], [9, 12, 10]])
def test_shares_of_many_steps(mga, dev, dtype, ps, new):
    """Heads of 128: 48 times the same three sequences, so that every wave visits more steps than it holds pages for."""
    pool = Pool(dev, new, [10000, 6999, 9990], 8, 128, ps, seed=2, scales=(-7, -3))
    n, T = 48, sum(new)
    q = queries(pool, 16, 128, dtype, dev)
    cu = torch.tensor([0] + new * n, device=dev).cumsum(0).int()
    assert form(n * T, 3 * n, 16, 8, 10000)[:2] == ("shares", 1 if max(new) == 1 else 2)
    got = mga.paged_attention(q.repeat(n, 1, 1), pool.pages, pool.table.repeat(n, 1), cu, pool.len.repeat(n), 128 ** -0.5)
    got = got.view(n, T, 16, 128)
    for x in (got.amin(0), got.amax(0)):
        check_attention(x, q, pool, 128 ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps", [16, 64])
@pytest.mark.parametrize("new,cached", [([3, 2], [1400, 1100]), ([12, 9], [1300, 1100])])
def test_shares_with_holes_and_nan(mga, dev, dtype, ps, new, cached):
    """Heads of 128: missing pages and NaN in tiles of which several waves take a part."""
    pool = Pool(dev, new, cached, 2, 128, ps, seed=6, scales=(-6, -2))
    t0 = pool.table.cpu()
    last = cached[0] + new[0] - 2                      # seen by the first sequence's last two rows
    pool.v[t0[0, last // ps], 1, 3, last % ps] = 0x7f
    pool.k[t0[1, (cached[1] + 1) // ps], 0, (cached[1] + 1) % ps, 5] = 0xff
    for b in range(2):
        end = new[b] + cached[b]
        if end % ps:
            pool.v[t0[b, end // ps], :, :, end % ps:] = 0x7f
            pool.k[t0[b, end // ps], :, end % ps:] = 0xff
    pool.table[1, 700 // ps] = -1
    pool.table[0, 256 // ps] = pool.n
    assert form_of(pool, 8)[:2] == ("shares", 1 if max(new) < 9 else 2)
    q = queries(pool, 8, 128, dtype, dev)
    want = check_attention(attend(mga, pool, q), q, pool, 128 ** -0.5)
    nan = np.isnan(want)
    assert nan[new[0] - 2:new[0], 4:, 3].all() and not nan[:new[0] - 2].any() and nan[new[0] + 1:, :4].all()
    assert not nan[:new[0], :4].any() and not nan[new[0]].any()


# ---- probabilities in two parts ---------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,cached,width,want", [([1, 1], [20, 30], 2, ("tiles", 1)), ([9, 12], [20, 30], 2, ("tiles", 2)),
                                                   ([1, 1], [20, 30], 40, ("shares", 1)),
                                                   ([9, 12], [20, 30], 40, ("shares", 2))])
def test_bf16_probabilities_in_two_parts(mga, dev, D, new, cached, width, want, monkeypatch):
    """Over a streamed cache bf16 queries' probabilities are held to 16 bits: small sums of large terms are
    as exact as that. Scores of ordinary size, so that fp32's own error is below one part's."""
    monkeypatch.setitem(PARTS, torch.bfloat16, 2)
    for seed in range(4):
        pool = Pool(dev, new, cached, 2, D, 64, seed=seed, width=width, scales=(-8, -7))
        pool.k.copy_(torch.where((pool.k & 0x7f) > 0x38, pool.k & 0xbf, pool.k))   # magnitudes below 2
        assert form_of(pool, 8)[:2] == want
        q = queries(pool, 8, D, torch.bfloat16, dev, seed=seed)
        check_attention(attend(mga, pool, q, scale=8.0), q, pool, 8.0)


# ---- the adapter with gated projections ----------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_adapter_hands_the_gate_to_the_projections(mga, dev, dtype):
    """qwen3_attention_forward over the paged cache with the reference's projections (forward_qkv_proj and
    o_proj take gate_mask): what they give, appended and attended."""
    T, Hq, Hkv, D, hidden = 9, 4, 2, 64, 256

    def proj(n_in, n_out):
        m = mga.GatedLoRALinear(torch.nn.Linear(n_in, n_out, bias=False), 8, 16, 0.0, False, False)
        torch.nn.init.normal_(m.lora_B.weight, std=0.05)
        return m.to(device=dev, dtype=dtype).eval()

    qp, kp, vp, op = proj(hidden, Hq * D), proj(hidden, Hkv * D), proj(hidden, Hkv * D), proj(Hq * D, hidden)
    norm = lambda: types.SimpleNamespace(weight=torch.rand(D, device=dev).to(dtype) + 0.5, variance_epsilon=1e-6)   # noqa: E731
    module = types.SimpleNamespace(head_dim=D, layer_idx=0, sliding_window=None, scaling=D ** -0.5, q_norm=norm(), k_norm=norm(),
                                   forward_qkv_proj=lambda x, gate: (qp(x, gate), kp(x, gate), vp(x, gate)), o_proj=op)
    x = torch.randn(1, T, hidden, device=dev).to(dtype)
    cos, sin = torch.randn(2, 1, T, D, device=dev).to(dtype)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)   # noqa: E731
    table, cu, lengths = i(0, 1, 2, 3).view(2, 2), i(0, 4, T), i(0, 0)
    outs = []
    with torch.no_grad():
        for gate in (torch.tensor([1, 0, 1, 1, 0, 0, 1, 0, 1], device=dev).view(1, T, 1), torch.zeros(1, T, 1, device=dev), None):
            caches = [mga.PagedKVCache(4, 1, Hkv, D, page_size=16, device=dev) for _ in range(2)]
            caches[0].begin(table, cu, lengths)
            got, none = mga.qwen3_attention_forward(module, x, (cos, sin), None, gate, past_key_value=caches[0])
            assert none is None
            pages = caches[1].pages(0)
            q, k, v = (t.view(T, -1, D) for t in module.forward_qkv_proj(x, gate))
            q = mga.paged_append(k, v, pages, table, cu, lengths, query=q, cos=cos[0], sin=sin[0], q_weight=module.q_norm.weight,
                                 k_weight=module.k_norm.weight)
            o = mga.paged_attention(q, pages, table, cu, lengths, D ** -0.5).view(1, T, -1)
            assert torch.equal(got, op(o) if gate is None else op(o, gate))
            for a, b in zip(caches[0].pages(0), pages):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            outs.append(got)
    assert not torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], outs[2])
