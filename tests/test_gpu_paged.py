"""The paged 8-bit cache on the GPU against the float64 oracle (oracle/paged.py).

Appending. A value is computed in fp32 within ``e`` of the exact one and then rounded to
the nearest code, which is monotone: the code lies between the roundings of exact - e and
exact + e, under a scale that lies between those of the page's largest value less and plus
its e. e: a product and an fma for the rotation, 2^-24 of |x cos| + |x sin| each, doubled
for the order of the operations; with a norm (D + 8) 2^-24 more for the sum of squares,
the square root, the reciprocal and two products. Rows from before are rounded from whole
codes: equal. Query rows: one rounding, eps / 2, beside e.

Attention. With p the exact probabilities, |got - want| <= (ep + es) sum p |v| + eps / 2
|want|: ep the rounding of P, 2^-8 for one bf16 part, 2^-16 for two, 2^-24 for three; es
the error of fp32 scores and of their exponentials, 2 (D + 16) 2^-24 max |q| |k| scale
(log2 e, the offset and the product behind it are within those 16) + 2^-20, and n 2^-24
for the sums over n keys."""
import numpy as np
import pytest
import torch

from oracle import paged as po

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
E4M3 = torch.float8_e4m3fn
TABLE = po.e4m3_table()


def values(codes):
    return TABLE[codes.contiguous().view(torch.uint8).cpu().numpy().astype(np.int64)]


class Pool:
    """Pages of random codes, and a batch of sequences on them."""

    def __init__(self, dev, new, cached, Hkv, D, ps, seed=0, spare=2, width=None, scales=(-9, -3)):
        g = torch.Generator(device=dev).manual_seed(seed)
        need = [max(1, -(-(n + c) // ps)) for n, c in zip(new, cached)]
        n = sum(need) + spare
        code = lambda shape: torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.uint8)   # noqa: E731
        self.k, self.v = code((n, Hkv, ps, D)), code((n, Hkv, D, ps))
        for t in (self.k, self.v):   # no NaN, and magnitudes up to 2^6
            t.copy_(torch.where((t & 0x7f) > 0x68, t & 0x87, t))
        e = lambda: torch.randint(*scales, (n, Hkv), generator=g, device=dev)   # noqa: E731
        self.ks, self.vs = torch.exp2(e().float()), torch.exp2(e().float())
        order = torch.randperm(n, generator=g, device=dev).tolist()
        w = width or max(need)
        rows, at = [], 0
        for c in need:
            rows.append(order[at:at + c] + [-1] * (w - c))
            at += c
        self.table = torch.tensor(rows, dtype=torch.int32, device=dev)
        self.cu = torch.tensor(np.cumsum([0] + list(new)), dtype=torch.int32, device=dev)
        self.len = torch.tensor(cached, dtype=torch.int32, device=dev)
        self.ps, self.n, self.T = ps, n, sum(new)

    @property
    def pages(self):
        return self.k.view(E4M3), self.v.view(E4M3), self.ks, self.vs

    @property
    def batch(self):
        return self.table, self.cu, self.len

    def clone(self):
        c = object.__new__(Pool)
        c.__dict__ = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in self.__dict__.items()}
        return c

    def kv(self):
        """Values [page, Hkv, row, D] of keys and values."""
        s = lambda t: t.double().cpu().numpy()[..., None, None]   # noqa: E731
        return values(self.k) * s(self.ks), values(self.v.transpose(2, 3)) * s(self.vs)


# ---- attention ------------------------------------------------------------------------

PARTS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}


def check_attention(got, q, pool, scale):
    k, v = pool.kv()
    cu, lens, table = pool.cu.cpu().numpy(), pool.len.cpu().numpy(), pool.table.cpu().numpy()
    qd = q.double().cpu().numpy()
    want, weight = po.attend(qd, k, v, cu, lens, table, pool.ps, scale)
    D, n = q.shape[2], int((lens + np.diff(cu)).max())
    kmax = np.nanmax(np.sqrt((k * k).sum(-1)))
    qmax = np.sqrt((qd * qd).sum(-1)).max()
    es = 2 * (D + 16) * 2.0 ** -24 * qmax * kmax * scale + 2.0 ** -20 + n * 2.0 ** -24
    ep = 2.0 ** (-8 * PARTS[q.dtype])
    bound = (ep + es) * weight + torch.finfo(q.dtype).eps / 2 * np.abs(want) + torch.finfo(q.dtype).tiny
    g = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(g), np.isnan(want))
    err = np.where(np.isnan(want), 0, np.abs(g - want))
    assert (err <= np.where(np.isnan(bound), np.inf, bound)).all(), f"{np.nanmax(err / bound)} of the bound"
    return want


def queries(pool, Hq, D, dtype, dev, seed=5, extra=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(pool.T + extra, Hq, D, generator=g, device=dev) * 1.5).to(dtype)


def attend(mga, pool, q, scale=None, **kw):
    got = mga.paged_attention(q, pool.pages, *pool.batch, scale or q.shape[2] ** -0.5, **kw)
    torch.cuda.synchronize()
    return got


BATCHES = [([1], [0]), ([1], [1]), ([1], [63]), ([1], [64]), ([1], [200]), ([3], [126]), ([1, 1, 1], [5, 0, 130]),
           ([5, 1, 0, 9], [64, 300, 20, 0]), ([40], [0]), ([17, 2, 33], [15, 256, 1])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
def test_attention_batches(mga, dev, dtype, Hq, Hkv, D, ps):
    for i, (new, cached) in enumerate(BATCHES):
        print(f"case {new} {cached} {ps} {dtype}", flush=True)
        pool = Pool(dev, new, cached, Hkv, D, ps, seed=i)
        q = queries(pool, Hq, D, dtype, dev)
        check_attention(attend(mga, pool, q), q, pool, D ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D", [(3, 3, 64), (14, 2, 64), (5, 1, 128), (16, 1, 64), (24, 1, 128), (32, 1, 64), (2, 1, 128)])
def test_attention_head_groups(mga, dev, dtype, Hq, Hkv, D):
    for new, cached in [([1, 2], [70, 0]), ([9, 20], [100, 3]), ([70], [31])]:
        print(f"case {Hq} {Hkv} {D} {new} {dtype}", flush=True)
        pool = Pool(dev, new, cached, Hkv, D, 64, seed=Hq)
        q = queries(pool, Hq, D, dtype, dev)
        check_attention(attend(mga, pool, q), q, pool, D ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,cached", [([300], [0]), ([130, 1, 64], [500, 900, 64]), ([1, 1], [5000, 9]), ([2] * 70, [33] * 70)])
def test_attention_long(mga, dev, dtype, new, cached):
    pool = Pool(dev, new, cached, 1, 64, 64, seed=3)
    q = queries(pool, 2, 64, dtype, dev)
    check_attention(attend(mga, pool, q), q, pool, 0.125)


PROMPTS = [([700, 30, 500, 1, 333], [0, 77, 190, 400, 3]), ([1, 129, 64, 900, 65, 200], [1000, 0, 63, 64, 500, 1])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D,ps", [(16, 8, 64, 64), (32, 8, 128, 64), (32, 8, 64, 16), (24, 8, 128, 128), (40, 8, 64, 32)])
def test_attention_prompts(mga, dev, dtype, Hq, Hkv, D, ps):
    """Batches of prompts, with sequences of few tokens among them."""
    for i, (new, cached) in enumerate(PROMPTS):
        print(f"case {new} {cached} {Hq} {Hkv} {D} {ps} {dtype}", flush=True)
        pool = Pool(dev, new, cached, Hkv, D, ps, seed=i)
        q = queries(pool, Hq, D, dtype, dev, extra=3)
        got = attend(mga, pool, q)
        assert not got[pool.T:].any()
        check_attention(got, q, pool, D ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,ps", [(64, 64), (128, 16), (64, 128)])
def test_attention_prompts_with_holes_and_nan(mga, dev, dtype, D, ps):
    """Missing pages, NaN that some rows see, wide scores, in batches of prompts."""
    pool = Pool(dev, [700, 30, 500, 333], [0, 77, 190, 3], 8, D, ps, seed=6, scales=(-6, 0))
    t0 = pool.table.cpu()
    pool.v[t0[0, 130 // ps], 0, 3, 130 % ps] = 0x7f    # position 130: the later rows of the first sequence
    pool.v[t0[0, 699 // ps], 7, D - 1, 699 % ps] = 0xff
    pool.k[t0[2, 400 // ps], 5, 400 % ps, 5] = 0xff    # a key of the third
    pool.v[t0[1, 106 // ps], :, :, 107 % ps:] = 0x7f   # behind the second one's end
    pool.table[3, 100 // ps] = -1
    pool.table[2, 0] = pool.n
    q = queries(pool, 16, D, dtype, dev)
    got = attend(mga, pool, q)
    want = check_attention(got, q, pool, D ** -0.5)
    nan = np.isnan(want)
    assert nan[130:700, 0:2, 3].all() and not nan[:130].any() and nan[699, 14, D - 1] and not nan[698, 14, D - 1]
    pool.table[3, :] = -1
    assert not attend(mga, pool, q)[1230:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
def test_attention_many_long_sequences(mga, dev, dtype, ps):
    """Sequences that share their pages, of so many keys that every wave visits more steps than
    it holds pages for at once: 48 times the same three."""
    pool = Pool(dev, [1, 1, 1], [10000, 6999, 9990], 8, 64, ps, seed=2, scales=(-6, -2))
    q = queries(pool, 16, 64, dtype, dev)
    n = 48
    one = torch.arange(3 * n + 1, dtype=torch.int32, device=dev)
    got = mga.paged_attention(q.repeat(n, 1, 1), pool.pages, pool.table.repeat(n, 1), one, pool.len.repeat(n), 0.125)
    got = got.view(n, 3, 16, 64)
    for x in (got.amin(0), got.amax(0)):
        check_attention(x, q, pool, 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
def test_attention_prompts_behind_long_sequences(mga, dev, dtype, ps):
    """Prompts that visit more steps than the lanes hold pages for at once."""
    pool = Pool(dev, [1000, 900, 200], [4200, 100, 8300], 8, 64, ps, seed=2)
    q = queries(pool, 16, 64, dtype, dev)
    got = attend(mga, pool, q)
    for i in (0, 1, 2):   # the oracle for some rows of each: as sequences of their own
        first, n, c = int(pool.cu[i]), [1000, 900, 200][i], [4200, 100, 8300][i]
        at = torch.tensor([0, 1, 63, 64, n // 2, n - 2, n - 1], device=dev)
        some = pool.clone()
        some.table = pool.table[i:i + 1].repeat(7, 1)
        some.cu, some.len, some.T = torch.arange(8, dtype=torch.int32, device=dev), (c + at).int(), 7
        check_attention(got[first + at], q[first + at], some, 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_many_sequences(mga, dev, dtype):
    """More sequences than threads of a workgroup, some without tokens."""
    new = [i % 3 for i in range(700)]
    cached = [(i * 37) % 90 for i in range(700)]
    pool = Pool(dev, new, cached, 1, 64, 16, seed=9)
    q = queries(pool, 1, 64, dtype, dev)
    check_attention(attend(mga, pool, q), q, pool, 0.125)


@pytest.mark.parametrize("width", [None, 80])
def test_most_sequences(mga, dev, width):
    """4096 sequences, a third of them without tokens, appended to and attended over, in tiles and in
    shares; one more is refused."""
    new = [(0, 1, 2)[i % 3] for i in range(4096)]
    cached = [(i * 29) % 70 for i in range(4096)]
    pool = Pool(dev, new, cached, 1, 64, 16, seed=3, width=width)
    x, y = rows(pool.T, 1, 64, torch.bfloat16, dev, 1), rows(pool.T, 1, 64, torch.bfloat16, dev, 2)
    run_append(mga, pool, None, x, y)
    q = queries(pool, 2, 64, torch.bfloat16, dev)
    check_attention(attend(mga, pool, q), q, pool, 0.125)
    with pytest.raises(RuntimeError, match="4096"):
        mga.paged_attention(q, pool.pages, torch.cat([pool.table, pool.table[:1]]), torch.cat([pool.cu, pool.cu[-1:]]),
                            torch.cat([pool.len, pool.len[:1]]), 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_missing_pages(mga, dev, dtype):
    """Pages outside the cache are masked; a row with nothing else is zeros."""
    pool = Pool(dev, [2, 1, 3, 1], [100, 40, 0, 200], 2, 64, 32, seed=4)
    pool.table[0, 1] = -1
    pool.table[1, :] = 1 << 30
    pool.table[2, 0] = pool.n
    pool.table[3, 0] = -(1 << 31)
    q = queries(pool, 4, 64, dtype, dev)
    got = attend(mga, pool, q)
    check_attention(got, q, pool, 0.125)
    assert not got[2:6].any()
    # a table too narrow for its sequence
    pool.table = pool.table[:, :1].contiguous()
    check_attention(attend(mga, pool, q), q, pool, 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_nan_reaches_only_who_sees_it(mga, dev, dtype):
    pool = Pool(dev, [6, 20, 1], [60, 0, 70], 1, 64, 64, seed=6)
    t0 = pool.table.cpu()
    pool.v[t0[0, 0], 0, 3, 62] = 0x7f          # position 62: rows 2 .. 5 of the first sequence
    pool.k[t0[1, 0], 0, 7, 5] = 0xff           # position 7 of the second
    pool.v[t0[1, 0], 0, 60, 12] = 0xff         # position 12
    pool.v[t0[2, 1], 0, :, 7:] = 0x7f          # behind the third sequence's end
    pool.k[t0[2, 1], 0, 7:] = 0x7f
    q = queries(pool, 2, 64, dtype, dev)
    got = attend(mga, pool, q)
    want = check_attention(got, q, pool, 0.125)
    nan = np.isnan(want).any(-1).any(-1)
    assert nan.tolist() == [False] * 2 + [True] * 4 + [False] * 7 + [True] * 13 + [False]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
@pytest.mark.parametrize("Hq,new,cached", [(4, [1, 3], [70, 5]), (8, [5, 2], [1300, 17]), (16, [700, 900], [33, 500])])
def test_attention_of_pages_never_written(mga, dev, dtype, ps, Hq, new, cached):
    """Scales of pages that hold no token are anything, wherever the table names them; so are page
    0's where a page is missing."""
    Hkv = Hq // 2
    pool = Pool(dev, new, cached, Hkv, 64, ps, seed=4, spare=6, width=-(-1400 // ps) + 3)
    pool.table[1, 0] = -1
    q = queries(pool, Hq, 64, dtype, dev)
    want = attend(mga, pool, q)
    check_attention(want, q, pool, 0.125)
    used = torch.zeros(pool.n + 1, dtype=torch.bool, device=dev)
    used[pool.table.long()] = True      # -1: the last, which is none
    free = (~used[:-1]).nonzero().flatten()
    assert len(free) >= 6
    move = free[0].item()
    if used[0]:   # page 0 is to be one of them
        for t in (pool.k, pool.v, pool.ks, pool.vs):
            t[move] = t[0].clone()
        pool.table[pool.table == 0] = move
        free[0] = 0
    bad = torch.tensor([float("nan"), float("inf"), -1.0, 0.0, 3e38, float("nan")], device=dev)
    bad[0] = float("nan")
    for t in (pool.ks, pool.vs):
        t[free] = bad[torch.arange(len(free), device=dev) % 6][:, None]
    for b in range(2):                  # behind the tokens' pages
        n = -(-(new[b] + cached[b]) // ps)
        tail = pool.table.shape[1] - n
        pool.table[b, n:] = free[torch.arange(tail, device=dev) % len(free)].int()
    assert torch.equal(attend(mga, pool, q), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_wide_scores(mga, dev, dtype):
    """Scores hundreds of units apart, rising and falling along the sequence, and queries of
    zeros, infinity and NaN."""
    pool = Pool(dev, [4], [400], 1, 64, 64, seed=8, scales=(-4, 2))
    q = queries(pool, 2, 64, dtype, dev) * 3
    check_attention(attend(mga, pool, q), q, pool, 0.125)
    q[0] = 0
    got = attend(mga, pool, q)
    check_attention(got, q, pool, 0.125)
    q[1, 0, 5], q[2, 1, 7] = float("nan"), float("inf")
    bad = attend(mga, pool, q)
    assert torch.isnan(bad[1, 0]).all() and torch.isnan(bad[2, 1]).all()
    for t, h in ((0, 0), (0, 1), (1, 1), (2, 0), (3, 0), (3, 1)):
        assert torch.equal(bad[t, h], got[t, h])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,cached", [([4, 1], [90, 10]), ([4, 1], [1500, 10]), ([400, 900], [500, 0])])
def test_attention_small_queries(mga, dev, dtype, new, cached):
    """Queries below fp16's normal range, whose products with the keys are of ordinary size."""
    pool = Pool(dev, new, cached, 4, 64, 32, seed=8, scales=(-3, 3))
    q = (queries(pool, 16, 64, dtype, dev).float() * 2.0 ** -17).to(dtype)
    got = attend(mga, pool, q, scale=2.0 ** 11)
    check_attention(got, q, pool, 2.0 ** 11)
    assert (got[0].float() - got[0].float().mean(0)).abs().max() > 0.1   # the heads differ: the queries count


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_behind_the_last_sequence(mga, dev, dtype):
    pool = Pool(dev, [2, 3], [10, 70], 2, 64, 64)
    q = queries(pool, 4, 64, dtype, dev, extra=4)
    got = attend(mga, pool, q)
    assert not got[5:].any()
    check_attention(got[:5], q[:5], pool, 0.125)
    out = torch.full_like(got, 7)
    attend(mga, pool, q, out=out)
    assert torch.equal(out[:5], got[:5]) and (out[5:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_strides(mga, dev, dtype):
    pool = Pool(dev, [3, 4], [90, 10], 2, 64, 32, width=9)
    q = queries(pool, 4, 64, dtype, dev)
    want = attend(mga, pool, q)
    wide = torch.zeros(7, 12, 64, dtype=dtype, device=dev)
    wide[:, 8:] = q
    forms = [wide[:, 8:], q.transpose(0, 1).contiguous().transpose(0, 1), q.transpose(1, 2).contiguous().transpose(1, 2)]
    odd = torch.zeros(7 * 4 * 65 + 1, dtype=dtype, device=dev)[1:].view(7, 4, 65)[:, :, :64]
    odd.copy_(q)
    for x in forms + [odd]:
        assert torch.equal(attend(mga, pool, x), want)
        out = torch.zeros(4, 7, 64, dtype=dtype, device=dev).transpose(0, 1)
        assert attend(mga, pool, x, out=out) is out and torch.equal(out, want)
    table = torch.full((2, 20), -1, dtype=torch.int32, device=dev)[:, 3:12]
    table.copy_(pool.table)
    pool.table = table
    assert torch.equal(attend(mga, pool, q), want)
    one = attend(mga, pool, q[:1].expand(7, 4, 64))   # a stride of 0
    assert torch.equal(one, attend(mga, pool, q[:1].expand(7, 4, 64).contiguous()))


def test_attention_repeats_bit_for_bit(mga, dev):
    pool = Pool(dev, [3, 1, 70], [3000, 20, 900], 2, 128, 64)
    q = queries(pool, 8, 128, torch.bfloat16, dev)
    first = attend(mga, pool, q)
    for _ in range(3):
        assert torch.equal(attend(mga, pool, q), first)


def test_attention_of_a_cache_past_2_31_bytes(mga, dev):
    """Pages past 2^31 and 2^32 bytes: the same codes give the same output."""
    Hkv, D, ps, n = 8, 128, 64, 70000      # 65536 bytes a page: 4.6 GB each
    small = Pool(dev, [2], [190], Hkv, D, ps, spare=0)
    k = torch.zeros(n, Hkv, ps, D, dtype=torch.uint8, device=dev)
    v = torch.zeros(n, Hkv, D, ps, dtype=torch.uint8, device=dev)
    ks, vs = torch.ones(n, Hkv, device=dev), torch.ones(n, Hkv, device=dev)
    at = torch.tensor([69999, 40000, 33000], device=dev)
    order = small.table[0].long()
    k[at], v[at], ks[at], vs[at] = small.k[order], small.v[order], small.ks[order], small.vs[order]
    q = queries(small, 32, D, torch.bfloat16, dev)
    got = mga.paged_attention(q, (k.view(E4M3), v.view(E4M3), ks, vs), at.int()[None], small.cu, small.len, D ** -0.5)
    assert torch.equal(got, attend(mga, small, q))
    # and appending there
    x = torch.randn(2, Hkv, D, device=dev).bfloat16()
    mga.paged_append(x, x, (k.view(E4M3), v.view(E4M3), ks, vs), at.int()[None], small.cu, small.len)
    mga.paged_append(x, x, small.pages, *small.batch)
    assert torch.equal(k[at], small.k[order]) and torch.equal(v[at], small.v[order]) and torch.equal(ks[at], small.ks[order])
    assert not k[69998].any() and not k[0].any()


# ---- appending -------------------------------------------------------------------------

def check_append(before, after, x_k, x_v, e_k, e_v):
    """x_*: exact rows [T, Hkv, D], e_* their fp32 errors."""
    cu, lens, table = before.cu.cpu().numpy(), before.len.cpu().numpy(), before.table.cpu().numpy()
    T = len(x_k)
    for x, e, was, now, s0, s1 in ((x_k, e_k, before.k, after.k, before.ks, after.ks),
                                   (x_v, e_v, before.v.transpose(2, 3), after.v.transpose(2, 3), before.vs, after.vs)):
        was8, now8 = (t.contiguous().cpu().numpy() for t in (was, now))
        s0, s1 = s0.double().cpu().numpy(), s1.double().cpu().numpy()
        rows = {}
        for t, b, pos, page, row in po.places(cu, lens, table, before.ps, before.n, T):
            if page is not None:
                rows.setdefault(page, []).append((row, t))
        for page in range(before.n):
            if page not in rows:
                assert np.array_equal(was8[page], now8[page]) and np.array_equal(s0[page], s1[page])
                continue
            r = [a for a, _ in rows[page]]
            t = [a for _, a in rows[page]]
            fin = np.isfinite(x[t])
            mag = np.where(fin, np.abs(x[t]), 0)
            err = np.where(fin, e[t], 0)
            lo, hi = (po.scale_of(np.maximum(mag + sign * err, 0).max((0, 2))) for sign in (-1, 1))
            old = s0[page] if min(r) else 0
            s = s1[page]
            assert (s >= np.maximum(lo, old)).all() and (s <= np.maximum(hi, old)).all()
            kept = [i for i in range(min(r))]
            if kept:
                again = po.round_e4m3(TABLE[was8[page][:, kept]] * (s0[page] / s)[:, None, None])
                assert np.array_equal(TABLE[now8[page][:, kept]], again, equal_nan=True)
            behind = [i for i in range(max(r) + 1, before.ps)]
            assert np.array_equal(was8[page][:, behind], now8[page][:, behind])
            got = TABLE[now8[page][:, r]].transpose(1, 0, 2)
            exact, within = x[t] / s[:, None], np.where(fin, e[t], 0) / s[:, None]
            assert np.array_equal(np.isnan(got), ~fin)
            ok = (got >= po.round_e4m3(exact - within)) & (got <= po.round_e4m3(exact + within))
            assert (ok | ~fin).all()


def run_append(mga, pool, q, k, v, qw=None, kw=None, cos=None, sin=None, eps=1e-6):
    before = pool.clone()
    got = mga.paged_append(k, v, pool.pages, *pool.batch, query=q, cos=cos, sin=sin, q_weight=qw, k_weight=kw, eps=eps)
    torch.cuda.synchronize()
    f = lambda t: None if t is None else t.double().cpu().numpy()   # noqa: E731
    D = k.shape[2]

    def error(x, w):
        y = po.prepared(x, w, eps=eps)
        rel = 2.0 ** -24 * ((D + 8 if w is not None else 0) + (4 if cos is not None else 0))
        if cos is None:
            return np.abs(y) * rel
        turned = np.concatenate([y[..., D // 2:], y[..., :D // 2]], -1)
        return (np.abs(y * f(cos)[:, None]) + np.abs(turned * f(sin)[:, None])) * rel

    with np.errstate(all="ignore"):
        x = po.prepared(f(k), f(kw), f(cos), f(sin), eps)
        check_append(before, pool, x, f(v), error(f(k), f(kw)), np.zeros(v.shape))
    if q is None:
        assert got is None
        return None
    live = min(int(pool.cu[-1]), len(q))
    want = po.prepared(f(q), f(qw), f(cos), f(sin), eps)
    e = error(f(q), f(qw))
    g = f(got)
    half = torch.finfo(q.dtype).eps / 2
    assert (np.abs(g - want)[:live] <= (e + half * (np.abs(want) + e) + torch.finfo(q.dtype).tiny)[:live]).all()
    assert not g[live:].any()
    return got


def rows(T, H, D, dtype, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(T, H, D, generator=g, device=dev) * torch.exp(torch.randn(H, D, generator=g, device=dev))).to(dtype)


def tables(T, D, dtype, dev):
    a = torch.arange(T, device=dev)[:, None] * 1.7 + torch.arange(D, device=dev)[None] * 0.3   # halves that differ, too
    return torch.cos(a).to(dtype), torch.sin(a).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("ps", [16, 32, 64, 128])
def test_append_batches(mga, dev, dtype, Hq, Hkv, D, ps):
    for i, (new, cached) in enumerate(BATCHES + [([300, 1], [7, 127]), ([256], [128])]):
        print(f"case {new} {cached} {ps} {dtype}", flush=True)
        pool = Pool(dev, new, cached, Hkv, D, ps, seed=i)
        T = pool.T
        q, k, v = rows(T, Hq, D, dtype, dev, i), rows(T, Hkv, D, dtype, dev, i + 50), rows(T, Hkv, D, dtype, dev, i + 90)
        w = (1 + 0.3 * torch.randn(2, D, device=dev)).to(dtype)
        cos, sin = tables(T, D, dtype if i % 2 else torch.float32, dev)
        if i % 3 == 0:
            run_append(mga, pool, q, k, v, w[0], w[1], cos, sin)
        elif i % 3 == 1:
            run_append(mga, pool, q, k, v, cos=cos, sin=sin)
        else:
            run_append(mga, pool, None, k, v, kw=w[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_append_few_tokens_on_average(mga, dev, dtype, D):
    """Batches of few tokens a sequence, with sequences of many or none, and many sequences."""
    many = [i % 3 for i in range(200)]
    for i, (new, cached) in enumerate([([30, 1, 1, 1, 1, 1, 1], [7, 64, 15, 0, 31, 100, 3]), (many, [(i * 29) % 70 for i in range(200)]),
                                       ([0, 0, 9, 0], [3, 16, 40, 0]), ([0, 1] * 40, [47] * 80)]):
        for ps in (16, 64):
            pool = Pool(dev, new, cached, 2, D, ps, seed=i, scales=(-14, -9))   # scales that have to grow
            T = pool.T
            q, k, v = (rows(T, h, D, dtype, dev, h + i) for h in (4, 2, 2))
            cos, sin = tables(T, D, dtype, dev)
            run_append(mga, pool, q, k, v, kw=(1 + 0.3 * torch.randn(D, device=dev)).to(dtype), cos=cos, sin=sin)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_token_by_token(mga, dev, dtype):
    """A scale that grows, stays, and begins anew with a page."""
    pool = Pool(dev, [1], [39], 1, 64, 16, seed=2, scales=(-14, -12))
    factor = [1e-4, 1.0, 1e-3, 30.0, 1e-2, 0.0, 1000.0, 1e-5, 1.0, 20000.0]
    pool.len[0] = 29
    for i, f in enumerate(factor):
        k, v = rows(1, 1, 64, dtype, dev, i) * f, rows(1, 1, 64, dtype, dev, i + 20) * f
        run_append(mga, pool, None, k.to(dtype), v.to(dtype))
        pool.len += 1


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_ends_of_the_types(mga, dev, dtype):
    big = torch.finfo(dtype).max
    for fill in ([big, -big, 1.0, 0.0], [float("inf"), 1.0, float("nan"), -2.0], [float("nan")] * 4, [0.0] * 4,
                 [-float("inf")] * 4, [448.0, 448.0, -448.0, 1.0], [torch.finfo(dtype).tiny, 0.0, -0.0, 1e-30]):
        for cached in (0, 5):
            pool = Pool(dev, [2], [cached], 1, 64, 16, seed=3)
            x = torch.tensor(fill, device=dev).repeat(32).view(2, 1, 64).to(dtype)
            run_append(mga, pool, None, x, x.flip(0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_strides_and_padding(mga, dev, dtype):
    """q, k, v as parts of one projection's rows, unaligned, expanded; rows behind the last
    sequence; pages that are not there."""
    T, Hq, Hkv, D = 9, 4, 2, 64
    base = Pool(dev, [3, 4], [30, 14], Hkv, D, 16, seed=5)
    base.T = T
    x = rows(T, Hq + 2 * Hkv, D, dtype, dev, 1)
    cos, sin = tables(T, D, dtype, dev)
    parts = x.split([Hq, Hkv, Hkv], 1)
    plain = base.clone()
    want = run_append(mga, plain, *(t.contiguous() for t in parts), cos=cos, sin=sin)
    buf = torch.zeros(T * (Hq + 2 * Hkv) * (D + 1) + 1, dtype=dtype, device=dev)[1:].view(T, -1, D + 1)[:, :, :D]
    buf.copy_(x)
    both = torch.zeros(T, 2, D + 3, dtype=dtype, device=dev)[:, :, 1:D + 1]
    both.copy_(torch.stack([cos, sin], 1))
    for given, c, s in ((parts, cos, sin), (buf.split([Hq, Hkv, Hkv], 1), cos, sin), (parts, both[:, 0], both[:, 1]),
                        ([t.transpose(1, 2).contiguous().transpose(1, 2) for t in parts], cos, sin)):
        pool = base.clone()
        got = run_append(mga, pool, *given, cos=c, sin=s)
        assert torch.equal(got, want) and torch.equal(pool.k, plain.k) and torch.equal(pool.v, plain.v)
    pool = base.clone()
    one = parts[1][:1].expand(T, Hkv, D)
    run_append(mga, pool, None, one, one)
    pool = base.clone()
    pool.table[0, 2], pool.table[1, 0] = -1, pool.n
    run_append(mga, pool, *parts, cos=cos, sin=sin)
    narrow = base.clone()
    narrow.table = narrow.table[:, :1].contiguous()
    run_append(mga, narrow, *parts, cos=cos, sin=sin)


def test_bookkeeping_out_of_range_stays_in_bounds(mga, dev):
    """Whatever cu_tokens and lengths hold, only the batch's pages and rows are touched."""
    for cu, lens in (([0, 5, 2], [10, 3]), ([-4, 2, 90], [0, 1]), ([0, 2, 4], [-7, 1 << 30]), ([3, 3, 3], [5, 5])):
        pool = Pool(dev, [2, 2], [40, 20], 1, 64, 16, seed=7)
        listed = set(pool.table.flatten().tolist())
        before = pool.clone()
        pool.cu, pool.len = (torch.tensor(t, dtype=torch.int32, device=dev) for t in (cu, lens))
        x = rows(4, 1, 64, torch.bfloat16, dev, 1)
        mga.paged_append(x, x, pool.pages, *pool.batch, query=x)
        out = attend(mga, pool, x)
        assert out.shape == x.shape
        for page in set(range(pool.n)) - listed:
            assert torch.equal(pool.k[page], before.k[page]) and torch.equal(pool.v[page], before.v[page])


# ---- forms, refusals -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
def test_native_and_python_forms(mga, dev, dtype, monkeypatch):
    base = Pool(dev, [5, 0, 20], [100, 4, 0], 2, 128, 32)
    T = base.T
    q, k, v = (rows(T, h, 128, dtype, dev, h) for h in (6, 2, 2))
    cos, sin = tables(T, 128, dtype, dev)
    w = (1 + 0.3 * torch.randn(2, 128, device=dev)).to(dtype)
    runs = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(mga._lib, "native", lambda *a: None)
        pool = base.clone()
        versions = [t._version for t in pool.pages]
        e = mga.paged_append(k, v, pool.pages, *pool.batch, query=q, cos=cos, sin=sin, q_weight=w[0], k_weight=w[1])
        assert mga.paged_append(k, v, pool.pages, *pool.batch) is None
        runs.append((e, attend(mga, pool, e), pool.k, pool.v, pool.ks, pool.vs))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("new,cached", [([3, 2], [90, 10]), ([3, 1], [3000, 700]), ([700, 900], [90, 0])])
def test_attention_in_place(mga, dev, new, cached):
    """out may be the query, or lie beside it in the rows of one buffer."""
    pool = Pool(dev, new, cached, 8, 64, 64, scales=(-6, -2))
    wide = torch.zeros(pool.T, 40, 64, dtype=torch.bfloat16, device=dev)
    wide[:, :16] = q = queries(pool, 16, 64, torch.bfloat16, dev)
    want = attend(mga, pool, q)
    assert torch.equal(attend(mga, pool, wide[:, :16], out=wide[:, 16:32]), want)
    assert torch.equal(wide[:, :16], q) and not wide[:, 32:].any()
    attend(mga, pool, q, out=q)
    assert torch.equal(q, want)
    with pytest.raises(RuntimeError, match="overlaps"):
        attend(mga, pool, wide[:, 8:24], out=wide[:, 16:32])


@pytest.mark.parametrize("native", [True, False])
def test_inference_mode(mga, dev, native, monkeypatch):
    if not native:
        monkeypatch.setattr(mga._lib, "native", lambda *a: None)
    with torch.inference_mode():
        pool = Pool(dev, [2, 3], [10, 20], 2, 64, 16)
        x, q = rows(5, 2, 64, torch.bfloat16, dev, 1), rows(5, 4, 64, torch.bfloat16, dev, 2)
        e = mga.paged_append(x, x, pool.pages, *pool.batch, query=q)
        assert attend(mga, pool, e).shape == q.shape
        logits = torch.randn(3, 50, device=dev)
        assert torch.equal(mga.adjust_logits(logits, torch.zeros(3, 1, dtype=torch.long, device=dev), presence=1.0, out=logits),
                           logits)


def test_refusals(mga, dev):
    pool = Pool(dev, [2], [10], 2, 64, 16)
    k, v, ks, vs = pool.pages
    x, q = rows(2, 2, 64, torch.bfloat16, dev, 1), rows(2, 4, 64, torch.bfloat16, dev, 2)
    cos, sin = tables(2, 64, torch.bfloat16, dev)
    app = lambda key=x, value=x, pages=pool.pages, batch=pool.batch, **kw: mga.paged_append(   # noqa: E731
        key, value, pages, *batch, **kw)
    att = lambda q=q, pages=pool.pages, batch=pool.batch, s=0.125, **kw: mga.paged_attention(   # noqa: E731
        q, pages, *batch, s, **kw)
    t, cu, ln = pool.batch
    for f in (app, att):
        with pytest.raises(ValueError, match="contiguous"):
            f(pages=(k.view(torch.uint8)[::2].view(E4M3), v, ks, vs))
        with pytest.raises(ValueError):
            f(pages=(k, k, ks, vs))
        with pytest.raises(ValueError):
            f(pages=(k, v, ks[:1], vs))
        with pytest.raises(TypeError):
            f(pages=(k.view(torch.uint8), v.view(torch.uint8), ks, vs))
        with pytest.raises(TypeError):
            f(pages=(k, v, ks.double(), vs))
        with pytest.raises(TypeError):
            f(batch=(t.long(), cu, ln))
        with pytest.raises(ValueError):
            f(batch=(t, cu[:1], ln))
        with pytest.raises(ValueError):
            f(batch=(t[0], cu, ln))
        with pytest.raises(ValueError):
            f(batch=(t[:, :0], cu, ln))
        with pytest.raises(RuntimeError, match="GPU"):
            f(batch=(t.cpu(), cu, ln))
    for kw in (dict(key=x[:, :1]), dict(value=x[:1]), dict(key=x[..., :32]), dict(key=x[0]), dict(query=q[:1]),
               dict(cos=cos), dict(cos=cos[:1], sin=sin), dict(q_weight=cos[0, :8], query=q), dict(k_weight=cos)):
        with pytest.raises(ValueError):
            app(**kw)
    for kw in (dict(key=x.double(), value=x.double()), dict(value=x.float()), dict(query=q.half()),
               dict(cos=cos.half(), sin=sin.half()), dict(cos=cos, sin=sin.float()), dict(k_weight=cos[0].float())):
        with pytest.raises(TypeError):
            app(**kw)
    for kw in (dict(q=q[:, :3]), dict(q=q[:, :0]), dict(q=q[0]), dict(q=q[..., :32]), dict(out=q[:1]), dict(out=q.float()),
               dict(out=torch.empty(2, 4, 72, device=dev, dtype=q.dtype)[..., 4:68])):
        with pytest.raises(ValueError):
            att(**kw)
    with pytest.raises(TypeError):
        att(q=q.double())
    for s in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(mga._lib.MGAError, match="scale"):
            att(s=s)
    with pytest.raises(mga._lib.MGAError, match="at most 32"):
        att(q=rows(2, 66, 64, torch.bfloat16, dev, 1))
    for f, a in ((app, x.clone().requires_grad_()), (att, q.clone().requires_grad_())):
        with pytest.raises(NotImplementedError, match="no_grad"):
            f(a)
        with torch.no_grad():
            f(a)
    with pytest.raises(ValueError, match="gradient"):
        att(out=torch.empty_like(q).requires_grad_())
    assert att(q=q[:0]).shape == (0, 4, 64) and app(key=x[:0], value=x[:0], query=q[:0]).shape == (0, 4, 64)
    with pytest.raises(RuntimeError, match="begin"):
        mga.PagedKVCache(4, 1, 2, 64).attend(0, q, 0.125)
