"""Token sampling on the GPU against the float64 oracle (oracle/vocab.py): equal
tokens. The oracle adds in extended precision; the kernel's sums are whole
multiples of 2^-45 of the largest weight, so the two differ only where u (or a
filter's border) lies within about 1e-11 of a border between tokens."""
import numpy as np
import pytest
import torch

from oracle import vocab as vo

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def logits(n, V, dtype, dev, seed=0, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + V)
    x = torch.randn(n, V, generator=g, device=dev) * spread
    at = torch.randint(V, (n, min(V, 50)), generator=g, device=dev)
    return x.scatter_add_(1, at, torch.rand(at.shape, generator=g, device=dev) * 8).to(dtype)


def uniform(n, dev, seed=0):
    return torch.rand(n, generator=torch.Generator(device=dev).manual_seed(seed), device=dev)


def check(mga, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    got = mga.sample_tokens(x, u, temperature, top_k, top_p, min_p)
    torch.cuda.synchronize()
    assert got.dtype == torch.int64 and got.shape == x.shape[:-1]
    n = u.numel()
    held = lambda v: np.broadcast_to(v.double().cpu().numpy().reshape(-1) if isinstance(v, torch.Tensor)   # noqa: E731
                                     else np.float64(np.float32(v)), (n,))
    t, k, p, m = held(temperature), held(top_k), held(top_p), held(min_p)
    rows, uu = x.double().cpu().numpy().reshape(n, -1), u.double().cpu().numpy().reshape(-1)
    want = [vo.sample_row(rows[i], uu[i], t[i], int(k[i]), p[i], m[i]) for i in range(n)]
    assert got.cpu().numpy().reshape(-1).tolist() == want
    return got


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=50, top_p=0.9), dict(temperature=1.3, top_p=0.95),
            dict(top_k=7), dict(min_p=0.05), dict(temperature=0.8, top_k=40, top_p=0.8, min_p=0.02), dict(top_k=2000),
            dict(top_k=1500, top_p=0.7), dict(top_p=0.5, min_p=0.1), dict(temperature=5.0, top_p=0.3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V", [(3, 1), (4, 7), (4, 64), (6, 1000), (4, 8193), (4, 32003), (3, 100003), (3, 151936),
                                 (2, 170001)])
def test_sizes_and_filters(mga, dev, dtype, n, V):
    x = logits(n, V, dtype, dev, seed=1)
    for i, s in enumerate(SETTINGS):
        print(f"case {n} {V} {dtype} {s}", flush=True)
        check(mga, x, uniform(n, dev, i), **s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_settings_of_each_row(mga, dev, dtype):
    n = 60
    x = logits(n, 3001, dtype, dev, seed=2)
    pick = torch.arange(n, device=dev)
    t = torch.tensor([0.0, 0.6, 1.0, 1.7], device=dev)[pick % 4]
    k = torch.tensor([0, 1, 3, 100, 5000], device=dev)[pick % 5]
    p = torch.tensor([1.0, 0.9, 0.4], device=dev)[pick % 3]
    m = torch.tensor([0.0, 0.01, 1.0], device=dev)[pick // 3 % 3]
    for kk in (k, k.int()):
        check(mga, x, uniform(n, dev, 3), t, kk, p, m)
    check(mga, x.reshape(5, 12, 3001), uniform(n, dev, 4).reshape(5, 12), t.reshape(5, 12), 0, p.reshape(5, 12))
    check(mga, x, uniform(n, dev, 5), t.double(), k, p[:1], m)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ends_of_the_uniform(mga, dev, dtype):
    """u at 0, next to 1, at and past its ends, NaN: the first and the last token of
    those that are left."""
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan"), 0.5], device=dev)
    x = logits(1, 9001, dtype, dev, seed=4).expand(7, 9001)
    for s in SETTINGS:
        print(f"case {dtype} {s}", flush=True)
        check(mga, x, u, **s)
    # the last columns are masked: u = 1 stops before them
    y = x.clone()
    y[:, 100:] = -float("inf")
    check(mga, y, u)
    check(mga, y, u, top_p=0.9)
    check(mga, y, u, top_k=3000)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_and_masked_values(mga, dev, dtype):
    V = 20011
    inf = float("inf")
    x = logits(8, V, dtype, dev, seed=5)
    x[0] = (x[0] * 0.25).round()
    x[1] = 2.0
    x[2] = -inf
    x[3, 3:] = -inf
    x[4] = float("nan")
    x[5, 4:] = float("nan")
    x[6, 7::11] = inf
    x[7, : V - 1] = -inf
    for i, s in enumerate(SETTINGS + [dict(top_k=64), dict(top_k=1024), dict(top_p=1e-6), dict(min_p=1.0),
                                      dict(temperature=1e-6), dict(temperature=1e-30), dict(temperature=1e30),
                                      dict(temperature=float("inf")), dict(min_p=1e-30)]):
        print(f"case {dtype} {s}", flush=True)
        check(mga, x, uniform(8, dev, 20 + i), **s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_far_from_zero(mga, dev, dtype):
    """Rows masked with the type's lowest value, all of them too, and rows whose
    largest logit is the type's largest."""
    V, low = 5003, torch.finfo(dtype).min
    x = logits(6, V, dtype, dev, seed=9)
    x[0] = low                              # nothing left: uniform
    x[1, :V // 2] = low
    x[2, 0::2] = low
    x[3] = low
    x[3, 77] = low / 2
    x[4, 1000::1000] = -low
    x[5] = low / 4 * (1 + torch.randint(0, 4, (V,), device=dev) / 4)
    for i, s in enumerate(SETTINGS):
        print(f"case {dtype} {s}", flush=True)
        check(mga, x, uniform(6, dev, i + 20), **s)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off", [0, 3])
def test_ties_at_the_threshold(mga, dev, dtype, off):
    """Rows of few values, of which a filter keeps a part of the last one's elements,
    more than are listed: those of the lowest columns, at the row's ends too."""
    V = 30011
    g = torch.Generator(device=dev).manual_seed(31)
    x = torch.randint(0, 3, (24, V + 8), generator=g, device=dev).to(dtype)[:, off:off + V]
    x[1] = 1.0
    u = torch.cat([uniform(20, dev, 32), torch.tensor([0.0, 0.999, 0.99999, 1.0], device=dev)])
    for s in (dict(top_k=15000), dict(top_k=29990), dict(top_k=4097), dict(top_p=0.95), dict(top_p=0.9999),
              dict(top_k=25000, top_p=0.99), dict(top_k=12000, min_p=0.3), dict(top_p=0.8, min_p=0.01)):
        print(f"case {dtype} {off} {s}", flush=True)
        check(mga, x, u, **s)


@pytest.mark.parametrize("dtype", DTYPES)
def test_whole_shares_of_equal_logits(mga, dev, dtype):
    """Half of an even number of equal largest logits is a whole number of them, at any
    value of theirs: top_p = 0.5 and u = 0.5 lie on borders between tokens, where only
    exact weights decide."""
    V = 12006
    for top in (1.0, 37.25, 150.5, 3e4, -2e4, torch.finfo(dtype).min / 4, torch.finfo(dtype).max):
        print(f"case {dtype} {top}", flush=True)
        x = torch.full((6, V), top, device=dev, dtype=dtype)
        x[1, ::2] = float("-inf")
        x[1, 0] = x[1, 1]
        x[1, 1] = float("-inf")
        x[2, 5000:] = float("-inf")
        x[3, 2::3] = torch.finfo(dtype).min if top > 0 else float("-inf")
        x[4, 100:] = float("-inf")
        x[5, 2:] = float("-inf")
        for s in (dict(top_p=0.5), dict(top_p=0.25), dict(top_p=0.5, temperature=0.3), dict(), dict(top_k=5000, top_p=0.5)):
            for u in (0.25, 0.5, 0.9999999):
                check(mga, x, torch.full((6,), u, device=dev), **s)


def test_borders(mga, dev):
    """Four equal tokens: half of their weight is two of them, just above is three;
    quarters of the uniform fall to the next token."""
    x = torch.full((1, 300), -float("inf"), device=dev)
    x[0, [5, 100, 200, 299]] = 1.25
    for p, n in ((0.25, 1), (0.5, 2), (0.5000001, 3), (0.75, 3), (0.9, 4)):
        hit = {int(check(mga, x, torch.tensor([u], device=dev), top_p=p)) for u in (0.0, 0.2, 0.4, 0.6, 0.8, 0.99)}
        assert hit <= {5, 100, 200, 299} and len(hit) == n
    for u, tok in ((0.0, 5), (0.25, 100), (0.5, 200), (0.75, 299), (0.7499999, 200)):
        assert int(check(mga, x, torch.tensor([u], device=dev))) == tok


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off", [1, 3, 8])
def test_strides(mga, dev, dtype, off):
    x = logits(6, 9001, dtype, dev, seed=off)
    u = uniform(6, dev, off)
    for s in SETTINGS[:6]:
        check(mga, x[:, off:off + 5003], u, **s)
        check(mga, x[:, ::2], u, **s)
        check(mga, x[::2], u[::2], **s)


def test_longest_row(mga, dev):
    for dtype in (torch.float16, torch.float32):
        x = logits(1, 1 << 20, dtype, dev, seed=7)
        for s in SETTINGS:
            print(f"case {dtype} {s}", flush=True)
            check(mga, x, uniform(1, dev, 8), **s)


def test_draws_follow_the_probabilities(mga, dev):
    """40 000 draws of 32 tokens, each count within 5 standard deviations."""
    n, V = 40000, 32
    x = logits(1, V, torch.float32, dev, seed=9)
    tok = mga.sample_tokens(x.expand(n, V), uniform(n, dev, 10), 1.5)
    p = torch.softmax(x[0].double() / 1.5, 0).cpu().numpy()
    c = np.bincount(tok.cpu().numpy(), minlength=V)
    assert (np.abs(c - n * p) <= 5 * np.sqrt(n * p * (1 - p)) + 1).all()


def test_refusals_and_empty(mga, dev):
    x, u = torch.randn(3, 50, device=dev), torch.rand(3, device=dev)
    assert mga.sample_tokens(x[:0], u[:0]).shape == (0,)
    assert mga.sample_tokens(x[0], u[0]).shape == ()
    with pytest.raises(TypeError):
        mga.sample_tokens(x, u.double())
    with pytest.raises(ValueError):
        mga.sample_tokens(x, u[:2])
    with pytest.raises(ValueError):
        mga.sample_tokens(x, u, torch.ones(2, device=dev))
    with pytest.raises(TypeError):
        mga.sample_tokens(x, u, 1.0, torch.ones(3, device=dev))
    with pytest.raises(TypeError):
        mga.sample_tokens(x, u, torch.ones(3, device=dev, dtype=torch.int64))
    with pytest.raises(TypeError):
        mga.sample_tokens(x.double(), u)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        mga.sample_tokens(x, u, torch.ones(3))
    with pytest.raises(ValueError, match="at most"):
        mga.sample_tokens(torch.zeros(1, (1 << 20) + 1, device=dev, dtype=torch.float16), u[:1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [8011, 30011])
def test_top_p_among_the_ties_of_top_k(mga, dev, dtype, V):
    """The border of top_k falls among equal logits, and top_p (below 1, yet so near it
    that the mass it needs is that of all of those elements, or of all but a few) leaves
    none of the others of that value in. 8 011 columns: no table for bf16 either."""
    g = torch.Generator(device=dev).manual_seed(41)
    x = torch.randint(0, 3, (6, V), generator=g, device=dev).to(dtype)
    x[0], x[1] = 1.0, -3.0
    x[2, ::2] = 5.0
    x[3, V // 3:] = -float("inf")
    u = torch.tensor([0.0, 0.3, 0.9, 0.999999, 0.99, 0.6], device=dev)
    for k in (1025, 2000, V // 2 + 7, V - 5):
        for p in (0.99, 0.9999, 0.99999994):
            for m in (0.0, 0.3):
                print(f"case {dtype} {V} {k} {p} {m}", flush=True)
                check(mga, x, u, top_k=k, top_p=p, min_p=m)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [300, 9001])
def test_infinity_beside_the_largest_number(mga, dev, dtype, V):
    """+inf alone is drawn, at any temperature, also where the type's largest number
    stands beside it."""
    x = logits(3, V, dtype, dev, seed=43)
    x[0, 3::5] = torch.finfo(dtype).max
    x[0, 7::50] = float("inf")
    x[1] = torch.finfo(dtype).max
    x[1, V - 2:] = float("inf")
    x[2, :] = float("inf")
    x[2, :5] = torch.finfo(dtype).max
    for s in SETTINGS + [dict(top_k=5, top_p=0.5), dict(top_p=0.75), dict(temperature=1e30, top_p=0.9)]:
        for t in (s.get("temperature", 1.0), float("inf")):
            for u in (0.0, 0.35, 0.999999):
                print(f"case {dtype} {V} {s} {t} {u}", flush=True)
                check(mga, x, torch.full((3,), u, device=dev), **dict(s, temperature=t))
    for m in (0.05, 1.0, 2.0):
        check(mga, x, torch.full((3,), 0.9, device=dev), float("inf"), 40, 1.0, m)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hole", [-float("inf"), float("nan")])
def test_top_k_among_logits_without_weight(mga, dev, dtype, hole):
    """The border of top_k falls among -inf or NaN: no logit is cut, the row's numbers
    may all be the type's lowest."""
    V, n = 32003, 20000
    g = torch.Generator(device=dev).manual_seed(47)
    x = torch.full((3, V), hole, device=dev, dtype=dtype)
    at = torch.randperm(V, generator=g, device=dev)[:n]
    x[0, at] = torch.finfo(dtype).min
    x[1, at] = torch.finfo(dtype).min
    x[1, at[::2]] = torch.finfo(dtype).min / 2
    x[2, at] = logits(1, n, dtype, dev, seed=48)[0]
    for u in (0.1, 0.5, 0.9, 0.999999):
        for s in (dict(top_k=25000), dict(top_k=n), dict(top_k=n + 1), dict(top_k=V - 1),
                  dict(top_k=25000, top_p=0.9999), dict(top_k=25000, min_p=0.5)):
            print(f"case {dtype} {hole} {u} {s}", flush=True)
            check(mga, x, torch.full((3,), u, device=dev), **s)
