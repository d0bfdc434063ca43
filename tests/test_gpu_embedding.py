"""Scaled embedding lookup and its gradient on the GPU against the float64 oracle
(oracle/vocab.py).

Tolerances. The lookup is one fp32 product and one rounding to the type:
eps / 2 relative (with 2^-23 for the product). A gradient row is a sum of n fp32
terms, each addition within 2^-24 of the sum of magnitudes so far: n 2^-24 times
the sum of |terms|, then the product with scale and one rounding."""
import numpy as np
import pytest
import torch

from oracle import vocab as vo

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def f64(t):
    return t.detach().double().cpu().numpy()


def table(V, H, dtype, dev, seed=0):
    return torch.randn(V, H, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(dtype)


def tokens(n, V, dev, seed=0, mask=0.5):
    """Half of them one token, in runs as in an MTP chunk; the rest spread."""
    g = torch.Generator(device=dev).manual_seed(seed + n)
    ids = torch.randint(V, (n,), generator=g, device=dev)
    runs = (torch.rand(n // 4 + 1, generator=g, device=dev) < mask).repeat_interleave(4)[:n]
    return torch.where(runs, V - 1, ids)


def close(got, want, bound, dtype):
    eps = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-38
    err = np.abs(f64(got) - want)
    assert (err <= eps * np.abs(want) * (1 + 1e-3) + bound + tiny).all(), float((err - bound).max())


def grad_bound(dy, ids, V, scale, pad=None):
    count = vo.embedding_grad(np.ones((len(ids), 1)), ids, V, 1.0, pad)
    return (count + 4) * 2.0 ** -24 * abs(scale) * vo.embedding_grad(np.abs(dy), ids, V, 1.0, pad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,H", [(1, 1, 1), (1, 5, 8), (7, 3, 5), (64, 10, 77), (65, 1000, 256), (130, 40, 1000),
                                   (1000, 17, 2560), (5120, 3001, 4096), (8192, 100, 64), (8193, 500, 40),
                                   (20000, 1024, 24), (17000, 1, 136)])
def test_lookup_and_gradient(mga, dev, dtype, n, V, H):
    print(f"case {n} {V} {H} {dtype}", flush=True)
    w = table(V, H, dtype, dev).requires_grad_()
    ids = tokens(n, V, dev)
    scale = [1.0, 16.0, 0.3][n % 3]
    out = mga.scaled_embedding(ids[None], w, scale)
    dy = table(n, H, dtype, dev, seed=1)[None]
    out.backward(dy)
    torch.cuda.synchronize()
    held = float(np.float32(scale))
    i = ids.cpu().numpy()
    close(out[0], vo.embedding(i, f64(w), held), np.float64(2.0 ** -23) * np.abs(f64(out[0])), dtype)
    close(w.grad, vo.embedding_grad(f64(dy[0]), i, V, held), grad_bound(f64(dy[0]), i, V, held), dtype)
    assert w.grad.shape == w.shape and w.grad.dtype == dtype
    again = mga.embedding_grad(dy, ids[None], V, scale)   # in a fixed order
    assert torch.equal(again, w.grad)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ids_outside_and_padding(mga, dev, dtype):
    V, H, n = 50, 72, 300
    w = table(V, H, dtype, dev).requires_grad_()
    ids = tokens(n, V, dev, seed=3)
    ids[::7], ids[1::7] = -1, V
    ids[2], ids[9] = 2 ** 31 - 1, -(2 ** 31)
    ids[16] = 2 ** 40 + 3
    i = ids.cpu().numpy()
    for t in (ids, ids.clamp(-(2 ** 31), 2 ** 31 - 1).int()):
        w.grad = None
        out = mga.scaled_embedding(t, w, 2.0, padding_idx=V - 1)
        dy = table(n, H, dtype, dev, seed=4)
        out.backward(dy)
        close(out, vo.embedding(t.cpu().numpy(), f64(w), 2.0), 0.0, dtype)
        close(w.grad, vo.embedding_grad(f64(dy), i, V, 2.0, V - 1), grad_bound(f64(dy), i, V, 2.0, V - 1), dtype)
        assert not w.grad[V - 1].any()
    none = mga.embedding_grad(dy, torch.full((n,), -1, device=dev), V)
    assert none.shape == (V, H) and not none.any()
    w.grad = None
    mga.scaled_embedding(ids, w, 2.0, padding_idx=-1).backward(dy)   # the last row, as torch counts
    assert not w.grad[V - 1].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", [64, 77])
def test_accumulate(mga, dev, dtype, H):
    """Chunks added into one buffer: touched rows only, in the gradients' type or
    fp32; rows without a token keep every bit, NaN among them."""
    V, n = 40, 500
    ids = [tokens(n, V - 10, dev, seed=s) + 5 for s in (1, 2)]
    dy = [table(n, H, dtype, dev, seed=s) for s in (3, 4)]
    for out_dtype in {dtype, torch.float32}:
        out = torch.full((V, H), float("nan"), device=dev, dtype=out_dtype)
        out[5:V - 5] = 0.25
        before = out.clone()
        want = np.where(np.isnan(f64(out)), np.nan, f64(out))
        bound = 0.0
        for i, d in zip(ids, dy):
            r = mga.embedding_grad(d, i, V, 0.5, out=out, accumulate=True)
            assert r is out
            want = want + vo.embedding_grad(f64(d), i.cpu().numpy(), V, 0.5)
            bound = bound + grad_bound(f64(d), i.cpu().numpy(), V, 0.5) \
                + torch.finfo(out_dtype).eps * (np.abs(np.nan_to_num(want)) + 1)
        touched = np.zeros(V, bool)
        touched[np.concatenate([i.cpu().numpy() for i in ids])] = True
        t = torch.tensor(touched, device=dev)
        close(out[t], want[touched], bound[touched], out_dtype)
        bits = torch.int32 if out_dtype == torch.float32 else torch.int16
        assert torch.equal(out[~t].view(bits), before[~t].view(bits))
    # fp32 sums of 16-bit gradients, everything written
    out = torch.full((V, H), float("nan"), device=dev)
    mga.embedding_grad(dy[0], ids[0], V, 1.0, out=out)
    close(out, vo.embedding_grad(f64(dy[0]), ids[0].cpu().numpy(), V, 1.0),
          grad_bound(f64(dy[0]), ids[0].cpu().numpy(), V, 1.0), torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(mga, dev, dtype):
    V, H, n = 60, 48, 200
    base = table(V, 2 * H + 1, dtype, dev)
    ids = tokens(2 * n, V, dev, seed=5)[::2]
    for w in (base[:, 1:H + 1], base[:, :H], base[:, ::2][:, :H], base.t()[:H].t()):
        w = w.detach().requires_grad_()
        out = mga.scaled_embedding(ids, w, 3.0)
        close(out, vo.embedding(ids.cpu().numpy(), f64(w), 3.0), 0.0, dtype)
        big = table(n, H + 3, dtype, dev, seed=6)
        for dy in (big[:, 3:], big[:, :H], big[:1, :H].expand(n, H), torch.ones((), device=dev, dtype=dtype).expand(n, H)):
            (g,) = torch.autograd.grad(out, w, dy, retain_graph=True)
            i = ids.cpu().numpy()
            close(g, vo.embedding_grad(f64(dy), i, V, 3.0), grad_bound(f64(dy), i, V, 3.0), dtype)
    out = torch.full((V, H + 5), 7.0, device=dev, dtype=dtype)
    view = out[:, 2:H + 2]
    mga.embedding_grad(big[:, :H], ids, V, 1.0, out=view)
    close(view, vo.embedding_grad(f64(big[:, :H]), ids.cpu().numpy(), V, 1.0),
          grad_bound(f64(big[:, :H]), ids.cpu().numpy(), V, 1.0), dtype)
    assert bool((out[:, :2] == 7).all()) and bool((out[:, H + 2:] == 7).all())


def test_no_tokens_and_refusals(mga, dev):
    w = table(10, 16, torch.float32, dev).requires_grad_()
    none = torch.zeros(2, 0, dtype=torch.long, device=dev)
    out = mga.scaled_embedding(none, w)
    assert out.shape == (2, 0, 16)
    out.sum().backward()
    assert w.grad.shape == w.shape and not w.grad.any()
    ids = torch.zeros(3, dtype=torch.long, device=dev)
    dy = torch.zeros(3, 16, device=dev)
    with pytest.raises(TypeError):
        mga.scaled_embedding(ids.float(), w)
    with pytest.raises(TypeError):
        mga.scaled_embedding(ids, w.double())
    with pytest.raises(ValueError):
        mga.scaled_embedding(ids, w[0])
    with pytest.raises(ValueError, match="padding_idx"):
        mga.scaled_embedding(ids, w, padding_idx=10)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        mga.scaled_embedding(ids.cpu(), w)
    with pytest.raises(ValueError):
        mga.embedding_grad(dy, ids[:2], 10)
    with pytest.raises(ValueError):
        mga.embedding_grad(dy, ids, 0)
    with pytest.raises(ValueError, match="accumulate"):
        mga.embedding_grad(dy, ids, 10, accumulate=True)
    with pytest.raises(ValueError):
        mga.embedding_grad(dy, ids, 10, out=torch.zeros(9, 16, device=dev))
    with pytest.raises(TypeError):
        mga.embedding_grad(dy, ids, 10, out=torch.zeros(10, 16, device=dev, dtype=torch.float16))
    with pytest.raises(ValueError):
        mga.embedding_grad(dy, ids, 10, out=torch.zeros(16, 10, device=dev).t())


def test_gradient_past_the_cache(mga, dev):
    """A table larger than the last-level cache, cleared past it."""
    V, H, n = 30011, 4096, 900
    ids = tokens(n, V, dev, seed=7)
    dy = table(n, H, torch.bfloat16, dev, seed=8)
    g = mga.embedding_grad(dy, ids, V, 1.0)
    rows = torch.unique(ids)
    want = vo.embedding_grad(f64(dy), np.searchsorted(rows.cpu().numpy(), ids.cpu().numpy()), len(rows), 1.0)
    bound = grad_bound(f64(dy), np.searchsorted(rows.cpu().numpy(), ids.cpu().numpy()), len(rows), 1.0)
    close(g[rows], want, bound, torch.bfloat16)
    g[rows] = 0
    assert not g.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,H", [(511, 5000, 3), (512, 9, 520), (513, 9, 520), (512, 1, 1), (300, 70000, 8),
                                   (40, 3, 70001), (1, 9000, 1), (200, 16500, 8192)])
def test_few_tokens(mga, dev, dtype, n, V, H):
    """About the number of tokens up to which one launch takes them all, with tables
    on both sides of the size to which it does; both types of ids, written into rows
    that lie apart, and added to, where rows without a token keep every bit."""
    print(f"case {n} {V} {H} {dtype}", flush=True)
    ids = tokens(n, V, dev, seed=9).int()
    ids[::11] = -1
    rows = torch.unique(ids[ids >= 0].long())
    i = np.where(ids.cpu().numpy() < 0, -1, np.searchsorted(rows.cpu().numpy(), ids.cpu().numpy()))
    dy = table(n, H, dtype, dev, seed=8)
    want, bound = vo.embedding_grad(f64(dy), i, len(rows), 2.0), grad_bound(f64(dy), i, len(rows), 2.0)
    buf = torch.full((V, H + 8), 7.0, device=dev, dtype=dtype)
    out = buf[:, :H]
    for given in (ids, ids.long()):
        out.fill_(float("nan"))
        mga.embedding_grad(dy, given, V, 2.0, out=out)
        close(out[rows], want, bound, dtype)
        assert bool((buf[:, H:] == 7).all())
        out[rows] = 0
        assert not out.any()
    out.fill_(float("nan"))
    out[rows] = 1.0
    mga.embedding_grad(dy, ids, V, 2.0, out=out, accumulate=True)
    close(out[rows], want + 1, bound + torch.finfo(dtype).eps * (np.abs(want) + 1), dtype)
    out[rows] = float("nan")
    assert bool(out.isnan().all())


def test_layer(mga, dev):
    base = torch.nn.Embedding(30, 24, padding_idx=3, device=dev)
    layer = mga.ScaledEmbedding.wrap(base, 4.0)
    ids = torch.randint(30, (2, 9), device=dev)
    a, b = layer(ids), base(ids) * 4.0
    assert torch.equal(a, b)
    (ga,) = torch.autograd.grad(a.square().sum(), layer.weight)
    (gb,) = torch.autograd.grad(b.square().sum(), base.weight)
    torch.testing.assert_close(ga, gb, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 700])
def test_gradients_of_one_column(mga, dev, dtype, n):
    """A table of one column: gradients whose last dimension carries a stride that is
    none (0 of an expanded one, a far one of a slice), of one token too."""
    V = 3
    w = table(V, 1, dtype, dev).requires_grad_()
    ids = torch.arange(n, device=dev) % 2
    i = ids.cpu().numpy()
    for t in (ids, ids[None], ids[:, None]):
        w.grad = None
        mga.scaled_embedding(t, w, 2.0).sum().backward()
        close(w.grad, vo.embedding_grad(np.ones((n, 1)), i, V, 2.0), 0.0, dtype)
    wide = table(n, 10, dtype, dev, seed=3)
    for dy in (wide[:, 3:4], wide[:, ::7][:, 1:], wide[:, :1], wide[:1, :1].expand(n, 1)):
        w.grad = None
        mga.scaled_embedding(ids, w, 2.0).backward(dy)
        close(w.grad, vo.embedding_grad(f64(dy), i, V, 2.0), grad_bound(f64(dy), i, V, 2.0), dtype)


def test_layer_of_a_frozen_model(mga, dev):
    """The hook by which a frozen model's inputs come to require gradients goes on
    working, and its handle removes it."""
    base = torch.nn.Embedding(30, 24, device=dev).requires_grad_(False)
    handle = base.register_forward_hook(lambda m, args, out: out.requires_grad_())
    layer = mga.ScaledEmbedding.wrap(base, 4.0)
    ids = torch.arange(30, device=dev)
    out = layer(ids)
    assert out.requires_grad and torch.equal(out, base.weight * 4.0)
    handle.remove()
    assert not layer(ids).requires_grad


def test_out_counts_as_written(mga, dev):
    """A graph that saved ``out`` before it was written refuses its backward."""
    ids, dy = torch.arange(4, device=dev), torch.ones(4, 8, device=dev)
    for accumulate in (False, True):
        out, w = torch.ones(6, 8, device=dev), torch.ones(6, 8, device=dev, requires_grad=True)
        y = (out * w).sum()
        mga.embedding_grad(dy, ids, 6, out=out, accumulate=accumulate)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    with torch.inference_mode():
        out = torch.zeros(6, 8, device=dev)
        mga.embedding_grad(dy, ids, 6, out=out)
    assert float(out.sum()) == 32
