"""Keys stored in the paged 8-bit cache have the code nearest to their value, and their page the
least scale, however near the value lies to the middle between two codes or to 448 times a
power of two.

A key is prepared in fp64: its error is (D + 16) 2^-53 of |x cos| + |x sin| (the sum of squares,
root, reciprocal, products and the rotation), so that a code may be the other one only
within that of a middle. Where the products are exact in 53 bits there is no error at all."""
import numpy as np
import pytest
import torch

from oracle import paged as po
from test_gpu_paged import DTYPES, Pool, TABLE, check_append, rows, tables

pytestmark = pytest.mark.gpu

STEPS = [-1.2, -0.9, -0.7, -0.5, -0.3, -0.1, 0.0, 0.1, 0.3, 0.5, 0.7, 0.9, 1.2]   # fp32 steps from the middle


def f64(t):
    return t.double().cpu().numpy()


def append(mga, dev, k, cos, sin, new, ps=16):
    """One head's keys [T, 1, D] as ``new`` tokens for each sequence, each in its page 0; codes' values
    and scales of each token, and that they are what the definition gives for the exact key."""
    T, _, D = k.shape
    pool = Pool(dev, new, [0] * len(new), 1, D, ps, seed=1)
    before = pool.clone()
    mga.paged_append(k, torch.zeros_like(k), pool.pages, *pool.batch, cos=cos, sin=sin)
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore"):
        exact = po.prepared(f64(k), cos=f64(cos), sin=f64(sin))
    check_append(before, pool, exact, np.zeros(k.shape), np.zeros(k.shape), np.zeros(k.shape))
    return pool, exact


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tokens", [1, 13])      # of a sequence: a wave a page, a workgroup a page
def test_keys_beside_the_middle_of_two_codes(mga, dev, dtype, D, tokens):
    """k cos - k' sin with cos = 1, k' = 1 and k a middle: sin is the distance from it."""
    v = np.sort(TABLE[:127])
    mid = ((v[1:] + v[:-1]) / 2)[1:]                     # of neighbours, from 1.5 2^-9 on
    half = D // 2
    mid = np.resize(np.concatenate([mid, -mid]), -(-2 * len(mid) // (half - 1)) * (half - 1)).reshape(-1, half - 1)
    T = len(mid) * len(STEPS)
    k, sin = np.ones((T, 1, D)), np.zeros((T, D))
    k[:, 0, 0] = 448                                     # with a scale of 1
    k[:, 0, 1:half] = np.repeat(mid, len(STEPS), 0)
    sin[:, 1:half] = np.tile(STEPS, len(mid))[:, None] * np.spacing(np.abs(k[:, 0, 1:half]).astype(np.float32))
    k = torch.tensor(k, dtype=dtype, device=dev)
    sin = torch.tensor(sin, dtype=torch.float32, device=dev)
    assert np.array_equal(np.abs(f64(k)[:, 0, 1:half]), np.abs(np.repeat(mid, len(STEPS), 0)))   # of few bits
    append(mga, dev, k, torch.ones_like(sin), sin, [tokens] * (T // tokens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 13])
def test_scales_beside_their_limit(mga, dev, dtype, tokens):
    """The page's largest key beside 448 times a power of two: the least scale that holds it."""
    D, powers = 64, [-20, -3, 0, 1, 7]
    T = len(powers) * len(STEPS) * tokens
    k, sin = np.zeros((T, 1, D)), np.zeros((T, D))
    top = np.repeat(448 * 2.0 ** np.array(powers), len(STEPS))
    by = np.tile(STEPS, len(powers)) * np.spacing(top.astype(np.float32))
    k[::tokens, 0, 5], k[::tokens, 0, 5 + D // 2] = top, 2.0 ** -12
    sin[::tokens, 5] = by * 2.0 ** 12
    k = torch.tensor(k, dtype=dtype, device=dev)
    sin = torch.tensor(sin, dtype=torch.float32, device=dev)
    append(mga, dev, k, torch.ones_like(sin), sin, [tokens] * (T // tokens))


@pytest.mark.parametrize("tokens", [1, 13])
def test_finite_keys_past_fp32(mga, dev, tokens):
    """A key that is finite in fp64 is not NaN: past 448 times the largest scale it has the largest code."""
    D, big = 64, float(torch.finfo(torch.float32).max)
    k = torch.full((13, 1, D), 1.0, device=dev)
    k[:, 0, :8] = torch.tensor([big, -big, big, big, 1e38, 3e38, -2e38, big], device=dev)
    cos, sin = torch.ones(13, D, device=dev), torch.zeros(13, D, device=dev)
    cos[:, :8] = torch.tensor([2.0, 2.0, 1.0, 1 + 2.0 ** -23, 1.5, 3.0, 1e10, 1e30], device=dev)
    pool, exact = append(mga, dev, k, cos, sin, [tokens] * (13 // tokens))
    assert np.isfinite(exact).all() and np.abs(exact).max() > big
    # and so is what an infinity or a NaN was not part of
    k[0, 0, 0] = float("inf")
    append(mga, dev, k, cos, sin, [tokens] * (13 // tokens))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,norm,new,cached", [(128, True, [700, 60], [37, 0]), (64, True, [1] * 300, list(range(300))),
                                               (64, False, [300, 300], [5, 100]), (128, False, [3] * 90, [20] * 90)])
def test_keys_to_fp64(mga, dev, dtype, D, norm, new, cached):
    eps = 2.0 ** -20
    pool = Pool(dev, new, cached, 4, D, 32, seed=3, scales=(-14, -9))
    before = pool.clone()
    k, v = rows(pool.T, 4, D, dtype, dev, 1), rows(pool.T, 4, D, dtype, dev, 2)
    w = (1 + 0.3 * torch.randn(D, device=dev)).to(dtype) if norm else None
    cos, sin = tables(pool.T, D, torch.float32, dev)
    mga.paged_append(k, v, pool.pages, *pool.batch, cos=cos, sin=sin, k_weight=w, eps=eps)
    torch.cuda.synchronize()
    y = po.prepared(f64(k), None if w is None else f64(w), eps=eps)
    turned = np.concatenate([y[..., D // 2:], y[..., :D // 2]], -1)
    e = (np.abs(y * f64(cos)[:, None]) + np.abs(turned * f64(sin)[:, None])) * (D + 16) * 2.0 ** -53
    exact = po.prepared(f64(k), None if w is None else f64(w), f64(cos), f64(sin), eps)
    check_append(before, pool, exact, f64(v), e, np.zeros(v.shape))
