"""A teacher's top logits and the cross-entropy against them on the GPU, against
the float64 oracle (oracle/vocab.py) on the same inputs.

Tolerances. Values and ids are equal. Sums of exponentials run over at most
V / 256 + 70 fp32 additions in a chain, each term within a few steps of 2^-24 of
its value (the exponent's argument, at most 60 where the term counts, times
2^-24): relative error d = (V / 256 + 200) 2^-24. A log-sum-exp is then within
d + 2^-22 |lse|, a row's loss within tau^2 (Q d + 2^-21 sum_k |terms|), and a
gradient element within |coef| d (Q p_j + sum q) of the exact one before its one
rounding (eps / 2 relative; half of fp16's smallest step, 2^-25, where it is
subnormal)."""
import numpy as np
import pytest
import torch

from oracle import vocab as vo

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def f64(t):
    return t.detach().double().cpu().numpy()


def logits(n, V, dtype, dev, seed=0, spread=2.0):
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + V)
    x = torch.randn(n, V, generator=g, device=dev) * spread
    at = torch.randint(V, (n, min(V, 50)), generator=g, device=dev)
    return x.scatter_add_(1, at, torch.rand(at.shape, generator=g, device=dev) * 10).to(dtype)


def chain(V):
    return (V / 256 + 200) * 2.0 ** -24


def check_top(mga, x, k, tau=1.0):
    got = mga.top_logits(x, k, temperature=tau)
    torch.cuda.synchronize()
    xr = f64(x).reshape(-1, x.shape[-1])
    values, ids, lse = vo.top_logits(xr, k, tau)
    assert got.values.dtype == x.dtype and got.ids.dtype == torch.int32 and got.lse.dtype == torch.float32
    assert got.values.shape == got.ids.shape == (*x.shape[:-1], k) and got.lse.shape == x.shape[:-1]
    assert np.array_equal(got.ids.cpu().numpy().reshape(-1, k), ids)
    assert np.array_equal(f64(got.values).reshape(-1, k), values, equal_nan=True)
    have = f64(got.lse).reshape(-1)
    fin = np.isfinite(lse)
    assert np.array_equal(have[~fin], lse[~fin], equal_nan=True)
    assert (np.abs(have[fin] - lse[fin]) <= chain(x.shape[-1]) + 2.0 ** -22 * np.abs(lse[fin])).all()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,k", [(1, 1, 1), (3, 7, 7), (2, 8, 3), (2, 64, 64), (5, 1000, 17), (3, 1024, 1024),
                                   (2, 4097, 300), (3, 32003, 20), (2, 40001, 257), (2, 100003, 64),
                                   (2, 151936, 64), (1, 170001, 1000), (1, 200704, 5)])
def test_sizes(mga, dev, dtype, n, V, k):
    print(f"case {n} {V} {k} {dtype}", flush=True)
    check_top(mga, logits(n, V, dtype, dev), k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_and_masked_values(mga, dev, dtype):
    """Rows of few distinct values, of one value, masked down to fewer than k, with
    infinities and NaN: more candidates than the list holds."""
    V, k = 20011, 64
    print(f"case {dtype}", flush=True)
    inf = float("inf")
    x = logits(9, V, dtype, dev, seed=3)
    x[0] = (x[0] * 0.25).round()            # some dozen values
    x[1] = 1.5                              # one
    x[2] = -inf                             # none
    x[3, 10:] = -inf                        # fewer than k
    x[4, 5:V - 3] = float("nan")            # NaN below them
    x[5] = float("nan")
    x[6, ::3] = inf
    x[7] = torch.where(torch.arange(V, device=dev) % 2 == 0, 0.0, -0.0).to(dtype)
    x[8, :] = -5.0
    x[8, V - 1] = -4.0
    for i in range(9):
        check_top(mga, x[i:i + 1], k)
    check_top(mga, x, 1)
    check_top(mga, x[:, :4999], 1024)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off", [1, 3, 8])
def test_strides(mga, dev, dtype, off):
    """Rows that begin off a 16-byte boundary, each at another offset, and columns
    that are not contiguous; the row behind the last is not read."""
    x = logits(5, 9001, dtype, dev, seed=off)
    check_top(mga, x[:, off:off + 5003], 9)
    check_top(mga, x[:, ::2], 9)
    check_top(mga, x[None, ::2], 5, tau=0.5)
    check_top(mga, x[:4].reshape(2, 2, 9001)[:, :, off:], 3, tau=3.0)
    check_top(mga, x[0].expand(3, 9001), 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_with_nan(mga, dev, dtype):
    """A NaN makes the log-sum-exp NaN, beside +inf too; +inf in the student's row makes
    loss and gradient NaN."""
    x = logits(4, 3001, dtype, dev, seed=21)
    x[0, 5], x[0, 9] = float("inf"), float("nan")
    x[1, 5:8] = float("inf")
    x[2, :] = float("inf")
    x[2, 7] = float("nan")
    t = check_top(mga, x, 4)
    assert t.lse.isnan().tolist() == [True, False, True, False]
    v = torch.zeros(4, 4, device=dev)
    for n in (1, 100):
        y, vals, ids = x[1:2].repeat(n, 1), v[:1].repeat(n, 1), t.ids[3:].repeat(n, 1)
        loss, g = mga.top_logits_loss_and_grad(y, vals, ids)
        ys = y.clone().requires_grad_()
        total = mga.top_logits_cross_entropy(ys, vals, ids)
        total.backward()
        assert bool(loss.isnan()) and bool(total.isnan()) and bool(g.isnan().all()) and bool(ys.grad.isnan().all())


def test_no_rows_and_refusals(mga, dev):
    x = torch.randn(2, 50, device=dev)
    r = mga.top_logits(x[:0], 4)
    assert r.values.shape == (0, 4) and r.lse.shape == (0,)
    for k in (0, -1, 51):
        with pytest.raises(ValueError, match="k must be"):
            mga.top_logits(x, k)
    with pytest.raises(ValueError, match="k must be"):
        mga.top_logits(torch.zeros(1, 3000, device=dev), 1025)
    with pytest.raises(ValueError, match="at most"):
        mga.top_logits(torch.zeros(1, (1 << 20) + 1, device=dev, dtype=torch.float16), 1)
    with pytest.raises(TypeError):
        mga.top_logits(x.double(), 3)
    with pytest.raises(ValueError):
        mga.top_logits(torch.zeros(3, 0, device=dev), 1)


# ---- the loss ------------------------------------------------------------------

def check_ce(mga, x, values, ids, lse=None, tau=1.0, go=0.375):
    V = x.shape[-1]
    xr = f64(x).reshape(-1, V)
    vr, ir = f64(values).reshape(len(xr), -1), ids.cpu().numpy().reshape(len(xr), -1)
    lr = None if lse is None else f64(lse).reshape(-1)
    want, grad = vo.top_ce(xr, vr, ir, lr, tau, go)
    q = vo.teacher_weights(vr, ir, V, lr, tau)
    Q = q.sum(1)
    xs = x.detach().clone().requires_grad_() if x.is_contiguous() else x.detach().requires_grad_()
    total = mga.top_logits_cross_entropy(xs, values, ids, lse, tau)
    (total * go).backward()
    total2, g2 = mga.top_logits_loss_and_grad(x, values, ids, lse, tau, scale=go)
    torch.cuda.synchronize()
    assert total.shape == total2.shape == () and g2.shape == x.shape and g2.dtype == x.dtype
    with np.errstate(invalid="ignore"):
        at = np.where((ir >= 0) & (ir < V), ir, 0)
        picked = np.take_along_axis(xr, at, 1) / tau
        norm = np.array([vo.logsumexp(r / tau) for r in xr])
        m = np.nanmax(np.where(np.isnan(xr), -np.inf, xr), 1) / tau
        size = q * (np.abs(m[:, None] - picked) + np.abs(norm - m)[:, None])
    tol = tau ** 2 * np.where(q > 0, chain(V) * q + 2.0 ** -21 * size, 0).sum()
    for t in (total, total2):
        if np.isfinite(want.sum()):
            bound = tol + 2.0 ** -22 * np.abs(want).sum() + 1e-30
            assert abs(float(t.detach()) - want.sum()) <= bound, (float(t), want.sum(), tol)
        else:
            assert float(t) == want.sum()
    eps = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-38
    with np.errstate(invalid="ignore", over="ignore"):
        p = np.where(norm[:, None] == -np.inf, 0.0, np.exp(xr / tau - norm[:, None]))
    tsum = np.zeros_like(grad)
    rows = np.repeat(np.arange(len(xr)), ir.shape[1])
    np.add.at(tsum, (rows, at.reshape(-1)), q.reshape(-1))
    slack = abs(go) * tau * chain(V) * (np.where(Q[:, None] > 0, Q[:, None] * p, 0) + tsum)
    for g in (xs.grad, g2):
        err = np.abs(f64(g).reshape(grad.shape) - grad)
        assert (err <= eps * np.abs(grad) * (1 + 1e-3) + slack + tiny).all(), float((err - slack).max())
    return total, xs.grad, g2


def teacher(mga, x, k, tau, seed=1):
    g = torch.Generator(device=x.device).manual_seed(seed)
    t = x.float() + torch.randn(x.shape, generator=g, device=x.device)
    return mga.top_logits(t.to(x.dtype), k, temperature=tau)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_lse", [True, False])
@pytest.mark.parametrize("n,V,k", [(1, 1, 1), (3, 7, 7), (4, 64, 9), (5, 1000, 33), (3, 8193, 64), (70, 4099, 5),
                                   (3, 32003, 300), (2, 151936, 64), (2, 170001, 8), (1030, 515, 16), (2, 2048, 1024)])
def test_loss_and_gradient(mga, dev, dtype, with_lse, n, V, k):
    print(f"case {n} {V} {k} {dtype} lse={with_lse}", flush=True)
    x = logits(n, V, dtype, dev, seed=5)
    tau = [1.0, 2.0, 0.5][V % 3]
    t = teacher(mga, x, k, tau)
    a = check_ce(mga, x[None], t.values[None], t.ids[None], t.lse[None] if with_lse else None, tau)
    b = check_ce(mga, x[None], t.values[None], t.ids[None], t.lse[None] if with_lse else None, tau)
    assert all(torch.equal(p, q) for p, q in zip(a, b))   # sums in a fixed order


@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_duplicates_and_masks(mga, dev, dtype):
    V, k = 5001, 8
    print(f"case {dtype}", flush=True)
    inf = float("inf")
    x = logits(9, V, dtype, dev, seed=6)
    t = teacher(mga, x, k, 1.0)
    ids, values, lse = t.ids.clone(), t.values.clone(), t.lse.clone()
    ids[0] = -1                             # a padded row, its logits NaN
    x[0] = float("nan")
    ids[1] = V                              # ids outside the row
    ids[2, 3:] = -7
    ids[3] = ids[3, :1]                     # one column k times
    values[4] = -inf                        # a teacher row masked out
    lse[4] = -inf
    values[5, 2:] = -inf
    x[5, ids[5, 4].long()] = -inf           # masked in both
    x[6, 0::2] = -inf                       # half the vocabulary masked
    ids[6] = (ids[6] | 1).clamp(max=V - 2)
    values[7, :] = values[7, 0]
    x[8] = torch.randn(V, device=dev).to(dtype) * 0.01 + (300 if dtype != torch.float16 else 200)   # far from zero
    check_ce(mga, x, values, ids)
    check_ce(mga, x, values, ids, lse)
    # a masked student logit that the teacher wants: infinite loss, finite gradient
    y = x[2:3].clone()
    y[0, ids[2, 0].long()] = -inf
    check_ce(mga, y, values[2:3], ids[2:3], lse[2:3])
    y[:] = -inf
    check_ce(mga, y, values[2:3], ids[2:3], lse[2:3])
    # NaN among the logits of a row that counts
    y = x[2:3].clone()
    y[0, 7] = float("nan")
    loss, g = mga.top_logits_loss_and_grad(y, values[2:3], ids[2:3])
    assert bool(loss.isnan()) and bool(g.isnan().all())
    assert bool(mga.top_logits_cross_entropy(y, values[2:3], ids[2:3]).isnan())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tau", [1.0, 4.0, 2.0 ** -20])
def test_rows_far_from_zero(mga, dev, dtype, tau):
    """Rows masked with the type's lowest value, all of them too, and rows of other
    values whose quotient by the temperature is far past fp32's whole numbers: the
    sums there are exact (equal elements count 1, others nothing)."""
    V, k = 5003, 6
    print(f"case {dtype} {tau}", flush=True)
    low = torch.finfo(dtype).min if tau >= 1 else max(torch.finfo(dtype).min, -1e30)
    x = logits(9, V, dtype, dev, seed=13)
    x[0] = low                              # nothing left: uniform
    x[1, :V // 2] = low                     # masked from the start,
    x[2, V // 2:] = low                     # to the end,
    x[3, 0::2] = low                        # and between
    x[4] = low
    x[4, 77] = low / 2
    x[5, 1000::1000] = -low                 # the largest value, five times
    x[6] = max(-1e12, low / 4) * (1 + torch.randint(0, 64, (V,), device=dev) * 2.0 ** -6)
    x[7] = 7e8 if dtype != torch.float16 else 6e4   # next to where counting begins (at tau = 1)
    x[7, 5::7] = float(x[7, 0]) * (1 + 2.0 ** -7)
    x[8] = -x[7]
    t = check_top(mga, x, k, tau)
    ids = t.ids.clone()
    ids[4, 1:] = -1
    ids[5, 5:] = -1
    values = torch.randn(9, k, device=dev).to(dtype) * min(tau, 1.0)
    for i in range(9):
        check_ce(mga, x[i:i + 1], values[i:i + 1], ids[i:i + 1], None, tau)
    check_ce(mga, x.repeat(12, 1), values.repeat(12, 1), ids.repeat(12, 1), None, tau)
    # NaN in such a row
    y = x[:1].clone()
    y[0, 7] = float("nan")
    for z in (y, y.repeat(100, 1)):
        loss, g = mga.top_logits_loss_and_grad(z, values[:1].expand(len(z), k), ids[:1].expand(len(z), k))
        assert bool(loss.isnan()) and bool(g.isnan().all())


@pytest.mark.parametrize("V", [5003, 170003])
def test_strides_and_types(mga, dev, V):
    """Student rows off a 16-byte boundary, columns that are not contiguous, strided
    teachers, int64 ids, values of another type than the student."""
    x = logits(6, V + 9, torch.bfloat16, dev, seed=8)
    t = teacher(mga, x[:, :V], 12, 1.0)
    wide = torch.zeros(6, 20, device=dev)
    wide[:, 3:15] = t.values.float()
    ids = torch.zeros(6, 30, device=dev, dtype=torch.int64)
    ids[:, 5:17] = t.ids
    check_ce(mga, x[:, 1:V + 1], wide[:, 3:15], ids[:, 5:17])
    check_ce(mga, x[:, 1:V + 1][::2], t.values.half()[::2], t.ids[::2], t.lse[::2])
    check_ce(mga, x[:, ::2][:, :V // 2], t.values, torch.where(t.ids < V // 2, t.ids, -1))
    check_ce(mga, x[:, :V].reshape(2, 3, V), t.values.reshape(2, 3, 12), t.ids.reshape(2, 3, 12))
    check_ce(mga, x[:4, :V].reshape(2, 2, V).transpose(0, 1), t.values[:4].reshape(2, 2, 12).transpose(0, 1),
             t.ids[:4].reshape(2, 2, 12).transpose(0, 1))


def test_gradient_by_differences(mga, dev):
    """fp32: central differences of the loss along random directions. The loss of 4
    rows of 64 is within 1e-6 relative, differences of 2e-2 then within 1e-3."""
    x = logits(4, 64, torch.float32, dev, seed=9)
    t = teacher(mga, x, 8, 1.0)
    _, g = mga.top_logits_loss_and_grad(x, t.values, t.ids, t.lse)
    gen = torch.Generator(device=dev).manual_seed(1)
    for _ in range(4):
        d = torch.randn(x.shape, generator=gen, device=dev) * 0.02
        num = mga.top_logits_cross_entropy(x + d, t.values, t.ids, t.lse) - \
            mga.top_logits_cross_entropy(x - d, t.values, t.ids, t.lse)
        # third order: |d|^3 / 6 summed over a row's softmax, below 1e-4 a row
        assert abs(float(num) / 2 - float((g * d).sum())) <= 1e-3


def test_all_logits_kept_is_the_soft_cross_entropy(mga, dev):
    x = logits(6, 1024, torch.float32, dev, seed=10)[None]
    t = logits(6, 1024, torch.float32, dev, seed=11)[None]
    top = mga.top_logits(t, 1024)
    a, b = (x.clone().requires_grad_() for _ in range(2))
    la = mga.top_logits_cross_entropy(a, top.values, top.ids, top.lse)
    lb = mga.StableSoftCrossEntropy.apply(b, t)
    la.backward()
    lb.backward()
    assert abs(float(la) - float(lb)) <= 1e-5 * float(lb)
    assert float((a.grad - b.grad).abs().max()) <= 4 * chain(1024)


def test_refusals_and_empty(mga, dev):
    x = torch.randn(3, 50, device=dev)
    v, i, lse = torch.randn(3, 4, device=dev), torch.zeros(3, 4, dtype=torch.int32, device=dev), torch.zeros(3, device=dev)
    for call in (mga.top_logits_cross_entropy, mga.top_logits_loss_and_grad):
        with pytest.raises(ValueError):
            call(x, v[:2], i)
        with pytest.raises(ValueError):
            call(x, v[:, :3], i)
        with pytest.raises(TypeError):
            call(x, v, i.float())
        with pytest.raises(TypeError):
            call(x, v.double(), i)
        with pytest.raises(TypeError):
            call(x.double(), v, i)
        with pytest.raises(ValueError):
            call(x, v, i, lse[:2])
        with pytest.raises(TypeError):
            call(x, v, i, lse.double())
        with pytest.raises(ValueError):
            call(x, v[:, :0], i[:, :0])
        with pytest.raises(ValueError):
            call(x, torch.zeros(3, 1025, device=dev), torch.zeros(3, 1025, dtype=torch.int64, device=dev))
        with pytest.raises(ValueError, match="temperature"):
            call(x, v, i, lse, 0.0)
    e = x[:0].requires_grad_()
    loss = mga.top_logits_cross_entropy(e, v[:0], i[:0])
    loss.backward()
    assert float(loss) == 0 and e.grad.shape == (0, 50)
    loss, g = mga.top_logits_loss_and_grad(x[:0], v[:0], i[:0])
    assert float(loss) == 0 and g.shape == (0, 50)


def test_gradient_past_the_cache(mga, dev):
    """More bytes than the last-level cache holds, and other kernels for fewer rows:
    a row's gradients on both sides are within half a step and the sums' slack of
    the exact one, so within eps |g| and twice the slack of each other."""
    V = 151936
    x = logits(700, V, torch.bfloat16, dev, seed=12)
    t = teacher(mga, x, 16, 1.0)
    xs = x.clone().requires_grad_()
    mga.top_logits_cross_entropy(xs, t.values, t.ids, t.lse).backward()
    _, g = mga.top_logits_loss_and_grad(x, t.values, t.ids, t.lse)
    for at in (0, 500):
        few = slice(at, at + 200)
        ys = x[few].clone().requires_grad_()
        mga.top_logits_cross_entropy(ys, t.values[few], t.ids[few], t.lse[few]).backward()
        _, h = mga.top_logits_loss_and_grad(x[few], t.values[few], t.ids[few], t.lse[few])
        kept = (t.values[few].float() - t.lse[few][:, None]).exp()
        q = torch.zeros(200, V, device=dev).scatter_(1, t.ids[few].long(), kept)
        slack = 2 * chain(V) * (torch.softmax(x[few].float(), -1) * q.sum(-1, keepdim=True) + q)
        for a, b in ((g[few], h), (xs.grad[few], ys.grad), (g[few], xs.grad[few])):
            d = (a.float() - b.float()).abs()
            assert bool((d <= 2.0 ** -7 * torch.maximum(a.abs(), b.abs()).float() + slack + 1e-30).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 100])
def test_student_rows_of_nan(mga, dev, dtype, n):
    """NaN in a row that counts gives NaN, for few rows and many: in a row of nothing
    else, beside -inf alone, and where the teacher wants a masked logit."""
    V, k = 3001, 4
    x = torch.full((3, V), float("nan"), device=dev, dtype=dtype)
    x[1, 5:] = -float("inf")
    x[2] = logits(1, V, dtype, dev, seed=31)[0]
    x[2, 1], x[2, 9] = float("nan"), -float("inf")
    ids = torch.full((3, k), 9, dtype=torch.int32, device=dev)
    values = torch.zeros(3, k, device=dev)
    for r in range(3):
        xs = x[r:r + 1].repeat(n, 1).requires_grad_()
        args = values[r:r + 1].repeat(n, 1), ids[r:r + 1].repeat(n, 1)
        loss, g = mga.top_logits_loss_and_grad(xs.detach(), *args)
        total = mga.top_logits_cross_entropy(xs, *args)
        total.backward()
        assert bool(loss.isnan()) and bool(total.isnan()), (r, float(loss), float(total.detach()))
        assert bool(g.isnan().all()) and bool(xs.grad.isnan().all()), r


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 100])
def test_quotients_by_the_temperature_past_fp32(mga, dev, dtype, n):
    """Teacher and student logits of the type's lowest value at temperature 1 / 2: a
    teacher's row of equal values has equal weights whatever the value, and a student's
    masked logit that the teacher wants a finite loss."""
    V, k, tau = 3001, 5, 0.5
    low = torch.finfo(dtype).min
    x = logits(n, V, dtype, dev, seed=33)
    ids = torch.arange(k, device=dev, dtype=torch.int32).expand(n, k) * 7
    zero = torch.zeros(n, k, device=dev, dtype=dtype)
    want = check_ce(mga, x, zero, ids, None, tau)
    for value in (low, -low):
        for got, w in zip(check_ce_calls(mga, x, torch.full_like(zero, value), ids, tau), want):
            assert torch.equal(got, w)
    part = torch.full_like(zero, low)
    part[:, 2] = low / 2                    # the only one with a weight
    for got, w in zip(check_ce_calls(mga, x, part, ids, tau), check_ce_calls(mga, x, zero[:, :1], ids[:, 2:3], tau)):
        assert torch.equal(got, w)
    x[0, 7], x[0, 14] = low, low / 2
    check_ce(mga, x, zero, ids, None, tau)


def check_ce_calls(mga, x, values, ids, tau, go=0.375):
    """What check_ce returns, without an oracle."""
    xs = x.detach().clone().requires_grad_()
    total = mga.top_logits_cross_entropy(xs, values, ids, None, tau)
    (total * go).backward()
    return total, xs.grad, mga.top_logits_loss_and_grad(x, values, ids, None, tau, scale=go)[1]


def test_logits_without_a_dimension_are_refused(mga, dev):
    x, i = torch.zeros((), device=dev), torch.zeros((), dtype=torch.int32, device=dev)
    for call in (lambda: mga.top_logits_cross_entropy(x, x, i), lambda: mga.top_logits_loss_and_grad(x, x, i),
                 lambda: mga.top_logits(x, 1), lambda: mga.sample_tokens(x, x)):
        with pytest.raises(ValueError):
            call()
