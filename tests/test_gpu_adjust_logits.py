"""adjust_logits on the GPU against the float64 oracle (oracle/vocab.py). Every value is
computed in fp32 from at most 4 + K operations, each off by 2^-24 of what it adds or scales,
and rounded once: |got - want| <= (4 + K) 2^-24 mag + eps / 2 |want|, mag the sum of the
magnitudes that went into it, with the first term rounded along with the value."""

import numpy as np
import pytest
import torch

from oracle import vocab as vo

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def case(n, V, L, K, dtype, dev, seed=0, mask=False, ids=torch.int64):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g, device=dev)   # noqa: E731
    a = dict(logits=(torch.randn(n, V, generator=g, device=dev) * 3).to(dtype))
    if L:
        a["tokens"] = (r(n, L).pow(3) * (V + 4) - 2).floor().to(ids)
        a["lengths"] = (r(n) * (L + 1)).int()
        a["prompt_lengths"] = (r(n) * (L + 1)).int()
        a |= dict(repetition=0.7 + r(n), frequency=r(n) - 0.2, presence=r(n) - 0.2)
    if K:
        a["bias_ids"] = (r(n, K).pow(2) * (V + 4) - 2).floor().to(ids)
        a["bias"] = torch.randn(n, K, generator=g, device=dev) * 5
    if mask:
        a["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (n, -(-V // 32)), generator=g, device=dev).int()
    return a


def check(got, a):
    f = lambda t: t.double().cpu().numpy() if isinstance(t, torch.Tensor) else t   # noqa: E731
    x = a["logits"]
    n = x.shape[:-1].numel()
    flat = lambda k: (lambda t: t.reshape(n, t.shape[-1]) if t.ndim > 1 else t)(f(a[k])) if k in a else None   # noqa: E731
    one = lambda k, d: np.reshape(f(a.get(k, d)), -1)   # noqa: E731
    want, mag = vo.adjust(flat("logits").reshape(n, -1), flat("tokens") if x.dim() > 1 or "tokens" not in a else flat("tokens")[None],
                          None if "lengths" not in a else one("lengths", 0),
                          None if "prompt_lengths" not in a else one("prompt_lengths", 0), one("repetition", 1.0),
                          one("frequency", 0.0), one("presence", 0.0), flat("bias_ids"), flat("bias"),
                          None if "allowed" not in a else a["allowed"].cpu().numpy().reshape(-1, a["allowed"].shape[-1]))
    # past the middle between the largest number and the next one that the exponent would
    # have, (1 + eps / 4) max or more for every type, rounding to nearest gives infinity
    over = np.isfinite(want) & (np.abs(want) > torch.finfo(x.dtype).max * (1 + torch.finfo(x.dtype).eps))
    want = np.where(over, np.copysign(np.inf, want), want)
    torch.cuda.synchronize()
    assert got.shape == x.shape and got.dtype == x.dtype
    g = f(got).reshape(n, -1)
    K = a["bias"].shape[-1] if "bias" in a else 0
    half = torch.finfo(x.dtype).eps / 2
    with np.errstate(all="ignore"):
        e = (4 + K) * 2.0 ** -24 * mag
        ok = np.abs(g - want) <= e + half * (np.abs(want) + e) + torch.finfo(x.dtype).tiny
    assert (ok | (g == want) | (np.isnan(g) & np.isnan(want))).all()


def run(mga, a, **kw):
    a = dict(a)
    return mga.adjust_logits(a.pop("logits"), a.pop("tokens", None), **a, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V", [(1, 1), (3, 7), (2, 64), (3, 1000), (5, 1023), (3, 1025), (4, 4096), (2, 32003), (1, 151936),
                                 (70, 151936 // 2 + 3)])
def test_sizes(mga, dev, dtype, n, V):
    for i, (L, K, mask) in enumerate([(0, 0, False), (1, 0, False), (300, 0, True), (0, 5, False), (1500, 700, True),
                                      (2049, 256, False)]):
        print(f"case {n} {V} {L} {K} {mask} {dtype}", flush=True)
        a = case(n, V, L, K, dtype, dev, i, mask, torch.int32 if i % 2 else torch.int64)
        check(run(mga, a), a)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_of_wide_tiles(mga, dev, dtype):
    """Enough rows for the wide tiles, with rows that begin anywhere within a vector."""
    for V in (8197, 12288, 20000):
        a = case(600, V, 64, 9, dtype, dev, V, True)
        check(run(mga, a), a)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,K", [(16383, 1024), (16384, 3), (20, 1025), (40000, 2000)])
def test_long_lists(mga, dev, dtype, L, K):
    """Histories and bias lists at and past the narrow form's ends; one token in all of a history."""
    for V in (50, 3001):
        a = case(3, V, L, K, dtype, dev, L, True)
        check(run(mga, a), a)
        a |= dict(tokens=torch.full((3, L), 17, device=dev), lengths=torch.tensor([L, L, L - 1], device=dev).int(),
                  prompt_lengths=torch.tensor([0, L, 1], device=dev).int())
        check(run(mga, a), a)


@pytest.mark.parametrize("dtype", DTYPES)
def test_settings(mga, dev, dtype):
    base = case(12, 500, 200, 0, dtype, dev, 3)
    check(run(mga, base | dict(repetition=1.3, frequency=0.4, presence=-0.3)), base | dict(repetition=1.3, frequency=0.4,
                                                                                          presence=-0.3))
    check(run(mga, base | dict(repetition=base["repetition"].double(), presence=base["presence"][:1])),
          base | dict(presence=base["presence"][:1]))
    odd = base["repetition"].clone()
    odd[:3] = torch.tensor([0.0, -2.0, float("nan")], device=dev)
    check(run(mga, base | dict(repetition=odd)), base | dict(repetition=odd))
    for drop in (["lengths"], ["prompt_lengths"], ["lengths", "prompt_lengths"]):
        a = {k: v for k, v in base.items() if k not in drop}
        check(run(mga, a), a)
    a = base | dict(lengths=torch.full((12,), 1000, device=dev).int(), prompt_lengths=torch.full((12,), -5, device=dev).int())
    check(run(mga, a), a)
    a = base | dict(tokens=torch.full((12, 200), 17, device=dev))    # one token, again and again
    check(run(mga, a), a)
    a = base | dict(tokens=torch.full((12, 200), (1 << 32) + 3, device=dev))   # outside, in 64 bits
    check(run(mga, a), a)


@pytest.mark.parametrize("dtype", DTYPES)
def test_shapes_and_shared_rows(mga, dev, dtype):
    a = case(12, 700, 50, 9, dtype, dev, 4, True)
    want = run(mga, a)
    lead = {k: v.reshape(3, 4, *v.shape[1:]) for k, v in a.items()}
    assert torch.equal(run(mga, lead).reshape(12, 700), want)
    first = {k: v[0] for k, v in a.items()}   # a row without a leading dimension
    assert torch.equal(run(mga, first), want[0])
    for k in ("bias_ids", "allowed"):
        shared = a | {k: a[k][0]}
        check(run(mga, shared), shared)
        assert torch.equal(run(mga, shared), run(mga, a | {k: a[k][:1].expand(12, -1)}))
    check(run(mga, a | dict(bias=a["bias"][0], bias_ids=a["bias_ids"][0])), a | dict(bias=a["bias"][0], bias_ids=a["bias_ids"][0]))
    empty = a | dict(tokens=a["tokens"][:, :0], bias=a["bias"][:, :0], bias_ids=a["bias_ids"][:, :0])
    check(run(mga, empty), empty)
    assert run(mga, {k: v[:0] for k, v in a.items()}).shape == (0, 700)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_out(mga, dev, dtype):
    for V in (701, 4104):
        a = case(9, V, 60, 9, dtype, dev, 5, True)
        want = run(mga, a)
        check(want, a)
        for shift in (0, 1, 3):
            wide = torch.zeros(9, V + 13, dtype=dtype, device=dev)[:, shift:shift + V]
            wide.copy_(a["logits"])
            out = torch.full((9, V + 5), 7, dtype=dtype, device=dev)
            got = run(mga, a | dict(logits=wide), out=out[:, shift:shift + V])
            assert torch.equal(got, want) and (out[:, :shift] == 7).all() and (out[:, shift + V:] == 7).all()
            assert run(mga, a | dict(logits=wide), out=wide) is wide and torch.equal(wide, want)   # in place
        cols = a["logits"].t().contiguous().t()
        assert torch.equal(run(mga, a | dict(logits=cols)), want)
        strided = {k: torch.stack([v, v], -1)[..., 0] if v.dim() == 2 and k != "logits" else v for k, v in a.items()}
        assert torch.equal(run(mga, strided), want)
        assert torch.equal(run(mga, a | dict(logits=a["logits"][:1].expand(9, V))),
                           run(mga, a | dict(logits=a["logits"][:1].expand(9, V).contiguous())))


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_not_finite(mga, dev, dtype):
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[inf, -inf, nan, 0.0, -0.0, torch.finfo(dtype).min, torch.finfo(dtype).max, 1.0]] * 3, device=dev).to(dtype)
    t = torch.arange(8, device=dev).expand(3, 8)
    a = dict(logits=x, tokens=t, repetition=1.5, frequency=0.5, presence=0.25)
    check(run(mga, a), a)
    a |= dict(allowed=torch.tensor([[0xff], [0], [0b11111010]], device=dev).int())
    got = run(mga, a)
    check(got, a)
    assert (got[1] == -inf).all() and got[2, 2] == -inf     # masked NaN among them
    assert mga.sample_tokens(got, torch.zeros(3, device=dev))[1] == -1
    a |= dict(bias_ids=torch.tensor([0, 2, 3, 3], device=dev), bias=torch.tensor([-inf, 1.0, -inf, 1.0], device=dev))
    check(run(mga, a), a)


def test_equal_ids_are_added_in_order(mga, dev):
    """1e8 + 1 - 1e8 in fp32: 0 in this order, 1 in another; across parts of the list, too."""
    K = 700
    ids = torch.full((K,), 3, device=dev)
    bias = torch.zeros(K, device=dev)
    bias[10], bias[300], bias[301], bias[650] = 1e8, 1.0, -1e8, 0.5
    got = mga.adjust_logits(torch.zeros(2, 9, device=dev), bias_ids=ids, bias=bias)
    assert got[0, 3] == 0.5 and got[1, 3] == 0.5
    a = case(40, 3000, 500, 600, torch.float32, dev, 8)
    first = run(mga, a)
    for _ in range(3):
        assert torch.equal(run(mga, a), first)


@pytest.mark.parametrize("dtype", DTYPES)
def test_native_and_python_forms(mga, dev, dtype, monkeypatch):
    a = case(6, 3001, 200, 20, dtype, dev, 9, True)
    native = run(mga, a)
    called = []
    f = mga._lib.load_torch_module().adjust_logits
    assert f(a["logits"], a["tokens"], a["lengths"], a["prompt_lengths"], a["repetition"], a["frequency"], a["presence"], 0.0,
             0.0, 0.0, a["bias_ids"], a["bias"], a["allowed"], None) is not None
    monkeypatch.setattr(mga._lib, "native", lambda *x: called.append(1))
    assert torch.equal(run(mga, a), native) and called


def test_past_2_31_elements(mga, dev):
    V = (1 << 30) - 3
    x = torch.zeros(3, V, dtype=torch.bfloat16, device=dev)
    x[2, -1], x[1, 5] = 4.0, -2.0
    t = torch.tensor([[5, V - 1]] * 3, device=dev)
    got = mga.adjust_logits(x, t, repetition=2.0, presence=1.0, out=x)
    assert got[2, -1] == 1.0 and got[1, 5] == -5.0 and got[0, 5] == -1.0 and got[2, 6] == 0
    assert int((got != 0).sum()) == 6


def test_refusals(mga, dev):
    a = case(4, 100, 10, 3, torch.bfloat16, dev, 1, True)
    x = a["logits"]
    bad = lambda **kw: run(mga, a | kw)   # noqa: E731
    for kw in (dict(lengths=a["lengths"][:2]), dict(tokens=a["tokens"][:2]), dict(tokens=a["tokens"][0]),
               dict(bias=a["bias"][:, :2]), dict(bias=None), dict(bias_ids=None), dict(allowed=a["allowed"][:, :3]),
               dict(allowed=a["allowed"][:3]), dict(repetition=torch.ones(3, device=dev)), dict(out=x[:2]),
               dict(out=x.float()), dict(out=torch.empty(100, 4, device=dev, dtype=x.dtype).t()),
               dict(tokens=None), dict(logits=x[:, :0]), dict(logits=torch.tensor(1.0, device=dev))):
        with pytest.raises(ValueError):
            bad(**kw)
    for kw in (dict(tokens=a["tokens"].float()), dict(lengths=a["lengths"].long()), dict(bias=a["bias"].double()),
               dict(bias_ids=a["bias_ids"].short()), dict(allowed=a["allowed"].long()), dict(logits=x.double()),
               dict(repetition=torch.ones(4, device=dev).int())):
        with pytest.raises(TypeError):
            bad(**kw)
    for kw in (dict(logits=x.cpu()), dict(tokens=a["tokens"].cpu()), dict(allowed=a["allowed"].cpu())):
        with pytest.raises(RuntimeError, match="GPU"):
            bad(**kw)
    for r in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(mga._lib.MGAError, match="repetition"):
            bad(repetition=r)
    both = torch.zeros(500, device=dev, dtype=x.dtype)
    with pytest.raises(mga._lib.MGAError, match="overlaps"):
        bad(logits=both[:400].view(4, 100), out=both[8:408].view(4, 100))
    with pytest.raises(NotImplementedError, match="no_grad"):
        bad(logits=x.clone().requires_grad_())
    with torch.no_grad():
        bad(logits=x.clone().requires_grad_())
