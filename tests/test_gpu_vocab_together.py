"""The vocabulary operators as they are used: a rollout from the teacher's logits to
the gradient of the embedding, native and Python forms, captured graphs, other
streams, tensors past 2^31 elements.

Equality is bit for bit where the same kernels run on the same values."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from oracle import vocab as vo
from test_gpu_embedding import close, grad_bound
from test_gpu_native_calls import both, grads
from test_gpu_top_logits import chain, check_ce, check_top, f64, logits

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def inputs(n, V, H, dtype, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = logits(n, V, dtype, dev, seed=seed)
    t = (x.float() + torch.randn(n, V, generator=g, device=dev)).to(dtype)
    u = torch.rand(n, generator=g, device=dev)
    w = torch.randn(V, H, generator=g, device=dev).to(dtype)
    dy = torch.randn(n, H, generator=g, device=dev).to(dtype)
    return x, t, u, w, dy


def everything(mga, x, t, u, w, dy, tau=2.0):
    """One call of each operator, no autograd."""
    top = mga.top_logits(t, min(9, t.shape[-1]), tau)
    loss, g = mga.top_logits_loss_and_grad(x, *top, temperature=tau, scale=0.25)
    fwd = mga.top_logits_cross_entropy(x, *top, tau)
    ids = mga.sample_tokens(x, u, 0.8, 40, 0.9, 0.01)
    e = mga.scaled_embedding(ids, w, 3.0)
    dw = mga.embedding_grad(dy, ids, w.shape[0], 3.0)
    mga.embedding_grad(dy, ids, w.shape[0], 3.0, out=dw, accumulate=True)
    return [*top, loss, g, fwd, ids, e, dw]


@pytest.mark.parametrize("dtype", DTYPES)
def test_rollout(mga, dev, dtype):
    """Teacher's logits -> tokens -> embedding -> student's logits -> loss against the
    teacher's top logits -> gradient of the embedding, each stage against the oracle
    on the stage's own inputs."""
    print(f"case {dtype}", flush=True)
    B, S, V, H, k, tau = 2, 37, 1003, 64, 12, 2.0
    x, _, u, w, _ = inputs(B * S, V, H, dtype, dev, seed=3)
    teacher = x.reshape(B, S, V)
    top = check_top(mga, teacher, k, tau)
    ids = mga.sample_tokens(teacher, u.reshape(B, S), 0.7, 50, 0.9)
    want = [vo.sample_row(r, float(v), np.float64(np.float32(0.7)), 50, np.float64(np.float32(0.9)))
            for r, v in zip(f64(x), f64(u))]
    assert ids.cpu().numpy().reshape(-1).tolist() == want
    ids[1, -3:] = 5                                   # padding
    layer = mga.ScaledEmbedding(V, H, padding_idx=5, scale=4.0, device=dev, dtype=dtype)
    with torch.no_grad():
        layer.weight.copy_(w)
    e = layer(ids)
    e.retain_grad()
    close(e, vo.embedding(ids.cpu().numpy(), f64(w), 4.0).reshape(B, S, H), 0.0, dtype)
    head = torch.randn(H, V, generator=torch.Generator(device=dev).manual_seed(9), device=dev).to(dtype) / 8
    student = torch.matmul(e.reshape(-1, H), head).reshape(B, S, V)
    student.retain_grad()
    keep = torch.where(torch.arange(S, device=dev)[None, :, None] < S - 3, top.ids, -1)
    mga.top_logits_cross_entropy(student, top.values, keep, top.lse, tau).backward()
    _, g, g2 = check_ce(mga, student.detach(), top.values, keep, top.lse, tau, go=1.0)
    assert torch.equal(student.grad, g) and not student.grad[:, S - 3:].any()
    i, de = ids.cpu().numpy().reshape(-1), f64(e.grad).reshape(-1, H)
    close(layer.weight.grad, vo.embedding_grad(de, i, V, 4.0, 5), grad_bound(de, i, V, 4.0, 5), dtype)
    assert not layer.weight.grad[5].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [5, 130])
def test_native_and_python_forms(mga, dev, monkeypatch, dtype, n):
    V, H = 3001, 72
    x, t, u, w, dy = inputs(n, V, H, dtype, dev, seed=4)

    def run():
        out = everything(mga, x, t, u, w, dy)
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = mga.top_logits_cross_entropy(xs, *out[:3], 2.0)
        e = mga.scaled_embedding(out[6], ws, 3.0, padding_idx=1)
        temperature, top_k = u + 0.1, (u * 100).int()
        return out + [loss, e, *grads([loss, e], [xs, ws], [torch.full((), 0.5, device=dev), dy]),
                      mga.sample_tokens(x, u, temperature, top_k, u, u * 0.1)]

    taken = both(mga, monkeypatch, run)
    names = {name for name, done in taken if done}
    assert names == {"top_logits", "top_logits_step", "top_logits_ce", "sample", "embedding"}
    assert all(done for _, done in taken)


def capture(work):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    return graph, out


def scribble(out):
    for o in out:
        o.fill_(float("nan") if o.dtype.is_floating_point else -7)


@pytest.mark.parametrize("n", [7, 150])
def test_captured_graphs(mga, dev, n):
    """Two graphs of all operators, replayed in turn on changing inputs with eager
    calls between, against the eager results."""
    sets = [inputs(n, 5003, 136, dt, dev, seed=s) for s, dt in ((5, torch.bfloat16), (6, torch.float32))]
    graphs = [capture(lambda s=s: everything(mga, *s)) for s in sets]
    for rep in range(4):
        fresh = [inputs(n, 5003, 136, s[0].dtype, dev, seed=10 + rep) for s in sets]
        want = [everything(mga, *f) for f in fresh]
        for s, f in zip(sets, fresh):
            for a, b in zip(s, f):
                a.copy_(b)
        for _, out in graphs:
            scribble(out)
        torch.cuda.synchronize()
        for graph, _ in graphs if rep % 2 else reversed(graphs):
            graph.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            for i, (a, b) in enumerate(zip(out, w)):
                assert torch.equal(a, b), (rep, i)


def test_captured_backward(mga, dev):
    """Forward and backward of both differentiable operators in one graph; refused
    while an eager graph of the same leaf lives, captured after it is gone."""
    n, V, H = 20, 2003, 64
    x, t, u, w, dy = inputs(n, V, H, torch.bfloat16, dev, seed=7)
    top = mga.top_logits(t, 8)
    ids = torch.randint(V, (n,), device=dev)
    xs, ws = x.requires_grad_(), w.requires_grad_()

    def work():
        loss = mga.top_logits_cross_entropy(xs, *top)
        e = mga.scaled_embedding(ids, ws, 2.0)
        return [loss.detach(), e.detach(), *torch.autograd.grad([loss, e], [xs, ws], [torch.ones_like(loss), dy])]

    want = [o.clone() for o in work()]
    eager = mga.scaled_embedding(ids, ws, 2.0), mga.top_logits_cross_entropy(xs, *top)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = u * 2
        with pytest.raises(RuntimeError, match="scaled_embedding: under graph capture"):
            mga.scaled_embedding(ids, ws, 2.0)
        with pytest.raises(RuntimeError, match="top_logits_cross_entropy: under graph capture"):
            mga.top_logits_cross_entropy(xs, *top)
        with torch.no_grad():
            e = mga.scaled_embedding(ids, ws, 2.0)
    graph.replay()
    assert torch.equal(y, u * 2) and torch.equal(e, eager[0])
    del eager
    graph, out = capture(work)
    for rep in range(3):
        scribble(out)
        work()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(out, want)):
            assert torch.equal(a, b), (rep, i)


def test_other_streams(mga, dev):
    """Calls on two streams at once, behind the work that makes their inputs."""
    sets = [inputs(n, 20011, 256, torch.bfloat16, dev, seed=n) for n in (40, 200)]
    want = [everything(mga, *s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                big = torch.zeros(64 << 20, device=dev)
                made = [a * 1 + big[0].to(a.dtype) for a in s]   # ready only behind the fill
                got.append(everything(mga, *made))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        for j, (a, b) in enumerate(zip(out, want[i % 2])):
            assert torch.equal(a, b), (i, j)


@pytest.mark.parametrize("dtype", DTYPES)
def test_broadcast_inputs(mga, dev, dtype):
    """Gradients of inputs that were expanded: the sum over what they were expanded
    to, which torch adds from the operators' own dense gradients."""
    V, H, n = 515, 24, 6
    x, t, u, w, dy = inputs(n, V, H, dtype, dev, seed=8)
    top = mga.top_logits(t, 5)
    one = x[:1].clone().requires_grad_()
    mga.top_logits_cross_entropy(one.expand(n, V), *top).backward()
    row = w[:1].clone().requires_grad_()
    ids = torch.randint(V, (n,), device=dev)
    e = mga.scaled_embedding(ids, row.expand(V, H), 2.0)
    e.backward(dy)
    _, g, _ = check_ce(mga, x[:1].expand(n, V).contiguous(), *top, go=1.0)
    eps = torch.finfo(dtype).eps
    # both sums hold n rounded rows: added in fp32 and rounded, or in steps of dtype
    for got, parts in ((one.grad, g), (row.grad, mga.embedding_grad(dy, ids, V, 2.0))):
        bound = eps * (parts.float().abs().sum(0) * (2 + len(parts) / 64)) + 1e-30
        assert bool(((got[0].float() - parts.float().sum(0)).abs() <= bound).all())


def test_sizes_past_32_bits_are_refused(mga, dev):
    n = 1 << 31
    x, ids = torch.zeros(1, 1, device=dev).expand(n, 1), torch.zeros(1, dtype=torch.int32, device=dev).expand(n)
    top = torch.zeros(1, 1, device=dev).expand(n, 1), torch.zeros(1, 1, dtype=torch.int32, device=dev).expand(n, 1)
    w = torch.zeros(3, 1, device=dev)
    for call in (lambda: mga.top_logits(x, 1), lambda: mga.sample_tokens(x, x[:, 0]),
                 lambda: mga.top_logits_cross_entropy(x, *top), lambda: mga.top_logits_loss_and_grad(x, *top),
                 lambda: mga.scaled_embedding(ids, w), lambda: mga.embedding_grad(x, ids, 3),
                 lambda: mga.embedding_grad(w, ids[:3], n), lambda: mga.scaled_embedding(ids[:3], x)):
        with pytest.raises(ValueError):
            call()


def test_past_2_31_elements(mga, dev):
    """The last rows of tensors of more than 2^31 elements are the same rows alone."""
    V, n = 151936, 14200
    x = torch.zeros(n, V, device=dev, dtype=torch.bfloat16)
    last = slice(n - 120, n)
    x[last] = logits(120, V, torch.bfloat16, dev, seed=9)
    u = torch.rand(n, device=dev)
    print("top_logits", flush=True)
    a, b = mga.top_logits(x, 20), mga.top_logits(x[last].clone(), 20)
    for p, q in zip(a, b):
        assert torch.equal(p[last], q)
    print("sample", flush=True)
    few = mga.sample_tokens(x[last].clone(), u[last], 0.9, 0, 0.95)
    assert torch.equal(mga.sample_tokens(x, u, 0.9, 0, 0.95)[last], few)
    print("step", flush=True)
    _, g = mga.top_logits_loss_and_grad(x, *a)
    _, h = mga.top_logits_loss_and_grad(x[last].clone(), *(t[last] for t in a))
    assert torch.equal(g[last], h)
    del g
    print("loss", flush=True)
    x.requires_grad_()
    mga.top_logits_cross_entropy(x, *a).backward()
    y = x.detach()[last].clone().requires_grad_()
    mga.top_logits_cross_entropy(y, *(t[last] for t in a)).backward()
    d = (x.grad[last].float() - y.grad.float()).abs()   # the same sums in the forward; column ranges in the backward
    assert torch.equal(x.grad[last], y.grad) or float(d.max()) <= 2 * chain(V)
    del x, y, a, b, d
    torch.cuda.empty_cache()
    print("embedding", flush=True)
    V, H, n = 300000, 8192, 700
    w = torch.zeros(V, H, device=dev, dtype=torch.bfloat16)
    w[-500:] = torch.randn(500, H, device=dev).bfloat16()
    ids = torch.randint(V - 500, V, (n,), device=dev)
    e = mga.scaled_embedding(ids, w, 2.0)
    assert torch.equal(e, mga.scaled_embedding(ids - (V - 500), w[-500:].clone(), 2.0))
    dw = mga.embedding_grad(e, ids, V, out=w)
    assert dw is w and torch.equal(dw[-500:], mga.embedding_grad(e, ids - (V - 500), 500))
    assert not dw[:-500].any()


def test_capture_refused_in_every_form(mga, dev):
    """While an eager graph of the leaf lives, a differentiable call under capture is
    refused also where the operands are not those that the native forms take; nothing
    of it is refused without a gradient, outside a capture or after that graph is gone."""
    n, V, H = 20, 2003, 64
    x, t, u, w, dy = inputs(n, V, H, torch.bfloat16, dev, seed=17)
    top = mga.top_logits(t, 8)
    ids = torch.randint(V, (2 * n,), device=dev)[::2]
    lse = torch.stack([top.lse, top.lse], 1)[:, 0]
    xs, ws = x.requires_grad_(), w.requires_grad_()
    wide = torch.stack([x, x], -1)[..., 0].detach().requires_grad_()
    calls = [("scaled_embedding", ws, lambda: mga.scaled_embedding(ids, ws, 2.0)),
             ("top_logits_cross_entropy", xs, lambda: mga.top_logits_cross_entropy(xs, top.values, top.ids, lse)),
             ("top_logits_cross_entropy", xs, lambda: mga.TopLogitsCrossEntropy.apply(xs, *top, 1.0)),
             ("top_logits_cross_entropy", wide, lambda: mga.top_logits_cross_entropy(wide, *top))]
    for name, leaf, call in calls:
        want = call().detach()
        eager = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = u * 2
            with pytest.raises(RuntimeError, match=name + ": under graph capture"):
                call()
            with torch.no_grad():
                e = call()
        graph.replay()
        assert torch.equal(y, u * 2) and torch.equal(e, want) and torch.equal(call(), want)
        del eager
        graph, out = capture(lambda: [call().detach()])
        for _ in range(3):
            scribble(out)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want)


@pytest.mark.parametrize("form", ["native", "python"])
def test_second_derivatives_are_refused(mga, dev, monkeypatch, form):
    """A gradient with a graph of its own has the ordinary values; to differentiate it
    again is refused instead of leaving its part out, also beside other terms. What
    does not go through a second derivative of these operators is not refused."""
    if form == "python":
        monkeypatch.setattr(mga._lib, "native", lambda *args: None)
    n, V, H = 12, 301, 16
    x, t, u, w, dy = inputs(n, V, H, torch.float32, dev, seed=19)
    top = mga.top_logits(t, 5)
    ids = torch.arange(n, device=dev) % 7
    xs, ws = x.requires_grad_(), w.requires_grad_()
    (want,) = torch.autograd.grad(mga.top_logits_cross_entropy(xs, *top), xs)
    (g,) = torch.autograd.grad(mga.top_logits_cross_entropy(xs, *top), xs, create_graph=True)
    assert torch.equal(g, want) and g.requires_grad
    with pytest.raises(RuntimeError, match="top_logits_cross_entropy: no second derivatives"):
        g.square().sum().backward()
    (g,) = torch.autograd.grad(mga.top_logits_cross_entropy(xs, *top) + xs.pow(3).sum(), xs, create_graph=True)
    with pytest.raises(RuntimeError, match="top_logits_cross_entropy: no second derivatives"):
        g.sum().backward()
    e = mga.scaled_embedding(ids, ws, 3.0)
    (want,) = torch.autograd.grad(e.square().sum(), ws, retain_graph=True)
    (g,) = torch.autograd.grad(e.square().sum(), ws, create_graph=True)
    assert torch.equal(g, want)
    with pytest.raises(RuntimeError, match="scaled_embedding: no second derivatives"):
        g.sum().backward()
    e = mga.scaled_embedding(ids, ws, 3.0)
    (g,) = torch.autograd.grad(e, ws, dy, create_graph=True)   # of a constant: no graph behind it
    assert not g.requires_grad
    ws.grad = None
    e = mga.scaled_embedding(ids, ws, 3.0)                      # a penalty on the gradient of what was looked up
    (g,) = torch.autograd.grad(e.pow(3).sum(), e, create_graph=True)
    g.square().sum().backward()                                 # of 9 e^4
    de = 36 * f64(e) ** 3
    got = f64(ws.grad)
    want = vo.embedding_grad(de, ids.cpu().numpy(), V, 3.0)
    # the powers' roundings (some 8 of 2^-24) beside the sum's
    bound = grad_bound(de, ids.cpu().numpy(), V, 3.0) + 2.0 ** -20 * vo.embedding_grad(abs(de), ids.cpu().numpy(), V, 3.0)
    assert (np.abs(got - want) <= bound + 1e-30).all()
    for leaf, call in ((xs, lambda a: mga.top_logits_cross_entropy(a, *top)), (ws, lambda a: mga.scaled_embedding(ids, a))):
        with forward_ad.dual_level(), pytest.raises(RuntimeError):
            call(forward_ad.make_dual(leaf.detach(), torch.ones_like(leaf)))
