"""Arguments that the vocabulary operators' C entry points refuse before any device
work, each with a message (so these run without a GPU), and CPU tensors at the
Python entry points."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(64)


def refused(mga, rc, text=b""):
    assert rc == mga._lib.MGA_ERR_INVALID
    msg = mga.load_library().mga_last_error()
    assert msg and text in msg


def _top(lib, **kw):
    a = dict(x=P, rs=100, n=2, v=100, dtype=0, k=4, t=1.0, values=P, ids=P, lse=None)
    a.update(kw)
    return lib.mga_top_logits(a["x"], a["rs"], a["n"], a["v"], a["dtype"], a["k"], a["t"], a["values"], a["ids"],
                              a["lse"], None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(rs=99), dict(n=0), dict(v=0), dict(dtype=3), dict(k=0), dict(k=101),
                                dict(v=2000, rs=2000, k=1025), dict(v=(1 << 20) + 1, rs=1 << 21), dict(t=0.0),
                                dict(t=-1.0), dict(t=float("inf")), dict(t=float("nan")), dict(t=1e-30),
                                dict(values=None),
                                dict(ids=None), dict(x=ctypes.c_void_p(65)), dict(x=ctypes.c_void_p(66), dtype=1)])
def test_top_logits(mga, kw):
    refused(mga, _top(mga.load_library(), **kw))


def _fwd(lib, step=False, **kw):
    a = dict(x=P, rs=100, values=P, vrs=4, vd=0, ids=P, irs=4, i64=0, lse=None, n=2, v=100, k=4, t=1.0, scale=1.0,
             dtype=0, q=P, stats=P, loss=P, sum=P, grad=ctypes.c_void_p(1 << 20), gs=100, ws=P)
    a.update(kw)
    head = (a["x"], a["rs"], a["values"], a["vrs"], a["vd"], a["ids"], a["irs"], a["i64"], a["lse"], a["n"], a["v"],
            a["k"], a["t"])
    if step:
        return lib.mga_top_logits_ce_step(*head, a["scale"], a["dtype"], a["loss"], a["sum"], a["grad"], a["gs"],
                                          a["ws"], None)
    return lib.mga_top_logits_ce_fwd(*head, a["dtype"], a["q"], a["stats"], a["loss"], a["sum"], a["ws"], None)


COMMON = [dict(x=None), dict(rs=99), dict(n=0), dict(dtype=5), dict(k=0), dict(k=1025, vrs=1025, irs=1025),
          dict(t=0.0), dict(t=float("nan")), dict(ids=None), dict(irs=3), dict(ids=ctypes.c_void_p(68), i64=1),
          dict(values=None), dict(vrs=3), dict(vd=7), dict(loss=None), dict(sum=None), dict(ws=None),
          dict(ws=ctypes.c_void_p(72)), dict(t=1e-30), dict(t=1e30)]


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("kw", COMMON)
def test_top_logits_ce(mga, kw, step):
    refused(mga, _fwd(mga.load_library(), step, **kw))


def test_top_logits_ce_outputs(mga):
    lib = mga.load_library()
    refused(mga, _fwd(lib, stats=None), b"stats")
    refused(mga, _fwd(lib, True, grad=None), b"grad")
    refused(mga, _fwd(lib, True, gs=99), b"grad")
    refused(mga, _fwd(lib, True, grad=P), b"overlaps")
    refused(mga, _fwd(lib, True, grad=ctypes.c_void_p(64 + 2 * 199)), b"overlaps")
    bwd = lambda **kw: lib.mga_top_logits_ce_bwd(   # noqa: E731
        P, 100, P, 4, 0, kw.get("q", P), kw.get("stats", P), 2, 100, 4, 1.0, 0, kw.get("go", P), kw.get("grad", P),
        kw.get("gs", 100), None)
    for kw in (dict(q=None), dict(stats=None), dict(go=None), dict(grad=None), dict(gs=50)):
        refused(mga, bwd(**kw))


@pytest.mark.parametrize("kw", [dict(x=None), dict(rs=9), dict(n=0), dict(v=(1 << 20) + 1, rs=1 << 21), dict(dtype=4),
                                dict(u=None), dict(token=None)])
def test_sample(mga, kw):
    a = dict(x=P, rs=10, n=1, v=10, dtype=0, u=P, token=P)
    a.update(kw)
    refused(mga, mga.load_library().mga_sample(a["x"], a["rs"], a["n"], a["v"], a["dtype"], a["u"], None, 1.0, None, 0,
                                               None, 1.0, None, 0.0, a["token"], None))


@pytest.mark.parametrize("kw", [dict(ids=None), dict(n=-1), dict(w=None), dict(rs=7), dict(v=0), dict(h=0),
                                dict(dtype=3), dict(out=None), dict(ors=7), dict(ids=ctypes.c_void_p(68), i64=1),
                                dict(n=2 ** 31 - 1, h=4096, rs=4096, ors=4096)])
def test_embedding_fwd(mga, kw):
    a = dict(ids=P, i64=0, n=3, w=P, rs=8, v=10, h=8, dtype=0, out=P, ors=8)
    a.update(kw)
    refused(mga, mga.load_library().mga_embedding_fwd(a["ids"], a["i64"], a["n"], a["w"], a["rs"], a["v"], a["h"], 1.0,
                                                      a["dtype"], a["out"], a["ors"], None))


@pytest.mark.parametrize("kw", [dict(dy=None), dict(drs=7), dict(ids=None), dict(n=-1), dict(v=0), dict(h=0),
                                dict(dtype=3), dict(dw=None), dict(wrs=7), dict(wd=2), dict(dtype=1, wd=0),
                                dict(ws=None), dict(wn=0), dict(ws=ctypes.c_void_p(72))])
def test_embedding_bwd(mga, kw):
    lib = mga.load_library()
    a = dict(dy=P, drs=8, ids=P, i64=0, n=3, v=10, h=8, dtype=0, dw=P, wrs=8, wd=0, ws=P,
             wn=int(lib.mga_embedding_workspace_bytes(3, 8)))
    a.update(kw)
    refused(mga, lib.mga_embedding_bwd(a["dy"], a["drs"], a["ids"], a["i64"], a["n"], 1.0, -1, a["v"], a["h"],
                                       a["dtype"], a["dw"], a["wrs"], a["wd"], 0, a["ws"], a["wn"], None))


def test_too_many_rows(mga):
    lib, n = mga.load_library(), 1 << 22
    refused(mga, _top(lib, n=n), b"rows")
    for step in (False, True):
        refused(mga, _fwd(lib, step, n=n, grad=ctypes.c_void_p(1 << 40)), b"rows")
    refused(mga, lib.mga_sample(P, 10, n, 10, 0, P, None, 1.0, None, 0, None, 1.0, None, 0.0, P, None), b"rows")
    far = ctypes.c_void_p(1 << 40)
    refused(mga, lib.mga_embedding_fwd(P, 0, 1 << 26, P, 8, 10, 8, 1.0, 0, far, 8, None), b"too many")
    refused(mga, lib.mga_embedding_bwd(P, 8, P, 0, 1 << 30, 1.0, -1, 10, 8, 0, far, 8, 0, 0, P, 1 << 40, None), b"ids")


def test_overlaps(mga):
    lib, at = mga.load_library(), ctypes.c_void_p(64 + 2 * (199 - 4))
    refused(mga, lib.mga_top_logits_ce_bwd(P, 100, P, 4, 0, P, P, 2, 100, 4, 1.0, 0, P, at, 100, None), b"overlaps")
    refused(mga, lib.mga_embedding_fwd(P, 0, 3, P, 8, 25, 8, 1.0, 0, at, 8, None), b"overlaps")
    refused(mga, lib.mga_embedding_bwd(P, 8, P, 0, 25, 1.0, -1, 10, 8, 0, at, 8, 0, 0, P, 1 << 20, None), b"overlaps")


def test_workspace_sizes_of_no_work(mga):
    lib = mga.load_library()
    assert lib.mga_embedding_workspace_bytes(0, 8) == 0
    assert lib.mga_top_logits_ce_workspace_floats(0, 8) == 0
    assert lib.mga_top_logits_ce_step_workspace_floats(4, 8, 0) == 0


def test_cpu_tensors(mga):
    x, ids = torch.randn(2, 9), torch.zeros(2, 3, dtype=torch.int32)
    for call in (lambda: mga.top_logits(x, 3), lambda: mga.top_logits_cross_entropy(x, torch.zeros(2, 3), ids),
                 lambda: mga.top_logits_loss_and_grad(x, torch.zeros(2, 3), ids),
                 lambda: mga.sample_tokens(x, torch.zeros(2)), lambda: mga.scaled_embedding(ids, x),
                 lambda: mga.embedding_grad(torch.zeros(2, 3, 4), ids, 5)):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-30, 1e30):
        with pytest.raises(ValueError, match="temperature"):
            mga.top_logits_cross_entropy(x, torch.zeros(2, 3), ids, None, t)


def test_layer_keeps_the_parameter(mga):
    base = torch.nn.Embedding(6, 4, padding_idx=2)
    layer = mga.ScaledEmbedding.wrap(base, 3.0)
    assert layer.weight is base.weight and layer.padding_idx == 2 and layer.scale == 3.0
    assert list(layer.state_dict()) == list(base.state_dict())
    own = mga.ScaledEmbedding(6, 4, scale=2.0, dtype=torch.bfloat16)
    assert own.weight.dtype == torch.bfloat16 and list(own.state_dict()) == ["weight"]
    with pytest.raises(NotImplementedError):
        mga.ScaledEmbedding.wrap(torch.nn.Embedding(6, 4, max_norm=1.0))


def test_columns_next_to_2_31(mga):
    """The loss's last column range would end past 2^31, its 32-bit length be that of a
    whole range: elements behind the row, which the backward writes."""
    lib, far = mga.load_library(), ctypes.c_void_p(1 << 40)
    for v in ((1 << 30) + 1, 2147383647, (1 << 31) - 1):
        for step in (False, True):
            refused(mga, _fwd(lib, step, n=1, v=v, rs=v, gs=v, grad=far), b"columns")
        refused(mga, lib.mga_top_logits_ce_bwd(P, v, P, 4, 0, P, P, 1, v, 4, 1.0, 0, P, far, v, None), b"columns")


def test_layer_keeps_what_the_base_carries(mga):
    base = torch.nn.Embedding(6, 4).eval()
    base.note = "mine"
    seen = []
    handles = [base.register_forward_pre_hook(lambda m, args: seen.append("pre")),
               base.register_forward_hook(lambda m, args, out: seen.append("post")),
               base.register_full_backward_hook(lambda m, gi, go: None),
               base._register_state_dict_hook(lambda m, sd, prefix, meta: sd.update(extra=1) or sd)]
    layer = mga.ScaledEmbedding.wrap(base, 3.0)
    assert not layer.training and layer.note == "mine" and "extra" in layer.state_dict()
    assert len(layer._forward_hooks) == len(layer._backward_hooks) == 1
    with pytest.raises(RuntimeError, match="GPU tensor"):
        layer(torch.zeros(2, dtype=torch.long))
    assert seen == ["pre"]
    for h in handles:
        h.remove()
    assert not layer._forward_hooks and not layer._forward_pre_hooks and not layer._backward_hooks
    layer.weight = torch.nn.Parameter(torch.zeros(6, 4))   # of the layer alone
    assert layer.weight is not base.weight


def test_layers_that_are_not_wrapped(mga):
    class Scaled(torch.nn.Embedding):
        def forward(self, ids):
            return super().forward(ids) * 2

    class Named(torch.nn.Embedding):
        pass

    patched = torch.nn.Embedding(6, 4)
    patched.forward = lambda ids: None
    normed = torch.nn.utils.parametrizations.weight_norm(torch.nn.Embedding(6, 4))
    for base, text in ((Scaled(6, 4), "forward of its own"), (patched, "forward of its own"),
                       (mga.ScaledEmbedding(6, 4, scale=2.0), "forward of its own"), (normed, "parameter")):
        with pytest.raises(NotImplementedError, match=text):
            mga.ScaledEmbedding.wrap(base)
    assert mga.ScaledEmbedding.wrap(Named(6, 4)).num_embeddings == 6


def test_launches_of_2_32_threads(mga):
    """The smallest numbers of ids that are refused, and those that would make a launch
    of exactly 2^32 threads (in the backward behind others that were queued)."""
    lib, far = mga.load_library(), ctypes.c_void_p(1 << 44)
    for n, h in (((1 << 26) - 3, 8), ((1 << 26) - 1, 1024), ((1 << 25) - 1, 1025), ((1 << 26) // 3, 3000)):
        refused(mga, lib.mga_embedding_fwd(P, 0, n, P, h, 10, h, 1.0, 0, far, h, None), b"too many")
    for n in ((1 << 26) + 1, (1 << 30) - 63, (1 << 30) - 1):
        refused(mga, lib.mga_embedding_bwd(P, 8, P, 0, n, 1.0, -1, 10, 8, 0, far, 8, 0, 0, P, 1 << 40, None), b"ids")


def test_layer_does_not_keep_a_compiled_forward(mga):
    base = torch.nn.Embedding(6, 4)
    base._compiled_call_impl = lambda ids: "base"   # as Module.compile() leaves it
    with pytest.raises(RuntimeError, match="GPU tensor"):
        mga.ScaledEmbedding.wrap(base, 3.0)(torch.zeros(2, dtype=torch.long))
    assert base(torch.zeros(2, dtype=torch.long)) == "base"


def test_soft_ce_columns_next_to_2_31(mga):
    lib, far = mga.load_library(), ctypes.c_void_p(1 << 40)
    for v in ((1 << 30) + 1, 2147383647, (1 << 31) - 1):
        refused(mga, lib.mga_soft_ce_fwd(P, v, P, v, 1, v, 0, P, P, P, None), b"columns")
        refused(mga, lib.mga_soft_ce_loss(P, v, P, v, 1, v, 0, P, P, P, P, None), b"columns")
        refused(mga, lib.mga_soft_ce_bwd(P, v, P, v, 1, v, 0, P, P, far, v, None), b"columns")
