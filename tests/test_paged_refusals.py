"""Arguments that the paged cache's C entry points refuse before any device work, each
with a message (so these run without a GPU), and CPU tensors at the Python entry points."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(64)


def refused(mga, rc, text=b""):
    assert rc == mga._lib.MGA_ERR_INVALID
    msg = mga.load_library().mga_last_error()
    assert msg and text in msg


PAGED = [dict(T=-1), dict(B=0), dict(B=4097), dict(D=96), dict(Hq=3), dict(Hkv=0), dict(dtype=3), dict(ps=48),
         dict(ps=256), dict(n=0), dict(width=0), dict(trs=3), dict(width=1 << 25, trs=1 << 25), dict(kp=None), dict(vp=None),
         dict(kp=ctypes.c_void_p(72)), dict(ks=None), dict(vs=None), dict(table=None), dict(cu=None), dict(lens=None),
         dict(n=1 << 30)]


LONG = dict(width=1000, trs=1000)   # sequences that need a workspace


def _args(**kw):
    a = dict(k=P, ss=256, hs=128, v=P, q=P, qw=None, kw=None, cos=None, sin=None, cs=128, c32=0, eps=1e-6, T=2, B=1, Hq=4,
             Hkv=2, D=128, dtype=0, kp=P, vp=P, ks=P, vs=P, n=4, ps=64, table=P, trs=4, width=4, cu=P, lens=P, qo=P,
             scale=0.1, out=ctypes.c_void_p(1 << 20), ws=P, nb=1 << 40)
    a.update(kw)
    return a


def _append(lib, **kw):
    a = _args(**kw)
    return lib.mga_paged_append(a["k"], a["ss"], a["hs"], a["v"], a["ss"], a["hs"], a["q"], 512, 128, a["qw"], a["kw"],
                                a["cos"], a["sin"], a["cs"], a["c32"], a["eps"], a["T"], a["B"], a["Hq"], a["Hkv"], a["D"],
                                a["dtype"], a["kp"], a["vp"], a["ks"], a["vs"], a["n"], a["ps"], a["table"], a["trs"],
                                a["width"], a["cu"], a["lens"], a["qo"], 512, 128, None)


def _attend(lib, **kw):
    a = _args(**kw)
    return lib.mga_paged_attn(a["q"], a["ss"], a["hs"], a["kp"], a["vp"], a["ks"], a["vs"], a["n"], a["ps"], a["table"],
                              a["trs"], a["width"], a["cu"], a["lens"], a["T"], a["B"], a["Hq"], a["Hkv"], a["D"],
                              a["dtype"], a["scale"], a["out"], 512, 128, 1, a["ws"], a["nb"], None)


@pytest.mark.parametrize("kw", PAGED + [dict(k=None), dict(v=None), dict(k=ctypes.c_void_p(65)), dict(ss=-1), dict(qo=None),
                                        dict(cos=P), dict(sin=P), dict(cos=P, sin=ctypes.c_void_p(65)),
                                        dict(eps=-1.0), dict(eps=float("nan")), dict(kw=ctypes.c_void_p(65)),
                                        dict(T=1 << 24)])
def test_append(mga, kw):
    refused(mga, _append(mga.load_library(), **kw))


@pytest.mark.parametrize("kw", PAGED + [dict(q=None), dict(out=None), dict(q=ctypes.c_void_p(72)), dict(ss=100),
                                        dict(hs=-128), dict(out=ctypes.c_void_p(66)), dict(Hq=66), dict(scale=0.0),
                                        dict(scale=float("inf")), dict(scale=float("nan")), LONG | dict(ws=None), LONG | dict(nb=100),
                                        LONG | dict(ws=ctypes.c_void_p(72)), dict(T=1 << 28, width=1 << 22, trs=1 << 22)])
def test_attend(mga, kw):
    refused(mga, _attend(mga.load_library(), **kw))


# q: 2 tokens of 4 heads of 128 bf16 at 64, strides 256 and 128
@pytest.mark.parametrize("kw", [dict(out=P), dict(out=ctypes.c_void_p(64 + 16)), dict(out=ctypes.c_void_p(64 + 1024)),
                                dict(q=ctypes.c_void_p(64 + 1536), out=P, ss=512), dict(ss=512, out=ctypes.c_void_p(64 + 16))])
def test_attend_out_overlaps_q(mga, kw):
    refused(mga, _attend(mga.load_library(), **kw), b"overlaps")


def test_no_tokens(mga):
    lib = mga.load_library()
    assert _append(lib, T=0) == 0 and _attend(lib, T=0) == 0
    assert lib.mga_paged_attn_workspace_bytes(0, 1, 4, 2, 128, 64, 4, 0) == 0
    assert lib.mga_paged_attn_workspace_bytes(1, 1, 4, 2, 128, 64, 1000, 0) > 0


def test_cpu_tensors(mga):
    pages = (torch.zeros(1, 1, 64, 64, dtype=torch.uint8).view(torch.float8_e4m3fn),
             torch.zeros(1, 1, 64, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(1, 1), torch.ones(1, 1))
    table, cu, lens = torch.zeros(1, 1).int(), torch.tensor([0, 1]).int(), torch.zeros(1).int()
    x = torch.zeros(1, 1, 64)
    with pytest.raises(RuntimeError, match="GPU"):
        mga.paged_append(x, x, pages, table, cu, lens)
    with pytest.raises(RuntimeError, match="GPU"):
        mga.paged_attention(x, pages, table, cu, lens, 0.125)
    with pytest.raises(RuntimeError, match="GPU"):
        mga.PagedKVCache(1, 1, 1, 64, device="cpu")
    for kw in (dict(page_size=48), dict(head_dim=80), dict(num_pages=0)):
        with pytest.raises(ValueError):
            mga.PagedKVCache(**{**dict(num_pages=1, num_layers=1, num_kv_heads=1, head_dim=64, device="cpu"), **kw})
    with pytest.raises(NotImplementedError, match="no_grad"):
        mga.paged_attention(x.requires_grad_(), pages, table, cu, lens, 0.125)
