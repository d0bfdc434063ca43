"""Arguments that mga_adjust_logits refuses before any device work, each with a message
(so these run without a GPU), and CPU tensors at the Python entry point."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(64)


@pytest.mark.parametrize("kw", [dict(x=None), dict(rs=99), dict(n=0), dict(v=0), dict(dtype=3), dict(n=1 << 22),
                                dict(v=(1 << 30) + 1, rs=1 << 31, ors=1 << 31), dict(x=ctypes.c_void_p(65)), dict(out=None),
                                dict(ors=99), dict(tokens=None), dict(tokens=ctypes.c_void_p(68)), dict(trs=3), dict(L=-1),
                                dict(L=1 << 30, trs=1 << 31), dict(K=-1), dict(bias_ids=None), dict(bias=None), dict(bias=ctypes.c_void_p(66)), dict(brs=2),
                                dict(vrs=2), dict(allowed=ctypes.c_void_p(66)), dict(ars=3), dict(r=0.0), dict(r=-1.0),
                                dict(r=float("nan")), dict(r=float("inf")), dict(out=ctypes.c_void_p(66)),
                                dict(out=ctypes.c_void_p(64 + 2 * 199)), dict(out=P, ors=101),
                                dict(n=(1 << 22) - 1, v=1 << 16, rs=1 << 16, ors=1 << 16, out=ctypes.c_void_p(1 << 50))])
def test_adjust_logits(mga, kw):
    a = dict(x=P, rs=100, n=2, v=100, dtype=0, tokens=P, t64=1, trs=4, L=4, r=1.0, bias_ids=P, brs=3, bias=P, vrs=3, K=3,
             allowed=P, ars=4, out=ctypes.c_void_p(1 << 20), ors=100)
    a.update(kw)
    lib = mga.load_library()
    rc = lib.mga_adjust_logits(a["x"], a["rs"], a["n"], a["v"], a["dtype"], a["tokens"], a["t64"], a["trs"], a["L"], None, None,
                               None, a["r"], None, 0.0, None, 0.0, a["bias_ids"], 0, a["brs"], a["bias"], a["vrs"], a["K"],
                               a["allowed"], a["ars"], a["out"], a["ors"], None)
    assert rc == mga._lib.MGA_ERR_INVALID and lib.mga_last_error()


def test_cpu_tensors(mga):
    with pytest.raises(RuntimeError, match="GPU"):
        mga.adjust_logits(torch.zeros(2, 10))
