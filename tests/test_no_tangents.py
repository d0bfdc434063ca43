"""The operators of a decoding step compute no derivative: an operand that asks for one is refused,
in forward mode as in reverse."""
import pytest
import torch
from torch.autograd import forward_ad


def operands(dev):
    e4m3 = torch.float8_e4m3fn
    f = lambda *s: torch.ones(*s, device=dev)   # noqa: E731
    code = torch.zeros(1, 1, 64, 64, dtype=torch.uint8, device=dev).view(e4m3)
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)   # noqa: E731
    x = dict(key=f(1, 1, 64), value=f(1, 1, 64), query=f(1, 2, 64), cos=f(1, 64), sin=f(1, 64), q_weight=f(64), k_weight=f(64),
             k_scale=f(1, 1), v_scale=f(1, 1), out=f(1, 2, 64))
    return x, code, (i(0)[None], i(0, 1), i(0))


def calls(mga, dev):
    """(name of the operand, call with operands by name)."""
    x, code, batch = operands(dev)

    def append(key, value, k_scale, v_scale, out, **kw):
        return mga.paged_append(key, value, (code, code.clone(), k_scale, v_scale), *batch, **kw)

    def attend(query, k_scale, v_scale, out, **kw):
        return mga.paged_attention(query, (code, code, k_scale, v_scale), *batch, 0.125, out=out)

    def adjust(**kw):
        return mga.adjust_logits(bias_ids=torch.tensor([1], device=dev), **kw)

    y = dict(logits=torch.ones(2, 5, device=dev), bias=torch.ones(1, device=dev), out=torch.ones(2, 5, device=dev))
    y |= {k: torch.ones(2, device=dev) for k in ("repetition", "frequency", "presence")}
    return [(f, x, n) for f, names in ((append, [n for n in x if n != "out"]), (attend, ["query", "k_scale", "v_scale", "out"]))
            for n in names] + [(adjust, y, n) for n in y]


def check(mga, dev):
    for f, x, name in calls(mga, dev):
        # without gradients forward mode still counts
        with forward_ad.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(**{**x, name: forward_ad.make_dual(x[name], torch.ones_like(x[name]))})
        if name != "out":
            with pytest.raises(NotImplementedError, match="no_grad"):
                f(**{**x, name: x[name].clone().requires_grad_()})


def test_cpu(mga):
    check(mga, torch.device("cpu"))
    for f, x, name in calls(mga, torch.device("cpu")):
        if name != "out":
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.func.jvp(lambda t: f(**{**x, name: t}), (x[name],), (torch.ones_like(x[name]),))   # noqa: B023


@pytest.mark.gpu
def test_gpu(mga, dev):
    check(mga, dev)
    for f, x, _ in calls(mga, dev):   # and without a tangent, also within a level
        with forward_ad.dual_level(), torch.no_grad():
            f(**x)
