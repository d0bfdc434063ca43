"""The oracle of the vocabulary operators (oracle/vocab.py) against other
formulations of the same definitions: torch's log_softmax and autograd, finite
differences, counted draws."""
import numpy as np
import pytest
import torch

from oracle import soft_ce as sc
from oracle import vocab as vo


def test_order_of_ties_nan_and_signed_zeros():
    x = [0.0, -0.0, np.nan, 3.0, -np.inf, 3.0, np.inf]
    assert list(vo.order(x)) == [6, 3, 5, 0, 1, 4, 2]


def test_top_logits_against_torch():
    x = np.random.default_rng(0).normal(size=(5, 101))
    values, ids, lse = vo.top_logits(x, 9, 2.0)
    tv, ti = torch.topk(torch.tensor(x), 9)
    assert np.array_equal(ids, ti.numpy()) and np.array_equal(values, tv.numpy())
    np.testing.assert_allclose(lse, torch.logsumexp(torch.tensor(x) / 2.0, -1).numpy(), rtol=1e-13)


@pytest.mark.parametrize("with_lse", [False, True])
@pytest.mark.parametrize("tau", [1.0, 2.0])
def test_top_ce_against_autograd(with_lse, tau):
    rng = np.random.default_rng(1)
    x, t = rng.normal(size=(4, 50)) * 2, rng.normal(size=(4, 50)) * 2
    values, ids, lse = vo.top_logits(t, 6, tau)
    ids[1, 4:] = -1                      # padding
    ids[2, 3] = ids[2, 0]                # one column twice
    ids[3] = 50                          # nothing left
    loss, grad = vo.top_ce(x, values, ids, lse if with_lse else None, tau, 0.5)
    xt = torch.tensor(x, requires_grad=True)
    total = 0.0
    for r in range(3):
        ok = torch.tensor(ids[r] >= 0)
        s = torch.tensor(values[r]) / tau
        q = torch.exp(s - lse[r])[ok] if with_lse else torch.softmax(s[ok], 0)
        lp = torch.log_softmax(xt[r] / tau, 0)[torch.tensor(ids[r])[ok]]
        row = -tau ** 2 * (q * lp).sum()
        assert abs(row.item() - loss[r]) < 1e-12
        total = total + row
    (total * 0.5).backward()
    np.testing.assert_allclose(grad, xt.grad.numpy(), atol=1e-13)
    assert loss[3] == 0 and not grad[3].any()


def test_top_ce_with_all_logits_is_the_soft_cross_entropy():
    rng = np.random.default_rng(2)
    x, t = rng.normal(size=(3, 40)), rng.normal(size=(3, 40))
    values, ids, lse = vo.top_logits(t, 40)
    for norm in (None, lse):
        loss, grad = vo.top_ce(x, values, ids, norm)
        np.testing.assert_allclose(loss, sc.soft_ce_rows(x, t)[0], rtol=1e-12)
        np.testing.assert_allclose(grad, sc.soft_ce_grad(x, t), atol=1e-14)


def test_top_ce_gradient_by_differences():
    rng = np.random.default_rng(3)
    x = rng.normal(size=(1, 12))
    values, ids = rng.normal(size=(1, 3)), np.array([[4, 4, 9]])
    _, grad = vo.top_ce(x, values, ids, None, 0.7)
    for j in range(12):
        d = np.zeros_like(x)
        d[0, j] = 1e-6
        num = (vo.top_ce(x + d, values, ids, None, 0.7)[0] - vo.top_ce(x - d, values, ids, None, 0.7)[0]) / 2e-6
        assert abs(num[0] - grad[0, j]) < 1e-8


def test_masked_rows_and_logits():
    inf = np.inf
    x = np.array([[np.nan, 1.0, 2.0], [-inf, 0.0, 0.0], [-inf, -inf, -inf]])
    values, ids = np.array([[1.0, 1.0], [1.0, -inf], [0.0, 0.0]]), np.array([[-1, 7], [1, 0], [0, 1]])
    loss, grad = vo.top_ce(x, values, ids)
    assert loss[0] == 0 and not grad[0].any()           # no entry left: whatever the logits hold
    assert abs(loss[1] - np.log(2)) < 1e-15             # an entry of weight 0 at a masked logit
    assert loss[2] == inf and list(grad[2]) == [-0.5, -0.5, 0]
    assert not vo.teacher_weights(values, ids, 3, lse=[-inf] * 3).any()


def test_sample_row_frequencies_and_filters():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.2, 0.1]))
    us = (np.arange(1000) + 0.5) / 1000
    count = lambda **kw: np.bincount([vo.sample_row(x, u, **kw) for u in us], minlength=5)   # noqa: E731
    assert list(count()) == [100, 400, 200, 200, 100]
    assert list(np.nonzero(count(top_k=2))[0]) == [1, 2]              # of two equal ones the lower column
    assert list(np.nonzero(count(top_p=0.55))[0]) == [1, 2]
    assert list(np.nonzero(count(min_p=0.4))[0]) == [1, 2, 3]
    assert list(np.nonzero(count(top_p=0.0))[0]) == [1]
    assert list(np.nonzero(count(temperature=0.0))[0]) == [1]
    assert vo.sample_row([-np.inf, np.nan], 0.5) == -1
    assert vo.sample_row([0.0, np.inf, np.inf], 0.6) == 2
    assert vo.sample_row([0.0, 1.0, -np.inf], 1.0) == 1               # u = 1: the last that is left


def test_embedding_against_torch():
    rng = np.random.default_rng(4)
    w, ids, dy = rng.normal(size=(7, 3)), rng.integers(0, 7, 20), rng.normal(size=(20, 3))
    wt = torch.tensor(w, requires_grad=True)
    out = torch.nn.functional.embedding(torch.tensor(ids), wt, padding_idx=2) * 1.5
    out.backward(torch.tensor(dy))
    np.testing.assert_allclose(vo.embedding(ids, w, 1.5), out.detach().numpy(), rtol=1e-15)
    np.testing.assert_allclose(vo.embedding_grad(dy, ids, 7, 1.5, 2), wt.grad.numpy(), atol=1e-14)
    ids[3], ids[4] = -1, 7
    assert not vo.embedding(ids, w, 1.5)[3:5].any()
    keep = np.delete(np.arange(20), [3, 4])
    np.testing.assert_allclose(vo.embedding_grad(dy, ids, 7, 1.5), vo.embedding_grad(dy[keep], ids[keep], 7, 1.5),
                               atol=1e-14)
