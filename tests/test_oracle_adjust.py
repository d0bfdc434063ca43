"""The oracle of adjust_logits against another formulation."""
import numpy as np
import torch

from oracle import vocab as vo


def test_against_scatter():
    rng = np.random.default_rng(0)
    N, V, L, K = 5, 50, 40, 7
    x = rng.normal(size=(N, V))
    tokens = rng.integers(-2, V + 2, size=(N, L))
    lengths, prompts = rng.integers(0, L + 1, N), rng.integers(0, L, N)
    rep, freq, pres = 1 + rng.random(N), rng.random(N), rng.random(N)
    ids, bias = rng.integers(-1, V + 1, size=(N, K)), rng.normal(size=(N, K))
    words = rng.integers(-2 ** 31, 2 ** 31, size=(N, 2)).astype(np.int32)
    got, mag = vo.adjust(x, tokens, lengths, prompts, rep, freq, pres, ids, bias, words)
    t = torch.tensor(tokens) + 2
    at = torch.arange(L)[None]
    live = at < torch.tensor(lengths)[:, None]
    out = live & (at >= torch.tensor(prompts)[:, None])
    count = lambda w: torch.zeros(N, V + 4).scatter_add_(1, t, w.float())[:, 2:-2].numpy()   # noqa: E731
    seen, c = count(live) > 0, count(out)
    y = np.where(seen, np.where(x > 0, x / rep[:, None], x * rep[:, None]), x) - freq[:, None] * c - pres[:, None] * (c > 0)
    y += torch.zeros(N, V + 2).double().scatter_add_(1, torch.tensor(ids) + 1, torch.tensor(bias))[:, 1:-1].numpy()
    bits = np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")[:, :V]
    assert np.allclose(got, np.where(bits, y, -np.inf), atol=1e-12)
    assert (mag >= np.abs(np.where(bits, got, 0)) - 1e-12).all()
