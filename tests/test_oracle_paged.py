"""The paged cache's oracle against other formulations."""
import numpy as np
import pytest
import torch

from oracle import paged as po


def test_e4m3_against_torch():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert np.array_equal(po.e4m3_table(), codes.float().numpy().astype(np.float64), equal_nan=True)
    g = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(20000, generator=g) * 2.0 ** torch.randint(-12, 7, (20000,), generator=g),
                   torch.tensor([0.0, 448.0, -448.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 17.0, 19.0])]).clamp(-448, 448)
    assert np.array_equal(po.round_e4m3(x.double().numpy()), x.to(torch.float8_e4m3fn).double().numpy())
    # halfway between neighbours
    v = np.sort(po.e4m3_table()[:127])
    mid = torch.tensor((v[1:] + v[:-1]) / 2).float()
    assert np.array_equal(po.round_e4m3(mid.double().numpy()), mid.to(torch.float8_e4m3fn).double().numpy())


@pytest.mark.parametrize("amax,want", [(448.0, 0), (448.0001, 1), (447.0, 0), (224.0, -1), (225.0, 0), (1.0, -8), (1.75, -8),
                                       (1.7500001, -7), (0.0, -100), (1e-38, -100), (3e38, 119)])
def test_scale(amax, want):
    s = po.scale_of(amax)
    assert s == 2.0 ** want
    if -100 < want < 119:
        assert amax <= 448 * s and amax > 224 * s


def test_rotation_is_a_turn_of_pairs():
    rng = np.random.default_rng(0)
    x, angle = rng.normal(size=(3, 2, 8)), rng.normal(size=(3, 4))
    cos, sin = np.cos(np.concatenate([angle, angle], -1)), np.sin(np.concatenate([angle, angle], -1))
    z = (x[..., :4] + 1j * x[..., 4:]) * np.exp(1j * angle)[:, None]
    got = po.prepared(x, cos=cos, sin=sin)
    assert np.allclose(got, np.concatenate([z.real, z.imag], -1), atol=1e-14)
    w = rng.normal(size=8)
    y = torch.nn.functional.rms_norm(torch.tensor(x), (8,), torch.tensor(w), 1e-3).numpy()
    assert np.allclose(po.prepared(x, w, eps=1e-3), y, atol=1e-14)


def test_attention_of_one_sequence():
    rng = np.random.default_rng(1)
    D, ps, n, L = 8, 4, 3, 9
    k, v = rng.normal(size=(2, 5, 1, ps, D))
    table = [[3, 0, 4, 99]]
    q = rng.normal(size=(n, 2, D))
    out, _ = po.attend(q, k, v, [0, n], [L - n], table, ps, 0.3)
    kk, vv = (np.concatenate([t[p, 0] for p in (3, 0, 4)])[:L] for t in (k, v))
    mask = torch.tril(torch.ones(n, L, dtype=torch.bool), diagonal=L - n)
    want = torch.nn.functional.scaled_dot_product_attention(
        torch.tensor(q).transpose(0, 1), *(torch.tensor(t).expand(2, -1, -1) for t in (kk, vv)), attn_mask=mask, scale=0.3)
    assert np.allclose(out, want.transpose(0, 1).numpy(), atol=1e-13)
    # a page that is not there is masked
    out, _ = po.attend(q, k, v, [0, n], [13], table, ps, 0.3)
    full, _ = po.attend(q, k, v, [0, n], [11 - n + 1], [[3, 0, 4]], ps, 0.3)
    assert np.allclose(out[-1], full[-1])
    assert not po.attend(q, k, v, [0, n], [0], [[-1]], ps, 0.3)[0].any()
