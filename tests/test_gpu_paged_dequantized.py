"""What ``PagedKVCache.dequantized`` reads of a sequence."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_positions_without_a_page(mga, dev):
    cache = mga.PagedKVCache(5, 1, 2, 64, page_size=16, device=dev)
    p = cache.pages(0)
    for t in (p.k, p.v):
        t.view(torch.uint8).copy_(torch.randint(0, 0x60, t.shape, device=dev, dtype=torch.uint8))
    for t in (p.k_scale, p.v_scale):
        t.copy_(torch.exp2(torch.randint(-9, 3, t.shape, device=dev).float()))
    row = torch.tensor([4, -1, 2, 5, 0, 1 << 30, -(1 << 31)], dtype=torch.int32, device=dev)
    for ids in (row, row.cpu(), row.long()):
        k, v = cache.dequantized(0, ids, 100)
        assert k.shape == v.shape == (2, 100, 64)
        for t, codes, scale in ((k, p.k, p.k_scale), (v, p.v.transpose(2, 3), p.v_scale)):
            for i, page in enumerate(row.tolist()):
                got = t[:, 16 * i:16 * i + 16]
                want = codes[page].float() * scale[page][:, None, None] if 0 <= page < 5 else torch.zeros(2, 16, 64, device=dev)
                assert torch.equal(got, want[:, :got.shape[1]])
    assert cache.dequantized(0, row, 0)[0].shape == (2, 0, 64)
    assert cache.dequantized(0, row[:0], 0)[1].shape == (2, 0, 64)


def test_refusals(mga, dev):
    cache = mga.PagedKVCache(5, 1, 2, 64, page_size=16, device=dev)
    row = torch.zeros(2, dtype=torch.int32, device=dev)
    for ids, n in ((row, 33), (row, -1), (row[None], 5), (row[:0], 1)):
        with pytest.raises(ValueError, match="tokens in a table row"):
            cache.dequantized(0, ids, n)
