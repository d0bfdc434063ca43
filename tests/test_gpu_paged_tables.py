"""Block tables as a program slices them, in the native and the Python forms."""
import pytest
import torch

from test_gpu_paged import Pool, attend, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_a_column_as_the_table_of_one_sequence(mga, dev, native, monkeypatch):
    """A row of a table of one sequence may carry any stride."""
    if not native:
        monkeypatch.setattr(mga._lib, "native", lambda *a: None)
    pool = Pool(dev, [3], [150], 2, 64, 16)
    q = queries(pool, 4, 64, torch.bfloat16, dev)
    x = torch.randn(3, 2, 64, device=dev).bfloat16()
    want, stored = attend(mga, pool, q), pool.clone()
    mga.paged_append(x, x, stored.pages, *stored.batch)
    column = pool.table[0].clone()[:, None]      # [pages, 1], the sequences' tables as columns
    for table in (column.t(), pool.table[0].expand(1, -1), torch.as_strided(pool.table, pool.table.shape, (0, 1))):
        assert table.shape == pool.table.shape and table.stride(0) < table.shape[1] or table.stride(0) == table.shape[1]
        p = pool.clone()
        p.table = table
        assert torch.equal(attend(mga, p, q), want)
        out = torch.empty_like(q)
        assert torch.equal(attend(mga, p, q, out=out), want)
        assert mga.paged_append(x, x, p.pages, *p.batch) is None
        assert torch.equal(p.k, stored.k) and torch.equal(p.v, stored.v)
