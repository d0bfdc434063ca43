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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,Hq,Hkv,D", [(5, 40, 2, 64), (300, 6, 2, 128)])
def test_queries_prepared_in_place(mga, dev, dtype, T, Hq, Hkv, D):
    """The C entry with query_out = query, the first heads of a projection's rows."""
    pool = Pool(dev, [T], [20], Hkv, D, 16)
    x = torch.randn(T, Hq + 2 * Hkv, D, device=dev).to(dtype)
    q, k, v = x.split([Hq, Hkv, Hkv], 1)
    cos, sin = torch.randn(2, T, D, device=dev).to(dtype)
    w = torch.rand(D, device=dev).to(dtype)
    other, rest = pool.clone(), x[:, Hq:].clone()
    want = mga.paged_append(k, v, other.pages, *other.batch, query=q, cos=cos, sin=sin, q_weight=w)
    at = lambda t: (t.data_ptr(), t.stride(0), t.stride(1))   # noqa: E731
    mga._lib.call("mga_paged_append", *at(k), *at(v), *at(q), w.data_ptr(), None, cos.data_ptr(), sin.data_ptr(), D, 0, 1e-6, T,
                  1, Hq, Hkv, D, mga.ops.dtype_code(dtype), *(t.data_ptr() for t in pool.pages), pool.n, 16,
                  pool.table.data_ptr(), pool.table.shape[1], pool.table.shape[1], pool.cu.data_ptr(), pool.len.data_ptr(),
                  *at(q), torch.cuda.current_stream(dev).cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(q, want) and torch.equal(x[:, Hq:], rest)
    assert torch.equal(pool.k, other.k) and torch.equal(pool.v, other.v) and torch.equal(pool.ks, other.ks)
