"""Outputs of the paged cache's C entry points that overlap themselves are refused
before any device work (so these run without a GPU)."""
import ctypes
import itertools

import pytest

from test_paged_refusals import refused

D = 64


def _attend(lib, ss, hs, T, H, q=ctypes.c_void_p(1 << 40)):
    p = ctypes.c_void_p(64)
    return lib.mga_paged_attn(q, H * D, D, p, p, p, p, 4, 64, p, 4, 4, p, p, T, 1, H, 1, D, 0, 0.1, ctypes.c_void_p(1 << 20),
                              ss, hs, 1, None, 0, None)


def _append(lib, ss, hs, T, H):
    p = ctypes.c_void_p(64)
    return lib.mga_paged_append(p, D, D, p, D, D, ctypes.c_void_p(1 << 40), H * D, D, None, None, None, None, 0, 0, 1e-6, T, 1,
                                H, 1, D, 0, p, p, p, p, 4, 64, p, 4, 4, p, p, ctypes.c_void_p(1 << 20), ss, hs, None)


# strides in halves of a row
@pytest.mark.parametrize("T,H", [(2, 1), (1, 2), (3, 2), (2, 5), (4, 3)])
def test_rows_that_overlap(mga, T, H):
    """Exactly the layouts in which two rows share an element, by their elements."""
    lib = mga.load_library()
    apart = 0
    for ss, hs in itertools.product(range(0, 14), repeat=2):
        cells = [t * ss + h * hs + c for t in range(T) for h in range(H) for c in range(2)]
        if len(set(cells)) < len(cells):
            refused(mga, _attend(lib, ss * D // 2, hs * D // 2, T, H), b"rows of out overlap")
            refused(mga, _append(lib, ss * D // 2, hs * D // 2, T, H), b"rows of query_out overlap")
        else:   # refused for what comes behind this check
            apart += 1
            refused(mga, _attend(lib, ss * D // 2, hs * D // 2, T, H, ctypes.c_void_p((1 << 20) + 16)), b"out overlaps q")
    assert apart > 10


# rows of one buffer from 1 << 20 on: 4 query heads, 2 of keys, 2 of values, then room for 4 more
Q, K, V, MORE = (ctypes.c_void_p((1 << 20) + 2 * D * h) for h in (0, 4, 6, 8))


@pytest.mark.parametrize("out,ss,hs,ok", [(Q, 12, 1, True), (MORE, 12, 1, True), (K, 12, 1, False), (V, 12, 1, False),
                                          (ctypes.c_void_p((1 << 20) + 2 * D), 12, 1, False), (Q, 24, 1, False), (Q, 12, 2, False),
                                          (ctypes.c_void_p((1 << 20) + 2 * D * 11), 12, 1, False),
                                          (ctypes.c_void_p((1 << 20) + 2 * D * 36), 4, 1, True)])
def test_query_out_beside_the_operands(mga, out, ss, hs, ok):
    p = ctypes.c_void_p(64)
    rc = mga.load_library().mga_paged_append(K, 12 * D, D, V, 12 * D, D, Q, 12 * D, D, None, None, None, None, 0, 0,
                                             -1.0 if ok else 1e-6, 3, 1, 4, 2, D, 0, p, p, p, p, 4, 64, p, 4, 4, p, p, out,
                                             ss * D, hs * D, None)
    refused(mga, rc, b"eps" if ok else b"query_out overlaps")   # a good one for its eps, behind this check
