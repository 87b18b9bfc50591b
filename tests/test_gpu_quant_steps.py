"""Attention over the quantised cache in steps at the ends of what its sizes may be."""
import pytest
import torch

from test_gpu_quant_cache import BF16, DEV, attend, check, random_pages, status, step
from test_gpu_quant_edges import queries

from kipp_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [None, 60])
def test_many_entries_of_a_long_table(window):
    """One entry of 512 tokens among 64, and tables with room for 2^20 keys: what every entry might have passes the 32 bits of a launch's
    counts, what they have does not."""
    layout, nq, nkv, D, page = [(50 + 3 * i, 1) for i in range(30)] + [(1000, 512)] + [(i, 1) for i in range(33)], 64, 8, 128, 16
    meta, table, n_pages = step(layout, page, 1, width=65536)
    pages, k, v = random_pages(n_pages, nkv, page, D, 4, 1)
    q = queries(meta, nq, D, 1)
    out, st = attend(pages, meta, q, nq, D ** -0.5, window, impl="direct")
    assert st.tolist() == [0] * 4
    check(out, q, meta, table, k, v, layout, nkv, page, window, D ** -0.5, lambda e: False)
