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


@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 70, 10 ** 9, -5])
@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("impl", ["direct", "portion"])
def test_lengths_far_behind_the_table(impl, window, length):
    """An entry said to have more cached than any table holds is reported, one below nothing has no result or any; the others are not
    touched by it."""
    layout, nq, nkv, D, page = [(301, 70), (90, 80), (40, 1), (77, 1)], 8, 2, 128, 16
    meta, table, n_pages = step(layout, page, 3)
    pages, k, v = random_pages(n_pages, nkv, page, D, 4, 3)
    q = queries(meta, nq, D, 3)
    for entry in (1, 3):
        meta.context_len[entry] = length
        got, st = attend(pages, meta, q, nq, D ** -0.5, window, impl=impl)
        meta.context_len[entry] = layout[entry][0]
        assert length < 0 or st.tolist() == [3, 0, 0, 0]
        assert st.tolist()[1:] == [0, 0, 0] and torch.isfinite(got).all()
        at = 0
        for e, (_, n) in enumerate(layout):                 # (how a row is cut into parts depends on all lengths)
            if e != entry:
                check(got[at:], q[at:], meta, table[e:], k, v, layout[e:e + 1], nkv, page, window, D ** -0.5, lambda e: False)
            at += n


@pytest.mark.parametrize("impl,bad", [("direct", float("nan")), ("direct", float("inf")), ("direct", -float("inf")), ("portion", float("nan")),
                                      (None, float("nan"))])
@pytest.mark.parametrize("layout", [[(40, 1), (3000, 1)], [(300, 1)] * 90 + [(40, 2), (900, 1)], [(0, 70), (9000, 1), (400, 130), (5000, 3)]])
def test_queries_that_are_no_numbers(impl, bad, layout):
    """Their results are no numbers either, in however many parts their keys are; the other queries have their results.  (The prompt kernel
    takes an infinite query as it is: a row whose keys all have the other sign there scores -inf everywhere, as one that sees nothing.
    The kernel of CUDA cores behind "read" leaves out scores that are no numbers, here as over the plain cache.)"""
    nq, nkv, D, page = 32, 8, 128, 16
    meta, table, n_pages = step(layout, page, 3)
    if impl == "portion" and meta.n_prefill_items128 == 0:
        return
    pages, k, v = random_pages(n_pages, nkv, page, D, 4, 3)
    q = queries(meta, nq, D, 3)
    clean, _ = attend(pages, meta, q, nq, D ** -0.5, impl=impl)
    hit = torch.zeros(meta.tokens, nq, dtype=torch.bool, device=DEV)
    hit[::3, 5] = hit[-1, 31] = hit[0, 0] = True
    q[:, :, 7] = torch.where(hit, torch.tensor(bad, dtype=BF16, device=DEV), q[:, :, 7])
    got, st = attend(pages, meta, q, nq, D ** -0.5, impl=impl)
    assert st.tolist() == [0] * 4
    assert torch.equal(got[~hit], clean[~hit]) and torch.isnan(got[hit]).all()


@pytest.mark.parametrize("D", [128, 96])
def test_a_lone_row_of_any_stride(D):
    """One token's projection as a transposed column, whose first stride is 1: what the same row gives as it is."""
    nq, nkv, page = 4, 2, 16
    meta, table, n_pages = step([(20, 1)], page, 1)
    column = torch.randn((nq + 2 * nkv) * D, 1, generator=torch.Generator().manual_seed(1)).to(BF16).to(DEV)
    row = column.t()
    assert row.shape[0] == 1 and row.stride() == (1, 1)
    results = []
    for qkv in (row, column.flatten()[None].contiguous()):
        pages, st = K.QuantizedPages.zeros(n_pages, nkv, page, D, 8, DEV), status()
        q = torch.zeros(1, nq, D, dtype=BF16, device=DEV)
        K.qk_norm_rope_write_quantized(qkv, q, pages, None, None, 1e-6, None, 0, meta.positions, meta.entry_of_token, meta.block_tables[0], 1, nq,
                                       True, st)
        assert st.tolist() == [0] * 4 and bool(pages.k_codes.any())
        results.append((q, pages.k_codes, pages.k_scales, pages.v_codes, pages.v_scales))
    assert all(torch.equal(a, b) for a, b in zip(*results))
