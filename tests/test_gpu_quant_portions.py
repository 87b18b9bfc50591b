"""Portions of prompts over the quantised cache, in every form that takes them: pages that are not there, steps of mixed entries, steps
whose pages do not fit what may be read back at a time, lists of tiles."""
import pytest
import torch

from test_gpu_quant_cache import BF16, DEV, attend, check, random_pages, status, step
from test_gpu_quant_edges import queries

from kipp_b200 import kernels as K
from kipp_b200.kernels import cache_quant

pytestmark = pytest.mark.gpu
FORMS = [None, "portion", "read", "direct"]


def chosen(out, q, pages, meta, nq):
    return cache_quant._plan(out, q, pages, meta, meta.block_tables[0], nq)[1]


# ------------------------------------------------------------------ what is not there
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("impl", FORMS)
def test_pages_that_are_not_there(impl, window, bad):
    """A page that a token sees is reported, whatever the form; the other entries have their results."""
    layout, nq, nkv, D, page = [(301, 70), (500, 200), (40, 1), (0, 130)], 32, 2, 128, 16
    meta, table, n_pages = step(layout, page, 3)
    pages, k, v = random_pages(n_pages, nkv, page, D, 4, 3)
    q = queries(meta, nq, D, 3)
    assert chosen(q, q, pages, meta, nq) == "portion"
    clean, st = attend(pages, meta, q, nq, D ** -0.5, window, impl=impl)
    assert st.tolist() == [0] * 4
    first = meta.q_lens[0]
    last = first + meta.q_lens[1]
    for slot in (26, 43) if window else (0, 2, 31, 43):     # (the window's first page, the last one)
        meta.block_tables[0].copy_(table)
        meta.block_tables[0][1, slot] = bad
        got, st = attend(pages, meta, q, nq, D ** -0.5, window, impl=impl)
        assert st.tolist() == [3, 0, 0, 0], slot
        assert torch.equal(got[:first], clean[:first]) and torch.equal(got[last:], clean[last:]) and torch.isfinite(got).all()
    if window:                                              # before the window nothing need be mapped
        meta.block_tables[0].copy_(table)
        meta.block_tables[0][1, :25] = -1
        got, st = attend(pages, meta, q, nq, D ** -0.5, window, impl=impl)
        assert st.tolist() == [0] * 4 and torch.equal(got, clean)


@pytest.mark.parametrize("impl", FORMS)
def test_a_table_that_is_too_short_is_reported(impl):
    layout, nq, nkv, D, page = [(60, 70), (200, 100), (190, 2)], 32, 2, 128, 16
    meta, table, n_pages = step(layout, page, 3)
    pages, k, v = random_pages(n_pages, nkv, page, D, 8, 3)
    q = queries(meta, nq, D, 3)
    assert chosen(q, q, pages, meta, nq) == "portion"
    for width, want in ((19, 0), (18, 3), (12, 3)):         # the second entry's last token is in the 19th page
        short = meta.block_tables[0][:, :width].contiguous()
        out, st = torch.zeros_like(q), status()
        K.attention_quantized(out, q, pages, meta, short, nq, D ** -0.5, None, st, impl=impl)
        assert st.tolist() == [want, 0, 0, 0], width
        check(out, q, meta, table, k, v, layout[:1], nkv, page, None, D ** -0.5, lambda e: impl == "read")
        check(out[170:], q[170:], meta, table[2:], k, v, layout[2:], nkv, page, None, D ** -0.5, lambda e: impl == "read")


# ------------------------------------------------------------------ mixed steps
@pytest.mark.parametrize("window", [None, 90])
@pytest.mark.parametrize("bits", [4, 8])
def test_single_tokens_between_portions_are_not_read_back(bits, window):
    """What they see is neither read nor written for the prompt kernel: the kernel over codes serves them."""
    layout, nq, nkv, D, page = [(30, 100), (400, 1), (0, 0), (700, 1), (0, 130), (5, 2), (900, 1)], 32, 2, 128, 16
    meta, table, n_pages = step(layout, page, 3)
    pages, k, v = random_pages(n_pages, nkv, page, D, bits, 3)
    q = queries(meta, nq, D, 3)
    out, st = attend(pages, meta, q, nq, D ** -0.5, window, impl="portion")
    assert st.tolist() == [0] * 4
    check(out, q, meta, table, k, v, layout, nkv, page, window, D ** -0.5, lambda e: False)
    made, factors = torch.full_like(meta.block_tables[0], -7), torch.zeros(len(layout), nkv, 2, device=DEV)
    cache_quant._read_entries(pages, BF16, meta, meta.block_tables[0], 0, 6, window or 0, st, made, torch.cuda.current_stream().cuda_stream, factors)
    for e, (c, n) in enumerate(layout):
        lo = max(0, c - (window or 10 ** 6) + 1) // page
        needed = -(-(c + n) // page) - lo if n > 1 else 0
        assert int((made[e] >= 0).sum()) == needed and (e == 6) == bool((made[e] == -7).all()), e
    assert st.tolist() == [0] * 4
