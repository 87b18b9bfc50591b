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


@pytest.mark.parametrize("at_once", [1, 2, 3])
@pytest.mark.parametrize("D,nkv", [(128, 2), (64, 3)])
def test_portions_that_do_not_fit_together(D, nkv, at_once, monkeypatch):
    """Room for a few entries' pages only: they go several at a time, and each has what it has when all go at once, bit for bit, wherever
    the list has its tiles."""
    layout, nq, page = [(30, 100), (400, 1), (0, 0), (700, 1), (0, 130), (5, 2), (900, 1), (333, 260)], 16 * nkv, 16
    meta, table, n_pages = step(layout, page, 3)
    pages, k, v = random_pages(n_pages, nkv, page, D, 4, 3)
    q = queries(meta, nq, D, 3, spare=3)
    want, st = attend(pages, meta, q, nq, D ** -0.5, impl="portion")
    check(want, q, meta, table, k, v, layout, nkv, page, None, D ** -0.5, lambda e: False)
    monkeypatch.setattr(cache_quant, "READ_BYTES", at_once * 2 * nkv * page * D * 2 * table.shape[1])
    assert chosen(q, q, pages, meta, nq) == "portion"
    chunks = cache_quant._plan(q, q, pages, meta, meta.block_tables[0], nq)[2]
    assert chunks == {1: [(0, 1), (4, 1), (5, 1), (7, 1)], 2: [(0, 1), (4, 2), (7, 1)], 3: [(0, 1), (4, 2), (7, 1)]}[at_once]
    order = torch.randperm(meta.n_prefill_items128, generator=torch.Generator().manual_seed(1)).to(DEV)
    for tiles in (meta.prefill_work128, meta.prefill_work128.flip(0).contiguous(), meta.prefill_work128[order].contiguous()):
        meta.prefill_work128 = tiles
        for impl in (None, "portion"):
            out, st = attend(pages, meta, q, nq, D ** -0.5, impl=impl)
            assert st.tolist() == [0] * 4 and torch.equal(out, want) and (out[meta.tokens:] == 7).all()


def test_an_engine_whose_portions_do_not_fit_together():
    """320 key heads of 128: two portions behind 3,900 tokens would take 1.3 GB read back, more than goes at a time."""
    from gpu_util import part_engine
    from kipp_b200.engine import StepEntry
    from kipp_b200.parts import AttentionMixer, NoPositionEncoding, PreNormBlock, RMSNorm, SwiGLUFeedForward
    from tiny import nmse
    heads, long = 320, 3900
    block = PreNormBlock(RMSNorm(64, 1e-5), AttentionMixer(64, heads, heads, 128, NoPositionEncoding()), RMSNorm(64, 1e-5),
                         SwiGLUFeedForward(64, 16))
    eng, _ = part_engine("bfloat16", 64, block=block, kv_quant="int4", page_size=16, n_pages=640, max_requests=5)
    g = torch.Generator().manual_seed(5)
    text = {r: torch.randint(0, 32, (n,), generator=g).tolist() for r, n in (("a", long + 100), ("b", 40), ("c", 150))}
    text["a2"], text["c2"] = text["a"], text["c"]
    for r in ("a", "a2"):
        for at in range(0, long, 500):
            eng.step([StepEntry(r, text[r][at:min(at + 500, long)], [])], check=True)
    eng.step([StepEntry("b", text["b"][:-1], [])], check=True)
    eng.profile_start()
    got = eng.step([StepEntry("a", text["a"][long:], list(range(100))), StepEntry("b", text["b"][-1:], [0]),
                    StepEntry("c", text["c"], list(range(150)))], check=True).double().cpu()
    assert "attn_prefill_tc" in eng.profile_stop()
    for rows, r, new in ((got[:100], "a2", text["a"][long:]), (got[101:], "c2", text["c"])):
        want = eng.step([StepEntry(r, new, list(range(len(new))))], check=True).double().cpu()
        assert nmse(rows, want) <= 1e-4, r


@pytest.mark.parametrize("wrong", ["none", "long portions only", "empty", "more", "short", "int64", "strided", "elsewhere"])
def test_lists_of_tiles_that_are_not_the_step_s(wrong):
    """A list that cannot hold the tiles of every entry of more than one token: refused where portions are asked for, and otherwise the
    step stays on the codes; no row is left unwritten."""
    layout, nq, nkv, D, page = [(30, 300), (400, 1), (5, 40), (60, 2), (0, 130)], 32, 2, 128, 16
    meta, table, n_pages = step(layout, page, 3)
    pages, k, v = random_pages(n_pages, nkv, page, D, 4, 3)
    q = queries(meta, nq, D, 3)
    assert chosen(q, q, pages, meta, nq) == "portion"
    whole, n = meta.prefill_work128, meta.n_prefill_items128
    assert n == 3 + 1 + 1 + 2
    meta.prefill_work128, meta.n_prefill_items128 = {
        "none": (None, 0), "long portions only": (whole[[0, 1, 2, 5, 6]].contiguous(), 5), "empty": (whole, 0), "more": (whole, n + 1),
        "short": (whole[:-1], n), "int64": (whole.long(), n), "strided": (whole.repeat(1, 2)[:, :2], n), "elsewhere": (whole.cpu(), n)}[wrong]
    with pytest.raises(K.KernelError, match="list of the 128-token tiles"):
        attend(pages, meta, q, nq, D ** -0.5, impl="portion")
    assert chosen(q, q, pages, meta, nq) == "direct"
    out, st = attend(pages, meta, q, nq, D ** -0.5)
    assert st.tolist() == [0] * 4
    check(out, q, meta, table, k, v, layout, nkv, page, None, D ** -0.5, lambda e: False)
