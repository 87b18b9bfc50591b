"""The quantised cache on the GPU where it could go wrong: ends of the number range, rows that many blocks share, rows and pages that no
token sees, captured graphs, other streams, pools past 2^31 bytes."""
import pytest
import torch

import plain_quant as Q
from test_gpu_quant_cache import BF16, DEV, F32, attend, check, random_pages, status, step

from kipp_b200 import kernels as K
from kipp_b200.kernels import KernelError

pytestmark = pytest.mark.gpu


def queries(meta, nq, D, seed=0, spare=0, dtype=BF16):
    return (2 * torch.randn(meta.tokens + spare, nq, D, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


# ------------------------------------------------------------------ ends of the number range
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("k_power,v_power", [(40, 0), (-30, 0), (0, 50), (0, 60), (0, -40), (20, 56)])
def test_attention_of_large_and_small_numbers(bits, k_power, v_power):
    """Powers of two in the scales change nothing but the result's power."""
    layout, nq, nkv, D, page = [(300, 1), (900, 3)], 8, 2, 128, 16
    meta, table, n_pages = step(layout, page, 1)
    pages, k, v = random_pages(n_pages, nkv, page, D, bits, 1)
    v_power -= 3 if v_power == 60 else 0                    # (values of up to 2^3 beside the power: the format ends at 2^60)
    pages.k_scales.mul_(2.0 ** k_power)
    pages.v_scales.mul_(2.0 ** v_power)
    q = queries(meta, nq, D, 1)
    scale = D ** -0.5 * 2.0 ** -k_power
    out, st = attend(pages, meta, q, nq, scale, impl="direct")
    assert st.tolist() == [0] * 4
    check(out.float() * 2.0 ** -v_power, q, meta, table, k, v, layout, nkv, page, None, D ** -0.5, lambda e: False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("k_power,v_power,q_power", [(0, 0, 0), (40, 0, 0), (-40, 0, 20), (0, 57, -30), (0, -60, 10), (20, 56, 0)])
def test_prompts_of_large_and_small_numbers(bits, D, k_power, v_power, q_power):
    """The same of portions, whose pages are read back as float16, beside single tokens; one kv head 2^9 smaller than the other."""
    layout, nq, nkv, page = [(300, 100), (900, 1), (0, 130), (0, 0), (70, 2)], 8, 2, 16
    meta, table, n_pages = step(layout, page, 1)
    pages, k, v = random_pages(n_pages, nkv, page, D, bits, 1)
    for head, less in ((0, 0), (1, 9)):
        pages.k_scales[:, head].mul_(2.0 ** (k_power - less))
        pages.v_scales[:, head].mul_(2.0 ** (v_power - less))
    k[:, 1] *= 2.0 ** -9
    v[:, 1] *= 2.0 ** -9
    q = queries(meta, nq, D, 1)
    scale = D ** -0.5 * 2.0 ** (-k_power - q_power)
    out, st = attend(pages, meta, q * 2.0 ** q_power, nq, scale, impl="portion")
    assert st.tolist() == [0] * 4
    # (single tokens: the kernel over codes, see check)
    check(out.float() * 2.0 ** -v_power, q, meta, table, k, v, layout, nkv, page, None, D ** -0.5, lambda e: False,
          lambda e: 2.0 ** (-64 - v_power) if layout[e][1] == 1 else 0.0)


@pytest.mark.parametrize("bits", [4, 8])
def test_loud_queries_see_the_keys_as_they_are(bits):
    """Scores of some tens: keys rounded to bfloat16 would move the weights by up to a tenth, which the plain form's bound shows."""
    layout, nq, nkv, D, page = [(100, 200)], 8, 2, 128, 16
    meta, table, n_pages = step(layout, page, 1)
    pages, k, v = random_pages(n_pages, nkv, page, D, bits, 1)
    q = 4 * queries(meta, nq, D, 1)
    for impl in ("portion", "direct"):
        out, st = attend(pages, meta, q, nq, D ** -0.5, impl=impl)
        check(out, q, meta, table, k, v, layout, nkv, page, None, D ** -0.5, lambda e: False)


@pytest.mark.parametrize("impl", ["direct", "read", None])
@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_attention_of_other_scales(scale, impl):
    layout, nq, nkv, D, page = [(300, 1), (90, 3), (0, 70)], 8, 2, 128, 16
    meta, table, n_pages = step(layout, page, 1)
    pages, k, v = random_pages(n_pages, nkv, page, D, 4, 1)
    q = queries(meta, nq, D, 1)
    out, st = attend(pages, meta, q, nq, scale, 50, impl=impl)
    check(out, q, meta, table, k, v, layout, nkv, page, 50, scale, lambda e: impl == "read")
    with pytest.raises(KernelError):                        # (its maximum is that of the scores before the scale)
        attend(pages, meta, q, nq, scale, impl="portion")


# ------------------------------------------------------------------ how rows are shared
@pytest.mark.parametrize("window", [None, 500])
@pytest.mark.parametrize("D,nq,nkv,bits,entries,longest", [(128, 16, 8, 4, 70, 900), (128, 48, 4, 8, 75, 700), (64, 32, 16, 4, 45, 1100), (256, 8, 8, 8, 21, 600),
                                                           (256, 8, 8, 4, 40, 600), (128, 8, 1, 4, 1, 20000), (64, 4, 2, 8, 2, 20000), (256, 2, 1, 4, 1, 9000)])
def test_rows_that_blocks_share(D, nq, nkv, bits, entries, longest, window):
    """More rows than blocks, and fewer, whose parts are joined by another kernel: ragged, with entries of no token between."""
    page, g = 16, torch.Generator().manual_seed(entries)
    layout = [(int(longest * torch.rand(1, generator=g)) if i else longest, (1, 1, 0, 1, 1)[i % 5]) for i in range(entries)]
    meta, table, n_pages = step(layout, page, 1)
    pages, k, v = random_pages(n_pages, nkv, page, D, bits, 1)
    q = queries(meta, nq, D, 1)
    for _ in range(2):
        out, st = attend(pages, meta, q, nq, D ** -0.5, window)
        assert st.tolist() == [0] * 4
        check(out, q, meta, table, k, v, layout, nkv, page, window, D ** -0.5, lambda e: False)


@pytest.mark.parametrize("page", [16, 6])
@pytest.mark.parametrize("window", [None, 3, 130])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("group,tokens", [(1, 4), (1, 3), (2, 2), (3, 1), (4, 1), (5, 1), (1, 5)])
def test_columns_of_several_tokens(group, tokens, D, window, page):
    """Four columns and five of a kv head, of one token or of several, each with its own limits."""
    nkv, layout = 2, [(126, tokens), (0, tokens), (1000, 1), (255, tokens), (31, 0)]
    meta, table, n_pages = step(layout, page, 1)
    pages, k, v = random_pages(n_pages, nkv, page, D, 4, 1)
    q = queries(meta, nkv * group, D, 1)
    out, st = attend(pages, meta, q, nkv * group, D ** -0.5, window, impl="direct")
    assert st.tolist() == [0] * 4
    check(out, q, meta, table, k, v, layout, nkv, page, window, D ** -0.5, lambda e: False)


# ------------------------------------------------------------------ what no token sees
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("impl,page", [("direct", 16), ("direct", 5), ("read", 16), ("read", 5), ("portion", 16)])
def test_rows_that_no_token_sees_may_hold_anything(impl, bits, page):
    """Slots behind the last token, pages of nobody and pages before the window (which need not be mapped); rows of the result behind
    the last token stay."""
    layout, nq, nkv, D, window = [(301, 1), (0, 0), (700, 2), (63, 70), (0, 1), (0, 0)], 8, 2, 128, 40
    meta, table, n_pages = step(layout, page, 3)
    pages, k, v = random_pages(n_pages, nkv, page, D, bits, 3)
    q = queries(meta, nq, D, 3, spare=5)
    clean, st = attend(pages, meta, q, nq, D ** -0.5, window, impl=impl)
    check(clean, q, meta, table, k, v, layout, nkv, page, window, D ** -0.5, lambda e: impl == "read")
    seen = torch.zeros(n_pages, page, dtype=torch.bool)
    device_table = table.clone()
    for e, (c, n) in enumerate(layout):
        lo = max(0, c - window + 1) if n else c + n
        for j in range(lo, c + n):
            seen[table[e, j // page], j % page] = True
        device_table[e, :lo // page] = -1
    gone = (~seen).to(DEV)
    for codes, scales in ((pages.k_codes, pages.k_scales), (pages.v_codes, pages.v_scales)):
        codes.permute(0, 2, 1, 3)[gone] = 255
        scales.permute(0, 2, 1, 3)[gone] = float("nan")
    meta.block_tables[0].copy_(device_table)
    got, st = attend(pages, meta, q, nq, D ** -0.5, window, impl=impl)
    assert st.tolist() == [0] * 4
    assert torch.equal(got, clean) and (got[meta.tokens:] == 7).all()


@pytest.mark.parametrize("bad", [-1, 10 ** 6])
@pytest.mark.parametrize("page", [16, 5])
def test_pages_that_are_not_there(page, bad):
    """They are reported; the other entries have their results."""
    layout, nq, nkv, D = [(301, 1), (500, 1), (40, 3)], 8, 2, 128
    meta, table, n_pages = step(layout, page, 3)
    pages, k, v = random_pages(n_pages, nkv, page, D, 4, 3)
    q = queries(meta, nq, D, 3)
    clean, _ = attend(pages, meta, q, nq, D ** -0.5, impl="direct")
    meta.block_tables[0][1, 2] = bad
    got, st = attend(pages, meta, q, nq, D ** -0.5, impl="direct")
    assert st.tolist() == [3, 0, 0, 0]
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2:], clean[2:]) and torch.isfinite(got[1]).all()


def test_a_table_that_is_too_short_is_reported():
    layout, nq, nkv, D, page = [(60, 1), (200, 1)], 4, 2, 128, 16
    meta, table, n_pages = step(layout, page, 3)
    pages, k, v = random_pages(n_pages, nkv, page, D, 8, 3)
    q = queries(meta, nq, D, 3)
    short = meta.block_tables[0][:, :4].contiguous()
    out, st = torch.zeros_like(q), status()
    K.attention_quantized(out, q, pages, meta, short, nq, D ** -0.5, None, st, impl="direct")
    assert st.tolist() == [3, 0, 0, 0]
    check(out, q, meta, table, k, v, layout[:1], nkv, page, None, D ** -0.5, lambda e: False)


# ------------------------------------------------------------------ graphs and streams
def chain(qkv, q_out, pages, meta, lists, out, back, st, nq, scale):
    """A step as it is used: written, attended to, read back."""
    T, D = q_out.shape[0], pages.head_dim
    K.qk_norm_rope_write_quantized(qkv, q_out, pages, None, None, 1e-6, None, 0, meta.positions, meta.entry_of_token, meta.block_tables[0], T, nq,
                                   True, st)
    K.attention_quantized(out, q_out, pages, meta, meta.block_tables[0], nq, scale, None, st)
    K.read_quantized_pages(*back, pages, lists, st)


@pytest.mark.parametrize("bits,nkv,rows,width", [(4, 2, 3, 40), (8, 8, 70, 12)])
def test_captured_steps_follow_the_lists(bits, nkv, rows, width):
    """Two graphs (and the streams they run on) of a step that writes, attends and reads back, replayed in turn and at once while their
    lists change in place: what the same calls give one by one, and what the plain form gives."""
    D, nq, page = 128, 2 * nkv, 16
    g = torch.Generator().manual_seed(5)
    sides = []
    for side in range(2):
        meta, table, n_pages = step([(width * page - 1, 1)] * rows, page, side)
        pages, k, v = random_pages(n_pages, nkv, page, D, bits, side)
        T = meta.tokens
        qkv = torch.randn(T, (nq + 2 * nkv) * D, generator=g).to(BF16).to(DEV)
        q_out, out, st = torch.zeros(T, nq, D, dtype=BF16, device=DEV), torch.zeros(T, nq, D, dtype=BF16, device=DEV), status()
        lists = torch.zeros(2, dtype=torch.int32, device=DEV)
        back = [torch.zeros(2, nkv, page, D, device=DEV) for _ in range(2)]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        args = (qkv, q_out, pages, meta, lists, out, back, st, nq, D ** -0.5)
        with torch.cuda.stream(stream):
            chain(*args)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            chain(*args)
        sides.append((graph, stream, args, table, k, v))
    for turn in range(3):
        wants = []
        for side, (graph, stream, args, table, k, v) in enumerate(sides):
            qkv, q_out, pages, meta, lists, out, back, st, _, scale = args
            c = torch.randint(0, width * page - 1, (rows,), generator=g, dtype=torch.int32)
            c[0], c[1] = (0, 1, 127)[turn], (128, width * page - 1, 15)[turn]
            meta.context_len[:rows].copy_(c)
            meta.positions[:rows].copy_(c)
            lists.copy_(torch.tensor([table[0, c[0] // page], table[1, c[1] // page]]))
            qkv.copy_(torch.randn(qkv.shape, generator=g))
            torch.cuda.synchronize()
            before = [t.clone() for t in (pages.k_codes, pages.k_scales, pages.v_codes, pages.v_scales)]
            chain(*args)
            torch.cuda.synchronize()
            wants.append([t.clone() for t in (q_out, out, *back, pages.k_codes, pages.v_scales)])
            # the plain form
            x = qkv.cpu().float().reshape(rows, nq + 2 * nkv, D)
            exact = []
            for rows_of, old in ((x[:, nq:nq + nkv], k), (x[:, nq + nkv:], v)):
                codes, scales = Q.quantise(rows_of, bits)
                new = Q.values(codes, scales, bits)
                for e in range(rows):
                    old[table[e, c[e] // page], :, c[e] % page] = new[e]
                exact.append(old)
            layout = [(int(n), 1) for n in c]
            check(out, q_out, meta, table, *exact, layout, nkv, page, None, scale, lambda e: False)
            assert all(torch.equal(b.cpu(), e[lists.long().cpu()].float()) for b, e in zip(back, exact))
            assert st.tolist() == [0] * 4
            for t, old in zip((pages.k_codes, pages.k_scales, pages.v_codes, pages.v_scales), before):
                t.copy_(old)
            out.fill_(7)
        torch.cuda.synchronize()
        for _ in range(3):                                  # both at once (a step repeated finds its own rows and leaves them)
            for graph, stream, *_ in sides:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (graph, stream, args, *_), want in zip(sides, wants):
            qkv, q_out, pages, meta, lists, out, back, st, _, scale = args
            for got, w in zip((q_out, out, *back, pages.k_codes, pages.v_scales), want):
                assert torch.equal(got, w), turn
            assert st.tolist() == [0] * 4


def test_a_captured_prompt():
    """A portion that is read back for the prompt kernel, beside single tokens, captured and replayed."""
    layout, nq, nkv, D, page = [(130, 100), (77, 1), (0, 64)], 8, 2, 128, 16
    meta, table, n_pages = step(layout, page, 3)
    pages, k, v = random_pages(n_pages, nkv, page, D, 4, 3)
    q = queries(meta, nq, D, 3)
    want, st = attend(pages, meta, q, nq, D ** -0.5, impl="portion")
    out, st = torch.zeros_like(want), status()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.attention_quantized(out, q, pages, meta, meta.block_tables[0], nq, D ** -0.5, None, st, impl="portion")
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want) and st.tolist() == [0] * 4


def test_portions_of_pools_of_one_size(monkeypatch):
    """Pages read back for 4 heads of 4 pages, 2 of 8 and 1 of 16 are as many bytes, and may come to lie in the same memory (as here): how
    they are fetched must not be that of another step."""
    from kipp_b200.kernels import cache_quant
    D, page = 128, 16
    memory, read = torch.empty(2, 16 * page * D, dtype=BF16, device=DEV), cache_quant._read_entries

    def read_there(*args):
        pages = read(*args)
        for there, got in zip(memory, pages):
            there.copy_(got.flatten())
        return tuple(there.view(got.shape) for there, got in zip(memory, pages))
    monkeypatch.setattr(cache_quant, "_read_entries", read_there)
    for nkv, slots in ((4, 4), (1, 16), (2, 8), (4, 4)):
        layout = [(slots * page - 64, 64)]
        meta, table, n_pages = step(layout, page, slots, spare=0)
        pages, k, v = random_pages(n_pages, nkv, page, D, 8, slots)
        q = queries(meta, 4, D, slots)
        for _ in range(2):
            out, st = attend(pages, meta, q, 4, D ** -0.5, impl="portion")
            check(out, q, meta, table, k, v, layout, nkv, page, None, D ** -0.5, lambda e: False)


def test_long_portions_choose_the_prompt_kernel():
    """Where reading back pays, portions go that way by themselves; a few tokens and small steps stay on the codes."""
    from kipp_b200.kernels.cache_quant import _plan
    for layout, form in (([(100, 128), (0, 70), (50, 1)], "portion"), ([(100, 64)], "direct"), ([(9, 4)] * 30, "direct")):
        nq, nkv, D, page = 32, 2, 64, 16
        meta, table, n_pages = step(layout, page, 3)
        pages, k, v = random_pages(n_pages, nkv, page, D, 8, 3)
        q = queries(meta, nq, D, 3)
        assert _plan(q, q, pages, meta, meta.block_tables[0], nq, 1.0)[1] == form
        out, st = attend(pages, meta, q, nq, D ** -0.5)
        check(out, q, meta, table, k, v, layout, nkv, page, None, D ** -0.5, lambda e: False)


# ------------------------------------------------------------------ sizes
@pytest.mark.parametrize("bits", [4, 8])
def test_a_pool_past_2_31_bytes(bits):
    """Pages at the end of a pool whose codes pass 2^31 bytes (and, in 4 bits, 2^32 channels)."""
    D, nq, nkv, page = 128, 16, 8, 16
    n_pages = (2 ** 31 + 2 ** 24) // (nkv * page * D * bits // 8)
    big = K.QuantizedPages.zeros(n_pages, nkv, page, D, bits, DEV)
    layout = [(70, 1), (0, 5)]
    meta, table, small = step(layout, page, 1)
    pages, k, v = random_pages(small, nkv, page, D, bits, 1)
    shift = n_pages - small
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        getattr(big, name)[shift:] = getattr(pages, name)
    far = torch.where(table >= 0, table + shift, table).to(DEV)
    q = queries(meta, nq, D, 1)
    want, _ = attend(pages, meta, q, nq, D ** -0.5)
    out, st = torch.zeros_like(q), status()
    K.attention_quantized(out, q, big, meta, far, nq, D ** -0.5, None, st)
    assert torch.equal(out, want)
    x = torch.randn(meta.tokens, (nq + 2 * nkv) * D, device=DEV).to(BF16)
    for p, t in ((pages, meta.block_tables[0]), (big, far)):
        K.qk_norm_rope_write_quantized(x, out, p, None, None, 1e-6, None, 0, meta.positions, meta.entry_of_token, t, meta.tokens, nq, True, st)
    assert all(torch.equal(getattr(big, n)[shift:], getattr(pages, n)) for n in ("k_codes", "k_scales", "v_codes", "v_scales"))
    assert not big.k_codes[:shift].any() and not big.v_scales[:shift].any()
    order = torch.arange(small, dtype=torch.int32, device=DEV)
    a, b, c, d = (torch.empty(small, nkv, page, D, device=DEV) for _ in range(4))
    K.read_quantized_pages(a, b, pages, order, st)
    K.read_quantized_pages(c, d, big, order + shift, st)
    assert torch.equal(a, c) and torch.equal(b, d) and st.tolist() == [0] * 4


def test_more_pages_an_entry_than_a_grid_has_rows():
    """Pages of one token in a table of 70,000: the 32-bit path, which reads them back."""
    layout, nq, nkv, D, page = [(66000, 1), (3, 2)], 2, 1, 32, 1
    meta, table, n_pages = step(layout, page, 1, width=70000)
    pages, k, v = random_pages(n_pages, nkv, page, D, 8, 1)
    q = queries(meta, nq, D, 1, dtype=F32)
    out, st = attend(pages, meta, q, nq, D ** -0.5)
    assert st.tolist() == [0] * 4
    check(out, q, meta, table, k, v, layout, nkv, page, None, D ** -0.5, lambda e: True)


def test_tensors_at_odd_addresses():
    """Writing takes any address; reading back and attention refuse codes that 8- and 16-byte loads cannot take."""
    layout, nq, nkv, D, page = [(10, 3)], 2, 1, 64, 16
    meta, table, n_pages = step(layout, page, 1)
    even = K.QuantizedPages.zeros(n_pages, nkv, page, D, 8, DEV)
    raw = [torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape) for t in (even.k_codes, even.k_scales, even.v_codes, even.v_scales)]
    odd = K.QuantizedPages(*raw, 8)
    x = torch.randn(meta.tokens, (nq + 2 * nkv) * D, device=DEV).to(BF16)
    q, st = torch.zeros(meta.tokens, nq, D, dtype=BF16, device=DEV), status()
    for p in (even, odd):
        K.qk_norm_rope_write_quantized(x, q, p, None, None, 1e-6, None, 0, meta.positions, meta.entry_of_token, meta.block_tables[0], meta.tokens, nq,
                                       True, st)
    assert torch.equal(even.k_codes, odd.k_codes) and torch.equal(even.v_scales, odd.v_scales)
    out = torch.empty(1, nkv, page, D, device=DEV)
    with pytest.raises(KernelError):
        K.read_quantized_pages(out, out.clone(), odd, torch.zeros(1, dtype=torch.int32, device=DEV), st)
    for impl in (None, "direct", "read"):
        with pytest.raises(KernelError):
            K.attention_quantized(q.clone(), q, odd, meta, meta.block_tables[0], nq, 0.1, None, st, impl=impl)
