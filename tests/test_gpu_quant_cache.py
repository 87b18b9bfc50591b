"""The quantised cache on the GPU: what is written, read back and attended to, against plain_quant.py in 64 bits."""
import math

import plain_quant as Q
import pytest
import torch
from gpu_util import pack_meta

from kipp_b200 import kernels as K
from kipp_b200.kernels import cache_quant

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


def status():
    return torch.zeros(4, dtype=torch.int32, device=DEV)


def step(layout, page, seed=0, width=None, spare=2):
    """(meta, table on the CPU, pages of the pool) for entries of (cached, new) tokens, pages anywhere in the pool."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-(c + n) // page) for c, n in layout]
    n_pages = sum(need) + spare
    perm = torch.randperm(n_pages, generator=g).int()
    table = torch.full((len(layout), width or max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = perm[at:at + k]
        at += k
    meta = pack_meta([(i, [0] * n, []) for i, (_, n) in enumerate(layout)], [c for c, _ in layout], list(range(len(layout))),
                     [table.numpy()], torch.device(DEV))
    return meta, table, n_pages


def random_pages(n_pages, nkv, page, D, bits, seed=0):
    """A pool of quantised Gaussian rows, a few channels of the keys loud: the pages and what they stand for in float64."""
    g = torch.Generator().manual_seed(100 + seed)
    k = torch.randn(n_pages, nkv, page, D, generator=g) * (1 + 3 * (torch.rand(D, generator=g) < 0.05))
    v = torch.randn(n_pages, nkv, page, D, generator=g) * (0.3 + torch.rand(n_pages, nkv, page, 1, generator=g))
    kc, ks = Q.quantise(k, bits)
    vc, vs = Q.quantise(v, bits)
    pages = K.QuantizedPages(Q.pack(kc, bits).to(DEV), ks.to(DEV), Q.pack(vc, bits).to(DEV), vs.to(DEV), bits)
    return pages, Q.values(kc, ks, bits), Q.values(vc, vs, bits)


# ------------------------------------------------------------------ writing
WRITES = [dict(D=128, nq=4, nkv=2, rot=128, page=16, norm=True), dict(D=64, nq=3, nkv=1, rot=64, page=8, norm=True, pad=8),
          dict(D=256, nq=2, nkv=2, rot=256, page=4, norm=True, w16=True), dict(D=128, nq=2, nkv=1, rot=0, page=5, norm=False),
          dict(D=64, nq=2, nkv=2, rot=32, page=16, norm=True), dict(D=256, nq=2, nkv=1, rot=128, page=16, norm=True), dict(D=128, nq=3, nkv=1, rot=64, page=8, norm=False),
          dict(D=128, nq=2, nkv=1, rot=96, page=16, norm=True), dict(D=96, nq=3, nkv=1, rot=96, page=16, norm=True),
          dict(D=32, nq=1, nkv=1, rot=20, page=1, norm=False, pad=3), dict(D=512, nq=1, nkv=1, rot=512, page=2, norm=True),
          dict(D=128, nq=2, nkv=2, rot=128, page=16, norm=True, pad=1), dict(D=128, nq=4, nkv=2, rot=128, page=16, norm=False, long=70)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("case", WRITES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_write(case, bits, dtype):
    """Codes and scales are those of the plain form, bit for bit; the queries are off by their rounding at most."""
    D, nq, nkv, rot, page = (case[k] for k in ("D", "nq", "nkv", "rot", "page"))
    layout = [(13, 5), (40, 1), (0, case.get("long", 19))]
    meta, table, n_pages = step(layout, page, D)
    g = torch.Generator().manual_seed(D + bits)
    T, width = meta.tokens, (nq + 2 * nkv) * D
    wide = (torch.randn(T, width + case.get("pad", 0), generator=g) * torch.exp(torch.randn(T, 1, generator=g))).to(dtype)
    qkv = wide[:, :width]
    wdt = BF16 if case.get("w16") else F32
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(wdt) if case["norm"] else None for _ in range(2))
    angle = meta.positions.cpu().double()[:, None] * torch.pow(1e4, -torch.arange(rot // 2).double() / max(rot // 2, 1))
    cos_sin = torch.stack([angle.cos(), angle.sin()], -1).float() if rot else None
    pages = K.QuantizedPages.zeros(n_pages, nkv, page, D, bits, DEV)
    pages.k_codes.fill_(77); pages.v_scales.fill_(-3.0)
    q_out, st = torch.zeros(T, nq, D, dtype=dtype, device=DEV), status()
    on = lambda t: None if t is None else t.to(DEV)        # noqa: E731
    K.qk_norm_rope_write_quantized(on(wide)[:, :width], q_out, pages, on(qw), on(kw), 1e-6, None, rot, meta.positions,
                                   meta.entry_of_token, meta.block_tables[0], T, nq, True, st, cos_sin=on(cos_sin))
    assert st.tolist() == [0, 0, 0, 0]
    x = qkv.float().reshape(T, nq + 2 * nkv, D)
    want_q = Q.heads(x[:, :nq], qw, 1e-6, cos_sin, rot).to(dtype)
    # (the queries' sum of squares may be formed in 32 bits: 2^-22 of the row beside the rounding to their type)
    near_q = lambda got, want: ((got.cpu().double() - want.double()).abs() <= (2.0 ** -8 if dtype == BF16 else 2.0 ** -24) * want.double().abs()   # noqa: E731
                                + 2.0 ** -21 * want.double().abs().amax(-1, keepdim=True)).all()
    assert near_q(q_out, want_q)
    # (the plain form's own operations are those of the definition to rounding)
    if qw is not None and dtype == F32:
        exact = x[:, :nq].double() / ((x[:, :nq].double() ** 2).mean(-1, keepdim=True) + 1e-6).sqrt() * qw.double()
        if rot == 0:
            assert torch.allclose(want_q.double(), exact, rtol=8 * 2.0 ** -24, atol=0)
    kc, ks = Q.quantise(Q.heads(x[:, nq:nq + nkv], kw, 1e-6, cos_sin, rot), bits)
    vc, vs = Q.quantise(x[:, nq + nkv:], bits)
    pos, ent = meta.positions.tolist(), meta.entry_of_token.tolist()
    written = torch.zeros(n_pages, page, dtype=torch.bool)
    for t in range(T):
        p, s = int(table[ent[t], pos[t] // page]), pos[t] % page
        assert torch.equal(pages.k_scales[p, :, s].cpu(), ks[t]) and torch.equal(pages.v_scales[p, :, s].cpu(), vs[t]), t
        assert torch.equal(pages.k_codes[p, :, s].cpu(), Q.pack(kc[t], bits)) and torch.equal(pages.v_codes[p, :, s].cpu(), Q.pack(vc[t], bits)), t
        written[p, s] = True
    assert (pages.k_codes.cpu().permute(0, 2, 1, 3)[~written] == 77).all() and (pages.v_scales.cpu().permute(0, 2, 1, 3)[~written] == -3).all()
    # a run that reads another run's cache writes nothing
    before = pages.k_codes.clone()
    K.qk_norm_rope_write_quantized(on(-wide)[:, :width], q_out, pages, on(qw), on(kw), 1e-6, None, rot, meta.positions,
                                   meta.entry_of_token, meta.block_tables[0], T, nq, False, st, cos_sin=on(cos_sin))
    assert torch.equal(pages.k_codes, before) and near_q(q_out, -want_q)


@pytest.mark.parametrize("D", [64, 96])
@pytest.mark.parametrize("bits", [4, 8])
def test_write_of_special_values(D, bits):
    """Infinities and NaN, groups of zeros, numbers near both ends, and the positive one of two alike."""
    nq, nkv, page = 1, 1, 4
    meta, table, n_pages = step([(0, 9)], page, 1)
    x = torch.randn(9, 3, D, generator=torch.Generator().manual_seed(1))
    x[0, 1:] = 0
    x[1, 1, 3], x[1, 1, 4], x[1, 2, 0] = math.nan, math.inf, -math.inf
    x[2, 1:] = 3e38
    x[3, 1:] = 1e-42
    x[4, 1:] *= 1e-38
    x[5, 1, 0], x[5, 1, 1] = 9.0, -9.0
    x[6, 1:] = -1.0
    x[7, 1:] *= 1e20
    x[8, 1:] = (torch.arange(D) % 8 - 4).float() / 2
    pages, st = K.QuantizedPages.zeros(n_pages, nkv, page, D, bits, DEV), status()
    q_out = torch.zeros(9, nq, D, device=DEV)
    K.qk_norm_rope_write_quantized(x.flatten(1).to(DEV), q_out, pages, None, None, 1e-6, None, 0, meta.positions, meta.entry_of_token,
                                   meta.block_tables[0], 9, nq, True, st)
    for got_c, got_s, rows in ((pages.k_codes, pages.k_scales, x[:, 1:2]), (pages.v_codes, pages.v_scales, x[:, 2:])):
        c, s = Q.quantise(rows, bits)
        for t in range(9):
            p = int(table[0, t // page])
            assert torch.equal(got_s[p, :, t % page].cpu(), s[t]), t
            assert torch.equal(got_c[p, :, t % page].cpu(), Q.pack(c[t], bits)), t


@pytest.mark.parametrize("D", [128, 96])
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
def test_write_to_a_page_that_is_not_there(D, bad):
    meta, table, n_pages = step([(0, 6), (0, 6)], 4, 2)
    table[1, 0] = bad
    x = torch.randn(12, 3 * D, device=DEV)
    pages, st = K.QuantizedPages.zeros(n_pages, 1, 4, D, 8, DEV), status()
    K.qk_norm_rope_write_quantized(x, torch.empty(12, 1, D, device=DEV), pages, None, None, 1e-6, None, 0, meta.positions,
                                   meta.entry_of_token, table.to(DEV), 12, 1, True, st)
    assert st.tolist() == [2, 0, 0, 0]
    touched = (pages.k_scales != 0).any(-1).any(1).sum()
    assert int(touched) == 6 + 2                            # the first entry's tokens and the second's beyond its first page


# ------------------------------------------------------------------ reading back
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("shape", [(128, 2, 16), (64, 3, 8), (256, 1, 4), (96, 2, 5), (32, 1, 1), (512, 1, 3), (160, 1, 16)])
def test_read(shape, bits, out):
    """The values in float32 are exact; in bfloat16 they are those rounded once."""
    D, nkv, page = shape
    pages, k, v = random_pages(7, nkv, page, D, bits, D)
    order = torch.tensor([3, 0, 6, -1, 3, 7, 1], dtype=torch.int32, device=DEV)
    k_out = torch.full((7, nkv, page, D), 5.0, dtype=out, device=DEV)
    v_out, st = k_out.clone(), status()
    K.read_quantized_pages(k_out, v_out, pages, order, st)
    assert st.tolist() == [3, 0, 0, 0]                      # page 7 is past the pool
    for i, p in enumerate(order.tolist()):
        for got, want in ((k_out, k), (v_out, v)):
            assert torch.equal(got[i].cpu(), want[p].to(F32).to(out) if 0 <= p < 7 else torch.zeros(nkv, page, D, dtype=out)), i
    K.read_quantized_pages(k_out[:0], v_out[:0], pages, order[:0], st)


def test_read_of_more_pages_than_a_grid_has_rows():
    pages, k, v = random_pages(5, 1, 1, 32, 4)
    order = (torch.arange(66000) * 7 % 5).int()
    k_out = torch.empty(66000, 1, 1, 32, device=DEV)
    v_out = torch.empty_like(k_out)
    K.read_quantized_pages(k_out, v_out, pages, order.to(DEV), status())
    assert torch.equal(k_out.cpu(), k[order.long()].float()) and torch.equal(v_out.cpu(), v[order.long()].float())


# ------------------------------------------------------------------ attention
def attend(pages, meta, q, nq, scale, window=None, st=None, **more):
    out, st = torch.full_like(q, 7.0), status() if st is None else st
    K.attention_quantized(out, q, pages, meta, meta.block_tables[0], nq, scale, window, st, **more)
    return out, st


def check(out, q, meta, table, k, v, layout, nkv, page, window, scale, read_back, lost=lambda e: 0.0):
    """bfloat16: a weight and the result are rounded (2^-8 each, relative), a weight is off by what float32 leaves of its score, and sums
    of codes of up to 255 steps are formed in float32; float32: the score's and the sums' roundings alone.
    ``read_back(e)``: entry e's keys and values are read back first, rounded to q's type: it is those that the result is checked with.
    ``lost(e)``: what a key may lose beside that.  (The kernel over codes adds products of a weight, a scale and a code in units of
    2^-85; float32 ends at 2^-149, so that each is off by 2^-64 at most, whatever it stands for.)"""
    unit = 2.0 ** -8 if q.dtype == BF16 else 0.0
    exact_k, exact_v, t = k, v, 0
    for e, (start, n) in enumerate(layout):
        if n == 0:
            continue
        k, v = (a.to(q.dtype).double() if read_back(e) else a for a in (exact_k, exact_v))
        at = table[e, :-(-(start + n) // page)].long()
        rows = lambda a: a[at].permute(0, 2, 1, 3).flatten(0, 1)[:start + n]       # noqa: E731
        want, mass = Q.attention(q[t:t + n].cpu(), rows(k), rows(v), start, window or 0, scale)
        got = out[t:t + n].double().cpu()
        far = (got - want).abs() - (2.0 * unit * mass + unit * want.abs() + 2.0 ** -13 * mass + 2.0 ** -20 * rows(v).abs().max() + lost(e) * (start + n))
        assert float(far.max()) <= 0, (e, start, n, float(far.max()))
        t += n


LAYOUTS = [[(0, 70), (130, 1), (5, 2), (63, 66), (300, 1)], [(0, 1), (1, 1), (15, 1), (16, 1), (255, 1), (256, 1), (257, 1), (700, 1)],
           [(0, 200)], [(100, 3), (0, 4), (64, 8), (127, 2)], [(1000, 1)], [(2600, 1), (3, 1)], [(40, 1), (0, 0), (77, 1)]]
SHAPES = [dict(D=128, nq=8, nkv=2, page=16), dict(D=64, nq=6, nkv=2, page=8), dict(D=256, nq=8, nkv=1, page=32), dict(D=128, nq=5, nkv=1, page=5),
          dict(D=64, nq=16, nkv=1, page=64), dict(D=128, nq=3, nkv=3, page=1), dict(D=96, nq=4, nkv=2, page=16), dict(D=128, nq=20, nkv=1, page=16)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window", [None, 37])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(f"{k}{v}" for k, v in s.items()))
def test_attention(shape, bits, window, dtype):
    D, nq, nkv, page = (shape[k] for k in ("D", "nq", "nkv", "page"))
    for li, layout in enumerate(LAYOUTS):
        meta, table, n_pages = step(layout, page, li, width=None if li % 2 else 200 if page > 8 else None)
        pages, k, v = random_pages(n_pages, nkv, page, D, bits, li)
        q = (2 * torch.randn(meta.tokens, nq, D, generator=torch.Generator().manual_seed(li))).to(dtype).to(DEV)
        long = dtype == BF16 and D in (64, 128) and page in (8, 16, 32, 64) and max(n for _, n in layout) >= 64
        for impl in (None, "direct", "read") + ("portion",) * long if dtype == BF16 and D != 96 else (None,):
            out, st = attend(pages, meta, q, nq, D ** -0.5, window, impl=impl)
            assert st.tolist() == [0, 0, 0, 0]
            form = impl or cache_quant._plan(out, q, pages, meta, meta.block_tables[0], nq)[0]
            assert (form == "read") == (dtype == F32 or D == 96 or impl == "read")
            check(out, q, meta, table, k, v, layout, nkv, page, window, D ** -0.5, lambda e: form == "read")
            again, _ = attend(pages, meta, q, nq, D ** -0.5, window, impl=impl)
            assert torch.equal(out, again)                 # no sum depends on which block ends first
