"""What the operators of the quantised cache are measured on: keys and values held in 8 or 4 bits, written as a step
makes them, read back, and attended to.

The cache of one layer is four arrays: ``codes`` (bytes) and ``scales`` (bfloat16) of keys and of values,

    codes  [pages, kv heads, page size, D * bits / 8]      scales [pages, kv heads, page size, D / 32]

A head's D channels form G = D / 32 groups of 32: channel c belongs to group (c // 4) % G.  With L = 2^(bits - 1), a
group's scale is s = bfloat16(m / -L), m the group's element of the largest magnitude (the positive one of two alike),
and the code of x is clamp(rint(x / s), -L, L - 1) + L; it stands for (code - L) * s.  Four-bit codes lie two to a byte,
the even channel in the low half.

Three operators, told apart by ``"does"``:

* ``write``: a step's projection rows -> queries with norm and rotation, keys and values into the cache; the pages it
  wrote to are then read back (as a prompt step does before its attention), so that what was stored is among the outputs.
* ``read``: pages of the cache -> keys and values in bfloat16 or float32.
* ``attend``: causal grouped-query attention of a step's tokens over the cache, for single tokens, a few tokens and
  portions of prompts, with or without a window.

Sizes are those of the benchmark's table of layers (1b, 4b), and heads of 64 and 256 channels as the tests have them.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
HEADS = {"1b": (16, 4, 128), "4b": (32, 8, 128), "narrow": (12, 2, 64), "wide": (8, 1, 256)}   # q heads, kv heads, D
PAGE = 16
SPREAD = 0.6180339887


# ---- the cases -------------------------------------------------------------------------------------------
def case(does, size, bits, requests, context, tokens, **more):
    """``requests`` texts of up to ``context`` tokens each in the cache, each bringing up to ``tokens`` new ones."""
    out = dict(does=does, size=size, bits=bits, requests=requests, context=context, tokens=tokens, ragged=False,
               dtype="bfloat16", norm=True, rotary=1.0, pad=0, window=0, prompts=0, prompt=0)
    out.update(more)
    return out


def listed():
    return [
        # eight requests decode: what one layer of their step writes; launches and latency
        dict(case("write", "4b", 4, 8, 2000, 1, ragged=True), name="write 8 tokens, 4 bits"),
        # the benchmark's prompt
        dict(case("write", "4b", 8, 1, 0, 2048), name="write 2048 tokens, 8 bits"),
        # three odd prompts on the 32-bit path, half of each head rotated, the projection's rows wider than its heads
        dict(case("write", "narrow", 4, 3, 50, 1277, ragged=True, dtype="float32", norm=False, rotary=0.5, pad=12),
             name="write 3 prompts, float32"),
        # a short text of a small model read back
        dict(case("read", "1b", 8, 1, 77, 0), name="read 77 tokens, 8 bits"),
        # all that eight long requests have cached
        dict(case("read", "4b", 4, 8, 8100, 0), name="read 8x8100, 4 bits"),
        # thirteen odd texts, for the 32-bit path
        dict(case("read", "narrow", 8, 13, 5003, 0, ragged=True, dtype="float32"), name="read 13 ragged, float32"),
        # one user, a short exchange with a small model: latency
        dict(case("attend", "1b", 4, 1, 76, 1), name="attend 1x77, 4 bits"),
        # one user behind a long document
        dict(case("attend", "4b", 4, 1, 65535, 1), name="attend 1x65536, 4 bits"),
        # the benchmark's headline: eight requests near the end of their context
        dict(case("attend", "4b", 4, 8, 8100, 1), name="attend 8x8101, 4 bits"),
        # a loaded server
        dict(case("attend", "4b", 8, 64, 2048, 1), name="attend 64x2049, 8 bits"),
        # a draft of a few tokens checked for each of thirteen odd requests, in layers that see a window
        dict(case("attend", "narrow", 4, 13, 5003, 4, ragged=True, window=1024), name="attend 13 ragged x4, window"),
        # a portion of a long prompt behind what is cached of it
        dict(case("attend", "4b", 4, 1, 4096, 2048), name="attend 2048 behind 4096"),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    does = rng.choice(["write", "read", "attend", "attend", "attend"])
    size = rng.choice(["1b", "4b", "4b", "narrow", "wide"])
    bits = rng.choice([4, 8])
    ragged = rng.random() < 0.6
    window = rng.choice([0, 0, 0, _log(rng, 16, 4000)])
    if does == "write":
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        plan = dict(ragged=ragged, dtype=dtype, norm=rng.random() < 0.7, rotary=rng.choice([1.0, 1.0, 0.5, 0.0]),
                    pad=rng.choice([0, 0, 8, 20]))
        if rng.random() < 0.5:
            return case("write", size, bits, _log(rng, 1, 64), _log(rng, 1, 8000), 1, **plan)
        n = rng.randint(1, 4)
        return case("write", size, bits, n, rng.choice([0, _log(rng, 1, 500)]), _log(rng, 9, 2048 // n), **plan)
    if does == "read":
        n = _log(rng, 1, 64)
        return case("read", size, bits, n, _log(rng, 16, 65536 // n), 0, ragged=ragged, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    kind = rng.choice(["decode", "decode", "few", "portion", "mixed"])
    if kind in ("decode", "few"):
        n = _log(rng, 1, 64)
        return case("attend", size, bits, n, _log(rng, 1, 65536 // n), 1 if kind == "decode" else rng.randint(2, 8), ragged=ragged,
                    window=window)
    if kind == "portion":
        n = rng.randint(1, 3)
        return case("attend", size, bits, n, _log(rng, 1, 4096), _log(rng, 40, 2048 // n), ragged=ragged, window=window)
    n, k = _log(rng, 1, 12), rng.randint(1, 3)
    return case("attend", size, bits, n, _log(rng, 16, 3001), 1, ragged=ragged, window=window, prompts=k, prompt=_log(rng, 17, 700 // k))


def _lengths(n, longest, ragged):
    """n lengths: all the longest, or spread between a tenth of it and all of it."""
    if not ragged or n == 0:
        return [longest] * n
    return [longest] + [max(min(longest, 1), int(longest * (0.1 + 0.9 * ((i * SPREAD) % 1.0)))) for i in range(1, n)]


def layout(c):
    """(cached tokens, new tokens) of every entry of the step."""
    starts = _lengths(c["requests"], c["context"], c["ragged"])
    new = _lengths(c["requests"], c["tokens"], c["ragged"] and c["tokens"] > 8)
    return list(zip(starts, new)) + [(0, n) for n in _lengths(c["prompts"], c["prompt"], c["ragged"])]


# ---- preparation -------------------------------------------------------------------------------------------
def _quantise(x, bits):
    """Codes (packed) and scales of x [..., D] in float32."""
    D = x.shape[-1]
    G, L = D // 32, 1 << (bits - 1)
    v = x.reshape(*x.shape[:-1], 8, G, 4)
    hi, lo = v.amax((-3, -1)), v.amin((-3, -1))
    scale = (torch.where(hi >= -lo, hi, lo) / -L).to(BF16)
    q = v / scale.float().unsqueeze(-2).unsqueeze(-1)
    q = torch.where(torch.isfinite(q), q, 0.0).round().clamp(-L, L - 1).add(L).to(torch.uint8).reshape(x.shape)
    if bits == 4:
        q = q[..., 0::2] | (q[..., 1::2] << 4)
    return q.contiguous(), scale.contiguous()


def _tables(lens, device, gen):
    """A block table with every entry's pages somewhere in a pool, and the pool's number of pages."""
    need = [-(-max(n, 1) // PAGE) for n in lens]
    n_pages = sum(need) + 3
    perm = torch.randperm(n_pages, generator=gen, device=device).to(torch.int32)
    width = max(need)
    first = torch.tensor([0] + need[:-1], device=device).cumsum(0)
    slot = torch.arange(width, device=device)
    at = first[:, None] + slot
    known = slot < torch.tensor(need, device=device)[:, None]
    table = torch.where(known, perm[torch.where(known, at, 0)], torch.tensor(-1, dtype=torch.int32, device=device))
    return table.contiguous(), n_pages


def prepare(c, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    nq, nkv, D = HEADS[c["size"]]
    rand = lambda *shape: torch.randn(*shape, generator=gen, device=device, dtype=F32)      # noqa: E731
    dev = lambda a: torch.tensor(a, dtype=torch.int32, device=device)                       # noqa: E731
    dtype = getattr(torch, c["dtype"])
    entries = layout(c)
    starts, new = [s for s, _ in entries], [n for _, n in entries]
    table, n_pages = _tables([s + n for s, n in entries], device, gen)
    s = SimpleNamespace(c=c, nq=nq, nkv=nkv, D=D, bits=c["bits"], table=table, dtype=dtype, scale=D ** -0.5,
                        status=torch.zeros(4, dtype=torch.int32, device=device))
    # keys keep a few loud channels, values a few loud tokens, as trained models have them
    loud = 1 + 3 * (torch.rand(nkv, 1, D, generator=gen, device=device) < 0.05)
    keys = rand(n_pages, nkv, PAGE, D) * loud
    values = rand(n_pages, nkv, PAGE, D) * (1 + 4 * (torch.rand(n_pages, nkv, PAGE, 1, generator=gen, device=device) < 0.02))
    s.k_codes, s.k_scales = _quantise(keys, s.bits)
    s.v_codes, s.v_scales = _quantise(values, s.bits)
    del keys, values
    T = sum(new)
    s.positions = dev([a + i for a, n in entries for i in range(n)])
    s.entry_of_token = dev([e for e, n in enumerate(new) for _ in range(n)])
    if c["does"] == "read":
        used = torch.arange(table.shape[1], device=device) < dev([-(-n // PAGE) for n in starts])[:, None]
        s.pages = table[used].contiguous()
        s.k_out = torch.empty(s.pages.numel(), nkv, PAGE, D, dtype=dtype, device=device)
        s.v_out = torch.empty_like(s.k_out)
        return s
    if c["does"] == "write":
        width = (nq + 2 * nkv) * D
        s.qkv = rand(T, width + c["pad"]).to(dtype)[:, :width]
        s.rot = int(D * c["rotary"])
        half = s.rot // 2
        angle = s.positions[:, None].to(F64) * torch.pow(1e6, -torch.arange(half, device=device, dtype=F64) / max(half, 1))
        s.cos_sin = torch.stack([angle.cos(), angle.sin()], -1).to(F32).contiguous() if s.rot else None
        s.q_norm = 1 + 0.2 * rand(D) if c["norm"] else None
        s.k_norm = 1 + 0.2 * rand(D) if c["norm"] else None
        s.q_out = torch.empty(T, nq, D, dtype=dtype, device=device)
        touched = table[s.entry_of_token.long(), (s.positions // PAGE).long()]
        s.pages = torch.unique(touched)
        s.k_out = torch.empty(s.pages.numel(), nkv, PAGE, D, dtype=BF16, device=device)
        s.v_out = torch.empty_like(s.k_out)
        return s
    s.q = (rand(T, nq, D) * (1 + 2 * torch.rand(nq, 1, generator=gen, device=device))).to(dtype)
    s.out = torch.empty_like(s.q)
    first = [0]
    for n in new:
        first.append(first[-1] + n)
    tiles = [(e, t) for e, n in enumerate(new) if n > 1 for t in range(0, n, 128)]
    s.meta = SimpleNamespace(tokens=T, entries=len(entries), q_lens=new, kv_lens=[a + n for a, n in entries], positions=s.positions,
                             entry_of_token=s.entry_of_token, q_start=dev(first), context_len=dev(starts),
                             prefill_work128=dev(tiles).view(-1, 2) if tiles else None, n_prefill_items128=len(tiles))
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------
def _values(codes, scales, bits, D):
    """What codes [..., D * bits / 8] and scales [..., D / 32] stand for, in float32."""
    G, L = D // 32, 1 << (bits - 1)
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    v = (codes.to(F32) - L).unflatten(-1, (8, G, 4)) * scales.to(F32).unsqueeze(-2).unsqueeze(-1)
    return v.flatten(-3)


def _plain_write(s):
    T = s.positions.numel()
    x = s.qkv.float().reshape(T, s.nq + 2 * s.nkv, s.D)
    q, k, v = x[:, :s.nq], x[:, s.nq:s.nq + s.nkv], x[:, s.nq + s.nkv:]

    def turned(h, w):
        if w is not None:           # (the sum of squares in 64 bits: a code's border is near for some element)
            mean = h.double().square().mean(-1, keepdim=True).float()
            h = h * (1 / (mean + 1e-6).sqrt()) * w
        if s.rot:
            a, b = h[..., :s.rot // 2], h[..., s.rot // 2:s.rot]
            cs, sn = s.cos_sin[:, None, :, 0], s.cos_sin[:, None, :, 1]
            h = torch.cat([a * cs - b * sn, b * cs + a * sn, h[..., s.rot:]], -1)
        return h

    page = s.table[s.entry_of_token.long(), (s.positions // PAGE).long()].long()
    slot = (s.positions % PAGE).long()
    k_codes, k_scales = _quantise(turned(k, s.k_norm), s.bits)
    v_codes, v_scales = _quantise(v, s.bits)
    s.k_codes[page, :, slot], s.k_scales[page, :, slot] = k_codes, k_scales
    s.v_codes[page, :, slot], s.v_scales[page, :, slot] = v_codes, v_scales
    return turned(q, s.q_norm).to(s.dtype), *_plain_read(s, BF16)


def _plain_read(s, dtype):
    at = s.pages.long()
    return (_values(s.k_codes[at], s.k_scales[at], s.bits, s.D).to(dtype),
            _values(s.v_codes[at], s.v_scales[at], s.bits, s.D).to(dtype))


def _plain_attend(s):
    m = s.meta
    E, most, W = m.entries, max(m.q_lens), s.table.shape[1]
    at = s.table.clamp(min=0).long()
    k = _values(s.k_codes[at], s.k_scales[at], s.bits, s.D).permute(0, 2, 1, 3, 4).reshape(E, s.nkv, W * PAGE, s.D)
    v = _values(s.v_codes[at], s.v_scales[at], s.bits, s.D).permute(0, 2, 1, 3, 4).reshape(E, s.nkv, W * PAGE, s.D)
    e = s.entry_of_token.long()
    i = (s.positions - m.context_len[e]).long()
    q = torch.zeros(E, most, s.nq, s.D, dtype=F32, device=s.q.device)
    q[e, i] = s.q.float()
    q = q.reshape(E, most, s.nkv, -1, s.D).permute(0, 2, 3, 1, 4)                          # [E, kv, group, tokens, D]
    group = q.shape[2]
    score = (q.reshape(E, s.nkv, group * most, s.D) @ k.transpose(2, 3)) * s.scale
    pos = m.context_len[:, None] + torch.arange(most, device=q.device)
    j = torch.arange(W * PAGE, device=q.device)
    seen = j <= pos[:, :, None]
    if s.c["window"]:
        seen &= j > pos[:, :, None] - s.c["window"]
    seen = seen[:, None, None]
    score = score.view(E, s.nkv, group, most, -1).masked_fill_(~seen, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p / p.sum(-1, keepdim=True)).reshape(E, s.nkv, group * most, -1) @ v
    out = out.view(E, s.nkv, group, most, s.D).permute(0, 3, 1, 2, 4).reshape(E, most, s.nq, s.D)
    return out[e, i].to(s.dtype)


def run(s):
    c = s.c
    if own:
        from kipp_b200 import kernels
        pages = kernels.QuantizedPages(s.k_codes, s.k_scales, s.v_codes, s.v_scales, s.bits)
        if c["does"] == "write":
            kernels.qk_norm_rope_write_quantized(s.qkv, s.q_out, pages, s.q_norm, s.k_norm, 1e-6, None, s.rot, s.positions,
                                                 s.entry_of_token, s.table, s.positions.numel(), s.nq, True, s.status,
                                                 cos_sin=s.cos_sin)
            kernels.read_quantized_pages(s.k_out, s.v_out, pages, s.pages, s.status)
            return s.q_out, s.k_out, s.v_out
        if c["does"] == "read":
            kernels.read_quantized_pages(s.k_out, s.v_out, pages, s.pages, s.status)
            return s.k_out, s.v_out
        kernels.attention_quantized(s.out, s.q, pages, s.meta, s.table, s.nq, s.scale, c["window"] or None, s.status)
        return s.out
    if c["does"] == "write":
        return _plain_write(s)
    if c["does"] == "read":
        return _plain_read(s, s.dtype)
    return _plain_attend(s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------
def work(c):
    nq, nkv, D = HEADS[c["size"]]
    es = 4 if c["dtype"] == "float32" else 2
    row = 2 * nkv * (D * c["bits"] // 8 + D // 16)             # a token's keys and values as they are held
    entries = layout(c)
    T = sum(n for _, n in entries)
    pages = lambda n: -(-n // PAGE)                            # noqa: E731
    if c["does"] == "read":
        n = sum(pages(s) for s, _ in entries) * PAGE
        return {"bytes": n * (row + 2 * nkv * D * es), "flops": 2 * n * 2 * nkv * D}
    if c["does"] == "write":
        n = sum(pages(s + k) - s // PAGE for s, k in entries) * PAGE
        made = T * ((2 * nq + 2 * nkv) * D * es + int(D * c["rotary"]) * 4 + row)
        return {"bytes": made + n * (row + 2 * nkv * D * 2), "flops": T * (nq + nkv) * D * 6 + T * 2 * nkv * D * 3 + 2 * n * 2 * nkv * D}
    w = c["window"] or 1 << 40
    held = sum(min(s + n, w + n - 1) for s, n in entries)
    seen = sum(sum(min(s + i + 1, w) for i in range(n)) for s, n in entries)
    return {"bytes": held * row + 2 * T * nq * D * es, "flops": 4 * seen * nq * D}


# ---- the same in 64 bits, entry by entry ------------------------------------------------------------------------
def _stand_for(codes, scales, bits):
    """Values of rows of codes by looking every channel up: [rows, D] in 64 bits."""
    rows = codes.shape[0]
    D = codes.shape[1] * 8 // bits
    channel = torch.arange(D, device=codes.device)
    if bits == 8:
        code = codes[:, channel].to(F64)
    else:
        code = ((codes[:, channel // 2].to(torch.int64) >> (4 * (channel % 2))) & 15).to(F64)
    group = (channel // 4) % (D // 32)
    return (code - 2 ** (bits - 1)) * scales.to(F64).reshape(rows, -1)[:, group]


def _rounded(x, bits):
    """What rows [rows, D] become in the cache, in 64 bits."""
    D = x.shape[1]
    group = (torch.arange(D, device=x.device) // 4) % (D // 32)
    L = 2.0 ** (bits - 1)
    out = torch.zeros_like(x)
    for g in range(D // 32):
        part = x[:, group == g]
        top, low = part.max(1).values, part.min(1).values
        scale = (torch.where(top >= -low, top, low) / -L).to(F32).to(BF16).to(F64)[:, None]
        safe = torch.where(scale == 0, torch.ones_like(scale), scale)
        out[:, group == g] = torch.clamp(torch.round(part / safe), -L, L - 1) * scale
    return out


def exact(c, seed):
    s = prepare(c, seed)
    if c["does"] == "attend" and work(c)["flops"] > 2e12:
        return None
    if c["does"] == "attend":
        out = torch.empty(s.q.shape, dtype=F64, device=s.q.device)
        at = 0
        for e, (start, n) in enumerate(layout(c)):
            total = start + n
            pages = s.table[e, :-(-total // PAGE)].long()
            pos = torch.arange(start, total, device=s.q.device)
            j = torch.arange(total, device=s.q.device)
            hidden = j[None] > pos[:, None]
            if c["window"]:
                hidden |= j[None] <= pos[:, None] - c["window"]
            for g in range(s.nkv):
                rows = lambda a: a[pages, g].reshape(pages.numel() * PAGE, -1)[:total]              # noqa: E731
                k = _stand_for(rows(s.k_codes), rows(s.k_scales), s.bits)
                v = _stand_for(rows(s.v_codes), rows(s.v_scales), s.bits)
                for h in range(g * (s.nq // s.nkv), (g + 1) * (s.nq // s.nkv)):
                    w = (s.q[at:at + n, h].to(F64) @ k.T) * s.scale
                    w[hidden] = -math.inf
                    out[at:at + n, h] = torch.softmax(w, 1) @ v
            at += n
        return out
    if c["does"] == "write":
        T = s.positions.numel()
        x = s.qkv.to(F64).reshape(T, -1, s.D)
        made = []
        for h in range(s.nq + s.nkv):
            y = x[:, h]
            w = s.q_norm if h < s.nq else s.k_norm
            if w is not None:
                y = y / torch.sqrt(y.pow(2).sum(1, keepdim=True) / s.D + 1e-6) * w.to(F64)
            if s.rot:
                half, y = s.rot // 2, y.clone()
                cs, sn = s.cos_sin[..., 0].to(F64), s.cos_sin[..., 1].to(F64)
                a, b = y[:, :half].clone(), y[:, half:s.rot].clone()
                y[:, :half], y[:, half:s.rot] = a * cs - b * sn, a * sn + b * cs
            made.append(y)
        q = torch.stack(made[:s.nq], 1)
        outs = []
        place = {int(p): i for i, p in enumerate(s.pages.tolist())}
        page = s.table[s.entry_of_token.long(), (s.positions // PAGE).long()].tolist()
        row = torch.tensor([place[p] for p in page], device=x.device)
        slot = (s.positions % PAGE).long()
        for codes, scales, heads in ((s.k_codes, s.k_scales, made[s.nq:]), (s.v_codes, s.v_scales, [x[:, s.nq + s.nkv + g] for g in range(s.nkv)])):
            full = _stand_for(codes[s.pages.long()].flatten(0, 2), scales[s.pages.long()].flatten(0, 2), s.bits)
            full = full.view(s.pages.numel(), s.nkv, PAGE, s.D)
            for g in range(s.nkv):
                full[row, g, slot] = _rounded(heads[g], s.bits)
            outs.append(full)
        return q, outs[0], outs[1]
    at = s.pages.long()
    return tuple(_stand_for(a[at].flatten(0, 2), b[at].flatten(0, 2), s.bits).view(at.numel(), s.nkv, PAGE, s.D)
                 for a, b in ((s.k_codes, s.k_scales), (s.v_codes, s.v_scales)))
