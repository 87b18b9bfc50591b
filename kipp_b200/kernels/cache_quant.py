"""The quantised cache: keys and values held in 8 or 4 bits (layout and rounding: csrc/quant_format.cuh).

``qk_norm_rope_write_quantized`` is ``qk_norm_rope_write`` into such a cache, ``read_quantized_pages`` brings
pages of it back, ``attention_quantized`` is ``attention`` over it."""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from .ops import KernelError, _check, _fn, _ptr, c_float, c_int, c_void_p, dtype_code, rope_table

c_ll, c_char_p = ctypes.c_longlong, ctypes.c_char_p
READ_BYTES = 1 << 30          # most bytes of keys and values that attention reads back at a time (one entry's, where those are more)


class QuantizedPages:
    """One run's cache: codes uint8 ``[pages, n_kv, page_size, D * bits / 8]`` and scales bfloat16
    ``[pages, n_kv, page_size, D / 32]`` of keys and of values.  D is a multiple of 32, at most 512.  Launches go by the addresses
    that the tensors have when the object is made: they may be written to, but not exchanged, moved or resized."""

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor, bits: int):
        if bits != 4 and bits != 8:
            raise KernelError(f"a quantised cache holds 8 or 4 bits, not {bits}")
        u8, bf16 = torch.uint8, torch.bfloat16
        if k_codes.dtype != u8 or v_codes.dtype != u8 or k_scales.dtype != bf16 or v_scales.dtype != bf16:
            raise KernelError("QuantizedPages: codes are uint8 and scales bfloat16")
        shape, device = k_codes.shape, k_codes.get_device()
        if len(shape) != 4:
            raise KernelError("QuantizedPages: codes and scales are [pages, n_kv, page_size, ..]")
        n_pages, n_kv, page_size, row = shape
        D = row * 8 // bits
        if D % 32 or D > 512 or n_pages <= 0 or n_kv <= 0 or page_size <= 0 or D <= 0:
            raise KernelError(f"QuantizedPages: {n_pages} pages, {n_kv} heads, {page_size} tokens a page, {D} channels a head: heads are a "
                              "multiple of 32 channels, at most 512")
        s_shape = (n_pages, n_kv, page_size, D // 32)
        if v_codes.shape != shape or k_scales.shape != s_shape or v_scales.shape != s_shape:
            raise KernelError(f"QuantizedPages: keys and values must be alike, with scales {s_shape}")
        if not (k_codes.is_contiguous() and k_scales.is_contiguous() and v_codes.is_contiguous() and v_scales.is_contiguous()):
            raise KernelError("QuantizedPages: codes and scales must be contiguous")
        if k_scales.get_device() != device or v_codes.get_device() != device or v_scales.get_device() != device:
            raise KernelError("QuantizedPages: codes and scales must be on one device")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales, self.bits = k_codes, k_scales, v_codes, v_scales, bits
        self.n_pages, self.n_kv, self.page_size, self.head_dim = n_pages, n_kv, page_size, D
        self.device_index = device
        # (what a launch is given: the tensors are held, so the addresses stay)
        self.addresses = a, b, c, d = k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr()
        self.aligned = (a | b | c | d) % 16 == 0

    @classmethod
    def zeros(cls, n_pages: int, n_kv: int, page_size: int, head_dim: int, bits: int, device) -> "QuantizedPages":
        if bits not in (4, 8) or head_dim <= 0 or head_dim % 32:
            raise KernelError(f"a quantised cache holds 8 or 4 bits of heads of a multiple of 32 channels, not {bits} of {head_dim}")
        codes = lambda: torch.zeros(n_pages, n_kv, page_size, head_dim * bits // 8, dtype=torch.uint8, device=device)   # noqa: E731
        scales = lambda: torch.zeros(n_pages, n_kv, page_size, head_dim // 32, dtype=torch.bfloat16, device=device)     # noqa: E731
        return cls(codes(), scales(), codes(), scales(), bits)


_current_device, _current_stream, _I32 = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream, torch.int32


def _launch_stream(what: str, device: int, *tensors: torch.Tensor) -> int:
    """The current stream; every tensor must lie on the current device, where a launch goes whatever the tensors' own."""
    if device < 0:
        raise KernelError("kernels need CUDA tensors; there is no CPU path")
    for t in tensors:
        if t.get_device() != device:
            raise KernelError(f"{what}: the tensors are on several devices")
    if device != _current_device():
        raise KernelError(f"{what}: the tensors are on cuda:{device} and the current device is cuda:{_current_device()}")
    return _current_stream(device)


def _status(status: torch.Tensor, what: str) -> None:
    if status.dtype is not _I32 or status.numel() < 4 or not status.is_contiguous():
        raise KernelError(f"{what}: status must be a contiguous int32 tensor of 4 words")


def _lists(what: str, names: str, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype is not _I32 or not t.is_contiguous():
            raise KernelError(f"{what}: {names} must be contiguous int32 tensors")


# the structures of the C entry points (csrc/cache_quant.cu, csrc/attention_quant.cu): addresses, then sizes
_WRITE, _READ, _READ_ENTRIES, _ATTEND = (struct.Struct(f) for f in ("14Qq12if", "9Q7i", "13Q10i", "12Qq10if"))


_entries: dict = {}


def _call(lib: str, name: str, packed: bytes, what: str) -> None:
    f = _entries.get(name)
    if f is None:
        f = _entries[name] = _fn(lib, name, [c_char_p])
    _check(f(packed), what)


def qk_norm_rope_write_quantized(qkv: torch.Tensor, q_out: torch.Tensor, pages: QuantizedPages, q_norm_w: Optional[torch.Tensor],
                                 k_norm_w: Optional[torch.Tensor], eps: float, inv_freq: Optional[torch.Tensor], rotary_dim: int,
                                 positions: torch.Tensor, entry_of_token: torch.Tensor, block_table: torch.Tensor, tokens: int,
                                 n_q: int, write_cache: bool, status: torch.Tensor,
                                 cos_sin: Optional[torch.Tensor] = None) -> None:
    """Per-head RMSNorm of q and k, rotation, q to ``q_out`` [T, n_q, D], k and v as codes into ``pages`` through
    ``block_table`` [entries, width].  ``cos_sin`` is the step's ``rope_table``; without it the table is made here.
    A position whose page is not mapped is not written: status word 0 becomes 2.  Two tokens of a step must not have one place in the
    cache."""
    what, D, n_kv = "qk_norm_rope_write_quantized", pages.head_dim, pages.n_kv
    shape, dtype, q_norm, k_norm, table, norm_dtype = qkv.shape, qkv.dtype, 0, 0, 0, 0
    if len(shape) != 2 or shape[1] != (n_q + 2 * n_kv) * D or shape[0] < tokens:
        raise KernelError(f"{what}: qkv has the wrong shape")
    ld, one = qkv.stride()
    if one != 1:
        raise KernelError(f"{what}: qkv's rows must be contiguous")
    if shape[0] == 1:             # (the stride of a lone row says nothing)
        ld = shape[1]
    if q_out.dtype != dtype or not q_out.is_contiguous() or q_out.numel() < tokens * n_q * D:
        raise KernelError(f"{what}: q_out must be contiguous, of qkv's dtype and hold every query")
    _lists(what, "positions, entry_of_token and block_table", positions, entry_of_token, block_table)
    if positions.numel() < tokens or entry_of_token.numel() < tokens or block_table.dim() != 2:
        raise KernelError(f"{what}: a position and an entry for every token, and a table [entries, width]")
    if (q_norm_w is None) != (k_norm_w is None):
        raise KernelError(f"{what}: q and k norm weights must come together")
    device = pages.device_index
    if q_norm_w is None:
        stream = _launch_stream(what, device, qkv, q_out, positions, entry_of_token, block_table, status)
    else:
        stream = _launch_stream(what, device, qkv, q_out, positions, entry_of_token, block_table, status, q_norm_w, k_norm_w)
        if q_norm_w.dtype != k_norm_w.dtype or q_norm_w.numel() != D or k_norm_w.numel() != D or \
                not (q_norm_w.is_contiguous() and k_norm_w.is_contiguous()):
            raise KernelError(f"{what}: norm weights must be contiguous, alike and of the head's size")
        norm_dtype, q_norm, k_norm = dtype_code(q_norm_w.dtype), q_norm_w.data_ptr(), k_norm_w.data_ptr()
    if rotary_dim < 0 or rotary_dim % 2 or rotary_dim > D:
        raise KernelError(f"{what}: rotary_dim must be even and at most the head's size")
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.numel() * 2 != rotary_dim):
        raise KernelError(f"{what}: inv_freq must be float32 [rotary_dim / 2]")
    if rotary_dim > 0:
        if cos_sin is None:
            if inv_freq is None:
                raise KernelError(f"{what}: a rotation needs cos_sin or inv_freq")
            cos_sin = rope_table(positions, inv_freq, tokens)
        if cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous() or cos_sin.numel() < tokens * rotary_dim or \
                cos_sin.get_device() != device:
            raise KernelError(f"{what}: cos_sin must be contiguous float32 [tokens, rotary_dim / 2, 2] on the step's device")
        table = cos_sin.data_ptr()
    _status(status, what)
    _call("cache_quant", "kipp_quant_cache_write",
          _WRITE.pack(qkv.data_ptr(), q_out.data_ptr(), *pages.addresses, q_norm, k_norm, table, positions.data_ptr(),
                      entry_of_token.data_ptr(), block_table.data_ptr(), status.data_ptr(), stream, ld, pages.bits, pages.n_pages,
                      pages.page_size, dtype_code(dtype), norm_dtype, rotary_dim, block_table.shape[1], tokens, n_q, n_kv, D,
                      1 if write_cache else 0, eps), what)


def read_quantized_pages(k_out: torch.Tensor, v_out: torch.Tensor, pages: QuantizedPages, page_list: torch.Tensor,
                         status: torch.Tensor) -> None:
    """What the pages of ``page_list`` (int32, any number, any order) stand for, in bfloat16 or float32:
    ``k_out``, ``v_out`` [len(page_list), n_kv, page_size, D].  A negative number gives zeros, one past the
    pool zeros and status word 0 = 3."""
    what, n = "read_quantized_pages", page_list.numel()
    _lists(what, "page_list", page_list)
    shape = (n, pages.n_kv, pages.page_size, pages.head_dim)
    if k_out.shape != shape or v_out.shape != shape or k_out.dtype != v_out.dtype or not (k_out.is_contiguous() and v_out.is_contiguous()):
        raise KernelError(f"{what}: k_out and v_out must be contiguous, of one dtype and {shape}")
    _status(status, what)
    stream = _launch_stream(what, pages.device_index, k_out, v_out, page_list, status)
    _call("cache_quant", "kipp_quant_cache_read",
          _READ.pack(k_out.data_ptr(), v_out.data_ptr(), *pages.addresses, page_list.data_ptr(), status.data_ptr(), stream,
                     dtype_code(k_out.dtype), pages.bits, pages.n_pages, pages.page_size, n, pages.n_kv, pages.head_dim), what)


def _read_entries(pages: QuantizedPages, dtype: torch.dtype, meta, block_table: torch.Tensor, first: int, entries: int, window: int,
                  status: torch.Tensor, table: torch.Tensor, stream: int, factors: Optional[torch.Tensor] = None):
    """Pages of what ``entries`` entries from ``first`` on see, in ``dtype``, and their rows of ``table``.  With ``factors`` (float32
    [entries of the step, n_kv, 2], made here) the pages' 16 bits are float16, multiplied by those, and entries of one token are left out."""
    width = block_table.shape[1]
    k = torch.empty((entries * width, pages.n_kv, pages.page_size, pages.head_dim), dtype=dtype, device=table.device)
    v = torch.empty_like(k)
    _call("cache_quant", "kipp_quant_cache_read_entries",
          _READ_ENTRIES.pack(k.data_ptr(), v.data_ptr(), table.data_ptr(), *pages.addresses, meta.q_start.data_ptr(),
                             meta.context_len.data_ptr(), block_table.data_ptr(), status.data_ptr(), 0 if factors is None else factors.data_ptr(), stream,
                             dtype_code(dtype), pages.bits, pages.n_pages, pages.page_size, width, first, entries, window, pages.n_kv, pages.head_dim), "read_entries")
    return k, v


def _entries_at_once(pages: QuantizedPages, dtype: torch.dtype, width: int) -> int:
    """How many entries' pages may be read back together."""
    per = 2 * pages.n_kv * pages.page_size * pages.head_dim * dtype.itemsize * width
    return max(1, READ_BYTES // per)


PORTION_MIN = 64              # the longest entry's tokens from which on reading back for the prompt kernel may pay


def _portions_pay(q_lens, n_q: int, n_kv: int) -> bool:
    """Whether the entries of more than one token are read back for the prompt kernel of 128-token tiles, or run on the codes.  Per
    cached key the codes cost 4 ps a query; a wave of 296 tiles costs as much as 4,096 of them, however full it is, and reading back
    a key of a kv head as 64.  32 query and 8 key heads of 128: 64 and 128 tokens behind 4,096 keys 38 and 67 us on the codes, 91 and
    67 read back; four entries of 32 and 64 behind 2,048 (8 bits) 50 and 75, 62 and 62; 12 heads of 64, 64 tokens 10 and 27."""
    several = [n for n in q_lens if n > 1]
    tiles = sum((n + 127) // 128 for n in several)
    return n_q * sum(several) > 4096 * -(-n_q * tiles // 296) + 64 * n_kv * len(several)


_supported: dict = {}
_scratch_bytes: dict = {}


def _direct_ok(out: torch.Tensor, q: torch.Tensor, pages: QuantizedPages, n_q: int) -> bool:
    key = (pages.bits, pages.head_dim, n_q, pages.n_kv)
    if key not in _supported:
        _supported[key] = bool(_fn("attention_quant", "kipp_attn_quant_supported", [c_int] * 4)(*key))
    return q.dtype == torch.bfloat16 and _supported[key] and pages.aligned and (q.data_ptr() | out.data_ptr()) % 16 == 0


def _tiles_ok(meta, device: int) -> bool:
    """Whether the step has a list of 128-token tiles that can be that of every entry of more than one token."""
    work = getattr(meta, "prefill_work128", None)
    if work is None or work.dtype is not _I32 or not work.is_contiguous() or work.get_device() != device:
        return False
    tiles = sum((n + 127) // 128 for n in meta.q_lens if n > 1)
    return getattr(meta, "n_prefill_items128", 0) == tiles and work.numel() >= 2 * tiles


def _portion_chunks(q, pages, meta, block_table, n_q, scale):
    """The entries of more than one token as (first, number) of runs whose pages may be read back together, where the prompt kernel
    takes them and the step's list of tiles is theirs, or None.  (Entries of one token may lie between; they count as room, and are left out.)"""
    if not scale > 0:
        return None
    several = [e for e, n in enumerate(meta.q_lens) if n > 1]
    if not several or not _tiles_ok(meta, pages.device_index):
        return None
    from . import attention_bf16
    if not attention_bf16.prefill_tc_supported(pages.head_dim, n_q, pages.n_kv, pages.page_size):
        return None
    most, chunks = _entries_at_once(pages, q.dtype, block_table.shape[1]), []
    for e in several:
        if chunks and e - chunks[-1][0] < most:
            chunks[-1] = (chunks[-1][0], e + 1 - chunks[-1][0])
        else:
            chunks.append((e, 1))
    return chunks


def _plan(out, q, pages, meta, block_table, n_q, scale=1.0):
    """(form of the entries of one token, form of the others, the runs of entries that portions are read back in):
    forms "direct" (the kernel over codes), "portion" (read back, tcgen05 prompt kernel, for positive scales) and "read" (read back, CUDA cores).
    The prompt kernel reads a key and a value once for 128 tokens, the kernel over codes once for 8 or 16 columns."""
    if not _direct_ok(out, q, pages, n_q):
        return "read", "read", None
    if max(meta.q_lens) >= PORTION_MIN and _portions_pay(meta.q_lens, n_q, pages.n_kv):
        chunks = _portion_chunks(q, pages, meta, block_table, n_q, scale)
        if chunks is not None:
            return "direct", "portion", chunks
    return "direct", "direct", None


def attention_quantized(out: torch.Tensor, q: torch.Tensor, pages: QuantizedPages, meta, block_table: torch.Tensor, n_q: int,
                        scale: float, window: Optional[int], status: torch.Tensor, impl: Optional[str] = None) -> None:
    """Causal grouped-query attention of the step's tokens over a quantised cache.

    ``meta`` is the step's metadata as for ``attention`` (``tokens``, ``q_lens``, ``positions``, ``entry_of_token``,
    ``q_start``, ``context_len``, and for steps with entries of 64 tokens or more the list of the 128-token tiles of every entry of more
    than one token, ``prefill_work128`` int32 [tiles, (entry, first token)] in any order, and ``n_prefill_items128``; a step without
    that list, or with one of another length, stays on the codes).  bfloat16 with heads of 64, 128 or 256 runs on the codes themselves; long
    portions of prompts, other heads and float32 on pages that are read back.  A page that is not mapped, or past the pool, sets
    status word 0 to 3.  On the codes a weight is rounded to bfloat16 with its value's scale, in portions to float16, and the result
    to bfloat16; beside that a result is off by up to 2^-64 a key on the codes (values of 2^-40 and less feel it), and queries of 2^80 and
    more count as infinite there.  ``impl`` forces a form:
    "direct" or "read" for the whole step, "portion" (long portions') for every entry of more than one token."""
    what, D, n_kv, q_lens, tokens = "attention_quantized", pages.head_dim, pages.n_kv, meta.q_lens, meta.tokens
    window = int(window or 0)
    shape, entries, dtype = q.shape, len(q_lens), q.dtype
    dtype_code(dtype)
    if len(shape) != 3:
        raise KernelError(f"{what}: q must be [tokens, n_q, head_dim]")
    rows, heads, dims = shape
    if heads != n_q or dims != D or rows < tokens or n_q % n_kv or not q.is_contiguous():
        raise KernelError(f"{what}: q must be contiguous [tokens, n_q, head_dim] with n_q a multiple of the cache's heads")
    if out.dtype is not dtype or out.shape != shape or not out.is_contiguous():
        raise KernelError(f"{what}: out must be contiguous, of q's dtype and shape")
    if not 0 <= window < 1 << 31:
        raise KernelError(f"{what}: a window of {window} tokens")
    t_shape, q_start, context_len = block_table.shape, meta.q_start, meta.context_len
    if len(t_shape) != 2 or t_shape[0] < entries or t_shape[1] == 0 or sum(q_lens) != tokens:
        raise KernelError(f"{what}: a row of block_table for every entry, and as many tokens as the entries bring")
    _lists(what, "block_table, q_start and context_len", block_table, q_start, context_len)
    if q_start.numel() <= entries or context_len.numel() < entries:
        raise KernelError(f"{what}: the step's lists are shorter than the step")
    _status(status, what)
    stream = _launch_stream(what, pages.device_index, q, out, block_table, q_start, context_len, status)
    if tokens == 0:
        return
    if impl is None:
        single, several, chunks = _plan(out, q, pages, meta, block_table, n_q, scale)
    elif impl == "portion":
        single, several, chunks = "direct", "portion", _portion_chunks(q, pages, meta, block_table, n_q, scale)
        if chunks is None or not _direct_ok(out, q, pages, n_q):
            raise KernelError(f"{what}: portions are read back for bfloat16 heads of 64 or 128, 16-byte aligned, a positive scale and a "
                              "list of the 128-token tiles of every entry of more than one token")
    elif impl in ("direct", "read"):
        single, several, chunks = impl, impl, None
        if impl == "direct" and not _direct_ok(out, q, pages, n_q):
            raise KernelError(f"{what}: the kernel over codes takes bfloat16 heads of 64, 128 or 256, 16-byte aligned")
    else:
        raise KernelError(f"unknown attention implementation {impl!r}")
    if single == "read":
        _by_reading(out, q, pages, meta, block_table, n_q, scale, window, status, stream)
        return
    if several == "direct":
        _direct(out, q, pages, meta, block_table, n_q, scale, window, status, max(q_lens), stream)
        return
    if 1 in q_lens:
        _direct(out, q, pages, meta, block_table, n_q, scale, window, status, 1, stream)
    table = torch.empty_like(block_table)
    for first, entries in chunks:
        _portions(out, q, pages, meta, block_table, n_q, scale, window, status, first, entries, table, stream)


def _direct(out, q, pages, meta, block_table, n_q, scale, window, status, most: int, stream: int) -> None:
    """The entries of up to ``most`` tokens, over the codes."""
    D, width = pages.head_dim, block_table.shape[1]
    key = (D, width * pages.page_size)
    need = _scratch_bytes.get(key)
    if need is None:
        need = _scratch_bytes[key] = _fn("attention_quant", "kipp_attn_quant_scratch_bytes", [c_int, c_ll], restype=c_ll)(*key)
    # (a block of the caching allocator's, of q's type: new_empty is its cheapest way there)
    scratch = q.new_empty((need + 1) // 2) if need else None
    _call("attention_quant", "kipp_attn_quant",
          _ATTEND.pack(out.data_ptr(), q.data_ptr(), *pages.addresses, meta.q_start.data_ptr(), meta.context_len.data_ptr(),
                       block_table.data_ptr(), scratch.data_ptr() if need else 0, status.data_ptr(), stream, need, pages.bits, pages.n_pages,
                       pages.page_size, width, len(meta.q_lens), most, n_q, pages.n_kv, D, window, scale), "attn_quant")


def _portions(out, q, pages, meta, block_table, n_q, scale, window, status, first: int, entries: int, table, stream: int) -> None:
    """Those of ``entries`` entries from ``first`` on that bring more than one token: their pages read back as float16, and the prompt
    kernel over those."""
    factors = torch.empty((len(meta.q_lens), pages.n_kv, 2), dtype=torch.float32, device=q.device)
    k, v = _read_entries(pages, q.dtype, meta, block_table, first, entries, window, status, table, stream, factors)
    f = _fn("attention_tc", "kipp_attn_prefill_tc_half",
            [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int,
             c_void_p, c_int, c_int, c_int, c_int, c_float, c_int, c_void_p, c_int, c_int, c_void_p, c_void_p])
    _check(f(out.data_ptr(), q.data_ptr(), q.shape[0], k.data_ptr(), v.data_ptr(), k.shape[0], meta.q_start.data_ptr(),
             meta.context_len.data_ptr(), table.data_ptr(), table.shape[1], pages.page_size, _ptr(meta.prefill_work128),
             meta.n_prefill_items128, n_q, pages.n_kv, pages.head_dim, scale, window, factors.data_ptr(), first, entries, status.data_ptr(),
             stream), "attn_prefill_tc")


def _by_reading(out, q, pages, meta, block_table, n_q, scale, window, status, stream: int) -> None:
    """Every entry's pages read back, as many entries at a time as READ_BYTES allow, and the attention over them."""
    _lists("attention_quantized", "positions and entry_of_token", meta.positions, meta.entry_of_token)
    if min(meta.positions.numel(), meta.entry_of_token.numel()) < meta.tokens:
        raise KernelError("attention_quantized: the step's lists are shorter than the step")
    _launch_stream("attention_quantized", pages.device_index, meta.positions, meta.entry_of_token)
    D, n_kv, width = pages.head_dim, pages.n_kv, block_table.shape[1]
    table = torch.empty_like(block_table)
    step, at = _entries_at_once(pages, q.dtype, width), 0
    for first in range(0, len(meta.q_lens), step):
        lens = meta.q_lens[first:first + step]
        n = sum(lens)
        if n == 0:
            continue
        k, v = _read_entries(pages, q.dtype, meta, block_table, first, len(lens), window, status, table, stream)
        f = _fn("attention_simt", "kipp_paged_attention_simt",
                [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_int,
                 c_float, c_int, c_void_p, c_void_p])
        _check(f(_ptr(out[at:]), _ptr(q[at:]), _ptr(k), _ptr(v), dtype_code(q.dtype), _ptr(meta.positions[at:]), _ptr(meta.entry_of_token[at:]),
                 _ptr(table), width, pages.page_size, n, n_q, n_kv, D, float(scale), window, _ptr(status), stream), "attention_simt")
        at += n
