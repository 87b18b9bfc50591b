"""The quantised cache: keys and values held in 8 or 4 bits (layout and rounding: csrc/quant_format.cuh).

``qk_norm_rope_write_quantized`` is ``qk_norm_rope_write`` into such a cache, ``read_quantized_pages`` brings
pages of it back, ``attention_quantized`` is ``attention`` over it."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from .ops import KernelError, _check, _fn, _int32, _ptr, _stream, c_float, c_int, c_void_p, dtype_code, rope_table

c_ll = ctypes.c_longlong
READ_BYTES = 1 << 30          # most bytes of keys and values that attention reads back at a time


class QuantizedPages:
    """One run's cache: codes uint8 ``[pages, n_kv, page_size, D * bits / 8]`` and scales bfloat16
    ``[pages, n_kv, page_size, D / 32]`` of keys and of values.  D is a multiple of 32, at most 512."""

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor, bits: int):
        if bits not in (4, 8):
            raise KernelError(f"a quantised cache holds 8 or 4 bits, not {bits}")
        for codes, scales in ((k_codes, k_scales), (v_codes, v_scales)):
            if codes.dtype != torch.uint8 or scales.dtype != torch.bfloat16 or codes.dim() != 4 or scales.dim() != 4:
                raise KernelError("QuantizedPages: codes are uint8 and scales bfloat16, [pages, n_kv, page_size, ..] each")
            if not codes.is_contiguous() or not scales.is_contiguous() or codes.shape[:3] != scales.shape[:3] or \
                    codes.device != scales.device:
                raise KernelError("QuantizedPages: codes and scales must be contiguous, of the same pages and on one device")
        if k_codes.shape != v_codes.shape or k_scales.shape != v_scales.shape or k_codes.device != v_codes.device:
            raise KernelError("QuantizedPages: keys and values must be alike")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales, self.bits = k_codes, k_scales, v_codes, v_scales, bits
        self.n_pages, self.n_kv, self.page_size = k_codes.shape[:3]
        self.head_dim = k_codes.shape[3] * 8 // bits
        if self.head_dim % 32 or self.head_dim > 512 or self.head_dim == 0 or k_scales.shape[3] * 32 != self.head_dim:
            raise KernelError(f"QuantizedPages: {self.head_dim} channels and {k_scales.shape[3]} scales a head; heads are a multiple of "
                              "32 channels, at most 512, with a scale for every 32")
        if min(self.n_pages, self.n_kv, self.page_size) <= 0:
            raise KernelError("QuantizedPages: no pages")

    @classmethod
    def zeros(cls, n_pages: int, n_kv: int, page_size: int, head_dim: int, bits: int, device) -> "QuantizedPages":
        if bits not in (4, 8) or head_dim <= 0 or head_dim % 32:
            raise KernelError(f"a quantised cache holds 8 or 4 bits of heads of a multiple of 32 channels, not {bits} of {head_dim}")
        codes = lambda: torch.zeros(n_pages, n_kv, page_size, head_dim * bits // 8, dtype=torch.uint8, device=device)   # noqa: E731
        scales = lambda: torch.zeros(n_pages, n_kv, page_size, head_dim // 32, dtype=torch.bfloat16, device=device)     # noqa: E731
        return cls(codes(), scales(), codes(), scales(), bits)

    def pointers(self) -> tuple:
        return _ptr(self.k_codes), _ptr(self.k_scales), _ptr(self.v_codes), _ptr(self.v_scales), self.bits, self.n_pages, self.page_size


def _on(device: torch.device, what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Everything lies on the current device: a launch goes there, whatever the tensors' own."""
    if device.type != "cuda":
        raise KernelError("kernels need CUDA tensors; there is no CPU path")
    if any(t is not None and t.device != device for t in tensors):
        raise KernelError(f"{what}: the tensors are on several devices")
    if device.index != torch.cuda.current_device():
        raise KernelError(f"{what}: the tensors are on {device} and the current device is cuda:{torch.cuda.current_device()}")


def _status(status: torch.Tensor, what: str) -> None:
    if status.dtype != torch.int32 or status.numel() < 4 or not status.is_contiguous():
        raise KernelError(f"{what}: status must be a contiguous int32 tensor of 4 words")


def qk_norm_rope_write_quantized(qkv: torch.Tensor, q_out: torch.Tensor, pages: QuantizedPages, q_norm_w: Optional[torch.Tensor],
                                 k_norm_w: Optional[torch.Tensor], eps: float, inv_freq: Optional[torch.Tensor], rotary_dim: int,
                                 positions: torch.Tensor, entry_of_token: torch.Tensor, block_table: torch.Tensor, tokens: int,
                                 n_q: int, write_cache: bool, status: torch.Tensor,
                                 cos_sin: Optional[torch.Tensor] = None) -> None:
    """Per-head RMSNorm of q and k, rotation, q to ``q_out`` [T, n_q, D], k and v as codes into ``pages`` through
    ``block_table`` [entries, width].  ``cos_sin`` is the step's ``rope_table``; without it the table is made here.
    A position whose page is not mapped is not written: status word 0 becomes 2."""
    what, D, n_kv = "qk_norm_rope_write_quantized", pages.head_dim, pages.n_kv
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.shape[1] != (n_q + 2 * n_kv) * D or qkv.shape[0] < tokens:
        raise KernelError(f"{what}: qkv has the wrong shape")
    if q_out.dtype != qkv.dtype or not q_out.is_contiguous() or q_out.numel() < tokens * n_q * D:
        raise KernelError(f"{what}: q_out must be contiguous, of qkv's dtype and hold every query")
    for t, name in ((positions, "positions"), (entry_of_token, "entry_of_token"), (block_table, "block_table")):
        _int32(t, name)
    if positions.numel() < tokens or entry_of_token.numel() < tokens or block_table.dim() != 2:
        raise KernelError(f"{what}: a position and an entry for every token, and a table [entries, width]")
    norm_dtype = 0
    if (q_norm_w is None) != (k_norm_w is None):
        raise KernelError(f"{what}: q and k norm weights must come together")
    if q_norm_w is not None:
        if q_norm_w.dtype != k_norm_w.dtype or q_norm_w.numel() != D or k_norm_w.numel() != D or \
                not (q_norm_w.is_contiguous() and k_norm_w.is_contiguous()):
            raise KernelError(f"{what}: norm weights must be contiguous, alike and of the head's size")
        norm_dtype = dtype_code(q_norm_w.dtype)
    if rotary_dim < 0 or rotary_dim % 2 or rotary_dim > D:
        raise KernelError(f"{what}: rotary_dim must be even and at most the head's size")
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.numel() * 2 != rotary_dim):
        raise KernelError(f"{what}: inv_freq must be float32 [rotary_dim / 2]")
    if rotary_dim > 0 and cos_sin is None:
        if inv_freq is None:
            raise KernelError(f"{what}: a rotation needs cos_sin or inv_freq")
        cos_sin = rope_table(positions, inv_freq, tokens)
    if rotary_dim > 0 and (cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous() or cos_sin.numel() < tokens * rotary_dim):
        raise KernelError(f"{what}: cos_sin must be contiguous float32 [tokens, rotary_dim / 2, 2]")
    _status(status, what)
    _on(qkv.device, what, q_out, pages.k_codes, q_norm_w, k_norm_w, positions, entry_of_token, block_table, cos_sin, status)
    f = _fn("cache_quant", "kipp_quant_cache_write",
            [c_void_p, c_ll, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_int,
             c_float, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p])
    _check(f(_ptr(qkv), qkv.stride(0), _ptr(q_out), *pages.pointers(), dtype_code(qkv.dtype), _ptr(q_norm_w), _ptr(k_norm_w), norm_dtype,
             float(eps), _ptr(cos_sin) if rotary_dim else None, rotary_dim, _ptr(positions), _ptr(entry_of_token), _ptr(block_table),
             block_table.shape[1], tokens, n_q, n_kv, D, 1 if write_cache else 0, _ptr(status), _stream()), what)


def read_quantized_pages(k_out: torch.Tensor, v_out: torch.Tensor, pages: QuantizedPages, page_list: torch.Tensor,
                         status: torch.Tensor) -> None:
    """What the pages of ``page_list`` (int32, any number, any order) stand for, in bfloat16 or float32:
    ``k_out``, ``v_out`` [len(page_list), n_kv, page_size, D].  A negative number gives zeros, one past the
    pool zeros and status word 0 = 3."""
    what, n = "read_quantized_pages", page_list.numel()
    _int32(page_list, "page_list")
    shape = (n, pages.n_kv, pages.page_size, pages.head_dim)
    if tuple(k_out.shape) != shape or tuple(v_out.shape) != shape or k_out.dtype != v_out.dtype or \
            not (k_out.is_contiguous() and v_out.is_contiguous()):
        raise KernelError(f"{what}: k_out and v_out must be contiguous, of one dtype and {shape}")
    _status(status, what)
    _on(pages.k_codes.device, what, k_out, v_out, page_list, status)
    f = _fn("cache_quant", "kipp_quant_cache_read",
            [c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_int, c_int, c_int,
             c_void_p, c_void_p])
    _check(f(_ptr(k_out), _ptr(v_out), dtype_code(k_out.dtype), *pages.pointers(), _ptr(page_list), n, pages.n_kv, pages.head_dim,
             _ptr(status), _stream()), what)


def _read_entries(pages: QuantizedPages, dtype: torch.dtype, meta, block_table: torch.Tensor, first: int, entries: int, window: int,
                  status: torch.Tensor, table: torch.Tensor):
    """Pages of what ``entries`` entries from ``first`` on see, in ``dtype``, and their rows of ``table``."""
    shape = (entries * block_table.shape[1], pages.n_kv, pages.page_size, pages.head_dim)
    k, v = (torch.empty(shape, dtype=dtype, device=table.device) for _ in range(2))
    f = _fn("cache_quant", "kipp_quant_cache_read_entries",
            [c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p,
             c_int, c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p])
    _check(f(_ptr(k), _ptr(v), _ptr(table), dtype_code(dtype), *pages.pointers(), _ptr(meta.q_start), _ptr(meta.context_len),
             _ptr(block_table), block_table.shape[1], first, entries, window, pages.n_kv, pages.head_dim, _ptr(status), _stream()),
           "read_entries")
    return k, v


def _entries_at_once(pages: QuantizedPages, dtype: torch.dtype, width: int) -> int:
    """How many entries' pages may be read back together."""
    per = 2 * pages.n_kv * pages.page_size * pages.head_dim * dtype.itemsize * width
    return max(1, min(READ_BYTES // per, 65535 // width))


PORTION_MIN = 64              # an entry of as many tokens is read back for the prompt kernel of 128-token tiles


def _direct_ok(q: torch.Tensor, pages: QuantizedPages, n_q: int) -> bool:
    f = _fn("attention_quant", "kipp_attn_quant_supported", [c_int, c_int, c_int, c_int])
    return (q.dtype == torch.bfloat16 and bool(f(pages.bits, pages.head_dim, n_q, pages.n_kv))
            and all(t.data_ptr() % 16 == 0 for t in (q, pages.k_codes, pages.v_codes, pages.k_scales, pages.v_scales)))


def _plan(out, q, pages, meta, block_table, n_q):
    """(form of the entries of one token, form of the others, the entries of more than one token from the first to the last):
    forms "direct" (the kernel over codes), "portion" (read back, tcgen05 prompt kernel) and "read" (read back, CUDA cores).
    The prompt kernel reads a key and a value once for 128 tokens, the kernel over codes once for 8 or 16 columns."""
    if not _direct_ok(q, pages, n_q):
        return "read", "read", None
    several = [e for e, n in enumerate(meta.q_lens) if n > 1]
    if several and max(meta.q_lens) >= PORTION_MIN and getattr(meta, "prefill_work128", None) is not None:
        from . import attention_bf16
        span = (several[0], several[-1] + 1)
        if attention_bf16.prefill_tc_supported(pages.head_dim, n_q, pages.n_kv, pages.page_size) and out.data_ptr() % 16 == 0 and \
                span[1] - span[0] <= _entries_at_once(pages, q.dtype, block_table.shape[1]):
            return "direct", "portion", span
    return "direct", "direct", None


def attention_quantized(out: torch.Tensor, q: torch.Tensor, pages: QuantizedPages, meta, block_table: torch.Tensor, n_q: int,
                        scale: float, window: Optional[int], status: torch.Tensor, impl: Optional[str] = None) -> None:
    """Causal grouped-query attention of the step's tokens over a quantised cache.

    ``meta`` is the step's metadata as for ``attention`` (``tokens``, ``q_lens``, ``positions``, ``entry_of_token``,
    ``q_start``, ``context_len``, and where entries bring 64 tokens or more the list of their 128-token tiles,
    ``prefill_work128`` and ``n_prefill_items128``).  bfloat16 with heads of 64, 128 or 256 runs on the codes themselves; longer
    portions of prompts, other heads and float32 on pages that are read back.  ``impl`` forces a form for the whole step:
    "direct" or "read"."""
    what, D, n_kv, window = "attention_quantized", pages.head_dim, pages.n_kv, int(window or 0)
    dtype_code(q.dtype)
    if q.dim() != 3 or tuple(q.shape[1:]) != (n_q, D) or q.shape[0] < meta.tokens or not q.is_contiguous() or n_q % n_kv:
        raise KernelError(f"{what}: q must be contiguous [tokens, n_q, head_dim] with n_q a multiple of the cache's heads")
    if out.dtype != q.dtype or out.shape != q.shape or not out.is_contiguous():
        raise KernelError(f"{what}: out must be contiguous, of q's dtype and shape")
    if window < 0:
        raise KernelError(f"{what}: a window must not be negative")
    if block_table.dim() != 2 or block_table.shape[0] < len(meta.q_lens) or block_table.shape[1] == 0 or sum(meta.q_lens) != meta.tokens:
        raise KernelError(f"{what}: a row of block_table for every entry, and as many tokens as the entries bring")
    for t, name in ((block_table, "block_table"), (meta.positions, "positions"), (meta.entry_of_token, "entry_of_token"),
                    (meta.q_start, "q_start"), (meta.context_len, "context_len")):
        _int32(t, name)
    if meta.q_start.numel() <= len(meta.q_lens) or meta.context_len.numel() < len(meta.q_lens) or \
            min(meta.positions.numel(), meta.entry_of_token.numel()) < meta.tokens:
        raise KernelError(f"{what}: the step's lists are shorter than the step")
    _status(status, what)
    _on(q.device, what, out, pages.k_codes, block_table, meta.q_start, meta.context_len, meta.positions, meta.entry_of_token, status)
    if impl not in (None, "direct", "read"):
        raise KernelError(f"unknown attention implementation {impl!r}")
    if impl == "direct" and not _direct_ok(q, pages, n_q):
        raise KernelError(f"{what}: the kernel over codes takes bfloat16 heads of 64, 128 or 256, 16-byte aligned")
    if meta.tokens == 0:
        return
    single, several, span = _plan(out, q, pages, meta, block_table, n_q) if impl is None else (impl, impl, None)
    if single == "read":
        _by_reading(out, q, pages, meta, block_table, n_q, scale, window, status)
        return
    if several == "direct" or 1 in meta.q_lens:
        _direct(out, q, pages, meta, block_table, n_q, scale, window, status, max(meta.q_lens) if several == "direct" else 1)
    if several == "portion":
        _portions(out, q, pages, meta, block_table, n_q, scale, window, status, span)


def _direct(out, q, pages, meta, block_table, n_q, scale, window, status, most: int) -> None:
    """The entries of up to ``most`` tokens, over the codes."""
    need = _fn("attention_quant", "kipp_attn_quant_scratch_bytes", [c_int], restype=c_ll)(pages.head_dim)
    scratch = torch.empty(need, dtype=torch.uint8, device=q.device)
    f = _fn("attention_quant", "kipp_attn_quant",
            [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int,
             c_int, c_int, c_int, c_int, c_float, c_int, c_void_p, c_ll, c_void_p, c_void_p])
    _check(f(_ptr(out), _ptr(q), *pages.pointers(), _ptr(meta.q_start), _ptr(meta.context_len), _ptr(block_table), block_table.shape[1],
             len(meta.q_lens), most, n_q, pages.n_kv, pages.head_dim, float(scale), window, _ptr(scratch), need, _ptr(status), _stream()),
           "attn_quant")


def _portions(out, q, pages, meta, block_table, n_q, scale, window, status, span) -> None:
    """The entries of more than one token: their pages read back, and the prompt kernel over those."""
    table = torch.empty_like(block_table)
    k, v = _read_entries(pages, q.dtype, meta, block_table, span[0], span[1] - span[0], window, status, table)
    from . import attention_bf16
    attention_bf16.prefill_tc(out, q, k, v, meta, table, pages.page_size, n_q, pages.n_kv, pages.head_dim, scale, window, status)


def _by_reading(out, q, pages, meta, block_table, n_q, scale, window, status) -> None:
    """Every entry's pages read back, as many entries at a time as READ_BYTES allow, and the attention over them."""
    D, n_kv, width = pages.head_dim, pages.n_kv, block_table.shape[1]
    table = torch.empty_like(block_table)
    step, at = _entries_at_once(pages, q.dtype, width), 0
    for first in range(0, len(meta.q_lens), step):
        lens = meta.q_lens[first:first + step]
        n = sum(lens)
        if n == 0:
            continue
        k, v = _read_entries(pages, q.dtype, meta, block_table, first, len(lens), window, status, table)
        f = _fn("attention_simt", "kipp_paged_attention_simt",
                [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_int, c_int,
                 c_float, c_int, c_void_p, c_void_p])
        _check(f(_ptr(out[at:]), _ptr(q[at:]), _ptr(k), _ptr(v), dtype_code(q.dtype), _ptr(meta.positions[at:]), _ptr(meta.entry_of_token[at:]),
                 _ptr(table), width, pages.page_size, n, n_q, n_kv, D, float(scale), window, _ptr(status), _stream()), "attention_simt")
        at += n
