"""The paged cache in 8 bits: the write of new tokens, attention over it, pages read back.

Codes int8 [n_pages, n_kv_heads, 64, head_dim], scales float32 [n_pages, n_kv_heads]; a number is code * scale.  A scale is a power of
two, set by the largest number of its page and key head; it grows when a new token does not fit, and the tokens before it are
rounded again.  A page's scale starts afresh with the token in its first row.  A page that is given a number that is not finite
reads as NaN until it starts afresh.  The reference keeps its cache in 8 bits with a scale per position (QStream src/engine.c:240-293).
"""
from __future__ import annotations

import functools
from ctypes import c_float, c_int, c_longlong, c_void_p

import torch

from . import ops
from .q4 import TYPES, _refuse, launch_stream

PAGE_TOKENS = 64
MAX_SPLIT_CONTEXT = 4096 * 128      # what the merge of the keys' parts holds for any head size; longer contexts go a row at a time

_store = _read = _attention = _decode = _scratch = _prefill = None


def _bind():
    global _store, _read, _attention, _decode, _scratch, _prefill
    if _store is None:
        _read = ops.bind("qs_kv8_read_pages", [c_void_p, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p])
        _attention = ops.bind("qs_kv8_attention", [
            c_void_p, c_int, c_longlong, c_void_p, c_int, c_longlong, c_int, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_int, c_int,
            c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_float, c_int, c_int, c_int, c_void_p, c_float, c_int, c_void_p, c_void_p])
        _decode = ops.bind("qs_kv8_decode", [
            c_void_p, c_int, c_longlong, c_void_p, c_int, c_longlong, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p,
            c_int, c_int, c_int, c_int, c_float, c_int, c_int, c_int, c_void_p, c_float, c_int, c_void_p, c_void_p, c_void_p])
        _scratch = functools.lru_cache(maxsize=4096)(ops.bind("qs_kv8_decode_scratch", [c_int, c_int, c_int, c_int, c_int], c_longlong))
        _prefill = ops.bind("qs_kv8_prefill", [
            c_void_p, c_int, c_longlong, c_void_p, c_longlong, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_int, c_void_p,
            c_int, c_int, c_int, c_int, c_int, c_float, c_int, c_int, c_int, c_void_p, c_float, c_void_p, c_void_p])
        _store = ops.bind("qs_kv8_store", [
            c_void_p, c_longlong, c_void_p, c_longlong, c_void_p, c_longlong, c_void_p, c_longlong, c_void_p, c_longlong, c_float, c_int,
            c_int, c_int, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int,
            c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p])


def _check_cache(what, k_cache, v_cache, k_scale, v_scale, n_kv_heads, head_dim, v_head_dim, page_tokens) -> int:
    """The number of pages."""
    if page_tokens != PAGE_TOKENS:
        _refuse(f"{what}: pages of {page_tokens} tokens, the kernels are built for {PAGE_TOKENS}")
    shape = k_cache.shape
    n = shape[0] if len(shape) == 4 else 0
    if (n < 1 or n_kv_heads < 1 or head_dim < 1 or v_head_dim < 1 or shape != (n, n_kv_heads, PAGE_TOKENS, head_dim) or v_cache.shape != (n, n_kv_heads, PAGE_TOKENS, v_head_dim) or k_cache.dtype is not torch.int8
            or v_cache.dtype is not torch.int8 or not k_cache.is_contiguous() or not v_cache.is_contiguous()):
        _refuse(f"{what}: caches are contiguous int8 [pages, {n_kv_heads}, {PAGE_TOKENS}, {head_dim} and {v_head_dim}], got {k_cache.dtype} {tuple(shape)} and "
                f"{v_cache.dtype} {tuple(v_cache.shape)}")
    pages = (n, n_kv_heads)
    if (k_scale.shape != pages or v_scale.shape != pages or k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32
            or not k_scale.is_contiguous() or not v_scale.is_contiguous()):
        _refuse(f"{what}: scales are contiguous float32 {pages}, got {k_scale.dtype} {tuple(k_scale.shape)} and {v_scale.dtype} {tuple(v_scale.shape)}")
    return n


def _check_int32(what, name, t, dims, n=None):
    shape = t.shape
    if t.dtype is not torch.int32 or len(shape) != dims or not t.is_contiguous() or (n is not None and shape[0] != n) or (dims == 2 and 0 in shape):
        _refuse(f"{what}: {name} is a contiguous int32 tensor of {dims} dims{'' if n is None else f', {n} rows'}, got {t.dtype} {tuple(shape)}")


def _check_status(what, status):
    if status.dtype is not torch.int32 or status.numel() < 1:
        _refuse(f"{what}: the status word is int32")


def _at(t):
    return None if t is None else t.data_ptr()


def rope_store(q, k, v, n_heads, n_kv_heads, head_dim, rotary_dim, cos_sin, tok_slot, tok_pos, page_table, page_tokens, k_cache, v_cache,
               k_scale, v_scale, status, v_head_dim=None, v_first=None, v_mix=0.0, half_layout=False, q_out=None) -> None:
    """Rotate q (in place, or into `q_out`) and k, and write k and v into the 8-bit cache; arguments as for `ops.rope_store`, with the
    scales beside the caches.  Keys and values are rounded once, from 32 bits.  Rows with a slot below 0 are padding: their queries stay
    as they are, nothing is written for them.  A sequence's new tokens are consecutive rows with ascending positions; a second run of rows of a
    sequence for one page in the same call is not written, and status 5.  Two sequences may share pages that a call does not write; a page that both
    write to in one call holds neither's tokens reliably."""
    what = "kv8.rope_store"
    dv = int(v_head_dim or head_dim)
    n_pages = _check_cache(what, k_cache, v_cache, k_scale, v_scale, n_kv_heads, head_dim, dv, page_tokens)
    T, wk, ldk = ops._rows(k)
    _, wv, ldv = ops._rows(v)
    if k.dtype not in TYPES or v.dtype != k.dtype or v.shape[0] != T or wk != n_kv_heads * head_dim or wv != n_kv_heads * dv:
        _refuse(f"{what}: keys {k.dtype} {tuple(k.shape)} and values {v.dtype} {tuple(v.shape)} for {n_kv_heads} heads of {head_dim} and {dv}")
    if q is not None:
        q_out = q if q_out is None else q_out
        for t in (q, q_out):
            if t.dtype != k.dtype or ops._rows(t)[:2] != (T, n_heads * head_dim):
                _refuse(f"{what}: queries {t.dtype} {tuple(t.shape)} for {T} rows of {n_heads} heads of {head_dim}")
        if q_out is not q and q_out.data_ptr() == q.data_ptr() and q_out.stride(0) != q.stride(0):
            _refuse(f"{what}: q_out overlaps q")
    if v_first is not None and (v_first.dtype != k.dtype or ops._rows(v_first)[:2] != (T, wv)):
        _refuse(f"{what}: values to blend with are {v_first.dtype} {tuple(v_first.shape)}")
    if cos_sin is not None and (rotary_dim < 0 or rotary_dim % 2 or rotary_dim > head_dim or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous()
                                or cos_sin.dim() != 3 or tuple(cos_sin.shape[1:]) != (rotary_dim // 2, 2) or cos_sin.shape[0] < 1):
        _refuse(f"{what}: {rotary_dim} rotated dims of {head_dim} with a table {cos_sin.dtype} {tuple(cos_sin.shape)}")
    if head_dim % 2 or head_dim > 512 or dv > 512:
        _refuse(f"{what}: head sizes {head_dim} and {dv} (keys: even; up to 512)")
    _check_int32(what, "tok_slot", tok_slot, 1, T)
    _check_int32(what, "tok_pos", tok_pos, 1, T)
    _check_int32(what, "page_table", page_table, 2)
    _check_status(what, status)
    if T == 0:
        return
    stream = launch_stream(k.get_device(), v, q, q_out, v_first, cos_sin, tok_slot, tok_pos, page_table, k_cache, v_cache, k_scale, v_scale, status)
    if _store is None:
        _bind()
    slots, max_pages = page_table.shape
    ops.check(_store(_at(q_out), q_out.stride(0) if q is not None else 0, _at(q), q.stride(0) if q is not None else 0, k.data_ptr(), ldk, v.data_ptr(), ldv,
                     _at(v_first), v_first.stride(0) if v_first is not None else 0, float(v_mix), ops.dtype_code(k), T, n_heads if q is not None else 0,
                     n_kv_heads, head_dim, dv, rotary_dim if cos_sin is not None else 0, _at(cos_sin), cos_sin.shape[0] if cos_sin is not None else 0,
                     1 if half_layout else 0, tok_slot.data_ptr(), tok_pos.data_ptr(), page_table.data_ptr(), slots, max_pages, n_pages, k_cache.data_ptr(),
                     v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), status.data_ptr(), stream))


def read_pages(cache, scale, pages, dtype=torch.float32) -> torch.Tensor:
    """The numbers in the listed pages (int32): [n, n_kv_heads, 64, head_dim] of `dtype`, exact in float32 and in bfloat16.  A page that
    does not exist gives NaN."""
    what = "kv8.read_pages"
    if cache.dim() != 4 or scale.dim() != 2:
        _refuse(f"{what}: a cache {tuple(cache.shape)} with scales {tuple(scale.shape)}")
    _, heads, tokens, dim = cache.shape
    _check_cache(what, cache, cache, scale, scale, heads, dim, dim, tokens)
    _check_int32(what, "pages", pages, 1)
    if dtype not in TYPES:
        _refuse(f"{what}: numbers of {dtype}")
    n = pages.shape[0]
    total, heads, tokens, dim = cache.shape
    out = torch.empty((n, heads, tokens, dim), dtype=dtype, device=cache.device)
    stream = launch_stream(cache.get_device(), scale, pages)
    if _read is None:
        _bind()
    for a in range(0, n, 65535):
        b = min(n, a + 65535)
        to, ids = (out, pages) if b - a == n else (out[a:b], pages[a:b])
        ops.check(_read(to.data_ptr(), ops.dtype_code(out), cache.data_ptr(), scale.data_ptr(), ids.data_ptr(), b - a, total, heads, dim, stream))
    return out


def _check_attention(what, q, n_heads, n_kv_heads, head_dim, window, page_table, page_tokens, k_cache, v_cache, k_scale, v_scale, status, out, dv, softcap,
                     chunk, keep_first, sink, out_dtype):
    """(rows, pages, the output tensor) of a checked call."""
    n_pages = _check_cache(what, k_cache, v_cache, k_scale, v_scale, n_kv_heads, head_dim, dv, page_tokens)
    T, wq, _ = ops._rows(q)
    dtype = q.dtype
    if dtype not in TYPES or n_heads < 1 or n_heads % n_kv_heads or wq != n_heads * head_dim:
        _refuse(f"{what}: queries {q.dtype} {tuple(q.shape)} of {n_heads} heads of {head_dim} over {n_kv_heads} key heads")
    if head_dim > 512 or dv > 512:
        _refuse(f"{what}: head sizes {head_dim} and {dv} (up to 512)")
    if window < 0 or chunk < 0 or keep_first < 0 or (window > 0 and chunk > 0):
        _refuse(f"{what}: a window of {window}, chunks of {chunk}, {keep_first} kept first keys")
    if softcap < 0:
        _refuse(f"{what}: scores capped at {softcap}")
    if sink is not None and (sink.dtype != torch.float32 or sink.numel() != n_heads or not sink.is_contiguous()):
        _refuse(f"{what}: sinks are contiguous float32 [{n_heads}], got {sink.dtype} {tuple(sink.shape)}")
    want = out.dtype if out is not None else out_dtype or dtype
    if want not in TYPES or (dtype is torch.float32 and want is not dtype) or (out is not None and out_dtype not in (None, want)):
        _refuse(f"{what}: a result of {want} from queries of {q.dtype}")
    if out is None:
        out = torch.empty((T, n_heads * dv), dtype=want, device=q.device)
    elif tuple(out.shape) != (T, n_heads * dv) or out.stride(1) != 1:
        _refuse(f"{what}: the output view {tuple(out.shape)} does not fit")
    _check_int32(what, "page_table", page_table, 2)
    _check_status(what, status)
    return T, n_pages, out


def decode(q, n_heads, n_kv_heads, head_dim, scale, window, tok_slot, tok_pos, page_table, page_tokens, k_cache, v_cache, k_scale, v_scale,
           max_context, status, out=None, v_head_dim=None, softcap=0.0, chunk=0, keep_first=0, sink=None, out_dtype=None) -> torch.Tensor:
    """Each row of q [T, n_heads * head_dim] against the 8-bit cache of its sequence, up to the row's own position: softmax(scale q.K) V.
    Masks, cap and sinks as for `attention_bf16.decode`: a window of the last keys, beside it the first `keep_first`; chunks of positions;
    scores c tanh(s / c); exp(sink) in each head's sum.  Positions lie below `max_context`; a row beyond it, or beyond the page table,
    gives zeros and status 1, a page its sequence does not hold status 3.  Rows with a slot below 0 give zeros.

    Head sizes that are multiples of 16 up to 256 go to the tensor cores, a query as 16-bit floats over a power of two (numbers below 2^-14 of its largest are off
    by 2^-25 of it; float32 queries are two such floats, 22 bits), bfloat16 rows' weights as 16-bit floats; sums have 32 bits."""
    what = "kv8.decode"
    dv = int(v_head_dim or head_dim)
    T, n_pages, out = _check_attention(what, q, n_heads, n_kv_heads, head_dim, window, page_table, page_tokens, k_cache, v_cache, k_scale, v_scale, status, out, dv,
                              softcap, chunk, keep_first, sink, out_dtype)
    _check_int32(what, "tok_slot", tok_slot, 1, T)
    _check_int32(what, "tok_pos", tok_pos, 1, T)
    if max_context < 1:
        _refuse(f"{what}: a context of {max_context}")
    if T == 0:
        return out
    stream = launch_stream(q.get_device(), out, tok_slot, tok_pos, page_table, k_cache, v_cache, k_scale, v_scale, status, sink)
    if _decode is None:
        _bind()
    slots, max_pages = page_table.shape
    code, wide = ops.dtype_code(q), out.dtype is torch.float32
    cache = k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()
    if head_dim % 16 == 0 and dv % 16 == 0 and head_dim <= 256 and dv <= 256 and T <= 65535 and max_context <= MAX_SPLIT_CONTEXT:
        floats = _scratch(T, n_heads, head_dim, dv, max_context)
        partial = None
        if floats:
            partial = torch.empty((floats,), dtype=torch.float32, device=q.device)
            ops.count_launches(1)                       # split kernel + merge kernel
        ops.check(_decode(out.data_ptr(), 1 if wide else 0, out.stride(0), q.data_ptr(), code, q.stride(0), T, tok_slot.data_ptr(), tok_pos.data_ptr(),
                          page_table.data_ptr(), slots, max_pages, n_pages, *cache, n_heads, n_kv_heads, head_dim, dv, float(scale), int(window), int(chunk),
                          int(keep_first), _at(sink), float(softcap or 0.0), int(max_context), _at(partial), status.data_ptr(), stream))
        return out
    for a in range(0, T, 65535):
        b = min(T, a + 65535)
        ops.check(_attention(out[a:b].data_ptr(), ops.F32 if wide else ops.BF16, out.stride(0), q[a:b].data_ptr(), code, q.stride(0), b - a, tok_slot[a:b].data_ptr(),
                             tok_pos[a:b].data_ptr(), None, 0, page_table.data_ptr(), slots, max_pages, n_pages, *cache, n_heads, n_kv_heads, head_dim, dv,
                             float(scale), int(window), int(chunk), int(keep_first), _at(sink), float(softcap or 0.0), int(max_context), status.data_ptr(), stream))
    return out


def prefill(q, n_heads, n_kv_heads, head_dim, scale, window, tiles, page_table, page_tokens, k_cache, v_cache, k_scale, v_scale, status,
            padded=False, out=None, v_head_dim=None, softcap=0.0, chunk=0, keep_first=0, sink=None, out_dtype=None) -> torch.Tensor:
    """Many rows per sequence against the 8-bit cache.  `tiles` (int32 [n, 4]: first row, number of rows up to 128, position of the first row,
    slot) as from `attention_bf16.prefill_tiles`; rows that no tile covers are left as they are, or zeros with `padded`.  The rest as for `decode`.

    bfloat16 rows go to the tensor cores (head sizes that are multiples of 16 up to 256), their softmax weights rounded to bfloat16.  float32 rows and other head sizes take
    the plain kernel, a warp for a row and head: three prompts, 2,047 rows of 16 heads of 128: 5.9 ms, where bfloat16 rows take 39 us."""
    what = "kv8.prefill"
    dv = int(v_head_dim or head_dim)
    T, n_pages, out = _check_attention(what, q, n_heads, n_kv_heads, head_dim, window, page_table, page_tokens, k_cache, v_cache, k_scale, v_scale, status, out, dv,
                              softcap, chunk, keep_first, sink, out_dtype)
    _check_int32(what, "tiles", tiles, 2)
    if tiles.shape[1] != 4:
        _refuse(f"{what}: tiles are [n, 4], got {tuple(tiles.shape)}")
    if T == 0:
        return out
    stream = launch_stream(q.get_device(), out, tiles, page_table, k_cache, v_cache, k_scale, v_scale, status, sink)
    if _prefill is None:
        _bind()
    if padded:
        out.zero_()
    slots, max_pages = page_table.shape
    n, code, wide = tiles.shape[0], ops.dtype_code(q), out.dtype is torch.float32
    cache = k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()
    if (code == ops.BF16 and head_dim % 16 == 0 and dv % 16 == 0 and head_dim <= 256 and dv <= 256 and scale > 0 and n <= 65535
            and q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0 and out.stride(0) % (4 if wide else 8) == 0 and out.data_ptr() % 16 == 0):
        ops.check(_prefill(out.data_ptr(), 1 if wide else 0, out.stride(0), q.data_ptr(), q.stride(0), T, *cache, n_pages, page_table.data_ptr(), slots, max_pages,
                           tiles.data_ptr(), n, n_heads, n_kv_heads, head_dim, dv, float(scale), int(window), int(chunk), int(keep_first), _at(sink),
                           float(softcap or 0.0), status.data_ptr(), stream))
        return out
    for a in range(0, n, 511):
        b = min(n, a + 511)
        ops.check(_attention(out.data_ptr(), ops.F32 if wide else ops.BF16, out.stride(0), q.data_ptr(), code, q.stride(0), T, None, None, tiles[a:b].data_ptr(), b - a,
                             page_table.data_ptr(), slots, max_pages, n_pages, *cache, n_heads, n_kv_heads, head_dim, dv, float(scale), int(window), int(chunk),
                             int(keep_first), _at(sink), float(softcap or 0.0), 2147483647, status.data_ptr(), stream))
    return out
