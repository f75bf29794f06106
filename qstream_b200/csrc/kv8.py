"""The paged cache in 8 bits: the write of new tokens, attention over it, pages read back.

Codes int8 [n_pages, n_kv_heads, 64, head_dim], scales float32 [n_pages, n_kv_heads]; a number is code * scale.  A scale is a power of
two, set by the largest number of its page and key head; it grows when a new token does not fit, and the tokens before it are
rounded again.  A page's scale starts afresh with the token in its first row.  A page that is given a number that is not finite
reads as NaN until it starts afresh.  The reference keeps its cache in 8 bits with a scale per position (QStream src/engine.c:240-293).
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p

import torch

from ..errors import QsError, QStreamError
from . import ops
from .q4 import TYPES, _on_current_device, _refuse

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
        _scratch = ops.bind("qs_kv8_decode_scratch", [c_int, c_int, c_int, c_int, c_int], c_longlong)
        _prefill = ops.bind("qs_kv8_prefill", [
            c_void_p, c_int, c_longlong, c_void_p, c_longlong, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int, c_int, c_void_p,
            c_int, c_int, c_int, c_int, c_int, c_float, c_int, c_int, c_int, c_void_p, c_float, c_void_p, c_void_p])
        _store = ops.bind("qs_kv8_store", [
            c_void_p, c_longlong, c_void_p, c_longlong, c_void_p, c_longlong, c_void_p, c_longlong, c_void_p, c_longlong, c_float, c_int,
            c_int, c_int, c_int, c_int, c_int, c_int, c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int,
            c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p])


def _check_cache(what, k_cache, v_cache, k_scale, v_scale, n_kv_heads, head_dim, v_head_dim, page_tokens):
    if page_tokens != PAGE_TOKENS:
        _refuse(f"{what}: pages of {page_tokens} tokens, the kernels are built for {PAGE_TOKENS}")
    for name, cache, scale, dim in (("k", k_cache, k_scale, head_dim), ("v", v_cache, v_scale, v_head_dim)):
        if cache.dtype != torch.int8 or cache.dim() != 4 or tuple(cache.shape[1:]) != (n_kv_heads, PAGE_TOKENS, dim) or not cache.is_contiguous() or cache.shape[0] < 1:
            _refuse(f"{what}: {name}_cache is contiguous int8 [pages, {n_kv_heads}, {PAGE_TOKENS}, {dim}], got {cache.dtype} {tuple(cache.shape)}")
        if scale.dtype != torch.float32 or tuple(scale.shape) != tuple(cache.shape[:2]) or not scale.is_contiguous():
            _refuse(f"{what}: {name}_scale is contiguous float32 {tuple(cache.shape[:2])}, got {scale.dtype} {tuple(scale.shape)}")
    if k_cache.shape[0] != v_cache.shape[0]:
        _refuse(f"{what}: {k_cache.shape[0]} pages of keys and {v_cache.shape[0]} of values")


def _check_int32(what, name, t, dims, n=None):
    if t.dtype != torch.int32 or t.dim() != dims or not t.is_contiguous() or (n is not None and t.shape[0] != n) or (dims == 2 and 0 in t.shape):
        _refuse(f"{what}: {name} is a contiguous int32 tensor of {dims} dims{'' if n is None else f', {n} rows'}, got {t.dtype} {tuple(t.shape)}")


def _check_status(what, status):
    if status.dtype != torch.int32 or status.numel() < 1:
        _refuse(f"{what}: the status word is int32")


def rope_store(q, k, v, n_heads, n_kv_heads, head_dim, rotary_dim, cos_sin, tok_slot, tok_pos, page_table, page_tokens, k_cache, v_cache,
               k_scale, v_scale, status, v_head_dim=None, v_first=None, v_mix=0.0, half_layout=False, q_out=None) -> None:
    """Rotate q (in place, or into `q_out`) and k, and write k and v into the 8-bit cache; arguments as for `ops.rope_store`, with the
    scales beside the caches.  Keys and values are rounded once, from 32 bits.  Rows with a slot below 0 are padding: their queries stay
    as they are, nothing is written for them.  A sequence's new tokens are consecutive rows with ascending positions; a page that
    a second run of rows names in the same call gets the first run only, and status 5."""
    what = "kv8.rope_store"
    dv = int(v_head_dim or head_dim)
    _check_cache(what, k_cache, v_cache, k_scale, v_scale, n_kv_heads, head_dim, dv, page_tokens)
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
    _on_current_device(k, v, q, q_out, v_first, cos_sin, tok_slot, tok_pos, page_table, k_cache, v_cache, k_scale, v_scale, status)
    ops.ptr(k)
    _bind()
    ops.check(_store(ops.ptr(q_out), q_out.stride(0) if q is not None else 0, ops.ptr(q), q.stride(0) if q is not None else 0, ops.ptr(k), ldk, ops.ptr(v), ldv,
                     ops.ptr(v_first), v_first.stride(0) if v_first is not None else 0, float(v_mix), ops.dtype_code(k), T, n_heads if q is not None else 0,
                     n_kv_heads, head_dim, dv, rotary_dim if cos_sin is not None else 0, ops.ptr(cos_sin), cos_sin.shape[0] if cos_sin is not None else 0,
                     int(bool(half_layout)), ops.ptr(tok_slot), ops.ptr(tok_pos), ops.ptr(page_table), page_table.shape[0], page_table.shape[1],
                     k_cache.shape[0], ops.ptr(k_cache), ops.ptr(v_cache), ops.ptr(k_scale), ops.ptr(v_scale), ops.ptr(status), ops.stream()))


def read_pages(cache, scale, pages, dtype=torch.float32) -> torch.Tensor:
    """The numbers in the listed pages (int32): [n, n_kv_heads, 64, head_dim] of `dtype`, exact in float32 and in bfloat16.  A page that
    does not exist gives NaN."""
    what = "kv8.read_pages"
    if cache.dim() != 4 or scale.dim() != 2:
        _refuse(f"{what}: a cache {tuple(cache.shape)} with scales {tuple(scale.shape)}")
    _check_cache(what, cache, cache, scale, scale, cache.shape[1], cache.shape[3], cache.shape[3], cache.shape[2])
    _check_int32(what, "pages", pages, 1)
    if dtype not in TYPES:
        _refuse(f"{what}: numbers of {dtype}")
    n = pages.shape[0]
    out = torch.empty((n, *cache.shape[1:]), dtype=dtype, device=cache.device)
    _on_current_device(cache, scale, pages)
    ops.ptr(cache)
    _bind()
    for a in range(0, n, 65535):
        b = min(n, a + 65535)
        ops.check(_read(ops.ptr(out[a:b]), ops.dtype_code(out), ops.ptr(cache), ops.ptr(scale), ops.ptr(pages[a:b]), b - a, cache.shape[0], cache.shape[1],
                        cache.shape[3], ops.stream()))
    return out


def _check_attention(what, q, n_heads, n_kv_heads, head_dim, window, page_table, page_tokens, k_cache, v_cache, k_scale, v_scale, status, out, dv, softcap,
                     chunk, keep_first, sink, out_dtype):
    """(rows, the output tensor) of a checked call."""
    _check_cache(what, k_cache, v_cache, k_scale, v_scale, n_kv_heads, head_dim, dv, page_tokens)
    T, wq, _ = ops._rows(q)
    if q.dtype not in TYPES or n_heads < 1 or n_heads % n_kv_heads or wq != n_heads * head_dim:
        _refuse(f"{what}: queries {q.dtype} {tuple(q.shape)} of {n_heads} heads of {head_dim} over {n_kv_heads} key heads")
    if head_dim > 512 or dv > 512:
        _refuse(f"{what}: head sizes {head_dim} and {dv} (up to 512)")
    if window < 0 or chunk < 0 or keep_first < 0 or (window > 0 and chunk > 0):
        _refuse(f"{what}: a window of {window}, chunks of {chunk}, {keep_first} kept first keys")
    if softcap < 0:
        _refuse(f"{what}: scores capped at {softcap}")
    if sink is not None and (sink.dtype != torch.float32 or sink.numel() != n_heads or not sink.is_contiguous()):
        _refuse(f"{what}: sinks are contiguous float32 [{n_heads}], got {sink.dtype} {tuple(sink.shape)}")
    want = out.dtype if out is not None else out_dtype or q.dtype
    if want not in ((torch.float32,) if q.dtype == torch.float32 else TYPES) or (out is not None and out_dtype not in (None, out.dtype)):
        _refuse(f"{what}: a result of {want} from queries of {q.dtype}")
    if out is None:
        out = torch.empty((T, n_heads * dv), dtype=want, device=q.device)
    elif tuple(out.shape) != (T, n_heads * dv) or out.stride(1) != 1:
        _refuse(f"{what}: the output view {tuple(out.shape)} does not fit")
    _check_int32(what, "page_table", page_table, 2)
    _check_status(what, status)
    return T, out


def decode(q, n_heads, n_kv_heads, head_dim, scale, window, tok_slot, tok_pos, page_table, page_tokens, k_cache, v_cache, k_scale, v_scale,
           max_context, status, out=None, v_head_dim=None, softcap=0.0, chunk=0, keep_first=0, sink=None, out_dtype=None) -> torch.Tensor:
    """Each row of q [T, n_heads * head_dim] against the 8-bit cache of its sequence, up to the row's own position: softmax(scale q.K) V.
    Masks, cap and sinks as for `attention_bf16.decode`: a window of the last keys, beside it the first `keep_first`; chunks of positions;
    scores c tanh(s / c); exp(sink) in each head's sum.  Positions lie below `max_context`; a row beyond it, or beyond the page table,
    gives zeros and status 1, a page its sequence does not hold status 3.  Rows with a slot below 0 give zeros."""
    what = "kv8.decode"
    dv = int(v_head_dim or head_dim)
    T, out = _check_attention(what, q, n_heads, n_kv_heads, head_dim, window, page_table, page_tokens, k_cache, v_cache, k_scale, v_scale, status, out, dv,
                              softcap, chunk, keep_first, sink, out_dtype)
    _check_int32(what, "tok_slot", tok_slot, 1, T)
    _check_int32(what, "tok_pos", tok_pos, 1, T)
    if max_context < 1:
        _refuse(f"{what}: a context of {max_context}")
    if T == 0:
        return out
    _on_current_device(q, out, tok_slot, tok_pos, page_table, k_cache, v_cache, k_scale, v_scale, status, sink)
    ops.ptr(q)
    _bind()
    if head_dim % 16 == 0 and dv % 16 == 0 and head_dim <= 256 and dv <= 256 and T <= 65535 and max_context <= MAX_SPLIT_CONTEXT:
        floats = _scratch(T, n_heads, head_dim, dv, max_context)
        partial = torch.empty((floats,), dtype=torch.float32, device=q.device) if floats else None
        ops.check(_decode(ops.ptr(out), int(out.dtype == torch.float32), out.stride(0), ops.ptr(q), ops.dtype_code(q), q.stride(0), T, ops.ptr(tok_slot), ops.ptr(tok_pos),
                          ops.ptr(page_table), page_table.shape[0], page_table.shape[1], k_cache.shape[0], ops.ptr(k_cache), ops.ptr(v_cache), ops.ptr(k_scale),
                          ops.ptr(v_scale), n_heads, n_kv_heads, head_dim, dv, float(scale), int(window), int(chunk), int(keep_first), ops.ptr(sink),
                          float(softcap or 0.0), int(max_context), ops.ptr(partial), ops.ptr(status), ops.stream()))
        if partial is not None:
            ops.count_launches(1)                       # split kernel + merge kernel
        return out
    for a in range(0, T, 65535):
        b = min(T, a + 65535)
        ops.check(_attention(ops.ptr(out[a:b]), ops.dtype_code(out), out.stride(0), ops.ptr(q[a:b]), ops.dtype_code(q), q.stride(0), b - a, ops.ptr(tok_slot[a:b]),
                             ops.ptr(tok_pos[a:b]), None, 0, ops.ptr(page_table), page_table.shape[0], page_table.shape[1], k_cache.shape[0], ops.ptr(k_cache),
                             ops.ptr(v_cache), ops.ptr(k_scale), ops.ptr(v_scale), n_heads, n_kv_heads, head_dim, dv, float(scale), int(window), int(chunk),
                             int(keep_first), ops.ptr(sink), float(softcap or 0.0), int(max_context), ops.ptr(status), ops.stream()))
    return out


def prefill(q, n_heads, n_kv_heads, head_dim, scale, window, tiles, page_table, page_tokens, k_cache, v_cache, k_scale, v_scale, status,
            padded=False, out=None, v_head_dim=None, softcap=0.0, chunk=0, keep_first=0, sink=None, out_dtype=None) -> torch.Tensor:
    """Many rows per sequence against the 8-bit cache.  `tiles` (int32 [n, 4]: first row, number of rows up to 128, position of the first row,
    slot) as from `attention_bf16.prefill_tiles`; rows that no tile covers are left as they are, or zeros with `padded`.  The rest as for `decode`."""
    what = "kv8.prefill"
    dv = int(v_head_dim or head_dim)
    T, out = _check_attention(what, q, n_heads, n_kv_heads, head_dim, window, page_table, page_tokens, k_cache, v_cache, k_scale, v_scale, status, out, dv,
                              softcap, chunk, keep_first, sink, out_dtype)
    _check_int32(what, "tiles", tiles, 2)
    if tiles.shape[1] != 4:
        _refuse(f"{what}: tiles are [n, 4], got {tuple(tiles.shape)}")
    if T == 0:
        return out
    _on_current_device(q, out, tiles, page_table, k_cache, v_cache, k_scale, v_scale, status, sink)
    ops.ptr(q)
    _bind()
    if padded:
        out.zero_()
    wide = int(out.dtype == torch.float32)
    if (q.dtype == torch.bfloat16 and head_dim % 16 == 0 and dv % 16 == 0 and head_dim <= 256 and dv <= 256 and scale > 0 and tiles.shape[0] <= 65535
            and q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0 and out.stride(0) % (4 if wide else 8) == 0 and out.data_ptr() % 16 == 0):
        ops.check(_prefill(ops.ptr(out), wide, out.stride(0), ops.ptr(q), q.stride(0), T, ops.ptr(k_cache), ops.ptr(v_cache), ops.ptr(k_scale), ops.ptr(v_scale),
                           k_cache.shape[0], ops.ptr(page_table), page_table.shape[0], page_table.shape[1], ops.ptr(tiles), tiles.shape[0], n_heads, n_kv_heads,
                           head_dim, dv, float(scale), int(window), int(chunk), int(keep_first), ops.ptr(sink), float(softcap or 0.0), ops.ptr(status),
                           ops.stream()))
        return out
    for a in range(0, tiles.shape[0], 511):
        b = min(tiles.shape[0], a + 511)
        ops.check(_attention(ops.ptr(out), ops.dtype_code(out), out.stride(0), ops.ptr(q), ops.dtype_code(q), q.stride(0), T, None, None, ops.ptr(tiles[a:b]), b - a,
                             ops.ptr(page_table), page_table.shape[0], page_table.shape[1], k_cache.shape[0], ops.ptr(k_cache), ops.ptr(v_cache),
                             ops.ptr(k_scale), ops.ptr(v_scale), n_heads, n_kv_heads, head_dim, dv, float(scale), int(window), int(chunk), int(keep_first),
                             ops.ptr(sink), float(softcap or 0.0), 2147483647, ops.ptr(status), ops.stream()))
    return out
