"""What the calls over 4-bit weights and 8-bit pages refuse, before anything reaches a device."""
import copy

import pytest
import torch

from qstream_b200.csrc import kv8, q4
from qstream_b200.errors import QsError, QStreamError


def weight(n=40, k=100, group=32):
    c, s = q4.sizes(n, k, group)
    return q4.Weight4(torch.full(c, 0x88, dtype=torch.uint8), torch.zeros(s, dtype=torch.bfloat16), n, k, group)


def refused(code, call, *args, **kw):
    with pytest.raises(QStreamError) as e:
        call(*args, **kw)
    assert e.value.code == code, e.value


def test_a_packed_matrix_keeps_what_was_checked():
    w = weight()
    for name, value in (("codes", w.codes.clone()), ("scales", w.scales.clone()), ("out_features", 48), ("in_features", 128), ("group", 64), ("other", 1)):
        with pytest.raises(AttributeError):
            setattr(w, name, value)
    twin = copy.deepcopy(w)
    assert twin.shape == w.shape and twin.group == w.group and twin.codes.data_ptr() != w.codes.data_ptr() and torch.equal(twin.codes, w.codes)


def test_packed_matrices_that_do_not_fit():
    w = weight()
    assert w.shape == (40, 100) and w.numel() == 4000 and w.nbytes == 3 * 2 * 512 + 2 * 3 * 4 * 16
    for change in (dict(out_features=49), dict(in_features=129), dict(group=64), dict(group=48), dict(out_features=0), dict(codes=w.codes.int()),
                   dict(scales=w.scales.float()), dict(codes=w.codes.expand(3, 2, 32, 16)[:2]), dict(scales=w.scales.transpose(1, 2))):
        refused(QsError.QUANT_MISMATCH, q4.Weight4, **{**dict(codes=w.codes, scales=w.scales, out_features=40, in_features=100, group=32), **change})
    odd = torch.zeros(w.codes.numel() + 1, dtype=torch.uint8)[1:].view(w.codes.shape)
    if odd.data_ptr() % 16:
        refused(QsError.INVALID_INPUT, q4.Weight4, odd, w.scales, 40, 100, 32)


def test_matrices_that_cannot_be_rounded():
    m = torch.zeros(8, 64)
    refused(QsError.QUANT_MISMATCH, q4.quantize, m, 16)
    for bad in (m.half(), m[0], m.t(), m[:0], m[:, :0], m[:, ::2]):
        refused(QsError.INVALID_INPUT, q4.quantize, bad)
    refused(QsError.INVALID_INPUT, q4.quantize, m)                      # no CPU path


def test_products_that_are_refused():
    w, x = weight(), torch.zeros(3, 100)
    ok = torch.zeros(3, 40)
    for kw in (dict(x=torch.zeros(3, 99)), dict(x=x.half()), dict(x=x[0]), dict(x=torch.zeros(100, 3).t()), dict(activation="swish"), dict(bias=torch.zeros(39)),
               dict(bias=torch.zeros(40).half()), dict(bias=torch.zeros(80)[::2]), dict(residuals=(ok[:2],)), dict(residuals=(ok.bfloat16(),)),
               dict(residuals=(ok, ok, ok)), dict(residuals=(ok, torch.zeros(3, 50)[:, :40])), dict(out_dtype=torch.bfloat16), dict(out=torch.zeros(3, 41)),
               dict(out=torch.zeros(3, 40).bfloat16()), dict(out=torch.zeros(40, 3).t()), dict(out=ok, out_dtype=torch.bfloat16), dict(x=x)):
        refused(QsError.INVALID_INPUT, q4.linear, **{**dict(x=x, weight=w), **kw})
    assert q4.linear(x[:0], w).shape == (0, 40)
    wide = weight(16, 40000, 128)
    refused(QsError.INVALID_INPUT, q4.linear, torch.zeros(1, 40000), wide)


I = lambda *s: torch.zeros(s, dtype=torch.int32)           # noqa: E731,E741
CACHE = dict(k_cache=torch.zeros(5, 2, 64, 16, dtype=torch.int8), v_cache=torch.zeros(5, 2, 64, 8, dtype=torch.int8), k_scale=torch.zeros(5, 2), v_scale=torch.zeros(5, 2))
BAD_CACHE = [dict(k_cache=CACHE["k_cache"].short()), dict(k_cache=CACHE["k_cache"][:, :1]), dict(k_cache=CACHE["k_cache"][:4]), dict(v_cache=CACHE["v_cache"][..., :7]),
             dict(k_scale=torch.zeros(5, 3)), dict(v_scale=torch.zeros(5, 2).double()), dict(k_scale=torch.zeros(2, 5).t()), dict(page_tokens=32),
             dict(k_cache=CACHE["k_cache"][:0], v_cache=CACHE["v_cache"][:0], k_scale=torch.zeros(0, 2), v_scale=torch.zeros(0, 2)), dict(page_table=I(2, 3).long()),
             dict(n_kv_heads=0, **{n: t[:, :0] for n, t in CACHE.items()}), dict(page_table=I(6)), dict(page_table=I(0, 3)), dict(status=torch.zeros(1)), dict(status=I(0))]


def test_writes_that_are_refused():
    base = dict(q=torch.zeros(4, 4 * 16), k=torch.zeros(4, 2 * 16), v=torch.zeros(4, 2 * 8), n_heads=4, n_kv_heads=2, head_dim=16, rotary_dim=8, cos_sin=torch.zeros(9, 4, 2),
                tok_slot=I(4), tok_pos=I(4), page_table=I(2, 3), page_tokens=64, status=I(1), v_head_dim=8, **CACHE)
    for kw in BAD_CACHE + [dict(k=torch.zeros(4, 31)), dict(v=torch.zeros(3, 16)), dict(v=torch.zeros(4, 16).bfloat16()), dict(k=torch.zeros(4, 32).half(), v=torch.zeros(4, 16).half()),
                           dict(q=torch.zeros(4, 63)), dict(q=torch.zeros(4, 64).bfloat16()), dict(q_out=torch.zeros(5, 64)), dict(v_first=torch.zeros(4, 15)),
                           dict(rotary_dim=7, cos_sin=torch.zeros(9, 3, 2)), dict(rotary_dim=18, cos_sin=torch.zeros(9, 9, 2)), dict(cos_sin=torch.zeros(9, 4, 2).double()),
                           dict(cos_sin=torch.zeros(9, 5, 2)), dict(cos_sin=torch.zeros(0, 4, 2)), dict(tok_slot=I(5)), dict(tok_pos=I(4).long()), {}]:
        refused(QsError.INVALID_INPUT, kv8.rope_store, **{**base, **kw})           # {}: no CPU path
    odd = dict(k_cache=torch.zeros(5, 2, 64, 15, dtype=torch.int8), k=torch.zeros(4, 30), q=None, head_dim=15, cos_sin=None)
    refused(QsError.INVALID_INPUT, kv8.rope_store, **{**base, **odd})
    none = dict(q=torch.zeros(0, 64), k=torch.zeros(0, 32), v=torch.zeros(0, 16), tok_slot=I(0), tok_pos=I(0))
    assert kv8.rope_store(**{**base, **none}) is None


def test_attention_that_is_refused():
    base = dict(q=torch.zeros(4, 4 * 16), n_heads=4, n_kv_heads=2, head_dim=16, scale=0.25, window=0, page_table=I(2, 3), page_tokens=64, status=I(1), v_head_dim=8, **CACHE)
    common = BAD_CACHE + [dict(q=torch.zeros(4, 63)), dict(q=torch.zeros(4, 64).half()), dict(n_heads=3, q=torch.zeros(4, 48)), dict(window=-1), dict(window=3, chunk=4),
                          dict(chunk=-1), dict(keep_first=-2), dict(softcap=-1.0), dict(sink=torch.zeros(3)), dict(sink=torch.zeros(4).double()), dict(out=torch.zeros(4, 31)),
                          dict(out=torch.zeros(4, 32).bfloat16()), dict(out_dtype=torch.bfloat16), dict(out=torch.zeros(32, 4).t()), {}]
    for kw in common + [dict(tok_slot=I(3)), dict(tok_pos=I(4).long()), dict(max_context=0)]:
        refused(QsError.INVALID_INPUT, kv8.decode, **{**base, **dict(tok_slot=I(4), tok_pos=I(4), max_context=10), **kw})
    for kw in common + [dict(tiles=I(2, 3)), dict(tiles=I(4)), dict(tiles=I(2, 4).long())]:
        refused(QsError.INVALID_INPUT, kv8.prefill, **{**base, **dict(tiles=I(2, 4)), **kw})
    assert kv8.decode(**{**base, **dict(q=torch.zeros(0, 64), tok_slot=I(0), tok_pos=I(0), max_context=1)}).shape == (0, 32)


def test_pages_that_cannot_be_read():
    k, s = CACHE["k_cache"], CACHE["k_scale"]
    for args in ((k, s, I(2).long()), (k, s[:4], I(2)), (k.short(), s, I(2)), (k[0], s, I(2)), (k, s, I(2), torch.half), (k, s, I(2))):
        refused(QsError.INVALID_INPUT, kv8.read_pages, *args)
