"""Matrix products with 4-bit weights (csrc/q4.cu) against float64."""
import copy

import numpy as np
import pytest
import torch

import narrow_util as U
from qstream_b200.csrc import q4

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def normal(seed, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(16, 64), (1, 1), (17, 33), (40, 96), (31, 200), (64, 129), (100, 1000)])
def test_rounding_of_a_matrix(n, k, group, dtype):
    w = normal(n * 1000 + k + group, n, k, dtype=TYPES[dtype])
    w[0, : min(k, group)] = 0                               # a group of zeros
    if k > 2:
        w[-1, 1], w[-1, 2] = 9.0, -9.0                      # two of the largest magnitude: the first counts
    wide = torch.zeros(n, k + 5, dtype=TYPES[dtype], device="cuda")
    wide[:, :k] = w
    for matrix in (w, wide[:, :k]):                         # contiguous, and part of a wider one
        got = q4.quantize(matrix, group)
        codes, scales = U.unpack(got)
        want_codes, want_scales = U.codes_and_scales(w.float().cpu().numpy(), group)
        np.testing.assert_array_equal(scales[:n], want_scales)
        np.testing.assert_array_equal(codes[:n], want_codes)
        assert (codes[n:] == 8).all() and (scales[n:] == 0).all()
    # half a step of the group, a whole one where the largest value of the other sign finds no code; and the scale's own rounding
    err = np.abs(U.dense(got) - U.f64(w))
    step = np.repeat(np.abs(want_scales), group, axis=1)[:, :k]
    assert (err <= step * (1 + 8 * 2.0 ** -8)).all()


SHAPES = [(16, 64), (1, 1), (17, 33), (100, 96), (64, 1000), (300, 2048), (33, 4100)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", SHAPES)
def test_products(n, k, group, dtype):
    t = TYPES[dtype]
    w = q4.quantize(normal(n + k, n, k, std=0.05), group)
    dense = U.dense(w)
    for m in (1, 2, 3, 7, 8, 9, 16, 17, 31, 32, 33, 64, 65, 130):
        x = normal(m, m, k, dtype=t)
        want, bound = U.linear(U.f64(x), dense, out_bf16=t == torch.bfloat16)
        got = U.f64(q4.linear(x, w))
        assert got.shape == (m, n)
        assert (np.abs(got - want) <= bound).all(), (m, (np.abs(got - want) / bound).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_what_comes_behind_the_product(m, dtype):
    t, n, k = TYPES[dtype], 72, 320
    w = q4.quantize(normal(1, n, k, std=0.1), 64)
    dense, x = U.dense(w), normal(2, m, k, dtype=t)
    bias, r0, r1 = normal(3, n), normal(4, m, n, dtype=t), normal(5, m, n, dtype=t)
    for act in (None, "gelu_new", "silu"):
        for b in (None, bias, bias.bfloat16()):
            for res in ((), (r0,), (r0, r1), (None, r1)):
                for out_dtype in (None, torch.float32):
                    want, bound = U.linear(U.f64(x), dense, None if b is None else U.f64(b), act, [U.f64(r) for r in res if r is not None],
                                           t == torch.bfloat16 and out_dtype is None)
                    got = q4.linear(x, w, b, act, res, out_dtype)
                    assert got.dtype == (out_dtype or t)
                    assert (np.abs(U.f64(got) - want) <= bound).all(), (act, out_dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 3, 16, 70])
def test_views(m, dtype):
    """Rows and results inside wider tensors, at any offset; what lies beside them stays."""
    t, n, k = TYPES[dtype], 50, 136
    w = q4.quantize(normal(1, n, k, std=0.1), 32)
    wide = normal(2, m, k + 30, dtype=t)
    for at in (0, 1, 3, 8, 13):
        x = wide[:, at:at + k]
        out = torch.full((m, n + 20), 7.0, dtype=t, device="cuda")
        res = normal(3, m, n + 9, dtype=t)[:, 2:2 + n]
        q4.linear(x, w, residuals=(res,), out=out[:, 5:5 + n])
        want, bound = U.linear(U.f64(x), U.dense(w), residuals=[U.f64(res)], out_bf16=t == torch.bfloat16)
        assert (np.abs(U.f64(out[:, 5:5 + n]) - want) <= bound).all(), at
        assert (out[:, :5] == 7).all() and (out[:, 5 + n:] == 7).all()


def test_no_rows():
    w = q4.quantize(normal(1, 32, 64), 64)
    assert q4.linear(torch.zeros(0, 64, device="cuda"), w).shape == (0, 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 8, 33, 100])
def test_a_row_has_its_own_result(m, dtype):
    """Neither what the other rows hold nor what is not finite in them reaches a row."""
    t = TYPES[dtype]
    w = q4.quantize(normal(1, 200, 600, std=0.1), 64)
    x = normal(2, m, 600, dtype=t)
    before = q4.linear(x, w)
    if m > 1:
        y = x.clone()
        y[1:] = float("nan")
        y[-1] = float("inf")
        assert torch.equal(q4.linear(y, w)[0], before[0])
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[0, 5] = bad
        got = q4.linear(y, w)
        assert not torch.isfinite(got[0]).all() and torch.equal(got[1:], before[1:])
    assert torch.equal(q4.linear(x, w), before)             # the same bits again


def test_large_and_small_numbers():
    """Sums near the ends of the range of 32 bits: scales and rows of any size."""
    for size in (1e-30, 1e30):
        wf = normal(1, 48, 256) * size
        w = q4.quantize(wf, 64)
        x = normal(2, 5, 256) / size
        want, bound = U.linear(U.f64(x), U.dense(w))
        assert (np.abs(U.f64(q4.linear(x, w)) - want) <= bound).all()


def test_on_another_stream_and_in_a_graph():
    w = q4.quantize(normal(1, 512, 1024, std=0.1), 64)
    x = normal(2, 6, 1024, dtype=torch.bfloat16)
    want = q4.linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = q4.linear(x, w)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, xs, outs = [], [], []
    for i in range(2):                                      # two graphs of one matrix, replayed side by side
        xs.append(x.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(q4.linear(xs[i], w))
        graphs.append(g)
    xs[1].mul_(-1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], -want)


def test_a_float32_row_is_the_same_bits_in_any_batch():
    for k, group in ((2048, 64), (700, 32), (5000, 128)):
        w = q4.quantize(normal(k, 90, k, std=0.1), group)
        x = normal(2, 70, k)
        whole = q4.linear(x, w)
        for m in (1, 2, 3, 5, 6, 16, 33):
            assert torch.equal(q4.linear(x[:m], w), whole[:m])


def test_a_matrix_that_moves_is_read_where_it_lies():
    w = q4.quantize(normal(6, 90, 700, std=0.1), 64)
    twin = copy.deepcopy(w)
    x = normal(7, 3, 700)
    want = q4.linear(x, w)
    w.codes.data, w.scales.data = w.codes.data.clone(), w.scales.data.clone()
    assert torch.equal(q4.linear(x, w), want) and torch.equal(q4.linear(x, twin), want)
    w.codes.copy_(torch.full_like(w.codes, 0x88))
    assert (q4.linear(x, w) == 0).all() and torch.equal(q4.linear(x, twin), want)


@pytest.mark.parametrize("n,k", [(70, 16500), (33, 32768), (20, 9000)])
def test_many_columns(n, k):
    w = q4.quantize(normal(1, n, k, std=0.02), 64)
    for dtype in TYPES.values():
        for m in (1, 5, 12, 40):
            x = normal(m, m, k, dtype=dtype)
            want, bound = U.linear(U.f64(x), U.dense(w), out_bf16=dtype == torch.bfloat16)
            assert (np.abs(U.f64(q4.linear(x, w)) - want) <= bound).all(), m


@pytest.mark.parametrize("m,n,chunks", [(200, 2000, 47), (17, 9500, 93), (130, 20000, 5), (700, 1000, 23), (300, 19000, 7)])
def test_products_of_many_rows_whose_blocks_end_on_half_a_stage(m, n, chunks):
    """An odd number of chunks of 64 columns leaves half of a block's last stage unwritten; again and again, the same bits."""
    k = 64 * chunks
    w = q4.quantize(normal(n + k, n, k, std=0.05), 64)
    x = normal(m, m, k, dtype=torch.bfloat16)
    first = q4.linear(x, w)
    want, bound = U.linear(U.f64(x), U.dense(w), out_bf16=True)
    assert (np.abs(U.f64(first) - want) <= bound).all()
    for _ in range(100):
        assert torch.equal(q4.linear(x, w), first)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(17, 6000, 6016), (130, 2100, 2500), (300, 1000, 2048), (33, 1100, 17000), (1000, 130, 4800), (3000, 16, 12800)])
def test_products_of_many_rows(m, n, k, group):
    """Those that the 5th-generation tensor cores take, with ragged rows, columns and tiles, and what comes behind them."""
    w = q4.quantize(normal(n + k, n, k, std=0.05), group)
    dense = U.dense(w)
    wide = normal(m, m, k + 8, dtype=torch.bfloat16)
    bias, r0, r1 = normal(3, n), normal(4, m, n, dtype=torch.bfloat16), normal(5, m, n, dtype=torch.bfloat16)
    for at in (0, 8, 3):                                    # rows on 16-byte boundaries and off them
        x = wide[:, at:at + k] if at + k <= k + 8 else wide
        for args, kw in (((), {}), ((bias, "gelu_new", (r0, r1)), {}), ((bias, None, (r0,), torch.float32), {})):
            res = [U.f64(r) for r in args[2]] if len(args) > 2 else []
            want, bound = U.linear(U.f64(x), dense, U.f64(bias) if args else None, args[1] if args else None, res, out_bf16=len(args) < 4)
            got = U.f64(q4.linear(x, w, *args))
            assert (np.abs(got - want) <= bound).all(), (at, len(args), (np.abs(got - want) / bound).max())
    out = torch.full((m, n + 7), 7.0, dtype=torch.bfloat16, device="cuda")
    q4.linear(x, w, out=out[:, 3:3 + n])
    want, bound = U.linear(U.f64(x), dense, out_bf16=True)
    assert (np.abs(U.f64(out[:, 3:3 + n]) - want) <= bound).all() and (out[:, :3] == 7).all() and (out[:, 3 + n:] == 7).all()
    y = x.clone()
    y[0, 7], y[-1, 0] = float("nan"), float("inf")
    got = q4.linear(y, w)
    plain = q4.linear(x, w)
    assert not torch.isfinite(got[0]).any() and not torch.isfinite(got[-1]).all() and torch.equal(got[1:-1], plain[1:-1])
    # rows and scales of very different sizes keep their own precision
    z = x * torch.logspace(-30, 30, m, device="cuda")[:, None].bfloat16()
    big = q4.Weight4(w.codes, w.scales * torch.logspace(-2, 2, w.scales.shape[0], device="cuda")[:, None, None, None].bfloat16(), n, k, group)
    want, bound = U.linear(U.f64(z), U.dense(big), out_bf16=True)
    assert (np.abs(U.f64(q4.linear(z, big)) - want) <= bound).all()
