"""The operators over 4-bit weights and 8-bit pages at the ends of their ranges."""
import numpy as np
import pytest
import torch

import narrow_util as U
from qstream_b200.csrc import kv8, q4
from test_gpu_kv8 import MASKS

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def device(pages):
    return [torch.from_numpy(x).cuda() for x in pages[:4]], i32(pages[4])


def normal(seed, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def close(got, want, bound, what=None):
    err = np.abs(U.f64(got).reshape(want.shape) - want)
    assert (err <= bound).all(), (what, float(np.nanmax(err / np.maximum(bound, 1e-300))))


def reference(q, pages, slot, pos, per, scale, dtype, bf16_weights, **opts):
    """`narrow_util.attention`.  Prompts of bfloat16 rows on the tensor cores round each weight to bfloat16, by 2^-8 of it at most; their sum is taken of
    the weights before that.  So a result moves by 2^-8 of the sum of p |v|, which is the attention over the values' sizes."""
    want, bound = U.attention(q, pages[:2], pages[2:4], slot, pos, pages[4], per, scale, wide_weights=dtype == "f32" or bf16_weights, out_bf16=dtype == "bf16", **opts)
    if bf16_weights:
        sizes, more = U.attention(q, (pages[0], np.abs(pages[1])), pages[2:4], slot, pos, pages[4], per, scale, **opts)
        bound = bound + (1 + 2.0 ** -8) * 2.0 ** -8 * (sizes + more)
    return want, bound


class Scaled:
    """Keys of 2^e against queries of 2^-e, beside values of as much (as far as 150 of them have a sum): what attention makes of pages is what they read back as."""

    def __init__(self, e, size, dtype):
        rng = np.random.default_rng(size + 200 + e)
        self.size, self.dtype, self.e_v = size, dtype, min(max(e, -100), 112)
        kc, vc, ks, vs, table = U.paged(rng, [150, 64], 2, size, size)
        self.pages = kc, vc, np.full_like(ks, 2.0 ** e), np.full_like(vs, 2.0 ** self.e_v), table
        self.slot, self.pos = [0] * 20 + [1], list(range(130, 150)) + [63]
        self.q = (torch.tensor(rng.normal(size=(21, 4 * size))) * 2.0 ** (-e - 6)).to(TYPES[dtype]).cuda()
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(self, call, bf16_weights=False, **rows):
        dev, table = device(self.pages)
        got = call(self.q, 4, 2, self.size, self.size ** -0.5, 0, **rows, page_table=table, page_tokens=64, k_cache=dev[0], v_cache=dev[1], k_scale=dev[2], v_scale=dev[3],
                   status=self.status)
        want, bound = reference(U.f64(self.q).reshape(21, 4, self.size), self.pages, self.slot, self.pos, 2, self.size ** -0.5, self.dtype, bf16_weights)
        close(got, want, bound)
        assert int(self.status.item()) == 0

    def prompts(self):
        self.run(kv8.prefill, self.dtype == "bf16" and self.size % 16 == 0, tiles=i32([(0, 20, 130, 0), (20, 1, 63, 1)]))

    def single_tokens(self):
        self.run(kv8.decode, tok_slot=i32(self.slot), tok_pos=i32(self.pos), max_context=150)


EXPONENTS = [-126, -110, 0, 90, 100, 104, 105, 112, 120]


@pytest.mark.parametrize("size", [64, 80, 144])
@pytest.mark.parametrize("e", EXPONENTS)
def test_prompts_over_scales_of_any_size(e, size):
    Scaled(e, size, "bf16").prompts()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [64, 80, 144])
@pytest.mark.parametrize("e", EXPONENTS)
def test_single_tokens_over_scales_of_any_size(e, size, dtype):
    Scaled(e, size, dtype).single_tokens()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("e", EXPONENTS)
def test_the_plain_kernel_over_scales_of_any_size(e, dtype):
    """Head sizes that are no multiples of 16, and prompts of float32 rows."""
    Scaled(e, 20, dtype).prompts()
    Scaled(e, 20, dtype).single_tokens()
    if dtype == "f32":
        Scaled(e, 64, dtype).prompts()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [64, 128, 256])
def test_a_row_with_a_sink_does_not_depend_on_its_batch(size, dtype):
    """Contexts of one split, whose results need no merge, and of several: the same bits, whatever the sink counts beside the keys."""
    rng = np.random.default_rng(21)
    lens = [1000, 3, 64, 90, 128, 37]
    pages = U.paged(rng, lens, 2, size, size)
    dev, table = device(pages)
    q = torch.tensor(rng.normal(size=(6, 8 * size))).to(TYPES[dtype]).cuda()
    sink = torch.linspace(-3, 9, 8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(rows, reach, **kw):
        return kv8.decode(q[rows], 8, 2, size, size ** -0.5, 0, i32(rows), i32([lens[r] - 1 for r in rows]), table, 64, *dev, reach, status, sink=sink, **kw)

    for out_dtype in (None, torch.float32):
        whole = run(list(range(6)), 1000, out_dtype=out_dtype)
        for r in range(1, 6):
            for reach in (lens[r], 128, 256, 300):
                assert torch.equal(run([r], reach, out_dtype=out_dtype)[0], whole[r]), (r, reach)
    assert int(status.item()) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [64, 256, 20])                 # of a head: 256 and 128 keys to a split, and the plain kernel
@pytest.mark.parametrize("reach", [1, 100, 200, 256, 257, 600])
def test_positions_from_the_context_on_are_reported(reach, size, dtype):
    rng = np.random.default_rng(22)
    pages = U.paged(rng, [700, 700], 1, size, size)
    dev, table = device(pages)
    q = torch.tensor(rng.normal(size=(2, 2 * size))).to(TYPES[dtype]).cuda()
    run = lambda rows, pos, status: kv8.decode(q[rows], 2, 1, size, size ** -0.5, 0, i32(rows), i32(pos), table, 64, *dev, reach, status)   # noqa: E731
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    last = run([0], [reach - 1], status)
    assert int(status.item()) == 0
    want, bound = U.attention(U.f64(q[:1]).reshape(1, 2, size), pages[:2], pages[2:4], [0], [reach - 1], pages[4], 2, size ** -0.5, wide_weights=dtype == "f32", out_bf16=dtype == "bf16")
    close(last, want, bound)
    for beyond in (reach, reach + 1, 699):
        status.zero_()
        got = run([0, 1], [reach - 1, beyond], status)
        assert int(status.item()) == 1 and (got[1] == 0).all() and torch.equal(got[:1], last), beyond


@pytest.mark.parametrize("dtype", TYPES)
def test_tiles_at_the_end_of_32_bits_are_reported(dtype):
    """A first row or position whose sum with the number of rows has no place in 32 bits."""
    rng = np.random.default_rng(23)
    pages = U.paged(rng, [200], 1, 64, 64)
    dev, table = device(pages)
    q = torch.tensor(rng.normal(size=(20, 64))).to(TYPES[dtype]).cuda()
    top = 2 ** 31 - 1
    for bad in ((top, 5, 0, 0), (top - 4, 5, 0, 0), (top - 100, 128, 0, 0), (10, 5, top, 0), (10, 5, top - 3, 0), (10, top, 0, 0), (-2 ** 31, 5, 0, 0), (10, 5, -2 ** 31, 0)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.full((20, 64), 7.0, dtype=TYPES[dtype], device="cuda")
        kv8.prefill(q, 1, 1, 64, 0.125, 0, i32([bad]), table, 64, *dev, status, out=out)
        assert int(status.item()) == 1 and (out == 7).all(), bad


@pytest.mark.parametrize("m", [40, 130])
@pytest.mark.parametrize("x_size,w_size", [(2.0 ** -105, 2.0 ** 122), (2.0 ** 122, 2.0 ** -122), (2.0 ** -100, 2.0 ** 80), (2.0 ** 60, 2.0 ** 50), (2.0 ** -60, 2.0 ** -50)])
def test_powers_of_two_of_rows_and_matrix_far_apart(x_size, w_size, m):
    """Large scales beside small rows and the other way round, where the results lie within 32 bits."""
    n, k = 5000, 4096
    w = q4.quantize(normal(1, n, k) * w_size, 64)
    x = (normal(2, m, k) * x_size).bfloat16()
    assert torch.isfinite(w.scales.float()).all() and (w.scales != 0).any()
    want, bound = U.linear(U.f64(x), U.dense(w), out_bf16=True)
    got = U.f64(q4.linear(x, w, out_dtype=torch.float32))
    assert (np.abs(got - want) <= bound).all(), float(np.nanmax(np.abs(got - want) / bound))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(16, 64), (24, 100), (300, 64)])
def test_more_rows_than_a_grid_holds(n, k, dtype):
    t, m = TYPES[dtype], 140000
    w = q4.quantize(normal(1, n, k, std=0.1), 32)
    x, bias, r0 = normal(2, m, k, dtype=t), normal(3, n), normal(4, m, n, dtype=t)
    want, bound = U.linear(U.f64(x), U.dense(w), U.f64(bias), None, [U.f64(r0)], out_bf16=t == torch.bfloat16)
    got = q4.linear(x, w, bias, residuals=(r0,))
    assert (np.abs(U.f64(got) - want) <= bound).all()
    out = torch.full((m, n + 3), 7.0, dtype=t, device="cuda")
    assert q4.linear(x, w, bias, residuals=(None, r0), out=out[:, 1:1 + n]).data_ptr() == out[:, 1:].data_ptr()
    assert torch.equal(out[:, 1:1 + n], got) and (out[:, 0] == 7).all() and (out[:, 1 + n:] == 7).all()


@pytest.mark.parametrize("H,G,dk,dv", [(1, 1, 64, 64), (4, 2, 128, 128), (3, 1, 64, 32), (2, 1, 256, 256), (2, 2, 80, 48), (4, 1, 144, 192)])
def test_prompts_are_off_by_the_rounding_of_their_weights_and_no_more(H, G, dk, dv):
    new, held = [1, 130, 64, 300, 7], [0, 0, 63, 100, 250]
    lens = [a + b for a, b in zip(new, held)]
    rng = np.random.default_rng(H * dk + dv + 1)
    pages = U.paged(rng, lens, G, dk, dv)
    dev, table = device(pages)
    slot, pos, tiles, row = [], [], [], 0
    for i, (n, h) in enumerate(zip(new, held)):
        tiles += [(row + a, min(128, n - a), h + a, i) for a in range(0, n, 128)]
        slot, pos, row = slot + [i] * n, pos + list(range(h, h + n)), row + n
    q = torch.tensor(rng.normal(size=(row, H * dk))).bfloat16().cuda()
    sink = torch.tensor(rng.normal(size=H) + 1, dtype=torch.float32).cuda()
    for opts in MASKS:
        for s in (None, sink):
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            args = dict(opts)
            got = kv8.prefill(q, H, G, dk, dk ** -0.5, args.pop("window", 0), i32(tiles), table, 64, *dev, status, v_head_dim=dv, sink=s, **args)
            want, bound = reference(U.f64(q).reshape(row, H, dk), pages, slot, pos, H // G, dk ** -0.5, "bf16", True, sink=None if s is None else U.f64(s), **opts)
            close(got, want, bound, (opts, s is not None))
            assert np.median(bound) < 0.25 * np.median(np.abs(want))        # a kernel that returned something else would show
            assert int(status.item()) == 0


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [33, 200])
def test_products_of_many_rows_with_outliers(m, group):
    """Rows whose largest number meets weights of zero, beside numbers down to 2^-40 of it, and groups of very different scales in one row of the
    matrix.  As 16-bit floats a number is off by 2^-25 of its row's largest at most, and a weight by eight times 2^-25 of its row's largest scale."""
    n, k = 1200, 16384
    wf = normal(1, n, k) * torch.logspace(-9, 0, k // 128, base=10.0, device="cuda").repeat_interleave(128)
    wf[:, 7] = 0
    w = q4.quantize(wf, group)
    dense = U.dense(w)
    assert (dense[:, 7] == 0).all()
    x = (normal(2, m, k) * 2.0 ** -torch.randint(0, 40, (m, k), generator=torch.Generator().manual_seed(3)).cuda()).bfloat16()
    x[:, 7] = 2.0 ** 20 * (1 + torch.rand(m, generator=torch.Generator().manual_seed(4))).cuda()
    want, bound = U.linear(U.f64(x), dense, out_bf16=False)
    size, scale = np.abs(U.f64(x)), np.abs(U.unpack(w)[1][:n]).max(axis=1)
    off = 2.0 ** -25 * (size.max(axis=1)[:, None] * np.abs(dense).sum(axis=1)[None] + 8 * (1 + 2.0 ** -10) * size.sum(axis=1)[:, None] * scale[None])
    got = U.f64(q4.linear(x, w, out_dtype=torch.float32))
    assert (np.abs(got - want) <= bound + off).all(), float((np.abs(got - want) / (bound + off)).max())
    # up to 16 rows the numbers are taken as they are
    few = U.f64(q4.linear(x[:16], w, out_dtype=torch.float32))
    assert (np.abs(few - want[:16]) <= bound[:16]).all()
