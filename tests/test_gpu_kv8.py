"""The 8-bit cache (csrc/kv8.cu): the write of tokens against its definition, bit for bit; attention against float64."""
import numpy as np
import pytest
import torch

import narrow_util as U
from qstream_b200.csrc import attention_bf16, kv8

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def angles(n, rotary):
    a = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, rotary, 2) / rotary)
    return np.stack([np.cos(a), np.sin(a)], axis=-1).astype(np.float32)


class Cache:
    """Empty pages for some sequences, on the device and as numpy arrays that the definition fills."""

    def __init__(self, seqs, max_pages, heads, dk, dv, seed=0):
        n = seqs * max_pages + 2
        self.table = np.random.default_rng(seed).permutation(n)[:seqs * max_pages].reshape(seqs, max_pages).astype(np.int32)
        self.codes = [np.zeros((n, heads, 64, d), np.int8) for d in (dk, dv)]
        self.scales = [np.zeros((n, heads), np.float32) for _ in range(2)]
        self.dev = [torch.from_numpy(a).cuda() for a in self.codes + self.scales]
        self.table_dev = i32(self.table)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.heads, self.dk, self.dv = heads, dk, dv

    def write(self, slot, pos, k, v, q=None, rotary=0, half=False, first=None, mix=0.0, n_heads=0, q_out=None, table=None):
        cs = angles(4096, rotary) if rotary else None
        kv8.rope_store(q, k, v, n_heads, self.heads, self.dk, rotary, torch.from_numpy(cs).cuda() if rotary else None, i32(slot), i32(pos),
                       self.table_dev if table is None else i32(table), 64, *self.dev, self.status, v_head_dim=self.dv, v_first=first, v_mix=mix,
                       half_layout=half, q_out=q_out)
        kn, vn = (t.float().cpu().numpy().reshape(len(slot), self.heads, -1) for t in (k, v))
        if rotary:
            kn = U.rotate(kn, np.maximum(pos, 0), cs, rotary, half)
        if first is not None:
            vn = np.float32(1 - np.float32(mix)) * vn + np.float32(mix) * first.float().cpu().numpy().reshape(vn.shape)
        U.store(self.codes[0], self.scales[0], kn, slot, pos, self.table)
        U.store(self.codes[1], self.scales[1], vn, slot, pos, self.table)

    def same(self):
        for got, want in zip(self.dev, self.codes + self.scales):
            np.testing.assert_array_equal(got.cpu().numpy(), want)


def rows_of(rng, lens, held):
    """The rows of sequences 0, 1, ... that bring `lens` tokens to the `held` ones."""
    return [i for i, n in enumerate(lens) for _ in range(n)], [h + j for n, h in zip(lens, held) for j in range(n)]


def fresh(rng, rows, width, dtype, std=1.0):
    return torch.tensor(rng.normal(size=(rows, width)) * std).to(TYPES[dtype]).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dk,dv,rotary,half", [(2, 64, 64, 32, False), (1, 128, 80, 64, True), (3, 16, 24, 0, False), (1, 10, 7, 6, True), (2, 256, 256, 64, False),
                                                     (1, 96, 33, 96, True), (1, 512, 512, 2, False)])
def test_tokens_written_in_any_cutting(heads, dk, dv, rotary, half, dtype):
    """Prompts, single tokens, numbers that grow from call to call: codes and scales bit for bit."""
    rng = np.random.default_rng(heads + dk)
    c = Cache(3, 5, heads, dk, dv)
    held = [0, 0, 0]
    for step, lens in enumerate([(1, 70, 0), (1, 1, 130), (1, 1, 1), (62, 57, 0), (1, 1, 1), (64, 3, 60), (1, 1, 1), (1, 1, 1)]):
        slot, pos = rows_of(rng, lens, held)
        std = 0.2 * 1.7 ** step                         # every step brings larger numbers
        c.write(slot, pos, fresh(rng, len(slot), heads * dk, dtype, std), fresh(rng, len(slot), heads * dv, dtype, std), rotary=rotary, half=half)
        held = [a + b for a, b in zip(held, lens)]
        c.same()
    assert int(c.status.item()) == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_are_rotated_as_by_the_plain_cache_write(dtype):
    from qstream_b200.csrc import ops
    rng = np.random.default_rng(3)
    for half in (False, True):
        c = Cache(2, 3, 2, 64, 64)
        slot, pos = [0] * 5 + [1] * 3 + [-1] * 2, [3, 4, 5, 6, 7, 0, 1, 2, 0, 0]
        q, k = fresh(rng, 10, 6 * 64, dtype), fresh(rng, 10, 2 * 64, dtype)
        want = q.clone()
        cs = torch.from_numpy(angles(64, 32)).cuda()
        ops.rope_store(want, None, None, 6, 0, 64, 32, cs, i32(slot), i32(pos), None, 64, None, None, c.status, half_layout=half)
        apart = torch.full_like(q, 9.0)
        c.write(slot, pos, k, k, q=q, rotary=32, half=half, n_heads=6, q_out=apart)
        assert torch.equal(apart, want)                 # padding rows are copied
        c.write(slot, pos, k, k, q=q, rotary=32, half=half, n_heads=6)
        assert torch.equal(q, want)
        c.same()


def test_blended_values():
    rng = np.random.default_rng(4)
    c = Cache(1, 2, 2, 32, 48)
    k, v, first = fresh(rng, 9, 64, "bf16"), fresh(rng, 9, 96, "bf16"), fresh(rng, 9, 96, "bf16")
    c.write([0] * 9, list(range(9)), k, v, first=first, mix=0.3)
    c.same()


def test_rows_of_a_wider_product():
    """q, k and v as ranges of columns of one tensor, as a layer's product leaves them."""
    rng = np.random.default_rng(5)
    c = Cache(2, 3, 2, 64, 32)
    qkv = fresh(rng, 90, 4 * 64 + 128 + 64 + 3, "bf16")
    slot, pos = rows_of(rng, (80, 10), (0, 0))
    c.write(slot, pos, qkv[:, 256:384], qkv[:, 384:448], q=qkv[:, :256], rotary=16, n_heads=4)
    c.same()


def test_scales_at_the_ends_of_their_range():
    c = Cache(1, 1, 1, 4, 4)
    tiny, huge = np.float32(1e-41), np.float32(3.4e38)
    for row, x in enumerate(([0, 0, 0, 0], [tiny, 0, -tiny, 0], [2.0 ** -126] * 4, [1.0, 127.0, -127.0, 0.5], [127.00001, 0, 0, 0], [huge, 1, -huge, 0])):
        t = torch.tensor([x], dtype=torch.float32).cuda()
        c.write([0], [row], t, -t)
        c.same()


def test_numbers_that_are_not_finite_show():
    """A page that was given one reads as NaN, from its first row's next token on no more; other heads and pages stay."""
    rng = np.random.default_rng(6)
    c = Cache(1, 3, 2, 16, 16)
    for bad in (float("nan"), float("inf"), float("-inf")):
        c.write([0] * 70, list(range(70)), fresh(rng, 70, 32, "f32"), fresh(rng, 70, 32, "f32"))
        k, v = fresh(rng, 1, 32, "f32"), fresh(rng, 1, 32, "f32")
        k[0, 3], v[0, 20] = bad, bad
        c.write([0], [70], k, v)
        c.write([0], [71], fresh(rng, 1, 32, "f32"), fresh(rng, 1, 32, "f32"))
        c.same()
        page = i32([c.table[0, 0], c.table[0, 1]])
        got = kv8.read_pages(c.dev[0], c.dev[2], page)
        assert torch.isnan(got[1, 0]).all() and torch.isfinite(got[0]).all() and torch.isfinite(got[1, 1]).all()
        assert torch.isnan(kv8.read_pages(c.dev[1], c.dev[3], page)[1, 1]).all()


def test_rows_that_cannot_be_written_are_reported():
    rng = np.random.default_rng(7)
    for slot, pos, table, code in (([0, 1], [64 * 3, 0], None, 1), ([0, 1], [-1, 0], None, 1), ([2, 1], [0, 0], None, 1),
                                   ([0, 1], [64, 0], "holes", 2), ([0, 1], [0, 0], "far", 2)):
        c = Cache(2, 3, 1, 16, 16)
        t = c.table.copy()
        if table:
            t[0, :2] = [0 if code == 2 and table == "holes" else 10 ** 6, -1]
        before = [d.clone() for d in c.dev]
        k = fresh(rng, 2, 16, "f32")
        kv8.rope_store(None, k, k, 0, 1, 16, 0, None, i32(slot), i32(pos), i32(t), 64, *c.dev, c.status)
        assert int(c.status.item()) == code
        for got, was in zip(c.dev, before):             # the other row alone has been written
            changed = (got != was).flatten(1).any(dim=1).nonzero().flatten().tolist()
            assert set(changed) <= {int(t[1, 0])}
    # two runs of rows for one page; the same position twice
    for pos in ([5, 9], [5, 5], [9, 5]):
        c = Cache(1, 2, 1, 16, 16)
        k = fresh(rng, 2, 16, "f32")
        kv8.rope_store(None, k, k, 0, 1, 16, 0, None, i32([0, 0]), i32(pos), c.table_dev, 64, *c.dev, c.status)
        assert int(c.status.item()) == 5
        U.store(c.codes[0], c.scales[0], k[:1].cpu().numpy()[:, None], [0], pos[:1], c.table)
        np.testing.assert_array_equal(c.dev[0].cpu().numpy(), c.codes[0])


def test_pages_read_back():
    rng = np.random.default_rng(8)
    kc, vc, ks, vs, _ = U.paged(rng, [300], 3, 48, 20)
    for codes, scales in ((kc, ks), (vc, vs)):
        for dtype in TYPES.values():
            got = kv8.read_pages(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), i32([2, 0, 2, 99, -1]), dtype)
            want = codes[[2, 0, 2]].astype(np.float64) * scales[[2, 0, 2]].astype(np.float64)[..., None, None]
            np.testing.assert_array_equal(U.f64(got[:3]), want)             # exact in both types
            assert torch.isnan(got[3:]).all()
    assert kv8.read_pages(torch.from_numpy(kc).cuda(), torch.from_numpy(ks).cuda(), i32([]).reshape(0)).shape == (0, 3, 64, 48)


# ------------------------------------------------------------------------------------------------ attention

def device(pages):
    return [torch.from_numpy(x).cuda() for x in pages[:4]], i32(pages[4])


def check(got, want, bound, what=None):
    err = np.abs(U.f64(got).reshape(want.shape) - want)
    assert (err <= bound).all(), (what, float((err / np.maximum(bound, 1e-300)).max()))


MASKS = (dict(), dict(window=100), dict(window=1), dict(softcap=2.5), dict(chunk=96), dict(window=70, keep_first=5), dict(window=64, keep_first=200))
SIZES = [(1, 1, 64, 64), (2, 2, 128, 128), (16, 4, 128, 128), (5, 1, 64, 32), (8, 1, 80, 48), (9, 3, 256, 256), (12, 1, 96, 160), (2, 1, 512, 512), (3, 3, 20, 10), (4, 2, 24, 40),
         (32, 2, 64, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G,dk,dv", SIZES)
def test_single_tokens(H, G, dk, dv, dtype):
    lens = [1, 16, 17, 63, 64, 65, 130, 256, 257, 513, 700]
    rng = np.random.default_rng(H * dk + dv)
    pages = U.paged(rng, lens, G, dk, dv)
    dev, table = device(pages)
    slot, pos = list(range(len(lens))) + [-1], [n - 1 for n in lens] + [5]
    q = torch.tensor(rng.normal(size=(len(slot), H * dk))).to(TYPES[dtype]).cuda()
    sink = torch.tensor(rng.normal(size=H) + 1, dtype=torch.float32).cuda()
    for opts in MASKS:
        for s in (None, sink):
            for out_dtype in (None, torch.float32):
                status = torch.zeros(1, dtype=torch.int32, device="cuda")
                args = dict(opts)
                got = kv8.decode(q, H, G, dk, dk ** -0.5, args.pop("window", 0), i32(slot), i32(pos), table, 64, *dev, max(lens), status, v_head_dim=dv, sink=s,
                                 out_dtype=out_dtype, **args)
                assert int(status.item()) == 0 and got.dtype == (out_dtype or TYPES[dtype])
                want, bound = U.attention(U.f64(q).reshape(len(slot), H, dk), pages[:2], pages[2:4], slot, pos, pages[4], H // G, dk ** -0.5,
                                          sink=None if s is None else U.f64(s), wide_weights=dtype == "f32", out_bf16=got.dtype == torch.bfloat16, **opts)
                check(got, want, bound, (opts, s is not None, out_dtype))
                assert (got[-1] == 0).all()             # a row of no sequence


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G,dk,dv", [(1, 1, 64, 64), (4, 2, 128, 128), (3, 1, 64, 32), (2, 1, 256, 256), (2, 2, 80, 48), (2, 1, 20, 10), (2, 1, 320, 16)])
def test_prompts(H, G, dk, dv, dtype):
    """Prompts of unequal lengths, some behind cached tokens; rows between them belong to nobody."""
    new, held = [1, 130, 64, 300, 7], [0, 0, 63, 100, 250]
    lens = [a + b for a, b in zip(new, held)]
    rng = np.random.default_rng(H * dk + dv)
    pages = U.paged(rng, lens, G, dk, dv)
    dev, table = device(pages)
    slot, pos, tiles, row = [], [], [], 0
    for i, (n, h) in enumerate(zip(new, held)):
        tiles += [(row + a, min(128, n - a), h + a, i) for a in range(0, n, 128)] + [(0, 0, 0, 0)]
        slot += [i] * n + [-1] * (i == 2) * 3
        pos += list(range(h, h + n)) + [0] * (i == 2) * 3
        row = len(slot)
    q = torch.tensor(rng.normal(size=(len(slot), H * dk))).to(TYPES[dtype]).cuda()
    sink = torch.tensor(rng.normal(size=H) + 1, dtype=torch.float32).cuda()
    for opts in MASKS:
        for s in (None, sink):
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            args = dict(opts)
            out = torch.full((len(slot), H * dv), 7.0, dtype=TYPES[dtype], device="cuda")
            got = kv8.prefill(q, H, G, dk, dk ** -0.5, args.pop("window", 0), i32(tiles), table, 64, *dev, status, v_head_dim=dv, sink=s, out=out, **args)
            assert int(status.item()) == 0 and got is out
            want, bound = U.attention(U.f64(q).reshape(len(slot), H, dk), pages[:2], pages[2:4], slot, pos, pages[4], H // G, dk ** -0.5,
                                      sink=None if s is None else U.f64(s), wide_weights=dtype == "f32", out_bf16=dtype == "bf16", **opts)
            if dtype == "bf16":                         # weights rounded to bfloat16 on this path
                bound = bound + 2.0 ** -8 * 127 * float(pages[3].max())
            live = np.asarray(slot) >= 0
            check(got[torch.from_numpy(live).cuda()], want[live], bound[live], (opts, s is not None))
            assert (got[torch.from_numpy(~live).cuda()] == 7).all()
    got = kv8.prefill(q, H, G, dk, dk ** -0.5, 0, i32(tiles), table, 64, *dev, status, v_head_dim=dv, padded=True)
    assert (got[torch.from_numpy(~live).cuda()] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_seen_does_not_count(dtype):
    """Pages that read as NaN where a mask hides them, and what lies behind a sequence's end."""
    rng = np.random.default_rng(11)
    lens = [300]
    kc, vc, ks, vs, t = U.paged(rng, lens, 2, 64, 64)
    q = torch.tensor(rng.normal(size=(1, 4 * 64))).to(TYPES[dtype]).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def run(k_scale, v_scale, codes=(kc, vc), rows=q, pos=[299], tiles=None, window=0):
        (dev, table) = device((*codes, k_scale, v_scale, t))
        if tiles is not None:
            return kv8.prefill(rows, 4, 2, 64, 0.125, window, i32(tiles), table, 64, *dev, status)
        return kv8.decode(rows, 4, 2, 64, 0.125, window, i32([0] * len(pos)), i32(pos), table, 64, *dev, 320, status)

    plain = run(ks, vs, window=100)
    bad = ks.copy(), vs.copy()
    bad[0][t[0, :3]], bad[1][t[0, :3]] = np.nan, np.nan                         # positions 0 .. 191: outside the window of 100
    assert torch.equal(run(*bad, window=100), plain)
    seen = run(*bad)
    assert torch.isnan(seen).all()
    one = ks.copy(), vs.copy()
    one[1][t[0, 1], 1] = np.nan                                                 # values of one page, key head 1
    got = run(*one)
    assert torch.equal(got[:, :128], run(ks, vs)[:, :128]) and torch.isnan(got[:, 128:]).all()
    tail = kc.copy(), vc.copy()
    for c in tail:
        c[t[0, 4], :, 300 - 256:] = 77                                          # behind the end
    assert torch.equal(run(ks, vs, tail), run(ks, vs))
    # a prompt whose later rows see a page that reads as NaN: the earlier rows do not
    rows = torch.tensor(rng.normal(size=(128, 4 * 64))).to(TYPES[dtype]).cuda()
    tiles = [(0, 128, 64, 0)]
    late = ks.copy(), vs.copy()
    late[1][t[0, 2]] = np.nan                                                   # positions 128 .. 191
    got, want = run(*late, rows=rows, tiles=tiles), run(ks, vs, rows=rows, tiles=tiles)
    assert torch.equal(got[:64], want[:64]) and torch.isnan(got[64:]).all()
    late[0][t[0, 1]] = np.nan                                                   # the page of the first rows: with a window of 1 it is all they see
    got = run(late[0], vs, rows=rows, tiles=tiles, window=1)
    assert torch.isnan(got[:64]).all() and torch.isfinite(got[64:]).all()
    assert int(status.item()) == 0


def test_rows_that_cannot_be_read_are_reported():
    rng = np.random.default_rng(12)
    lens = [200, 70]
    pages = U.paged(rng, lens, 1, 64, 64)
    dev, table = device(pages)
    q = torch.tensor(rng.normal(size=(2, 64))).bfloat16().cuda()
    for slot, pos, reach, code in (([0, 5], [199, 3], 256, 1), ([0, 1], [199, -2], 256, 1), ([0, 1], [199, 999], 256, 1), ([0, 1], [199, 130], 256, 3)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = kv8.decode(q, 1, 1, 64, 0.125, 0, i32(slot), i32(pos), table, 64, *dev, reach, status)
        assert int(status.item()) == code
        alone = kv8.decode(q[:1], 1, 1, 64, 0.125, 0, i32([0]), i32([199]), table, 64, *dev, 256, status)
        assert torch.equal(got[:1], alone)
        if code == 1:
            assert (got[1] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_tiles_that_cannot_be_read_are_reported(dtype):
    rng = np.random.default_rng(17)
    pages = U.paged(rng, [200, 70], 1, 64, 64)
    dev, table = device(pages)
    q = torch.tensor(rng.normal(size=(20, 64))).to(TYPES[dtype]).cuda()
    good = (0, 10, 190, 0)
    for bad, code in (((10, 11, 0, 1), 1), ((-1, 5, 0, 1), 1), ((10, 5, 0, 2), 1), ((10, 5, 0, -1), 1), ((10, 5, -3, 1), 1), ((10, 5, 254, 0), 1), ((10, 5, 130, 1), 3)):
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.full((20, 64), 7.0, dtype=TYPES[dtype], device="cuda")
        kv8.prefill(q, 1, 1, 64, 0.125, 0, i32([good, bad]), table, 64, *dev, status, out=out)
        assert int(status.item()) == code, bad
        want, bound = U.attention(U.f64(q).reshape(20, 1, 64), pages[:2], pages[2:4], [0] * 10 + [-1] * 10, list(range(190, 200)) + [0] * 10, pages[4], 1, 0.125,
                                  wide_weights=dtype == "f32", out_bf16=dtype == "bf16")
        check(out[:10], want[:10], bound[:10] + (2.0 ** -8 * 127 * float(pages[3].max()) if dtype == "bf16" else 0))
        if code == 1:
            assert (out[10:] == 7).all()


def test_a_row_does_not_depend_on_its_batch():
    rng = np.random.default_rng(13)
    lens = [1000, 3, 517, 64, 2000, 129]
    pages = U.paged(rng, lens, 2, 128, 128)
    dev, table = device(pages)
    q = torch.tensor(rng.normal(size=(6, 8 * 128))).bfloat16().cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    run = lambda rows, reach: kv8.decode(q[rows], 8, 2, 128, 128 ** -0.5, 0, i32(rows), i32([lens[r] - 1 for r in rows]), table, 64, *dev, reach, status)   # noqa: E731
    whole = run(list(range(6)), 2000)
    for r in range(6):
        for reach in (lens[r], 2000, 2048):
            assert torch.equal(run([r], reach)[0], whole[r])


def test_long_cache():
    """Pages whose codes lie beyond 2^31 bytes, and a sequence of more than a hundred thousand keys."""
    rng = np.random.default_rng(14)
    heads, d, far = 8, 512, 9000                        # 9,000 pages of 256 KiB
    k = torch.zeros((far, heads, 64, d), dtype=torch.int8, device="cuda")
    v = torch.zeros((far, heads, 64, d), dtype=torch.int8, device="cuda")
    ks, vs = (torch.zeros((far, heads), device="cuda") for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    table = i32([[far - 1, 2, far - 2]])
    x, y = fresh(rng, 150, heads * d, "f32"), fresh(rng, 150, heads * d, "f32")
    kv8.rope_store(None, x, y, 0, heads, d, 0, None, i32([0] * 150), i32(range(150)), table, 64, k, v, ks, vs, status)
    codes, scales = [np.zeros((3, heads, 64, d), np.int8) for _ in range(2)], [np.zeros((3, heads), np.float32) for _ in range(2)]
    small = np.array([[0, 1, 2]])
    for i, t in enumerate((x, y)):
        U.store(codes[i], scales[i], t.cpu().numpy().reshape(150, heads, d), [0] * 150, list(range(150)), small)
        np.testing.assert_array_equal((k, v)[i][[far - 1, 2, far - 2]].cpu().numpy(), codes[i])
    q = fresh(rng, 1, heads * d, "f32")
    want, bound = U.attention(U.f64(q).reshape(1, heads, d), codes, scales, [0], [149], small, 1, d ** -0.5)
    check(kv8.decode(q, heads, heads, d, d ** -0.5, 0, i32([0]), i32([149]), table, 64, k, v, ks, vs, 150, status), want, bound)
    assert int(status.item()) == 0
    del k, v
    lens = [131072 + 77]
    pages = U.paged(rng, lens, 1, 64, 64)
    dev, table = device(pages)
    for dtype in TYPES:
        q = fresh(rng, 1, 4 * 64, dtype)
        want, bound = U.attention(U.f64(q).reshape(1, 4, 64), pages[:2], pages[2:4], [0], [lens[0] - 1], pages[4], 4, 0.125, wide_weights=dtype == "f32", out_bf16=dtype == "bf16")
        check(kv8.decode(q, 4, 1, 64, 0.125, 0, i32([0]), i32([lens[0] - 1]), table, 64, *dev, lens[0], status), want, bound)


def test_views_streams_and_graphs():
    """Queries and results inside wider tensors at any offset; another stream; two graphs over one cache replayed side by side."""
    rng = np.random.default_rng(15)
    lens = [400, 90]
    pages = U.paged(rng, lens, 2, 64, 64)
    dev, table = device(pages)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    slot, pos = i32([0, 1]), i32([399, 89])
    wide = torch.tensor(rng.normal(size=(2, 4 * 64 + 40))).bfloat16().cuda()
    for at in (0, 1, 8, 13):
        q = wide[:, at:at + 256]
        out = torch.full((2, 256 + 20), 7.0, dtype=torch.bfloat16, device="cuda")
        kv8.decode(q, 4, 2, 64, 0.125, 0, slot, pos, table, 64, *dev, 400, status, out=out[:, 3:259])
        want, bound = U.attention(U.f64(q).reshape(2, 4, 64), pages[:2], pages[2:4], [0, 1], [399, 89], pages[4], 2, 0.125, wide_weights=False, out_bf16=True)
        check(out[:, 3:259], want, bound, at)
        assert (out[:, :3] == 7).all() and (out[:, 259:] == 7).all()
        tiles = i32([(0, 1, 399, 0), (1, 1, 89, 1)])
        out = torch.full((2, 256 + 20), 7.0, dtype=torch.bfloat16, device="cuda")
        kv8.prefill(q, 4, 2, 64, 0.125, 0, tiles, table, 64, *dev, status, out=out[:, 3:259])
        check(out[:, 3:259], want, bound + 2.0 ** -8 * 127 * float(pages[3].max()), at)
        assert (out[:, :3] == 7).all() and (out[:, 259:] == 7).all()
    q = wide[:, :256].contiguous()
    call = lambda x: kv8.decode(x, 4, 2, 64, 0.125, 0, slot, pos, table, 64, *dev, 400, status)       # noqa: E731
    want = call(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(q)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, qs, outs = [], [], []
    for i in range(2):
        qs.append(q.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(qs[i]))
        graphs.append(g)
    qs[1].zero_()
    zero = call(torch.zeros_like(q))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], zero)


@pytest.mark.parametrize("dtype", TYPES)
def test_write_then_attend_as_a_step_does(dtype):
    """A prompt, then single tokens: write, attend, write, attend; the attention of every step over what the definition holds."""
    rng = np.random.default_rng(16)
    H, G, dk, dv, seqs = 4, 2, 64, 48, 3
    c = Cache(seqs, 4, G, dk, dv, seed=1)
    held = [0] * seqs
    for lens in ((100, 5, 64), (1, 1, 1), (1, 1, 1), (30, 1, 1), (1, 60, 1), (1, 1, 1)):
        slot, pos = rows_of(rng, lens, held)
        q, k, v = fresh(rng, len(slot), H * dk, dtype), fresh(rng, len(slot), G * dk, dtype), fresh(rng, len(slot), G * dv, dtype)
        c.write(slot, pos, k, v, q=q, rotary=32, half=True, n_heads=H)
        c.same()
        args = (H, G, dk, dk ** -0.5, 0)
        if max(lens) == 1:
            got = kv8.decode(q, *args, i32(slot), i32(pos), c.table_dev, 64, *c.dev, 256, c.status, v_head_dim=dv)
        else:
            batch = type("B", (), dict(slots=list(range(seqs)), new_tokens=list(lens), p0=held))()
            got = kv8.prefill(q, *args, attention_bf16.prefill_tiles(batch, q.device), c.table_dev, 64, *c.dev, c.status, v_head_dim=dv)
        want, bound = U.attention(U.f64(q).reshape(-1, H, dk), c.codes, c.scales, slot, pos, c.table, H // G, dk ** -0.5, wide_weights=dtype == "f32", out_bf16=dtype == "bf16")
        if dtype == "bf16" and max(lens) > 1:
            bound = bound + 2.0 ** -8 * 127 * float(c.scales[1].max())
        check(got, want, bound, lens)
        held = [a + b for a, b in zip(held, lens)]
    assert int(c.status.item()) == 0
