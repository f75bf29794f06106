"""Products with 4-bit weights whose rows are many: a block of the kernel for few rows of x walks over more tiles than it sums up at a time."""
import pytest
import torch

from qstream_b200.csrc import q4

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
# rows of the matrix from which each of the device's 148 SMs, a block to each, has nine tiles of 16 rows and more
NINE_TILES = 20000


def normal(seed, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * std).to(dtype)


def dense(w):
    """The matrix in float64, from the codes and scales as `q4.Weight4` describes them."""
    tiles, chunks = w.codes.shape[:2]
    nibbles = torch.stack([w.codes & 15, w.codes >> 4], dim=-1).view(tiles, chunks, 8, 4, 2, 2, 8)     # [tile][chunk][g][t][h][u][i]
    in_order = nibbles[..., [0, 4, 1, 5, 2, 6, 3, 7]]                       # columns 0 .. 7 of the code's eight
    codes = in_order.permute(0, 5, 2, 1, 4, 3, 6).reshape(tiles * 16, chunks * 64)
    scales = w.scales.permute(0, 3, 2, 1).reshape(tiles * 16, -1).double().repeat_interleave(w.group, dim=1)[:, :chunks * 64]
    return ((codes.double() - 8) * scales)[:w.out_features, :w.in_features]


def check(x, w, matrix):
    """Against float64, within the bound of `narrow_util.linear`."""
    got = q4.linear(x, w)
    y, size = x.double() @ matrix.T, x.double().abs() @ matrix.abs().T
    err = 2.0 ** -23 * (256 + x.shape[1] / 32) * size
    bound = err + (2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -24) * (y.abs() + err)
    wrong = (got.double() - y).abs() > bound
    assert not wrong.any(), (x.shape, x.dtype, w.shape, int(wrong.any(dim=0).sum()))
    assert torch.equal(q4.linear(x, w), got)


def small(m, n, k):
    """bfloat16 products of more than 16 rows stay with the kernel for few rows below this many multiplications."""
    return m <= 16 or m * n * k < 6e8


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("share", range(1, 17))
def test_every_share_of_a_tile(share, group):
    """1 to 16 warps share a tile's columns: 256 columns to a warp for up to 8 columns of rows of x (float32 rows are three columns), else 128."""
    for columns, rows in ((256, {"bf16": (1, 8)}), (128, {"bf16": (12, 17), "f32": (1, 3, 6)})):
        n, k = NINE_TILES, columns * share - 37
        w = q4.quantize(normal(share, n, k, std=0.05), group)
        matrix = dense(w)
        for dtype, ms in rows.items():
            for m in ms:
                if dtype == "f32" or small(m, n, k):
                    check(normal(m, m, k, dtype=TYPES[dtype]), w, matrix)


@pytest.mark.parametrize("n,k", [(50257, 768), (50257, 1280), (24576, 1152), (NINE_TILES, 256), (NINE_TILES, 640), (100003, 200), (160000, 64), (NINE_TILES, 5000), (37889, 1)])
def test_wide_matrices(n, k):
    w = q4.quantize(normal(k, n, k, std=0.05), 64)
    matrix = dense(w)
    for dtype, ms in (("bf16", (1, 8, 12, 40)), ("f32", (1, 3, 11))):
        for m in ms:
            if dtype == "f32" or small(m, n, k):
                check(normal(m, m, k, dtype=TYPES[dtype]), w, matrix)
