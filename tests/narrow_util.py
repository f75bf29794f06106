"""Plain forms of the operators over 4-bit weights and 8-bit pages, in numpy, from their definitions."""
import numpy as np
import torch

PAGE = 64


def f64(t):
    return t.detach().double().cpu().numpy()


# ------------------------------------------------------------------------------------------------ 4-bit weights

def codes_and_scales(w, group):
    """Codes (0 .. 15) and scales of a float32 matrix: m the group's element of the largest magnitude, s = bfloat16(-m / 8)."""
    n, k = w.shape
    kp = -(-k // 64) * 64
    groups = -(-kp // group)
    full = np.zeros((n, groups * group), np.float32)
    full[:, :k] = w
    g = full.reshape(n, groups, group)
    m = np.take_along_axis(g, np.abs(g).argmax(axis=2)[..., None], axis=2)[..., 0]
    s = torch.from_numpy(m * np.float32(-0.125)).bfloat16().float().numpy()
    s[m == 0] = 0
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s[..., None] != 0, np.clip(np.rint(g / s[..., None]), -8, 7), 0) + 8
    return c.reshape(n, -1)[:, :kp].astype(np.uint8), s


def unpack(weight):
    """(codes [rows, columns], scales [rows, groups]) of a Weight4, what fills up the tiles included."""
    b, s = weight.codes.cpu().numpy(), weight.scales.float().cpu().numpy()
    tiles, chunks, groups = b.shape[0], b.shape[1], s.shape[1]
    codes, scales = np.zeros((tiles * 16, chunks * 64), np.uint8), np.zeros((tiles * 16, groups), np.float32)
    for lane in range(32):
        g, t = divmod(lane, 4)
        for word in range(4):
            h, u = divmod(word, 2)
            for i, col in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
                codes[g + 8 * u::16, 32 * h + 8 * t + col::64] = b[:, :, lane, 4 * word + i // 2] >> (4 * (i % 2)) & 15
    for r in range(16):
        scales[r::16] = s[:, :, r % 8, r // 8]
    return codes, scales


def dense(weight):
    """The matrix in float64."""
    codes, scales = unpack(weight)
    w = (codes.astype(np.float64) - 8) * np.repeat(scales.astype(np.float64), weight.group, axis=1)[:, :codes.shape[1]]
    return w[:weight.out_features, :weight.in_features]


def gelu_new(y):
    return 0.5 * y * (1 + np.tanh(np.sqrt(2 / np.pi) * (y + 0.044715 * y ** 3)))


def linear(x, w, bias=None, act=None, residuals=(), out_bf16=False):
    """(result, bound of its error) for rows x and a dense matrix w, float64.
    A sum's terms are added within a group (128 at most), over the groups and over parts of them: each of at most 256 + K / 32 additions is off by
    2^-23 of the terms' magnitudes (an addition that cuts off; a rounded one by half).  The activation's slope is at most 1.13, its own
    error 2^-20 of the value and 2^-20; the last rounding half a step of the result's type."""
    y, size = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    err = 2.0 ** -23 * (256 + x.shape[1] / 32) * size
    if act == "gelu_new":
        y, err = gelu_new(y), 1.13 * err + 2.0 ** -20 * (np.abs(y) + 1)
    elif act == "silu":
        y, err = y / (1 + np.exp(-y)), 1.1 * err + 2.0 ** -20 * (np.abs(y) + 1)
    for r in residuals:
        y = y + r
        err = err + 2.0 ** -24 * (np.abs(y) + np.abs(r))
    return y, err + (2.0 ** -8 if out_bf16 else 2.0 ** -24) * (np.abs(y) + err)


# ------------------------------------------------------------------------------------------------ 8-bit pages

def power_of_two_for(most):
    """The smallest power of two (2^-126 at least) of which 127 reach `most`; 0 for 0."""
    if most == 0:
        return np.float32(0)
    f, e = np.frexp(np.float64(most))
    return np.float32(2.0 ** max(int(e) - 7 + int(f > 127 / 128), -126))


def rotate(x, pos, cos_sin, rotary, half):
    """Rotation of [rows, heads, d] in float32, every product and sum rounded by itself."""
    x = x.astype(np.float32).copy()
    c, s = cos_sin[pos][:, None, :, 0].astype(np.float32), cos_sin[pos][:, None, :, 1].astype(np.float32)
    a, b = (slice(0, rotary // 2), slice(rotary // 2, rotary)) if half else (slice(0, rotary, 2), slice(1, rotary, 2))
    xa, xb = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = xa * c - xb * s, xa * s + xb * c
    return x


def store(codes, scale, x, slot, pos, table):
    """Write rows x [rows, heads, d] (float32) into codes [pages, heads, 64, d] and scale [pages, heads], in place."""
    runs = {}
    for r, (i, p) in enumerate(zip(slot, pos)):
        if i >= 0:
            runs.setdefault((table[i][p // PAGE], p // PAGE, i), []).append(r)
    for (page, _, _), rows in runs.items():
        a = pos[rows[0]] % PAGE
        for h in range(codes.shape[1]):
            new = x[rows, h]
            before = scale[page, h] if a else np.float32(0)
            after = np.float32(np.nan) if not np.isfinite(new).all() or np.isnan(before) else max(before, power_of_two_for(np.abs(new).max()))
            scale[page, h] = after
            if np.isnan(after):
                codes[page, h, a:a + len(rows)] = 0
                continue
            if a and after != before:
                codes[page, h, :a] = np.rint(codes[page, h, :a].astype(np.float32) * (before / after))
            codes[page, h, a:a + len(rows)] = np.rint(new / after) if after > 0 else 0


def visible(pos, window=0, chunk=0, keep_first=0):
    """Which keys 0 .. pos the query at `pos` sees."""
    key = np.arange(pos + 1)
    first = pos - pos % chunk if chunk else max(0, pos - window + 1) if window else 0
    return (key >= first) | (key < (keep_first if window else 0))


def attention(q, codes, scales, slot, pos, table, per, scale, window=0, chunk=0, keep_first=0, softcap=0.0, sink=None, wide_weights=True, out_bf16=False):
    """(result [rows, heads, dv], bound of its error), float64; q [rows, heads, dk], codes and scales pairs of keys and values.
    A score is a sum of dk products, a result one of the keys: runs of at most 320 and 8 more per run joined; each addition is off by 2^-23 of
    its terms.  An error of the scores moves a weight by as much, relatively, and the weights' sum too; the exponential and the cap add 16
    roundings, and 2^-22 of the score's size where it is turned to base two.  Weights in 16 bits: 2^-11 more.  Queries as 16-bit numbers: 2^-24 of the largest."""
    (kc, vc), (ks, vs) = codes, scales
    rows, heads, _ = q.shape
    want, bound = np.zeros((rows, heads, vc.shape[-1])), np.zeros((rows, heads, 1))
    for r in range(rows):
        if slot[r] < 0:
            continue
        n = pos[r] + 1
        pages = np.asarray(table[slot[r]])[:-(-n // PAGE)]
        see = visible(pos[r], window, chunk, keep_first)
        for h in range(heads):
            g = h // per
            with np.errstate(invalid="ignore", over="ignore"):
                k, v = ((c[np.maximum(pages, 0), g].astype(np.float64) * s[np.maximum(pages, 0), g].astype(np.float64)[:, None, None]).reshape(-1, c.shape[-1])[:n][see]
                        for c, s in ((kc, ks), (vc, vs)))
                s = k @ q[r, h] * scale
                size = (np.abs(k) @ np.abs(q[r, h]) + 2.0 ** -1 * np.abs(k).sum(axis=1) * np.abs(q[r, h]).max()) * scale
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                m = s.max() if sink is None else max(s.max(), sink[h])
                p = np.exp(s - m)
                total = p.sum() + (0 if sink is None else np.exp(sink[h] - m))
                want[r, h] = p @ v / total
                bound[r, h] = (2.0 ** -23 * (2 * (k.shape[1] + 8) * size.max() + 2 * np.abs(s).max() + 400 + n / 32) + (0 if wide_weights else 2.0 ** -11)) * np.abs(v).max()
    return want, bound + (2.0 ** -8 if out_bf16 else 2.0 ** -24) * (np.abs(want) + bound)


def paged(rng, lens, heads, dk, dv, spare=1):
    """Random pages for sequences of the given lengths, in an order of their own: (key codes, value codes, key scales, value scales, table)."""
    need = [max(1, -(-n // PAGE)) for n in lens]
    n_pages = sum(need) + spare
    order = rng.permutation(n_pages)
    table, at = np.full((len(lens), max(need)), -1, np.int32), 0
    for i, p in enumerate(need):
        table[i, :p] = order[at:at + p]
        at += p
    draw = lambda d: np.clip(np.rint(rng.normal(size=(n_pages, heads, PAGE, d)) * 35), -127, 127).astype(np.int8)    # noqa: E731
    scale = lambda: (2.0 ** rng.integers(-7, -4, size=(n_pages, heads))).astype(np.float32)                          # noqa: E731
    return draw(dk), draw(dv), scale(), scale(), table


def bf16(x):
    """float64 numbers rounded to bfloat16."""
    return torch.tensor(np.asarray(x)).bfloat16().double().numpy()
