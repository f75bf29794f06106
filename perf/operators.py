"""Operators over narrow weights and a narrow cache, as a program calls them: matrix products with 4-bit weights and a scale for each
group of columns, the write of keys and values into a cache held in 8 bits with a scale for each page and key head, and attention over
that cache, for single tokens and for prompts.

    own               false: elementary torch operations in 32 bits; true: the library's kernels
    listed()          the cases that stand for the operators' use
    draw(rng)         one more of the same ranges
    prepare(c, seed)  weights, cache and inputs on the device, from the seed alone
    run(state)        one pass
    exact(c, seed)    its results in 64 bits
    work(c)           bytes and operations that no implementation can do without

Weights of 4 bits: w[n, k] = (code[n, k] - 8) * scale[n, k // group], code 0 .. 15, scale bfloat16.  A tile of 16 rows and 64 columns is
512 bytes, codes uint8 [rows / 16][columns / 64][32][16]: entry 4 g + t holds four words; word 2 h2 + h1 has the row g + 8 h1 and the columns
32 h2 + 8 t + (0, 2, 4, 6, 1, 3, 5, 7), lowest four bits first.  Scales [rows / 16][groups][8][2]: entry (g, h1) is the row g + 8 h1.  Rows and
columns are filled up to whole tiles with codes of 8 and scales of 0.

Cache in 8 bits: value = code * scale[page][head], code int8 -127 .. 127 in pages [page][head][64][dim], scale a power of two.
"""
from __future__ import annotations

import math
import zlib

import torch

own = False

DEVICE = "cuda"
PAGE = 64
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
SIZE = {"bfloat16": 2, "float32": 4}
COLUMNS = (0, 2, 4, 6, 1, 3, 5, 7)


def listed():
    return [
        # one user's token through an output projection of 4,096: the latency of a decode step
        {"name": "q4 1x4096x4096", "kind": "q4", "m": 1, "n": 4096, "k": 4096, "group": 64, "dtype": "bfloat16", "act": "none", "bias": False, "residual": False},
        # eight users' tokens through the up projection of a feed-forward, with its bias and activation
        {"name": "q4 8x16384x4096", "kind": "q4", "m": 8, "n": 16384, "k": 4096, "group": 64, "dtype": "bfloat16", "act": "gelu_new", "bias": True, "residual": False},
        # an odd batch through the down projection, the residual stream added on the way out
        {"name": "q4 33x4096x16384", "kind": "q4", "m": 33, "n": 4096, "k": 16384, "group": 128, "dtype": "bfloat16", "act": "none", "bias": True, "residual": True},
        # the 32-bit engine, which users run to check a model: three tokens, a feed-forward of 8/3 the width
        {"name": "q4 fp32 3x5461x2048", "kind": "q4", "m": 3, "n": 5461, "k": 2048, "group": 32, "dtype": "float32", "act": "none", "bias": False, "residual": False},
        # a prompt through the same kind of matrix
        {"name": "q4 700x8192x2048", "kind": "q4", "m": 700, "n": 8192, "k": 2048, "group": 64, "dtype": "bfloat16", "act": "none", "bias": False, "residual": False},
        # the cache write of a decode step of eight users with short conversations
        {"name": "store 8 rows", "kind": "store", "seqs": 8, "held": 150, "new": 8, "heads": 16, "kv_heads": 4, "dk": 128, "dv": 128, "rotary": 64, "half": True, "dtype": "bfloat16"},
        # the cache write of two long prompts
        {"name": "store 4082 rows", "kind": "store", "seqs": 2, "held": 0, "new": 4082, "heads": 16, "kv_heads": 16, "dk": 256, "dv": 256, "rotary": 64, "half": False, "dtype": "bfloat16"},
        # one user's token early in a conversation: the smallest attention call
        {"name": "decode 1x97", "kind": "decode", "seqs": 1, "held": 97, "pad": 0, "heads": 16, "kv_heads": 16, "dk": 256, "dv": 256, "window": 0, "softcap": 0.0, "dtype": "bfloat16"},
        # eight users in mid-conversation, a key head for every query head
        {"name": "decode 8x1024", "kind": "decode", "seqs": 8, "held": 8192, "pad": 0, "heads": 16, "kv_heads": 16, "dk": 256, "dv": 256, "window": 0, "softcap": 0.0, "dtype": "bfloat16"},
        # 31 users and one idle row, four query heads to a key head, capped scores
        {"name": "decode 32x2048 grouped", "kind": "decode", "seqs": 31, "held": 63488, "pad": 1, "heads": 16, "kv_heads": 4, "dk": 128, "dv": 128, "window": 0, "softcap": 30.0,
         "dtype": "bfloat16"},
        # one user with a long document behind them
        {"name": "decode 1x65536", "kind": "decode", "seqs": 1, "held": 65536, "pad": 0, "heads": 16, "kv_heads": 4, "dk": 128, "dv": 128, "window": 0, "softcap": 0.0, "dtype": "bfloat16"},
        # three users' prompts arriving together
        {"name": "prompt 3x682", "kind": "prompt", "seqs": 3, "held": 0, "new": 2047, "heads": 16, "kv_heads": 4, "dk": 128, "dv": 128, "window": 0, "softcap": 0.0, "dtype": "bfloat16"},
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    kind = rng.choice(("q4", "q4", "q4", "store", "decode", "decode", "prompt"))
    dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
    if kind == "q4":
        m = log(1, 700) if dtype == "bfloat16" else log(1, 64)
        most = min(16384 * 4096, 700 * 8192 * 2048 // m)
        k = rng.choice((2048, 4096, 5461, 8192, 16384, rng.randint(200, 16384)))
        n = max(16, min(log(64, 16384), most // k))
        return {"kind": kind, "m": m, "n": n, "k": k, "group": rng.choice((32, 64, 128)), "dtype": dtype, "act": rng.choice(("none", "none", "gelu_new")),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.3}
    heads, kv_heads, dk, dv = rng.choice(((16, 16, 256, 256), (16, 4, 128, 128), (32, 8, 64, 64), (12, 4, 128, 80), (8, 1, 128, 128)))
    shape = {"heads": heads, "kv_heads": kv_heads, "dk": dk, "dv": dv, "dtype": dtype}
    if kind == "store":
        seqs = rng.randint(1, 8)
        step = rng.random() < 0.5                       # a decode step, or prompts (some with tokens already cached)
        return {"kind": kind, "seqs": seqs, "held": log(1, 400) if step else rng.choice((0, rng.randint(1, 300))), "new": seqs if step else log(8, 2000), **shape,
                "rotary": 64, "half": rng.random() < 0.5}
    more = {"window": rng.choice((0, 0, rng.randint(1, 1500))), "softcap": rng.choice((0.0, 0.0, 30.0))}
    if kind == "decode":
        seqs = log(1, 32)
        return {"kind": kind, "seqs": seqs, "held": max(seqs, log(64, 16384)), "pad": rng.choice((0, 0, 3)), **shape, **more}
    return {"kind": kind, "seqs": rng.randint(1, 4), "held": rng.choice((0, 0, rng.randint(1, 300))), "new": log(8, 2047 if dtype == "bfloat16" else 500), **shape, **more}


# ---------------------------------------------------------------------------------------------------- inputs from a seed

def _generator(seed, name):
    return torch.Generator(device=DEVICE).manual_seed((seed * 1000003 + zlib.crc32(name.encode())) % (1 << 62))


def _normal(seed, name, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=_generator(seed, name), device=DEVICE, dtype=torch.float32) * std).to(dtype)


def _up(n, to):
    return -(-n // to) * to


def _shares(total, seqs):
    """`total` tokens over `seqs` sequences, unequally where there are several: 4 : 3 : 2 : 2 ..., at least one each."""
    shares = [max(2, 4 - i) for i in range(seqs)]
    total = max(total, seqs)
    out = [max(1, total * s // sum(shares)) for s in shares]
    out[0] += total - sum(out)
    return out


def _lengths(c):
    """(tokens held before the call, new tokens) of every sequence."""
    if c["kind"] == "decode":                           # the new token is the last of those held: it has been written already
        return [n - 1 for n in _shares(c["held"], c["seqs"])], [1] * c["seqs"]
    if c["kind"] == "store" and c["new"] == c["seqs"]:
        return [n % 400 for n in _shares(c["held"] * c["seqs"], c["seqs"])], [1] * c["seqs"]
    return [c["held"] * (i % 2 == 0) for i in range(c["seqs"])], _shares(c["new"], c["seqs"])


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _prepare_q4(c, seed):
    m, n, k, group, t = c["m"], c["n"], c["k"], c["group"], TYPES[c["dtype"]]
    np_, kp = _up(n, 16), _up(k, 64)
    # bell-shaped codes, as the rounding of a trained matrix leaves them
    codes = (torch.randn((np_, kp), generator=_generator(seed, "codes"), device=DEVICE) * 2.7).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    codes[n:] = 8
    codes[:, k:] = 8
    groups = _up(kp, group) // group
    scales = (torch.rand((np_, groups), generator=_generator(seed, "scales"), device=DEVICE) * 0.008 + 0.004).to(torch.bfloat16)
    scales[n:] = 0
    # the packed form: see the head of this file
    x = codes.view(np_ // 16, 2, 8, kp // 64, 2, 4, 8)[..., list(COLUMNS)]
    x = x.permute(0, 3, 2, 5, 4, 1, 6).reshape(np_ // 16, kp // 64, 32, 16, 2)
    packed = (x[..., 0] | (x[..., 1] << 4)).contiguous()
    s = scales.view(np_ // 16, 2, 8, groups).permute(0, 3, 2, 1).contiguous()
    return {"case": c, "codes": packed, "scales": s, "x": _normal(seed, "x", (m, k), t),
            "bias": _normal(seed, "bias", (n,), torch.float32, 0.1) if c["bias"] else None,
            "residual": _normal(seed, "residual", (m, n), t) if c["residual"] else None}


def _prepare_cache(c, seed):
    held, new = _lengths(c)
    total = [a + b for a, b in zip(held, new)]
    pages = [-(-n // PAGE) for n in total]
    n_pages, seqs, hk = sum(pages), c["seqs"], c["kv_heads"]
    order = torch.randperm(n_pages, generator=_generator(seed, "order"), device=DEVICE).to(torch.int32)
    table = torch.full((seqs, max(pages)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    slots = [i for i, b in enumerate(new) for _ in range(b)]
    pos = [a + j for a, b in zip(held, new) for j in range(b)]
    pad = c.get("pad", 0)
    rows = len(slots) + pad
    t = TYPES[c["dtype"]]
    state = {"case": c, "table": table, "order": order, "slot": _int32(slots + [-1] * pad), "pos": _int32(pos + [0] * pad), "longest": max(total),
             "status": torch.zeros(1, dtype=torch.int32, device=DEVICE), "q": _normal(seed, "q", (rows, c["heads"] * c["dk"]), t)}
    for name, d in (("k", c["dk"]), ("v", c["dv"])):
        scale = torch.exp2(torch.randint(-6, -4, (n_pages, hk), generator=_generator(seed, name + "s"), device=DEVICE).float())
        codes = torch.empty((n_pages, hk, PAGE, d), dtype=torch.int8, device=DEVICE)
        for a in range(0, n_pages, 256):                # normal numbers, rounded to the page's steps
            b = min(n_pages, a + 256)
            x = torch.randn((b - a, hk, PAGE, d), generator=_generator(seed, "%s%d" % (name, a)), device=DEVICE)
            codes[a:b] = (x / scale[a:b, :, None, None]).round_().clamp_(-127, 127).to(torch.int8)
        state[name + "_cache"], state[name + "_scale"] = codes, scale
    if c["kind"] == "store":
        state["k"] = _normal(seed, "new k", (rows, hk * c["dk"]), t, 1.3)
        state["v"] = _normal(seed, "new v", (rows, hk * c["dv"]), t)
        freq = 10000.0 ** (-torch.arange(0, c["rotary"], 2, dtype=torch.float64) / c["rotary"])
        angle = torch.arange(max(total), dtype=torch.float64)[:, None] * freq
        state["cos_sin"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float().to(DEVICE).contiguous()
        # what the pages hold beyond the cached tokens is nobody's: zeros
        tail = torch.arange(PAGE, device=DEVICE)
        at = 0
        for a, p in zip(held, pages):
            kept = (torch.arange(p, device=DEVICE)[:, None] * PAGE + tail) < a
            for name in ("k", "v"):
                state[name + "_cache"][order[at:at + p].long()] *= kept[:, None, :, None]
            at += p
        return state
    # the rows of every sequence, filled up with -1, and the tiles of 128 rows: the plan of the step
    longest, first, rows_of, tiles = max(new), 0, [], []
    for i, (a, b) in enumerate(zip(held, new)):
        rows_of.append(list(range(first, first + b)) + [-1] * (longest - b))
        tiles += [(first + j, min(128, b - j), a + j, i) for j in range(0, b, 128)]
        first += b
    tiles.sort(key=lambda x: -(x[1] + x[2]))
    return {**state, "rows_of": torch.tensor(rows_of, device=DEVICE), "tiles": _int32(tiles)}


def prepare(case, seed):
    return _prepare_q4(case, seed) if case["kind"] == "q4" else _prepare_cache(case, seed)


# ---------------------------------------------------------------------------------------------------- one pass

def _gelu(y):
    return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))


def _plain_q4(s):
    c, codes = s["case"], s["codes"]
    tiles, chunks = codes.shape[0], codes.shape[1]
    x = torch.stack([codes & 15, codes >> 4], dim=-1).view(tiles, chunks, 8, 4, 2, 2, 8)
    back = torch.empty_like(x)
    back[..., list(COLUMNS)] = x
    w = back.permute(0, 5, 2, 1, 4, 3, 6).reshape(tiles * 16, chunks * 64).float() - 8.0
    scale = s["scales"].permute(0, 3, 2, 1).reshape(tiles * 16, -1).float()
    w = w * scale.repeat_interleave(c["group"], dim=1)[:, :chunks * 64]
    y = s["x"].float() @ w[:c["n"], :c["k"]].t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["act"] == "gelu_new":
        y = _gelu(y)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _rotated(x, heads, d, cs, rotary, half):
    x = x.float().view(x.shape[0], heads, d)
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    if half:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        return torch.cat([a * c - b * n, a * n + b * c, x[..., rotary:]], dim=-1)
    a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
    return torch.cat([torch.stack([a * c - b * n, a * n + b * c], dim=-1).flatten(2), x[..., rotary:]], dim=-1)


def _plain_store(s):
    c = s["case"]
    hk, slot, pos = c["kv_heads"], s["slot"].long(), s["pos"].long()
    cs = s["cos_sin"][pos]
    q = _rotated(s["q"], c["heads"], c["dk"], cs, c["rotary"], c["half"]).flatten(1).to(s["q"].dtype)
    k = _rotated(s["k"], hk, c["dk"], cs, c["rotary"], c["half"])
    v = s["v"].float().view(-1, hk, c["dv"])
    page, row = s["table"].long()[slot, pos // PAGE], pos % PAGE
    n_pages = s["k_cache"].shape[0]
    first = torch.full((n_pages,), PAGE, device=DEVICE).scatter_reduce(0, page, row, "amin")      # the first row written now
    out = [q]
    for x, codes, scale in ((k, s["k_cache"], s["k_scale"]), (v, s["v_cache"], s["v_scale"])):
        most = torch.zeros((n_pages, hk), device=DEVICE).scatter_reduce(0, page[:, None].expand(-1, hk), x.abs().amax(dim=-1), "amax")
        f, e = torch.frexp(most)
        need = torch.where(most > 0, torch.ldexp(torch.ones_like(most), e - 7 + (f > 127 / 128).int()), torch.zeros_like(most))
        before = torch.where((first == 0)[:, None], torch.zeros_like(scale), scale)
        after = torch.maximum(before, need)
        shrink = torch.where(after > 0, before / after, torch.ones_like(after))
        old = (torch.arange(PAGE, device=DEVICE) < first[:, None])[:, None, :, None]
        new = torch.where(old, torch.round(codes.float() * shrink[:, :, None, None]), codes.float())
        new[page, :, row] = torch.round(x / after[page][..., None])
        out.append((new * after[:, :, None, None])[s["order"].long()].to(s["q"].dtype))
    return out


def _plain_attention(s):
    c = s["case"]
    hk, per, rows_of = c["kv_heads"], c["heads"] // c["kv_heads"], s["rows_of"]
    seqs, most = rows_of.shape
    live = rows_of >= 0
    rows = rows_of.clamp(min=0)
    pages = s["table"].long().clamp(min=0)
    k, v = ((s[n + "_cache"][pages].float() * s[n + "_scale"][pages][..., None, None]).transpose(2, 3).flatten(1, 2) for n in ("k", "v"))      # [seq, key, head, d]
    q = s["q"].float().view(-1, hk, per, c["dk"])[rows]                                             # [seq, row, head, query, d]
    score = torch.einsum("srhqd,skhd->shqrk", q, k) * c["dk"] ** -0.5
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    at, key = s["pos"].long()[rows][:, None, None, :, None], torch.arange(k.shape[1], device=DEVICE)
    seen = key <= at
    if c["window"]:
        seen = seen & (key > at - c["window"])
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    p = torch.exp(score - score.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    o = torch.einsum("shqrk,skhd->srhqd", p, v).flatten(2)
    out = torch.zeros((s["q"].shape[0], c["heads"] * c["dv"]), device=DEVICE)
    out[rows_of[live]] = o[live]
    return out.to(s["q"].dtype)


def _own_run(s):
    c = s["case"]
    if c["kind"] == "q4":
        from qstream_b200.csrc import q4
        w = q4.Weight4(s["codes"], s["scales"], c["n"], c["k"], c["group"])
        return q4.linear(s["x"], w, s["bias"], c["act"], () if s["residual"] is None else (s["residual"],))
    from qstream_b200.csrc import kv8
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if c["kind"] == "store":
        q = torch.empty_like(s["q"])
        kv8.rope_store(s["q"], s["k"], s["v"], c["heads"], c["kv_heads"], c["dk"], c["rotary"], s["cos_sin"], s["slot"], s["pos"], s["table"], PAGE, *cache,
                       s["status"], v_head_dim=c["dv"], half_layout=c["half"], q_out=q)
        return [q, kv8.read_pages(s["k_cache"], s["k_scale"], s["order"], s["q"].dtype), kv8.read_pages(s["v_cache"], s["v_scale"], s["order"], s["q"].dtype)]
    shape = (c["heads"], c["kv_heads"], c["dk"], c["dk"] ** -0.5, c["window"])
    if c["kind"] == "decode":
        return kv8.decode(s["q"], *shape, s["slot"], s["pos"], s["table"], PAGE, *cache, s["longest"], s["status"], v_head_dim=c["dv"], softcap=c["softcap"])
    return kv8.prefill(s["q"], *shape, s["tiles"], s["table"], PAGE, *cache, s["status"], v_head_dim=c["dv"], softcap=c["softcap"])


def run(state):
    if own:
        return _own_run(state)
    kind = state["case"]["kind"]
    return _plain_q4(state) if kind == "q4" else _plain_store(state) if kind == "store" else _plain_attention(state)


# ---------------------------------------------------------------------------------------------------- in 64 bits

def _exact_q4(c, s):
    m, n, k, group = c["m"], c["n"], c["k"], c["group"]
    bytes_ = s["codes"].cpu().numpy()
    scales = s["scales"].double().cpu().numpy()
    import numpy as np
    tiles, chunks = bytes_.shape[:2]
    w = np.zeros((tiles * 16, chunks * 64))
    for g in range(8):
        for t in range(4):
            for word in range(4):
                for j, column in enumerate(COLUMNS):
                    nibble = (bytes_[:, :, 4 * g + t, 4 * word + j // 2] >> (4 * (j % 2))) & 15
                    w[g + 8 * (word % 2)::16, 32 * (word // 2) + 8 * t + column::64] = nibble.astype(np.float64) - 8
    for row in range(16):
        w[row::16] *= np.repeat(scales[:, :, row % 8, row // 8], group, axis=1)[:, :chunks * 64]
    y = s["x"].double() @ torch.from_numpy(w[:n, :k].copy()).to(DEVICE).t()
    y = y + (0 if s["bias"] is None else s["bias"].double())
    if c["act"] == "gelu_new":
        y = y / 2 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    return y + (0 if s["residual"] is None else s["residual"].double())


def _exact_store(c, s):
    hk, rot = c["kv_heads"], c["rotary"]
    slot, pos, table = s["slot"].tolist(), s["pos"].tolist(), s["table"].tolist()
    angle = torch.atan2(s["cos_sin"][..., 1].double(), s["cos_sin"][..., 0].double())
    size = s["cos_sin"].double().norm(dim=-1)
    turn = torch.polar(size, angle)[s["pos"].long()][:, None]                                      # as complex numbers

    def rotate(x, heads):
        x = x.double().view(len(pos), heads, -1).clone()
        a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if c["half"] else (slice(0, rot, 2), slice(1, rot, 2))
        z = torch.complex(x[..., a], x[..., b]) * turn
        x[..., a], x[..., b] = z.real, z.imag
        return x

    out = [rotate(s["q"], c["heads"]).flatten(1)]
    runs, first = {}, {}
    for r, (i, p) in enumerate(zip(slot, pos)):
        runs.setdefault(table[i][p // PAGE], []).append(r)
        first.setdefault(table[i][p // PAGE], p % PAGE)
    for x, name in ((rotate(s["k"], hk), "k"), (s["v"].double().view(len(pos), hk, -1), "v")):
        codes, scale = s[name + "_cache"].double(), s[name + "_scale"].double()
        for page, rows in runs.items():
            a, n = first[page], len(rows)
            new = x[rows[0]:rows[-1] + 1].transpose(0, 1)
            most = new.abs().amax(dim=(1, 2))
            need = torch.exp2(torch.ceil(torch.log2(most / 127)))
            need = torch.where(most > 127 * need, need * 2, torch.where(most <= 127 * need / 2, need / 2, need))
            after = torch.maximum(need, scale[page] * (a > 0))
            codes[page, :, :a] = torch.round(codes[page, :, :a] * (scale[page] / after)[:, None, None])
            codes[page, :, a:a + n] = torch.round(new / after[:, None, None])
            scale[page] = after
        out.append(codes[s["order"].long()] * scale[s["order"].long()][:, :, None, None])
    return out


def _exact_attention(c, s):
    out = torch.zeros((s["q"].shape[0], c["heads"], c["dv"]), dtype=torch.float64, device=DEVICE)
    held, new = _lengths(c)
    first, per = 0, c["heads"] // c["kv_heads"]
    for i, (a, b) in enumerate(zip(held, new)):
        n = a + b
        pages = s["table"][i, :-(-n // PAGE)].long()
        at, key = torch.arange(a, n, device=DEVICE)[:, None], torch.arange(n, device=DEVICE)[None]
        hidden = (key > at) | (key <= at - c["window"]) if c["window"] else key > at
        for g in range(c["kv_heads"]):
            k, v = ((s[x + "_cache"][pages, g].double() * s[x + "_scale"][pages, g].double()[:, None, None]).flatten(0, 1)[:n] for x in ("k", "v"))
            for h in range(g * per, (g + 1) * per):
                score = s["q"][first:first + b, h * c["dk"]:(h + 1) * c["dk"]].double() @ k.t() / math.sqrt(c["dk"])
                if c["softcap"]:
                    score = c["softcap"] * torch.tanh(score / c["softcap"])
                out[first:first + b, h] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1) @ v
        first += b
    return out.flatten(1)


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_q4(case, s) if case["kind"] == "q4" else _exact_store(case, s) if case["kind"] == "store" else _exact_attention(case, s)


# ---------------------------------------------------------------------------------------------------- what cannot be done without

def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["kind"] == "q4":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": n * k // 2 + 2 * n * -(-k // c["group"]) + e * m * (k + n * (1 + c["residual"])) + 4 * n * c["bias"], "flops": 2 * m * n * k}
    held, new = _lengths(c)
    rows, hk, dk, dv = sum(new), c["kv_heads"], c["dk"], c["dv"]
    if c["kind"] == "store":
        pages = sum(-(-(a + b) // PAGE) for a, b in zip(held, new))
        moved = rows * e * (2 * c["heads"] * dk + hk * (dk + dv)) + rows * hk * (dk + dv)
        return {"bytes": moved + pages * hk * (PAGE * (dk + dv) * (1 + e) + 16), "flops": 6 * rows * (c["heads"] + hk) * c["rotary"]}
    # keys that some row sees, and pairs of a row and a key it sees
    keys = sum(min(a + b, c["window"] + b - 1) if c["window"] else a + b for a, b in zip(held, new))
    pairs = sum(min(p + 1, c["window"]) if c["window"] else p + 1 for a, b in zip(held, new) for p in range(a, a + b))
    return {"bytes": keys * hk * (dk + dv) + (keys // PAGE + 1) * hk * 8 + rows * c["heads"] * (dk + dv) * e, "flops": 2 * pairs * c["heads"] * (dk + dv)}
