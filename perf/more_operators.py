"""The calls that the performance of positions with several axes, of page tables
made on the GPU and of the cache in 4 bits is judged on.

``rope`` is the norm and rotation of a layer's queries and keys where each pair
of features follows one of three positions (time, height, width), as in prompts
with images (``train``: with the gradient).  ``reserve`` takes pages of a cache
for the new tokens of a batch and says where each goes.  ``append`` rounds the
keys and values of new tokens to 4 bits into such pages, and reads them back.
``paged`` is the attention of new tokens, one or a chunk per sequence, over
pages in 4 bits.

``new`` and ``lens`` hold, for each sequence, the number of new tokens and the
number of cached ones with the new ones among them.
"""
import importlib
import math
import random

import torch

own = False

_DTYPES = {"f16": torch.float16, "f32": torch.float32}
_EPS = 1e-6
_BASE = 10000.0
_GROUP = 32  # features that share a scale
_HALVES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of the 3 low bits of a code
# Where one magnitude ends and the next begins, and whether the border itself
# belongs to the next (ties go to the even code).
_BORDERS = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))
_MOST_SCALE = 10240.0


# ---- cases -----------------------------------------------------------------

def _rope(mode, dtype, B, S, H_q, H_kv, D, axes, fold, interleaved=False, w32=True):
    """``axes``: the pairs of each axis, as one text, or "a n": n pairs, the axes in turn."""
    return {"op": "rope", "mode": mode, "dtype": dtype, "B": B, "S": S, "H_q": H_q, "H_kv": H_kv, "D": D, "axes": axes,
            "fold": fold, "interleaved": interleaved, "w32": w32}


def _reserve(new, lens, page, width, finished=0, spare=64):
    """``lens``: cached tokens before the call; the first ``finished`` sequences
    without new tokens end; ``spare``: free pages beyond those needed."""
    return {"op": "reserve", "new": new, "lens": lens, "page": page, "width": width, "finished": finished, "spare": spare}


def _append(dtype, new, lens, H_q, H_kv, D_qk, D_v, page, axes, norm=False, interleaved=False):
    """``axes``: as in ``_rope``, or "" for the place in the sequence."""
    return {"op": "append", "dtype": dtype, "new": new, "lens": lens, "H_q": H_q, "H_kv": H_kv, "D_qk": D_qk, "D_v": D_v,
            "page": page, "axes": axes, "norm": norm, "interleaved": interleaved}


def _paged(dtype, new, lens, H_q, H_kv, D_qk, D_v, page, causal=True):
    return {"op": "paged", "dtype": dtype, "new": new, "lens": lens, "H_q": H_q, "H_kv": H_kv, "D_qk": D_qk, "D_v": D_v,
            "page": page, "causal": causal}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _spread(rng, n, lo, hi):
    """n lengths between lo and hi, spread over their logarithm, as one text."""
    return " ".join(str(_log(rng, lo, hi)) for _ in range(n))


def _ones(n):
    return " ".join(["1"] * n)


def listed():
    ragged = random.Random(23)
    long_lens = _spread(ragged, 64, 600, 16384)
    step_lens = _spread(ragged, 64, 50, 2000)
    rows = [
        # One generated token of 4 sequences, 32 query heads on 8: latency.
        ("rope_decode_f16", _rope("fwd", "f16", 4, 1, 32, 8, 128, "16 24 24", False, w32=False)),
        # Training on prompts with images: 4 sequences of 4096 tokens.
        ("rope_train_f16", _rope("train", "f16", 4, 4096, 32, 8, 128, "16 24 24", True)),
        # Full precision at a ragged length, the axes taking turns, neighbouring features paired.
        ("rope_train_f32", _rope("train", "f32", 8, 1000, 12, 12, 64, "a 32", True, True)),
        # A step of generation: 64 sequences, four of which have ended.
        ("reserve_decode", _reserve(" ".join(["0"] * 4 + ["1"] * 60), step_lens, 16, 160, finished=4)),
        # Prompts enter beside running sequences, pages of 64.
        ("reserve_prompts", _reserve("2048 4096 999 7500 1 1 1 1 1500 8000", "0 1904 0 0 333 4000 77 12 1833 0", 64, 160)),
        # One token of each of 64 sequences into pages of 16.
        ("append_decode_f16", _append("f16", _ones(64), step_lens, 32, 8, 128, 128, 16, "")),
        # Prompts with images of 4 sequences, keys and queries normed on the way.
        ("append_chunks_f16", _append("f16", "2048 4096 999 1500", "2048 6000 999 3333", 32, 8, 128, 128, 64, "16 24 24", True)),
        # Generation: one new token of 4 sequences with 16 heads each, 4096 cached.
        ("paged_decode_f16", _paged("f16", _ones(4), "4096 4096 4096 4096", 16, 16, 128, 128, 16)),
        # A serving batch: 64 sequences of very unequal length, shared heads.
        ("paged_decode_ragged_f16", _paged("f16", _ones(64), long_lens, 32, 8, 128, 128, 64)),
        # The next chunk of a long document: the largest call.
        ("paged_chunk_f16", _paged("f16", "512", "16000", 32, 8, 128, 128, 64)),
        # Chunks and single tokens in one batch, heads 64 wide.
        ("paged_mixed_f16", _paged("f16", "700 333 1 " + _ones(30), "1724 333 1 " + _spread(ragged, 30, 100, 4096), 16, 4, 64,
                                   64, 32)),
        # Full precision: a chunk and generation.
        ("paged_f32", _paged("f32", "300 1 1 1", "2300 1000 4001 517", 16, 4, 64, 64, 16)),
    ]
    return [dict(c, name=n) for n, c in rows]


def _draw_axes(rng, D):
    """Sections of D/2 pairs, or of fewer (the rest is not rotated), or the axes in turn."""
    pairs = rng.choice([D // 2, D // 2, D // 4])
    if rng.random() < 0.3:
        return "a %d" % pairs
    a = max(1, pairs // 4)
    b = (pairs - a) // 2
    return "%d %d %d" % (a, b, pairs - a - b)


def draw(rng):
    op = rng.choice(["rope", "rope", "reserve", "append", "paged", "paged", "paged"])
    dtype = rng.choice(["f16", "f16", "f16", "f32"])
    D = rng.choice([32, 64, 64, 96, 128, 128, 128])
    H_kv, G = rng.choice([1, 2, 4, 8, 8, 12, 16]), rng.choice([1, 1, 2, 3, 4, 8])
    if op == "rope":
        D = rng.choice([D, D, D, 80])
        mode = rng.choice(["fwd", "train", "train"])
        B, S = _log(rng, 1, 64), (1 if mode == "fwd" and rng.random() < 0.4 else _log(rng, 16, 8192))
        c = _rope(mode, dtype, B, S, H_kv * G, H_kv, D, _draw_axes(rng, D), rng.random() < 0.7, rng.random() < 0.3,
                  rng.random() < 0.5)
        while work(c)["bytes"] > 5e8:
            c["S"] = max(1, c["S"] * 2 // 3)
        return c
    page = rng.choice([16, 16, 32, 64, 128])
    kind = rng.choice(["decode", "decode", "chunks", "mixed"])
    few = H_kv * G <= 8
    if kind == "decode":
        N = _log(rng, 1, 512 if op == "reserve" else 128)
        new = [rng.choice([1, 1, 1, 1, 2, 4]) if few else 1 for _ in range(N)]
    elif kind == "chunks":
        N = rng.choice([1, 1, 2, 3, 5])
        new = [_log(rng, 33, 2048) for _ in range(N)]
    else:
        N = _log(rng, 3, 40)
        new = [_log(rng, 2, 700) if rng.random() < 0.2 else 1 for _ in range(N)]
    past = [0 if rng.random() < 0.1 else _log(rng, 1, 16384) for _ in new]
    text = lambda x: " ".join(map(str, x))  # noqa: E731
    if op == "reserve":
        finished = rng.choice([0, 0, 1, N // 4])
        for s in rng.sample(range(N), finished):
            new[s] = 0
        finished = sum(n == 0 for n in new)
        width = max(-(-(a + b) // page) for a, b in zip(past, new)) + rng.choice([0, 1, 7])
        # (now and then the pages run out)
        return _reserve(text(new), text(past), page, max(1, width), finished, rng.choice([100, 1, 0, 0, -3]))
    lens = [a + b for a, b in zip(past, new)]
    D_v = D if rng.random() < 0.8 else rng.choice([32, 64, 128])
    if op == "append":
        return _append(dtype, text(new), text(lens), H_kv * G, H_kv, D, D_v, page,
                       _draw_axes(rng, D) if rng.random() < 0.5 else "", rng.random() < 0.5, rng.random() < 0.3)
    most = 1.3e11 if dtype == "f16" else 3e10
    while True:
        c = _paged(dtype, text(new), text(lens), H_kv * G, H_kv, D, D_v, page, rng.random() < 0.9)
        w = work(c)
        if w["flops"] <= most and w["bytes"] <= 4e8:
            return c
        lens = [max(n, l * 2 // 3) for n, l in zip(new, lens)]
        if w["flops"] > most:
            new = [max(1, n * 3 // 4) for n in new]


def _ints(text):
    return [int(x) for x in text.split()]


def _axes_of(text):
    """The axis of every rotated pair."""
    if text.startswith("a"):
        return tuple(i % 3 for i in range(int(text.split()[1])))
    return tuple(a for a, n in enumerate(_ints(text)) for _ in range(n))


def _rotated_pairs(c):
    return len(_axes_of(c["axes"])) if c["axes"] else c["D_qk"] // 2


def work(case):
    c = case
    if c["op"] == "reserve":
        new, lens = _ints(c["new"]), _ints(c["lens"])
        pages = sum(-(-(a + b) // c["page"]) - -(-a // c["page"]) for a, b in zip(lens, new))
        gone = sum([-(-a // c["page"]) for a, b in zip(lens, new) if b == 0][:c["finished"]])
        # lengths, new lengths, ends; pages out of the stack into the table and back; what is written
        return {"bytes": 21 * len(new) + 8 * (pages + gone) + 12 * sum(new), "flops": 3 * sum(new)}
    e = 2 if c["dtype"] == "f16" else 4
    if c["op"] == "rope":
        n = c["B"] * c["S"] * (c["H_q"] + c["H_kv"]) * c["D"]
        table = 12 * c["B"] * c["S"] + 8 * c["S"] * len(_axes_of(c["axes"]))
        if c["mode"] == "fwd":  # x in, y out
            return {"bytes": 2 * n * e + table, "flops": 8 * n}
        return {"bytes": 5 * n * e + table, "flops": 24 * n}  # and x, dy in, dx out
    new, lens = _ints(c["new"]), _ints(c["lens"])
    T = sum(new)
    byte = 0.5 + 1 / _GROUP  # of a cached value
    if c["op"] == "append":  # q in and out; k and v in, into the cache, out of it again
        q, kv = T * c["H_q"] * c["D_qk"], T * c["H_kv"] * (c["D_qk"] + c["D_v"])
        return {"bytes": 2 * q * e + kv * (2 * e + 2 * byte) + 8 * T * _rotated_pairs(c), "flops": (8 if c["norm"] else 4) * (q + kv)}
    kv = sum(lens) * c["H_kv"] * (c["D_qk"] + c["D_v"]) * byte
    qo = T * c["H_q"] * ((c["D_qk"] + c["D_v"]) * e + 4)
    pairs = sum(n * l - (n * (n - 1) // 2 if c["causal"] else 0) for n, l in zip(new, lens))
    return {"bytes": kv + qo, "flops": 2 * pairs * c["H_q"] * (c["D_qk"] + c["D_v"])}


# ---- inputs ----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, spread=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * spread).to(dtype)


def _tables(n, R):
    """cos and sin of the angles position * base^(-2i/R), formed in 64 bits."""
    freq = _BASE ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    angle = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _weights(g, c, width):
    dt = torch.float32 if c.get("w32", True) else _DTYPES[c["dtype"]]
    return tuple((1 + 0.2 * torch.randn((width,), generator=g, device="cuda")).to(dt) for _ in range(2))


def _grid_positions(first, n):
    """Positions [3, n] of n tokens from place ``first`` on: text, with images of
    16 x 24 patches in between (text counts on all three axes alike)."""
    place = torch.arange(first, first + n, device="cuda")
    block, at = place // 512, place % 512
    start = block * (512 - 384 + 24)  # where a block of text and image begins
    image = at < 384
    text = start + 24 + at - 384
    t = torch.where(image, start, text)
    h = torch.where(image, start + at // 24, text)
    w = torch.where(image, start + at % 24, text)
    return torch.stack((t, h, w)).int()


def _int_tensor(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _batch(c, seed):
    """A page table whose pages lie in no order, the lengths, and the number of pages."""
    new, lens = _ints(c["new"]), _ints(c["lens"])
    used = [-(-l // c["page"]) for l in lens]
    rng = random.Random(seed)
    order = list(range(sum(used) + 3))
    rng.shuffle(order)
    width, at, rows = max(used), 0, []
    for u in used:
        rows.append(order[at:at + u] + [0] * (width - u))
        at += u
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return {"page_table": _int_tensor(rows), "q_starts": _int_tensor(starts), "kv_lens": _int_tensor(lens), "starts": starts,
            "lens": lens, "pages": len(order), "max_new": max(new)}


def _prepare_reserve(c, seed):
    new, lens, page, width = _ints(c["new"]), _ints(c["lens"]), c["page"], c["width"]
    used = [-(-l // page) for l in lens]
    need = sum(-(-(l + n) // page) - u for l, n, u in zip(lens, new, used))
    free = max(0, need + c["spare"])
    rng = random.Random(seed)
    order = list(range(sum(used) + free))
    rng.shuffle(order)
    at, rows = 0, []
    for u in used:
        rows.append((order[at:at + u] + [-1] * width)[:width])
        at += u
    ends = [s for s, n in enumerate(new) if n == 0][:c["finished"]]
    return {"page_table": _int_tensor(rows), "kv_lens": _int_tensor(lens), "new_lens": _int_tensor(new),
            # the stack: free pages first, room for all of them
            "free_pages": _int_tensor(order[at:] + [0] * at), "free_count": _int_tensor([free]),
            "finished": torch.tensor([s in set(ends) for s in range(len(new))], device="cuda"), "total": sum(new)}


def prepare(case, seed):
    c = case
    state = {"case": c, "op": importlib.import_module("tf-custom-flash-attention_amd") if own else None}
    if c["op"] == "reserve":
        return {**state, **_prepare_reserve(c, seed)}
    dt, g = _DTYPES[c["dtype"]], _generator(seed)
    if c["op"] == "rope":
        B, S, H_q, H_kv, D = c["B"], c["S"], c["H_q"], c["H_kv"], c["D"]
        # q and k are parts of one projection's output
        qk = _normal(g, (B, S, H_q + H_kv, D), dt, 1.5)
        state["q"], state["k"] = qk[:, :, :H_q], qk[:, :, H_q:]
        state["q_weight"], state["k_weight"] = _weights(g, c, D)
        state["axes"] = _axes_of(c["axes"])
        firsts = [random.Random(seed + b).randrange(1000) for b in range(B)]
        state["positions"] = torch.stack([_grid_positions(f, S) for f in firsts], 1).contiguous()  # [3, B, S]
        state["cos"], state["sin"] = _tables(1000 + S, 2 * len(state["axes"]))
        if c["mode"] == "train":
            for name, H in (("d_q", H_q), ("d_k", H_kv)):
                state[name] = _normal(g, (B * H, S, D) if c["fold"] else (B, S, H, D), dt)
        return state
    state.update(_batch(c, seed))
    T, H_q, H_kv, D_qk, D_v, page = state["starts"][-1], c["H_q"], c["H_kv"], c["D_qk"], c["D_v"], c["page"]
    state["q"] = _normal(g, (T, H_q, D_qk), dt)
    for name, D in (("k", D_qk), ("v", D_v)):
        cache = torch.zeros((state["pages"], H_kv, page, D // 2 + D // _GROUP), dtype=torch.uint8, device="cuda")
        if c["op"] == "paged" or max(state["lens"]) > state["max_new"]:
            for a in range(0, state["pages"], 4096):  # pages at a time
                part = cache[a:a + 4096]
                x = _normal(g, (part.shape[0], H_kv, page, D), torch.float32)
                codes, scales = _codes(x)
                (_put_k if name == "k" else _put_v)(part, codes, scales)
        state[name + "_cache"] = cache
    if c["op"] == "append":
        state["k"], state["v"] = _normal(g, (T, H_kv, D_qk), dt), _normal(g, (T, H_kv, D_v), dt)
        state["q_weight"], state["k_weight"] = _weights(g, c, D_qk) if c["norm"] else (None, None)
        state["cos"], state["sin"] = _tables(max(state["lens"]), 2 * _rotated_pairs(c))
        state["axes"] = _axes_of(c["axes"]) if c["axes"] else None
        parts = [(l - (e - s), e - s) for s, e, l in zip(state["starts"], state["starts"][1:], state["lens"])]
        state["positions"] = torch.cat([_grid_positions(*p) for p in parts], 1).contiguous() if c["axes"] else None
    return state


# ---- 4 bits: how a cache holds its values ---------------------------------------
#
# k_cache and v_cache: uint8 [pages, heads, page, D/2 + D/32].  The bytes of a page's
# head are its codes, then its scales:
#   k  codes [page][D/2], the lower half of a byte the feature before; scales [page][D/32]
#   v  codes [page/8][D][4], 8 tokens of a feature, the lower half the token before;
#      scales [page/8][D/32][8]
# A code is sign (8) and magnitude (_HALVES); a scale the upper byte of an fp16.

def _codes(x):
    """Codes and scales (bytes) of fp32 x [..., D], 32 neighbouring features a scale."""
    g = x.unflatten(-1, (-1, _GROUP))
    most = g.abs().amax(-1)  # (a NaN comes out)
    s = (most / 6).clamp_max(_MOST_SCALE).to(torch.float8_e5m2)
    s = torch.where(most.isfinite(), s.view(torch.uint8), 0x7F)  # infinities and NaN: all 32 are NaN
    f = s.view(torch.float8_e5m2).float().unsqueeze(-1)
    mag, code = g.abs(), torch.zeros(g.shape, dtype=torch.uint8, device=x.device)
    for border, with_it in _BORDERS:
        code += (mag >= border * f) & (f > 0) if with_it else mag > border * f
    code = torch.where((f > 0), code, torch.zeros_like(code))
    code |= torch.signbit(g).byte() * 8
    return code.flatten(-2), s


def _split(cache, D):
    """A cache's codes and scales, each [pages, heads, bytes]."""
    flat = cache.flatten(2)
    n = cache.shape[2] * D // 2
    return flat[:, :, :n], flat[:, :, n:]


def _width(cache):
    return cache.shape[3] * _GROUP // (_GROUP // 2 + 1)


def _put_k(cache, codes, scales):
    c, s = _split(cache, codes.shape[-1])
    c.copy_((codes[..., ::2] | codes[..., 1::2] << 4).flatten(2))
    s.copy_(scales.flatten(2))


def _put_v(cache, codes, scales):
    c, s = _split(cache, codes.shape[-1])
    by8 = codes.unflatten(2, (-1, 8)).transpose(3, 4)  # [pages, heads, page / 8, D, 8]
    c.copy_((by8[..., ::2] | by8[..., 1::2] << 4).flatten(2))
    s.copy_(scales.unflatten(2, (-1, 8)).transpose(3, 4).flatten(2))


def _halves_of(byte):
    return torch.stack((byte & 15, byte >> 4), -1).flatten(-2)


def _values(codes, scales):
    """fp32 values of codes [..., D] and scales [..., D/32]."""
    table = torch.tensor(_HALVES + tuple(-h for h in _HALVES), device=codes.device)
    x = table[codes.int()].unflatten(-1, (-1, _GROUP))
    return (x * scales.contiguous().view(torch.float8_e5m2).float().unsqueeze(-1)).flatten(-2)


def _page_values(cache, pages, is_v):
    """fp32 values [len(pages), heads, page, D] of some pages."""
    part, D = cache[pages], _width(cache)
    page = part.shape[2]
    c, s = _split(part, D)
    if is_v:
        c = _halves_of(c.unflatten(2, (page // 8, D, 4))).transpose(3, 4).flatten(2, 3)
        s = s.unflatten(2, (page // 8, D // _GROUP, 8)).transpose(3, 4).flatten(2, 3)
    else:
        c, s = _halves_of(c.unflatten(2, (page, D // 2))), s.unflatten(2, (page, D // _GROUP))
    return _values(c, s)


def _store_tokens(cache, x, pages, slots, is_v):
    """fp32 rows x [n, heads, D] to their places."""
    codes, scales = _codes(x)
    D, page = x.shape[-1], cache.shape[2]
    c, s = _split(cache, D)
    if not is_v:
        c.unflatten(2, (page, D // 2))[pages, :, slots] = codes[..., ::2] | codes[..., 1::2] << 4
        s.unflatten(2, (page, D // _GROUP))[pages, :, slots] = scales
        return
    c = c.unflatten(2, (page // 8, D, 4))
    for odd in (0, 1):  # (two tokens share a byte)
        i = (slots % 2 == odd).nonzero().squeeze(1)
        at = (pages[i], slice(None), slots[i] // 8, slice(None), slots[i] % 8 // 2)
        c[at] = (c[at] & 15) | codes[i] << 4 if odd else (c[at] & 240) | codes[i]
    s.unflatten(2, (page // 8, D // _GROUP, 8))[pages, :, slots // 8, :, slots % 8] = scales


def _load_tokens(cache, pages, slots, is_v):
    """Their fp32 values again, [n, heads, D]."""
    D, page = _width(cache), cache.shape[2]
    c, s = _split(cache, D)
    if not is_v:
        return _values(_halves_of(c.unflatten(2, (page, D // 2))[pages, :, slots]), s.unflatten(2, (page, -1))[pages, :, slots])
    byte = c.unflatten(2, (page // 8, D, 4))[pages, :, slots // 8, :, slots % 8 // 2]
    codes = byte >> (slots % 2 * 4).to(torch.uint8)[:, None, None] & 15
    return _values(codes, s.unflatten(2, (page // 8, D // _GROUP, 8))[pages, :, slots // 8, :, slots % 8])


# ---- plain forms -----------------------------------------------------------

def _halves(x, R, interleaved):
    if interleaved:
        return x[..., 0:R:2], x[..., 1:R:2]
    return x[..., :R // 2], x[..., R // 2:R]


def _joined(a, b, rest, interleaved):
    pair = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((pair, rest), -1)


def _rotated(x, cos, sin, R, interleaved):
    a, b = _halves(x, R, interleaved)
    return _joined(a * cos - b * sin, b * cos + a * sin, x[..., R:], interleaved)


def _by_axes(table, positions, axes):
    """table[positions[axes[i]]][i] for every pair i: [..., pairs]."""
    rows = positions[torch.tensor(axes, device="cuda")].movedim(0, -1).long()
    return table[rows, torch.arange(len(axes), device="cuda")]


def _folded(x, fold):  # [B, S, H, D] -> [B * H, S, D]
    return x.permute(0, 2, 1, 3).flatten(0, 1).contiguous() if fold else x


def _plain_rope(st):
    c = st["case"]
    R, inter = 2 * len(st["axes"]), c["interleaved"]
    cos, sin = (_by_axes(st[t], st["positions"], st["axes"]).unsqueeze(2) for t in ("cos", "sin"))
    outs, grads, weights = [], [], []
    for name, H in (("q", c["H_q"]), ("k", c["H_kv"])):
        x, w = st[name].float(), st[name + "_weight"].float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        xr = x * r
        outs.append(_folded(_rotated(xr * w, cos, sin, R, inter).to(st[name].dtype), c["fold"]))
        if c["mode"] == "train":
            dy = st["d_" + name].float()
            if c["fold"]:
                dy = dy.unflatten(0, (c["B"], H)).permute(0, 2, 1, 3)
            dn = _rotated(dy, cos, -sin, R, inter)
            weights.append((dn * xr).sum((0, 1, 2), dtype=torch.float64).to(st[name + "_weight"].dtype))
            dn = dn * w
            grads.append((r * (dn - xr * (dn * xr).mean(-1, keepdim=True))).to(st[name].dtype))
    return outs + grads + weights


def _plain_reserve(st):
    page, table, stack = st["case"]["page"], st["page_table"], st["free_pages"]
    N, width = table.shape
    column = torch.arange(width, device="cuda")
    old, new, count = st["kv_lens"].long(), st["new_lens"].long(), st["free_count"].long()
    back = table[st["finished"][:, None] & (column < (old[:, None] + page - 1) // page) & (table >= 0)]
    stack[torch.arange(back.numel(), device="cuda") + count] = back
    count = count + back.numel()
    old = torch.where(st["finished"], 0, old)
    want = (column >= (old[:, None] + page - 1) // page) & (column < (old[:, None] + new[:, None] + page - 1) // page)
    at = count - want.flatten().cumsum(0).view(N, width)
    table.copy_(torch.where(want, torch.where(at >= 0, stack[at.clamp_min(0)], -1), table))
    ends = new.cumsum(0)
    starts = torch.cat((ends.new_zeros(1), ends))
    seq = torch.repeat_interleave(torch.arange(N, device="cuda"), new, output_size=st["total"])
    place = old[seq] + torch.arange(st["total"], device="cuda") - starts[seq]
    pages = table[seq, place // page].long()
    slots = torch.where(pages >= 0, pages * page + place % page, -1)
    return [starts.int(), (old + new).int(), (count - want.sum()).clamp_min(0).int(), place.int(), slots, table, stack]


def _places(st):
    """Place in the sequence, page and row of every new token."""
    page = st["case"]["page"]
    runs = list(zip(st["starts"], st["starts"][1:], st["lens"]))
    pos = torch.cat([torch.arange(l - (e - s), l, device="cuda") for s, e, l in runs])
    seq = torch.cat([torch.full((e - s,), i, device="cuda") for i, (s, e, _) in enumerate(runs)])
    return pos, st["page_table"][seq, pos // page].long(), pos % page


def _plain_append(st):
    c = st["case"]
    pos, pages, slots = _places(st)
    rows = {}
    # (the keys in 64 bits: a value next to a border between two codes decides for one)
    for name, form in (("q", torch.float32), ("k", torch.float64)):
        x = st[name].to(form)
        if c["norm"]:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS) * st[name + "_weight"].to(form)
        cos, sin = (_by_axes(st[t], st["positions"], st["axes"]) if st["axes"] else st[t][pos] for t in ("cos", "sin"))
        rows[name] = _rotated(x, cos[:, None].to(form), sin[:, None].to(form), 2 * _rotated_pairs(c), c["interleaved"])
    _store_tokens(st["k_cache"], rows["k"].float(), pages, slots, False)
    _store_tokens(st["v_cache"], st["v"].float(), pages, slots, True)
    return [rows["q"].to(st["q"].dtype)] + [_load_tokens(st[n], pages, slots, n == "v_cache").half()
                                            for n in ("k_cache", "v_cache")]


def _plain_paged(st):
    c = st["case"]
    page, H_kv, G = c["page"], c["H_kv"], c["H_q"] // c["H_kv"]
    os, stats = [], []
    for s, (b, e, l) in enumerate(zip(st["starts"], st["starts"][1:], st["lens"])):
        pages = st["page_table"][s, :-(-l // page)].long()
        # [H_kv, l, D]
        k, v = (_page_values(st[x], pages, x == "v_cache").transpose(0, 1).flatten(1, 2)[:, :l].contiguous()
                for x in ("k_cache", "v_cache"))
        n = e - b
        q = st["q"][b:e].float().unflatten(1, (H_kv, G)).permute(1, 2, 0, 3).flatten(1, 2)  # [H_kv, G n, D]
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) * c["D_qk"] ** -0.5
        if c["causal"]:
            i, j = torch.arange(n, device="cuda"), torch.arange(l, device="cuda")
            hidden = j[None, :] > i[:, None] + (l - n)
            x = x.masked_fill_(hidden.repeat(G, 1), float("-inf"))
        m = x.amax(-1, keepdim=True)
        x = x.sub_(m).exp_()
        total = x.sum(-1, keepdim=True)
        o = torch.matmul(x, v) / total
        os.append(o.unflatten(1, (G, n)).permute(2, 0, 1, 3).flatten(1, 2).to(st["q"].dtype))
        stats.append((m + total.log()).squeeze(-1).unflatten(1, (G, n)).permute(2, 0, 1).flatten(1, 2))
    return [torch.cat(os), torch.cat(stats)]


# ---- one pass --------------------------------------------------------------

def run(state):
    st, c, op = state, state["case"], state["op"]
    if op is None:
        return {"rope": _plain_rope, "reserve": _plain_reserve, "append": _plain_append, "paged": _plain_paged}[c["op"]](st)
    if c["op"] == "rope":
        args = dict(q_weight=st["q_weight"], k_weight=st["k_weight"], positions=st["positions"], eps=_EPS,
                    interleaved=c["interleaved"], fold_heads=c["fold"], axes=st["axes"])
        outs = op.qk_norm_rope(st["q"], st["k"], st["cos"], st["sin"], **args)
        if c["mode"] == "train":
            outs += op.qk_norm_rope_grad(st["d_q"], st["d_k"], st["q"], st["k"], st["cos"], st["sin"], **args)
        return list(outs)
    if c["op"] == "reserve":
        step = op.kv_reserve(st["page_table"], st["kv_lens"], st["new_lens"], st["free_pages"], st["free_count"], c["page"],
                             st["total"], finished=st["finished"])
        return [step.q_starts, step.kv_lens, step.free_count, step.positions, step.slots, st["page_table"], st["free_pages"]]
    where = (st["k_cache"], st["v_cache"], st["page_table"], st["q_starts"], st["kv_lens"])
    if c["op"] == "append":
        q = op.kv_append_fp4(st["k"], st["v"], *where, cos=st["cos"], sin=st["sin"], q=st["q"], q_weight=st["q_weight"],
                             k_weight=st["k_weight"], norm=c["norm"], eps=_EPS, interleaved=c["interleaved"],
                             positions=st["positions"], axes=st["axes"])
        return [q, *op.kv_read_fp4(*where, st["starts"][-1])]
    return list(op.paged_sdpa_fp4(st["q"], *where, scale=c["D_qk"] ** -0.5, causal_mask=c["causal"], max_q_len=st["max_new"]))


# ---- the definition in 64 bits ----------------------------------------------

def _turn64(x, cos, sin, R, interleaved):
    """x [..., D] with the pairs of its first R features as complex numbers,
    each times cos + i sin."""
    if interleaved:
        a, b = list(range(0, R, 2)), list(range(1, R, 2))
    else:
        a, b = list(range(R // 2)), list(range(R // 2, R))
    y = torch.complex(x[..., a], x[..., b]) * torch.complex(cos.double(), sin.double())
    out = x.clone()
    out[..., a], out[..., b] = y.real, y.imag
    return out


def _norm64(x, w):
    out = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + _EPS)
    return out if w is None else out * w


def _angles64(st, pos):
    """cos and sin [..., pairs], pair by pair."""
    n = st["cos"].shape[1]
    rows = [st["positions"][st["axes"][i]].long() if st["axes"] else pos for i in range(n)]
    return tuple(torch.stack([st[t][r, i] for i, r in enumerate(rows)], -1) for t in ("cos", "sin"))


def _exact_rope(st):
    c = st["case"]
    cos, sin = (x.unsqueeze(2) for x in _angles64(st, None))
    train = c["mode"] == "train"
    outs, grads, weights = [], [], []
    for name in ("q", "k"):
        x = st[name].double().requires_grad_(train)
        w = st[name + "_weight"].double().requires_grad_(train)
        y = _turn64(_norm64(x, w), cos, sin, 2 * len(st["axes"]), c["interleaved"])
        if c["fold"]:
            y = y.transpose(1, 2).reshape(-1, c["S"], c["D"])
        outs.append(y.detach())
        if train:
            dx, dw = torch.autograd.grad(y, (x, w), st["d_" + name].double())
            grads.append(dx)
            weights.append(dw)
    return outs + grads + weights


def _rounded64(x):
    """What 4 bits hold of x [..., D], by distance to each of the 15 values."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // _GROUP, _GROUP)
    most = g.abs().max(-1, keepdim=True).values / 6
    e = torch.floor(torch.log2(most.clamp_min(2.0 ** -14)))
    step = torch.exp2(e - 2)  # a scale has 3 significant bits
    s = (torch.round(most / step) * step).clamp_max(_MOST_SCALE)  # (ties to even)
    y = torch.where(s > 0, g / s.clamp_min(2.0 ** -20), 0.0)
    a = y.abs().clamp_max(6.0)
    unit = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()  # distance of neighbours
    return (torch.round(a / unit) * unit * torch.sign(y) * s).reshape(x.shape)


def _exact_append(st):
    c = st["case"]
    firsts = [(st["starts"][s], st["starts"][s + 1], l) for s, l in enumerate(st["lens"])]
    pos = torch.cat([torch.arange(l - e + b, l, device="cuda") for b, e, l in firsts])
    cos, sin = (x[:, None] for x in _angles64(st, pos))
    out = []
    for name in ("q", "k"):
        x = st[name].double()
        if c["norm"]:
            x = _norm64(x, st[name + "_weight"].double())
        out.append(_turn64(x, cos, sin, 2 * _rotated_pairs(c), c["interleaved"]))
    return [out[0], _rounded64(out[1].float().double()), _rounded64(st["v"].double())]


def _cached64(st, name, s, h, l):
    """The l cached rows of one sequence and head, byte by byte."""
    page, cache = st["case"]["page"], st[name]
    D = cache.shape[3] * 32 // 17
    tok = torch.arange(l, device="cuda")
    row = cache[st["page_table"][s].long()[torch.div(tok, page, rounding_mode="floor")], h].reshape(l, -1)
    slot, d = (tok % page)[:, None], torch.arange(D, device="cuda")[None, :]
    if name == "k_cache":
        byte, odd = slot * (D // 2) + d // 2, d % 2
        scale = page * D // 2 + slot * (D // 32) + d // 32
    else:
        byte, odd = (slot // 8 * D + d) * 4 + slot % 8 // 2, slot % 2
        scale = page * D // 2 + (slot // 8 * (D // 32) + d // 32) * 8 + slot % 8
    code = torch.gather(row, 1, byte.expand(l, D)).int()
    code = torch.where(odd.expand(l, D) == 1, code // 16, code % 16)
    low = code % 8
    mag = torch.where(low < 2, low * 0.5, (1 + (low % 2) * 0.5) * torch.exp2(low // 2 - 1.0)).double()
    b = torch.gather(row, 1, scale.expand(l, D)).int()
    e = b // 4
    s64 = torch.where(e > 0, (1 + b % 4 / 4) * torch.exp2(e - 15.0), b % 4 * 2.0 ** -16).double()
    return torch.where(code >= 8, -mag, mag) * s64


def _exact_paged(st):
    c = st["case"]
    G = c["H_q"] // c["H_kv"]
    T = st["starts"][-1]
    o = torch.zeros((T, c["H_q"], c["D_v"]), dtype=torch.float64, device="cuda")
    stats = torch.zeros((T, c["H_q"]), dtype=torch.float64, device="cuda")
    for s, l in enumerate(st["lens"]):
        first, last = st["starts"][s], st["starts"][s + 1]
        key = torch.arange(l, device="cuda")
        for h in range(c["H_kv"]):
            k, v = _cached64(st, "k_cache", s, h, l), _cached64(st, "v_cache", s, h, l)
            heads = slice(h * G, (h + 1) * G)
            for b in range(first, last, 1024):  # queries at a time
                e = min(b + 1024, last)
                z = torch.mm(st["q"][b:e, heads].double().reshape(-1, c["D_qk"]), k.t().contiguous())
                z = z.reshape(e - b, G, l) * (1.0 / math.sqrt(c["D_qk"]))
                if c["causal"]:
                    seen = torch.arange(b, e, device="cuda") - first + (l - (last - first))
                    z = torch.where(key[None, None, :] <= seen[:, None, None], z, float("-inf"))
                lse = torch.logsumexp(z, -1)
                p = torch.exp(z - lse[..., None])
                o[b:e, heads] = torch.mm(p.reshape(-1, l), v).reshape(e - b, G, c["D_v"])
                stats[b:e, heads] = lse
    return [o, stats]


def exact(case, seed):
    global own
    if case["op"] == "reserve":
        return None
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    return {"rope": _exact_rope, "append": _exact_append, "paged": _exact_paged}[case["op"]](st)
