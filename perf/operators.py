"""The calls that the performance of the operators around ``sdpa`` is judged on.

``norm_rope`` is what a layer does to its queries and keys before attention:
the norm of each head, the rotation by position, and the layout that attention
reads (``train``: with the gradient; ``fwd``: without).  ``append`` puts the
keys and values of new tokens into the pages of a cache, rotated, with the
queries rotated in the same call.  ``paged`` is the attention of new tokens,
one or a chunk per sequence, over such a cache.

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


# ---- cases -----------------------------------------------------------------

def _norm_rope(mode, dtype, B, S, H_q, H_kv, D, R, fold, interleaved=False, w32=True, start=0):
    """``start``: the position of the first token (0: positions are left out,
    the sequence starts there)."""
    return {"op": "norm_rope", "mode": mode, "dtype": dtype, "B": B, "S": S, "H_q": H_q, "H_kv": H_kv, "D": D, "R": R,
            "fold": fold, "interleaved": interleaved, "w32": w32, "start": start}


def _spread(rng, n, lo, hi):
    """n lengths between lo and hi, spread over their logarithm, as one text."""
    return " ".join(str(_log(rng, lo, hi)) for _ in range(n))


def _append(dtype, new, lens, H_q, H_kv, D_qk, D_v, page, R, norm=False, interleaved=False):
    return {"op": "append", "dtype": dtype, "new": new, "lens": lens, "H_q": H_q, "H_kv": H_kv, "D_qk": D_qk, "D_v": D_v,
            "page": page, "R": R, "norm": norm, "interleaved": interleaved}


def _paged(dtype, new, lens, H_q, H_kv, D_qk, D_v, page, causal=True):
    return {"op": "paged", "dtype": dtype, "new": new, "lens": lens, "H_q": H_q, "H_kv": H_kv, "D_qk": D_qk, "D_v": D_v,
            "page": page, "causal": causal}


def listed():
    ragged = random.Random(11)
    long_lens = _spread(ragged, 64, 600, 16384)
    mixed_new = "700 333 1 " + " ".join(["1"] * 30)
    mixed_lens = "1724 333 1 " + _spread(ragged, 30, 100, 4096)
    rows = [
        # One generated token of 4 sequences, 32 query heads on 8 key heads: a
        # few microseconds, where latency counts.
        ("norm_rope_decode_f16", _norm_rope("fwd", "f16", 4, 1, 32, 8, 128, 128, False, w32=False, start=1203)),
        # A training step of the benchmark's attention layer: 4 sequences of
        # 4096 tokens, 32 heads of 128.
        ("norm_rope_train_f16", _norm_rope("train", "f16", 4, 4096, 32, 32, 128, 128, True)),
        # Full-precision training at a ragged length, half of each head rotated.
        ("norm_rope_train_f32", _norm_rope("train", "f32", 8, 1000, 12, 12, 64, 32, True)),
        # One token of each of 64 sequences into pages of 16.
        ("append_decode_f16", _append("f16", " ".join(["1"] * 64), _spread(ragged, 64, 50, 2000), 32, 8, 128, 128, 16, 128)),
        # Prompts of 4 sequences, keys and queries normed on the way.
        ("append_chunks_f16", _append("f16", "2048 4096 999 1500", "2048 6000 999 3333", 32, 8, 128, 128, 64, 128, True)),
        # Full precision, neighbouring features paired, heads 80 wide.
        ("append_f32", _append("f32", "129 1 500 64", "400 77 500 1000", 16, 16, 80, 64, 32, 80, False, True)),
        # Generation: one new token of 4 sequences with 16 heads each, 4096 cached.
        ("paged_decode_f16", _paged("f16", "1 1 1 1", "4096 4096 4096 4096", 16, 16, 128, 128, 16)),
        # A serving batch: 64 sequences of very unequal length, shared heads.
        ("paged_decode_ragged_f16", _paged("f16", " ".join(["1"] * 64), long_lens, 32, 8, 128, 128, 64)),
        # The next chunk of a long document.
        ("paged_chunk_f16", _paged("f16", "512", "16000", 32, 8, 128, 128, 64)),
        # Chunks and single tokens in one batch, heads 64 wide.
        ("paged_mixed_f16", _paged("f16", mixed_new, mixed_lens, 16, 4, 64, 64, 32)),
        # Four whole prompts: the largest call.
        ("paged_prompts_f16", _paged("f16", "4096 4096 4096 4096", "4096 4096 4096 4096", 32, 8, 128, 128, 128)),
        # Full precision: a chunk and generation.
        ("paged_f32", _paged("f32", "300 1 1 1", "2300 1000 4001 517", 16, 4, 64, 64, 16)),
    ]
    return [dict(c, name=n) for n, c in rows]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "norm_rope", "append", "paged", "paged", "paged"])
    dtype = rng.choice(["f16", "f16", "f16", "f32"])
    D = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
    H_kv, G = rng.choice([1, 2, 4, 8, 8, 12, 16]), rng.choice([1, 1, 2, 3, 4, 8])
    if op == "norm_rope":
        mode = rng.choice(["fwd", "train", "train"])
        B, S = _log(rng, 1, 64), (1 if mode == "fwd" and rng.random() < 0.4 else _log(rng, 16, 8192))
        c = _norm_rope(mode, dtype, B, S, H_kv * G, H_kv, D, rng.choice([D, D, D // 2]), rng.random() < 0.7,
                       rng.random() < 0.3, rng.random() < 0.5, rng.choice([0, 0, _log(rng, 1, 20000)]))
        while work(c)["bytes"] > 1.2e9:
            c["S"] = max(1, c["S"] * 2 // 3)
        return c
    page = rng.choice([16, 16, 32, 64, 128])
    kind = rng.choice(["decode", "decode", "chunks", "mixed"])
    few = H_kv * G <= 8
    if kind == "decode":
        N = _log(rng, 1, 128)
        new = [rng.choice([1, 1, 1, 1, 2, 4]) if few else 1 for _ in range(N)]
    elif kind == "chunks":
        N = rng.choice([1, 1, 2, 3, 5])
        new = [_log(rng, 33, 2048) for _ in range(N)]
    else:
        N = _log(rng, 3, 40)
        new = [_log(rng, 2, 700) if rng.random() < 0.2 else 1 for _ in range(N)]
    lens = [n + (0 if rng.random() < 0.1 else _log(rng, 1, 16384)) for n in new]
    D_v = D if rng.random() < 0.8 else rng.choice([32, 64, 128])
    if op == "append":
        return _append(dtype, " ".join(map(str, new)), " ".join(map(str, lens)), H_kv * G, H_kv, D, D_v, page,
                       rng.choice([D, D, D // 2]), rng.random() < 0.5, rng.random() < 0.3)
    most = 4e11 if dtype == "f16" else 6e10
    while True:
        c = _paged(dtype, " ".join(map(str, new)), " ".join(map(str, lens)), H_kv * G, H_kv, D, D_v, page,
                   rng.random() < 0.9)
        w = work(c)
        if w["flops"] <= most and w["bytes"] <= 1.2e9:
            return c
        lens = [max(n, l * 2 // 3) for n, l in zip(new, lens)]
        if w["flops"] > most:
            new = [max(1, n * 3 // 4) for n in new]


def _ints(text):
    return [int(x) for x in text.split()]


def work(case):
    c = case
    e = 2 if c["dtype"] == "f16" else 4
    if c["op"] == "norm_rope":
        n = c["B"] * c["S"] * (c["H_q"] + c["H_kv"]) * c["D"]
        table = 4 * c["S"] * c["R"]
        if c["mode"] == "fwd":  # x in, y out
            return {"bytes": 2 * n * e + table, "flops": 8 * n}
        return {"bytes": 5 * n * e + table, "flops": 24 * n}  # and x, dy in, dx out
    new, lens = _ints(c["new"]), _ints(c["lens"])
    T = sum(new)
    if c["op"] == "append":  # k, v and q in and out
        n = T * ((c["H_kv"] + c["H_q"]) * c["D_qk"] + c["H_kv"] * c["D_v"])
        return {"bytes": 2 * n * e + 4 * T * c["R"], "flops": (8 if c["norm"] else 4) * n}
    kv = sum(lens) * c["H_kv"] * (c["D_qk"] + c["D_v"]) * e
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


def _pages(c, seed):
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
    table, starts_t, lens_t = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (rows, starts, lens))
    return {"page_table": table, "q_starts": starts_t, "kv_lens": lens_t, "starts": starts, "lens": lens,
            "pages": len(order), "max_new": max(new)}


def prepare(case, seed):
    c = case
    dt, g = _DTYPES[c["dtype"]], _generator(seed)
    state = {"case": c, "op": importlib.import_module("tf-custom-flash-attention_amd") if own else None}
    if c["op"] == "norm_rope":
        B, S, H_q, H_kv, D = c["B"], c["S"], c["H_q"], c["H_kv"], c["D"]
        # q and k are parts of one projection's output
        qk = _normal(g, (B, S, H_q + H_kv, D), dt, 1.5)
        state["q"], state["k"] = qk[:, :, :H_q], qk[:, :, H_q:]
        state["q_weight"], state["k_weight"] = _weights(g, c, D)
        state["cos"], state["sin"] = _tables(c["start"] + S, c["R"])
        state["positions"] = None if c["start"] == 0 else torch.arange(c["start"], c["start"] + S, dtype=torch.int32,
                                                                       device="cuda")
        if c["mode"] == "train":
            for name, H in (("d_q", H_q), ("d_k", H_kv)):
                state[name] = _normal(g, (B * H, S, D) if c["fold"] else (B, S, H, D), dt)
        return state
    state.update(_pages(c, seed))
    T, H_q, H_kv, D_qk, D_v, page = state["starts"][-1], c["H_q"], c["H_kv"], c["D_qk"], c["D_v"], c["page"]
    state["q"] = _normal(g, (T, H_q, D_qk), dt)
    state["k_cache"] = _normal(g, (state["pages"], H_kv, page, D_qk), dt)
    state["v_cache"] = _normal(g, (state["pages"], H_kv, page, D_v), dt)
    if c["op"] == "append":
        state["k"], state["v"] = _normal(g, (T, H_kv, D_qk), dt), _normal(g, (T, H_kv, D_v), dt)
        state["q_weight"], state["k_weight"] = _weights(g, c, D_qk) if c["norm"] else (None, None)
        state["cos"], state["sin"] = _tables(max(state["lens"]), c["R"])
    return state


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


def _folded(x, fold):  # [B, S, H, D] -> [B * H, S, D]
    return x.permute(0, 2, 1, 3).flatten(0, 1).contiguous() if fold else x


def _plain_norm_rope(st):
    c = st["case"]
    S, R, inter = c["S"], c["R"], c["interleaved"]
    at = slice(c["start"], c["start"] + S)
    cos, sin = st["cos"][at, None, :], st["sin"][at, None, :]
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


def _plain_append(st):
    c = st["case"]
    starts, lens = st["starts"], st["lens"]
    pos = torch.cat([torch.arange(l - (e - s), l, device="cuda") for s, e, l in zip(starts, starts[1:], lens)])
    cos, sin = st["cos"][pos, None, :], st["sin"][pos, None, :]
    rows = []
    for name in ("q", "k"):
        x = st[name].float()
        if c["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * st[name + "_weight"].float()
        rows.append(_rotated(x, cos, sin, c["R"], c["interleaved"]).to(st[name].dtype))
    page = c["page"]
    for s, (b, e) in enumerate(zip(starts, starts[1:])):
        p = pos[b:e]
        pages, slots = st["page_table"][s].long()[p // page], p % page
        st["k_cache"][pages, :, slots] = rows[1][b:e]
        st["v_cache"][pages, :, slots] = st["v"][b:e]
    return [rows[0], st["k_cache"], st["v_cache"]]


def _plain_paged(st):
    c = st["case"]
    page, H_kv, G = c["page"], c["H_kv"], c["H_q"] // c["H_kv"]
    os, stats = [], []
    for s, (b, e, l) in enumerate(zip(st["starts"], st["starts"][1:], st["lens"])):
        pages = st["page_table"][s, :-(-l // page)].long()
        # [H_kv, l, D]
        k, v = (st[x][pages].float().transpose(0, 1).flatten(1, 2)[:, :l].contiguous() for x in ("k_cache", "v_cache"))
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
        return {"norm_rope": _plain_norm_rope, "append": _plain_append, "paged": _plain_paged}[c["op"]](st)
    if c["op"] == "norm_rope":
        args = dict(q_weight=st["q_weight"], k_weight=st["k_weight"], positions=st["positions"], eps=_EPS,
                    interleaved=c["interleaved"], fold_heads=c["fold"])
        outs = op.qk_norm_rope(st["q"], st["k"], st["cos"], st["sin"], **args)
        if c["mode"] == "train":
            outs += op.qk_norm_rope_grad(st["d_q"], st["d_k"], st["q"], st["k"], st["cos"], st["sin"], **args)
        return list(outs)
    where = (st["k_cache"], st["v_cache"], st["page_table"], st["q_starts"], st["kv_lens"])
    if c["op"] == "append":
        q = op.kv_append(st["k"], st["v"], *where, cos=st["cos"], sin=st["sin"], q=st["q"], q_weight=st["q_weight"],
                         k_weight=st["k_weight"], norm=c["norm"], eps=_EPS, interleaved=c["interleaved"])
        return [q, st["k_cache"], st["v_cache"]]
    return list(op.paged_sdpa(st["q"], *where, scale=c["D_qk"] ** -0.5, causal_mask=c["causal"], max_q_len=st["max_new"]))


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


def _exact_norm_rope(st):
    c = st["case"]
    at = torch.arange(c["start"], c["start"] + c["S"], device="cuda")
    cos, sin = st["cos"][at].unsqueeze(1), st["sin"][at].unsqueeze(1)
    train = c["mode"] == "train"
    outs, grads, weights = [], [], []
    for name in ("q", "k"):
        x = st[name].double().requires_grad_(train)
        w = st[name + "_weight"].double().requires_grad_(train)
        y = _turn64(_norm64(x, w), cos, sin, c["R"], c["interleaved"])
        if c["fold"]:
            y = y.transpose(1, 2).reshape(-1, c["S"], c["D"])
        outs.append(y.detach())
        if train:
            dx, dw = torch.autograd.grad(y, (x, w), st["d_" + name].double())
            grads.append(dx)
            weights.append(dw)
    return outs + grads + weights


def _exact_append(st):
    c = st["case"]
    caches = {"k": st["k_cache"].double(), "v": st["v_cache"].double()}
    q_out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    for s, l in enumerate(st["lens"]):
        rows = slice(st["starts"][s], st["starts"][s + 1])
        n = rows.stop - rows.start
        where = torch.arange(l - n, l, device="cuda")
        cos, sin = (st[t].index_select(0, where).unsqueeze(1) for t in ("cos", "sin"))
        q, k = (st[t][rows].double() for t in ("q", "k"))
        if c["norm"]:
            q, k = _norm64(q, st["q_weight"].double()), _norm64(k, st["k_weight"].double())
        q_out[rows] = _turn64(q, cos, sin, c["R"], c["interleaved"])
        k = _turn64(k, cos, sin, c["R"], c["interleaved"])
        page = st["page_table"][s].index_select(0, torch.div(where, c["page"], rounding_mode="floor")).long()
        slot = page * c["page"] + torch.remainder(where, c["page"])  # row of [pages * page, H_kv, D]
        for t, x in (("k", k), ("v", st["v"][rows].double())):
            cache = caches[t].transpose(1, 2)
            flat = cache.reshape(-1, *cache.shape[2:])
            flat[slot] = x
            caches[t] = flat.reshape(cache.shape).transpose(1, 2).contiguous()
    return [q_out, caches["k"], caches["v"]]


def _exact_paged(st):
    c = st["case"]
    G, page = c["H_q"] // c["H_kv"], c["page"]
    T = st["starts"][-1]
    o = torch.zeros((T, c["H_q"], c["D_v"]), dtype=torch.float64, device="cuda")
    stats = torch.zeros((T, c["H_q"]), dtype=torch.float64, device="cuda")
    for s, l in enumerate(st["lens"]):
        first, last = st["starts"][s], st["starts"][s + 1]
        key = torch.arange(l, device="cuda")
        at = st["page_table"][s].long()[torch.div(key, page, rounding_mode="floor")]
        for h in range(c["H_kv"]):
            k = st["k_cache"][at, h, key % page].double()
            v = st["v_cache"][at, h, key % page].double()
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
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    return {"norm_rope": _exact_norm_rope, "append": _exact_append, "paged": _exact_paged}[case["op"]](st)
