"""kv_append against the definition in 64 bits (bounds: test_norm_rope_gpu.py),
and what it must leave alone."""
import ctypes

import pytest
import torch

import _heads as R64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32

# dtype, new tokens, cached tokens with them, H_q, H_kv, D_qk, D_v, page, R, interleaved, norm, tokens behind the last
CASES = [
    (F16, (1,), (1,), 1, 1, 64, 64, 16, 64, False, False, 0),
    (F16, (1, 1, 1, 1, 1), (17, 16, 1, 100, 33), 32, 8, 128, 128, 16, 128, False, False, 0),
    (F16, (40, 0, 1, 0, 33), (40, 9, 70, 0, 64), 6, 3, 80, 64, 32, 40, False, True, 3),  # sequences without tokens
    (F16, (15, 18), (31, 50), 2, 1, 128, 32, 16, 128, True, True, 0),  # across pages, one key head
    (F16, (7, 5), (9, 37), 3, 3, 36, 20, 16, 20, False, True, 1),      # no whole chunks
    (F16, (9,), (20,), 0, 2, 33, 1, 16, 10, True, False, 0),           # no queries, odd widths
    (F32, (3, 64), (3, 1000), 4, 2, 64, 64, 64, 64, False, True, 2),
    (F32, (21, 1), (40, 16), 5, 5, 128, 128, 16, 0, False, False, 0),  # not rotated: a copy
    (F32, (6, 2), (6, 30), 2, 2, 18, 22, 16, 6, True, True, 0),
    (F16, (1500, 700), (1500, 2048), 16, 4, 64, 64, 128, 64, False, False, 0),  # four rows per group of lanes
    (F16, tuple([1] * 70 + [3] * 70), tuple(range(3, 143)), 2, 1, 64, 64, 16, 64, False, False, 0),  # 140 sequences
]


def _batch(new, lens, page, seed=0, extra=4):
    used = [-(-l // page) for l in lens]
    width = max(max(used), 1)
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(used) + extra, generator=g).tolist()
    table, at = [], 0
    for u in used:
        table.append(order[at:at + u] + [-7] * (width - u))  # (columns behind the last page are not read)
        at += u
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    return i32(table), i32(starts), i32(lens), sum(used) + extra


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c)[:90])
def test_append(pkg, case):
    T, new, lens, H_q, H_kv, D, D_v, page, R, inter, norm, behind = case
    table, starts, kv_lens, pages = _batch(new, lens, page)
    g = torch.Generator().manual_seed(1)
    n = sum(new) + behind
    qkv = torch.randn((n, H_q + H_kv, D), generator=g).to(T)
    v = torch.randn((n, H_kv, D_v), generator=g).to(T)
    kc, vc = (torch.randn((pages, H_kv, page, d), generator=g).to(T) for d in (D, D_v))
    w = [(1 + 0.3 * torch.randn((D,), generator=g)).to(F32) for _ in range(2)] if norm else [None, None]
    cos, sin = R64.tables(max(lens), R) if R else (None, None)
    dev = lambda t: None if t is None else t.to(DEV)
    gx, gkc, gvc = dev(qkv), dev(kc), dev(vc)
    q_out = pkg.kv_append(gx[:, H_q:], dev(v), gkc, gvc, dev(table), dev(starts), dev(kv_lens), dev(cos), dev(sin),
                          q=gx[:, :H_q] if H_q else None, q_weight=dev(w[0]), k_weight=dev(w[1]), norm=norm,
                          interleaved=inter)
    # the definition
    u = R64.U32
    rel, tiny = R64.half_step(T)
    want_k, want_v = kc.double(), vc.double()
    bound_k = torch.zeros_like(want_k)
    want_q, bound_q = torch.zeros((n, H_q, D), dtype=torch.float64), torch.zeros((n, H_q, D), dtype=torch.float64)
    for s, (m, l) in enumerate(zip(new, lens)):
        for i in range(m):
            t, pos = int(starts[s]) + i, l - m + i
            pg, slot = int(table[s, pos // page]), pos % page
            x = qkv[t].double()
            heads = torch.cat([R64.norm(x[:H_q], w[0].double(), 1e-6), R64.norm(x[H_q:], w[1].double(), 1e-6)]) if norm else x
            c, sn = (cos[pos].double(), sin[pos].double()) if R else (torch.zeros(0).double(), torch.zeros(0).double())
            y = R64.turn(heads, c, sn, inter)
            b = torch.zeros_like(y) if not R and not norm else rel * y.abs() + 32 * u * R64.pair_size(heads, R, inter) + tiny
            want_q[t], bound_q[t] = y[:H_q], b[:H_q]
            want_k[pg, :, slot], bound_k[pg, :, slot] = y[H_q:], b[H_q:]
            want_v[pg, :, slot] = v[t].double()
    assert R64.worst(gkc, want_k, bound_k) <= 1  # every other row as it was
    assert torch.equal(gvc.cpu(), want_v.to(T))
    if H_q:
        live = slice(0, sum(new))
        assert R64.worst(q_out[live], want_q[live], bound_q[live]) <= 1
    else:
        assert q_out is None


def test_places_that_do_not_exist(pkg):
    """Tokens past the table, on pages that are none, before the first token:
    not appended, their query rows NaN; positions outside of the tables: NaN."""
    page, H, D = 16, 2, 32
    new, lens = (4, 2, 2, 3), (34, 20, 1, 12)
    table = torch.tensor([[0, 1], [2, 9], [3, 4], [5, -1]], dtype=torch.int32)  # 9: there are 9 pages
    starts = torch.tensor([0, 4, 6, 8, 11], dtype=torch.int32)
    kv = torch.tensor(lens, dtype=torch.int32)
    g = torch.Generator().manual_seed(0)
    x = torch.randn((11, 3 * H, D), generator=g).half().to(DEV)
    cache = torch.randn((9, H, page, D), generator=g).half().to(DEV)
    kc, vc = cache.clone(), cache.clone()
    cos, sin = (t.to(DEV) for t in R64.tables(11, D))
    args = [t.to(DEV) for t in (table, starts, kv)]
    q = pkg.kv_append(x[:, H:2 * H], x[:, 2 * H:], kc, vc, *args, cos, sin, q=x[:, :H])
    ok = torch.zeros(11, dtype=torch.bool)
    # sequence 0: places 30, 31 hold, 32 and 33 are past the table's two columns;
    # 1: 18, 19 on page 9; 2: places -1 and 0; 3: 9, 10, 11
    placed = torch.zeros(11, dtype=torch.bool)
    placed[[0, 1, 7, 8, 9, 10]] = True
    ok[[7, 8, 9]] = True  # positions 0, 9, 10 inside the 11 rows of the tables
    assert torch.equal(torch.isnan(q).all(-1).all(-1).cpu(), ~ok) and not torch.isnan(q[ok.to(DEV)]).any()
    changed_v = (vc != cache).any(-1).any(1).nonzero().tolist()
    assert changed_v == [[1, 14], [1, 15], [3, 0], [5, 9], [5, 10], [5, 11]]
    bad_k = torch.isnan(kc).any(-1).any(1).nonzero().tolist()
    assert bad_k == [[1, 14], [1, 15], [5, 11]]


def test_rows_behind_the_last_sequence(pkg):
    """The C entry with a result of its own leaves rows behind the last
    sequence, and the whole of it where there are no sequences."""
    L = pkg.library()
    H, D, page = 2, 32, 16
    x = torch.randn((5, H, D), device=DEV).half()
    out = torch.full((5, H, D), 7.0, device=DEV, dtype=F16)
    cache = torch.zeros((2, H, page, D), device=DEV, dtype=F16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    table, starts, lens = i32([[0], [1]]), i32([0, 1, 3]), i32([1, 2])

    def call(N):
        return L.sdpa_hip_kv_append(1, x.data_ptr(), None, x.data_ptr(), None, cache.data_ptr(), cache.data_ptr(),
                                    x.data_ptr(), None, out.data_ptr(), None, None, None, 0, None, None, 0,
                                    table.data_ptr(), 1, starts.data_ptr(), lens.data_ptr(), N, 5, 1, 2, page, H, H, D, D,
                                    0, 1e-6, 0, 0, torch.cuda.current_stream().cuda_stream)

    assert call(0) == 0 and bool((out == 7).all())
    assert call(2) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[:3], x[:3]) and bool((out[3:] == 7).all())


def test_cache_past_32_bits(pkg):
    """Rows of a cache of more than 2^32 bytes, in its last page."""
    H, D, page = 4, 128, 256
    pages = 2 ** 32 // (H * D * page * 2) + 3
    cache = torch.zeros((pages, H, page, D), device=DEV, dtype=F16)
    x = torch.randn((2, H, D), device=DEV).half()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    args = (i32([[pages - 1], [0]]), i32([0, 1, 2]), i32([page, 1]))
    pkg.kv_append(x, x, cache, cache, *args)  # (k and v alike, so that one cache does)
    assert torch.equal(cache[pages - 1, :, page - 1], x[0]) and torch.equal(cache[0, :, 0], x[1])
    assert int((cache != 0).any(-1).sum()) == 2 * H


def test_captured_append_follows_the_lengths(pkg):
    """One captured generation step: lengths and tokens change between replays."""
    page, H, D = 16, 2, 64
    table = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32, device=DEV)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    lens = torch.tensor([1, 14], dtype=torch.int32, device=DEV)
    x = torch.randn((2, 3 * H, D), device=DEV).half()
    cos, sin = (t.to(DEV) for t in R64.tables(40, D))
    caches = [torch.zeros((4, H, page, D), device=DEV, dtype=F16) for _ in range(4)]
    step = lambda a, b: pkg.kv_append(x[:, H:2 * H], x[:, 2 * H:], a, b, table, starts, lens, cos, sin, q=x[:, :H])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0].clone(), caches[1].clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = step(caches[0], caches[1])
    for i in range(5):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)).half())
        lens += 1
        want = step(caches[2], caches[3])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, want) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


def test_layouts_of_the_batch(pkg):
    """A first sequence that does not begin at the first token, a table that is part
    of a wider one, results in the place of the queries (C entry)."""
    page, H, D = 16, 2, 64
    x = torch.randn((7, 3 * H, D), device=DEV).half()
    cos, sin = (t.to(DEV) for t in R64.tables(60, D))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    table, starts, lens = i32([[9, 0, 1, 2], [9, 3, 4, 5]]), i32([2, 4, 5]), i32([34, 17])
    kc, vc = (torch.zeros((6, H, page, D), device=DEV, dtype=F16) for _ in range(2))
    q = pkg.kv_append(x[:, H:2 * H], x[:, 2 * H:], kc, vc, table[:, 1:], starts, lens, cos, sin, q=x[:, :H])
    places = [(2, 0), (2, 1), (4, 0)]  # tokens 2, 3 at 32, 33 of the first; 4 at 16 of the second
    assert (vc != 0).any(-1).any(1).nonzero().tolist() == sorted(map(list, places))
    for t, (pg, slot) in zip((2, 3, 4), places):
        assert torch.equal(vc[pg, :, slot], x[t, 2 * H:])
    y = x.clone()
    k2, v2 = torch.zeros_like(kc), torch.zeros_like(vc)
    st = (ctypes.c_int64 * 2)(*y.stride()[:2])
    part = [y[:, i * H:(i + 1) * H].data_ptr() for i in range(3)]
    rc = pkg.library().sdpa_hip_kv_append(1, part[1], st, part[2], st, k2.data_ptr(), v2.data_ptr(), part[0], st, part[0], st,
                                          None, None, 0, cos.data_ptr(), sin.data_ptr(), 60, table[:, 1:].data_ptr(), 4,
                                          starts.data_ptr(), lens.data_ptr(), 2, 7, 3, 6, page, H, H, D, D, D, 1e-6, 0, 0,
                                          torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert torch.equal(k2, kc) and torch.equal(v2, vc) and torch.equal(y[2:5, :H], q[2:5])
    y[2:5, :H] = x[2:5, :H]
    assert torch.equal(y, x)  # other tokens, keys and values stay
