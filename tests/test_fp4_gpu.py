"""kv_append_fp4 and kv_read_fp4 against the definition of the cache in 4 bits
(_fp4.py): bytes and values are equal, not near."""
import pytest
import torch

import _fp4 as F
import _heads as R64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
I32 = torch.int32
NAN, INF = float("nan"), float("inf")


def _same(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def _batch(new, lens, page, seed=0, extra=4):
    used = [-(-l // page) for l in lens]
    width = max(max(used), 1)
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(used) + extra, generator=g).tolist()
    table, at = [], 0
    for u in used:
        table.append(order[at:at + u] + [-7] * (width - u))
        at += u
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    i32 = lambda x: torch.tensor(x, dtype=I32)
    return i32(table), i32(starts), i32(lens), sum(used) + extra


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _one_page(pkg, x, T):
    """Rows x [n, D] as keys and as values of one sequence: the caches, and what is read back."""
    n, D = x.shape
    page = max(16, 1 << (n - 1).bit_length())
    kc, vc = (c.fill_(0xFF) for c in pkg.fp4_cache(1, 1, page, D, D, device=DEV))
    batch = _dev(*(torch.tensor(t, dtype=I32) for t in ([[0]], [0, n], [n])))
    rows = x.to(T).to(DEV)[:, None]
    pkg.kv_append_fp4(rows, rows, kc, vc, *batch)
    return kc, vc, pkg.kv_read_fp4(kc, vc, *batch, n, T)


@pytest.mark.parametrize("T", (F16, F32))
def test_rounding(pkg, T):
    """Ties and their neighbours in codes and scales, scales below their normal range, the
    largest, groups of zeros and of infinities and NaN; keys and values alike."""
    g = torch.Generator().manual_seed(0)
    rows = []
    for s in (1.0, 1.25, 1.5, 1.75, 2.0 ** -14, 1.5 * 2.0 ** -15, 2.0 ** -16, 3 * 2.0 ** -16, 1024.0, 8192.0):
        ties = torch.tensor([0, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, .5, 1, 1.5, 2, 3, 4, 6, 5.5]) * s
        rows.append(torch.cat((ties, -ties.flip(0))))
        rows.append(torch.cat((torch.nextafter(ties.to(T), torch.tensor(0.).to(T)), torch.nextafter(ties.to(T), torch.tensor(9e4).to(T)))))
        rows[-1][14] = 6 * s
    for m in (6.75, 8.25, 9.75, 11.25, 6.75 * 2.0 ** -13, 9 * 2.0 ** -17, 15 * 2.0 ** -17, 2.0 ** -18, 60000., 65504.):  # largest: ties of scales
        rows.append(torch.rand(32, generator=g) * m)
        rows[-1][7] = m
        rows.append(rows[-1].to(T))
        rows[-1][7] = torch.nextafter(torch.tensor(m).to(T), torch.tensor(0.).to(T))
    rows.append(torch.zeros(32))
    rows.append(-torch.zeros(32))
    for bad in (INF, -INF, NAN):
        rows.append(torch.randn(32, generator=g))
        rows[-1][9] = bad
    if T == F32:
        for big in (1e5, 1e30, 3.4e38, 1e-30, 1e-44):
            rows.append(torch.randn(32, generator=g).clamp(-1, 1) * big)
    rows += list((torch.randn((300, 32), generator=g) * torch.exp(3 * torch.randn((300, 1), generator=g))).to(T))
    x = torch.stack([r.float() for r in rows]).to(T).float()
    wide = torch.cat((x, torch.randn(x.shape, generator=g)), 1)  # (a group does not touch the next)
    kc, vc, (k, v) = _one_page(pkg, wide, T)
    codes, scales = F.encode(wide.to(T))
    want = F.decode(codes, scales)
    n = len(wide)
    for cache, got, is_v in ((kc, k, False), (vc, v, True)):
        c, s = F.unpack(cache, is_v)
        assert torch.equal(s[0, 0, :n], scales)
        fine = ~torch.isnan(want)
        assert torch.equal(c[0, 0, :n][fine], codes[fine])
        assert _same(got[:, 0].double().cpu(), want)
        # what is behind the tokens stays as it was
        assert bool((c[0, 0, n:] == 15).all()) and bool((s[0, 0, n:] == 255).all())


# dtype, new tokens, cached tokens with them, H_q, H_kv, D_qk, D_v, page, R, interleaved, norm, tokens behind the last
CASES = [
    (F16, (1,), (1,), 1, 1, 64, 64, 16, 64, False, False, 0),
    (F16, (1, 1, 1, 1, 1), (17, 16, 1, 100, 33), 32, 8, 128, 128, 16, 128, False, False, 0),
    (F16, (40, 0, 1, 0, 33), (40, 9, 70, 0, 64), 6, 3, 96, 64, 32, 40, False, True, 3),
    (F16, (15, 18), (31, 50), 2, 1, 128, 32, 16, 128, True, True, 0),
    (F16, (7, 5, 3), (9, 37, 6), 3, 3, 32, 96, 16, 20, False, True, 1),    # inside one word; pairs that are no whole chunks
    (F16, (9,), (20,), 0, 2, 64, 128, 16, 10, True, False, 0),
    (F32, (3, 64), (3, 1000), 4, 2, 64, 64, 64, 64, False, True, 2),
    (F32, (21, 1), (40, 16), 5, 5, 128, 128, 16, 0, False, False, 0),
    (F32, (6, 2), (6, 30), 2, 2, 96, 32, 16, 6, True, True, 0),
    (F16, (1500, 700), (1500, 2048), 16, 8, 64, 64, 128, 64, False, False, 0),     # windows of 8 tokens
    (F32, (1100, 3, 1, 900), (1103, 3, 70, 950), 2, 8, 128, 32, 16, 128, False, True, 5),
    (F16, tuple([1] * 70 + [3] * 70), tuple(range(3, 143)), 2, 1, 64, 64, 16, 64, False, False, 0),
    (F16, tuple([1, 2, 5] * 400), tuple(5 + i % 90 for i in range(1200)), 1, 4, 32, 32, 16, 32, False, False, 0),
]


def _keys64(x, w, pos, cos, sin, inter, norm):
    """Keys [n, H, D] in 64 bits, turned by places or positions."""
    y = x.double()
    if norm:
        y = R64.norm(y, w.double(), 1e-6)
    if cos is None:
        return y
    return R64.turn(y, cos[pos].double()[:, None], sin[pos].double()[:, None], inter)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c)[:90])
def test_append_and_read(pkg, case):
    T, new, lens, H_q, H_kv, D, D_v, page, R, inter, norm, behind = case
    table, starts, kv_lens, pages = _batch(new, lens, page)
    g = torch.Generator().manual_seed(1)
    n = sum(new) + behind
    x = torch.randn((n, H_q + H_kv, D), generator=g).to(T)
    v = torch.randn((n, H_kv, D_v), generator=g).to(T)
    kc, vc = F.random_cache(g, pages, H_kv, page, D, False), F.random_cache(g, pages, H_kv, page, D_v, True)
    w = [(1 + 0.3 * torch.randn((D,), generator=g)).to(F32) for _ in range(2)] if norm else [None, None]
    cos, sin = R64.tables(max(lens), R) if R else (None, None)
    gx, gv, gkc, gvc, *rest = _dev(x, v, kc, vc, table, starts, kv_lens, cos, sin)
    kw = dict(q=gx[:, :H_q] if H_q else None, q_weight=_dev(w[0])[0], k_weight=_dev(w[1])[0], norm=norm, interleaved=inter)
    q_out = pkg.kv_append_fp4(gx[:, H_q:], gv, gkc, gvc, *rest, **kw)
    # queries as in the append to a cache of T
    dense = [torch.zeros((pages, H_kv, page, d), dtype=T, device=DEV) for d in (D, D_v)]
    other = pkg.kv_append(gx[:, H_q:], gv, *dense, *rest, **kw)
    live = sum(new)
    assert q_out is None if not H_q else torch.equal(q_out[:live], other[:live])
    # the new tokens' codes, every other as it was
    pos = torch.cat([torch.arange(l - m, l) for m, l in zip(new, lens)])
    seq = torch.cat([torch.full((m,), s) for s, m in enumerate(new)])
    pg, slot = table[seq, pos // page].long(), pos % page
    back = pkg.kv_read_fp4(gkc, gvc, *rest[:3], n, T)
    for before, cache, rows, is_v, got in ((kc, gkc, _keys64(x[:live, H_q:], w[1], pos, cos, sin, inter, norm), False, back[0]),
                                           (vc, gvc, v[:live], True, back[1])):
        want_c, want_s = F.unpack(before, is_v)
        codes, scales = F.encode(rows)
        want_c[pg, :, slot], want_s[pg, :, slot] = codes, scales
        c, s = F.unpack(cache, is_v)
        assert torch.equal(s, want_s) and torch.equal(c, want_c)
        assert torch.equal(got[:live].double().cpu(), F.decode(codes, scales))
    # the other dtype reads the same values
    again = pkg.kv_read_fp4(gkc, gvc, *rest[:3], n, F32 if T == F16 else F16)
    assert all(torch.equal(a[:live].float(), b[:live].float()) for a, b in zip(again, back))


@pytest.mark.parametrize("T,axes", [(F16, tuple([0] * 16 + [1] * 24 + [2] * 24)), (F32, (0, 1, 2) * 21 + (3,)), (F16, None)])
def test_append_by_positions(pkg, T, axes):
    H_q, H_kv, D, page, n = 6, 2, 128, 16, 12
    new, lens = (1, 9, 2), (20, 33, 2)
    table, starts, kv, pages = _batch(new, lens, page)
    g = torch.Generator().manual_seed(1)
    x = torch.randn((n, H_q + 2 * H_kv, D), generator=g).to(T)
    cos, sin = R64.tables(90, 128)
    pos = torch.randint(0, 90, (4, n) if axes else (n,), generator=g, dtype=I32)
    kc, vc = pkg.fp4_cache(pages, H_kv, page, D, D, device=DEV)
    gx, *rest = _dev(x, table, starts, kv, cos, sin)
    q = pkg.kv_append_fp4(gx[:, H_q:-H_kv], gx[:, -H_kv:], kc, vc, *rest, q=gx[:, :H_q], positions=pos.to(DEV), axes=axes)
    rows = (pos if axes else pos[None]).long()
    c, s = (torch.stack([t.double()[rows[a], i] for i, a in enumerate(axes or (0,) * 64)], -1)[:, None] for t in (cos, sin))
    want = F.decode(*F.encode(R64.turn(x[:, H_q:-H_kv].double(), c, s, False)))
    k, v = pkg.kv_read_fp4(kc, vc, *rest[:3], n, T)
    assert torch.equal(k.double().cpu(), want) and torch.equal(v.double().cpu(), F.decode(*F.encode(x[:, -H_kv:])))
    y = R64.turn(x[:, :H_q].double(), c, s, False)
    rel, tiny = R64.half_step(T)
    assert R64.worst(q, y, rel * y.abs() + 32 * R64.U32 * R64.pair_size(x[:, :H_q].double(), 128, False) + tiny) <= 1


def test_places_that_do_not_exist(pkg):
    """Tokens past the table, on pages that are none, before the first token: not
    appended, their query rows NaN and NaN when read; bad positions make keys NaN."""
    page, H, D = 16, 2, 32
    new, lens = (4, 2, 2, 3), (34, 20, 1, 12)
    table = torch.tensor([[0, 1], [2, 9], [3, 4], [5, -1]], dtype=I32)  # 9: there are 9 pages
    starts = torch.tensor([0, 4, 6, 8, 11], dtype=I32)
    kv = torch.tensor(lens, dtype=I32)
    g = torch.Generator().manual_seed(0)
    x = torch.randn((11, 3 * H, D), generator=g).half()
    kc, vc = F.random_cache(g, 9, H, page, D, False), F.random_cache(g, 9, H, page, D, True)
    gx, gkc, gvc, *batch = _dev(x, kc, vc, table, starts, kv)
    cos, sin = (t.to(DEV) for t in R64.tables(32, D))
    q = pkg.kv_append_fp4(gx[:, H:2 * H], gx[:, 2 * H:], gkc, gvc, *batch, cos, sin, q=gx[:, :H])
    # places: 30 31 32 33 | 18 19 | -1 0 | 9 10 11
    lost = torch.tensor([0, 0, 1, 1, 1, 1, 1, 0, 0, 0, 0], dtype=torch.bool)
    assert torch.equal(torch.isnan(q).all(-1).all(-1).cpu(), lost) and not torch.isnan(q[~lost.to(DEV)]).any()
    k, v = pkg.kv_read_fp4(gkc, gvc, *batch, 11)
    for t in (k, v):
        assert torch.equal(torch.isnan(t).all(-1).all(-1).cpu(), lost) and not torch.isnan(t[~lost.to(DEV)]).any()
    where = [(1, 14), (1, 15), (3, 0), (5, 9), (5, 10), (5, 11)]
    for before, after, is_v in ((kc, gkc, False), (vc, gvc, True)):
        changed = (F.values(before, is_v) != F.values(after, is_v)).any(-1).any(1).nonzero().tolist()
        assert sorted(map(tuple, changed)) == where
    # a position outside of the tables
    pos = torch.tensor([0, 1, 2, 3, 4, 5, 6, 7, 40, -1, 8], dtype=I32, device=DEV)
    q = pkg.kv_append_fp4(gx[:, H:2 * H], gx[:, 2 * H:], gkc, gvc, *batch, cos, sin, q=gx[:, :H], positions=pos)
    k, v = pkg.kv_read_fp4(gkc, gvc, *batch, 11)
    assert torch.isnan(k[8:10]).all() and not torch.isnan(k[[0, 1, 7, 10]]).any() and not torch.isnan(v[8:]).any()


def test_infinities_stay_in_their_group(pkg):
    x = torch.randn((5, 3, 96)).half()
    clean = x.clone()
    x[2, 1, 40], x[4, 0, 95] = INF, NAN
    args = _dev(*(torch.tensor(t, dtype=I32) for t in ([[0]], [0, 5], [5])))
    outs = []
    for rows in (clean.to(DEV), x.to(DEV)):
        kc, vc = pkg.fp4_cache(1, 3, 16, 96, 96, device=DEV)
        pkg.kv_append_fp4(rows, rows, kc, vc, *args)
        outs.append(torch.stack(pkg.kv_read_fp4(kc, vc, *args, 5)))
    differ = (outs[0] != outs[1]).nonzero().tolist()
    want = [[i, 2, 1, d] for i in (0, 1) for d in range(32, 64)] + [[i, 4, 0, d] for i in (0, 1) for d in range(64, 96)]
    assert sorted(differ) == sorted(want) and torch.isnan(outs[1][:, 2, 1, 32:64]).all()


def test_strides_and_alignment(pkg):
    """Parts of a wider tensor, odd addresses, tokens far apart, features that are not dense."""
    H, D, n, page = 2, 64, 21, 16
    table, starts, kv, pages = _batch((n,), (30,), page)
    batch = _dev(table, starts, kv)
    cos, sin = (t.to(DEV) for t in R64.tables(30, D))
    x = torch.randn((n, 3 * H, D), device=DEV).half()

    def run(k, v, q):
        kc, vc = pkg.fp4_cache(pages, H, page, D, D, device=DEV)
        return [pkg.kv_append_fp4(k, v, kc, vc, *batch, cos, sin, q=q), kc, vc]

    parts = lambda t: (t[:, H:2 * H], t[:, 2 * H:], t[:, :H])
    want = run(*(p.contiguous() for p in parts(x)))
    assert all(torch.equal(a, b) for a, b in zip(run(*parts(x)), want))
    odd = torch.empty(x.numel() + 3, device=DEV, dtype=F16)[3:].view_as(x).copy_(x)
    got = run(*parts(odd))
    assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))
    turned = x.permute(0, 2, 1).contiguous().permute(0, 2, 1)
    assert all(torch.equal(a, b) for a, b in zip(run(*parts(turned)), want))
    wide = torch.zeros((n, 4, 3 * H, D), device=DEV, dtype=F16)
    wide[:, 1] = x
    assert all(torch.equal(a, b) for a, b in zip(run(*parts(wide[:, 1])), want))


def test_empty(pkg):
    kc, vc = pkg.fp4_cache(3, 2, 16, 32, 32, device=DEV)
    batch = _dev(*(torch.tensor(t, dtype=I32) for t in ([[0, 1]], [0, 0], [9])))
    k = torch.empty((0, 2, 32), dtype=F16, device=DEV)
    assert pkg.kv_append_fp4(k, k, kc, vc, *batch, q=k).shape == (0, 2, 32)
    assert pkg.kv_read_fp4(kc, vc, *batch, 0)[0].shape == (0, 2, 32)
    k = torch.ones((4, 2, 32), dtype=F16, device=DEV)  # tokens of no sequence
    pkg.kv_append_fp4(k, k, kc, vc, *batch)
    none = [torch.empty((0, 4), dtype=I32, device=DEV), torch.zeros(1, dtype=I32, device=DEV), torch.empty(0, dtype=I32, device=DEV)]
    pkg.kv_append_fp4(k, k, kc, vc, *none)
    assert not kc.any() and not vc.any()


def test_captured_and_on_another_stream(pkg):
    """A captured append follows lengths and tables that change; a stream of its own."""
    H, D, page = 2, 128, 16
    x = torch.randn((3, 4 * H, D), device=DEV).half()
    kc, vc = pkg.fp4_cache(9, H, page, D, D, device=DEV)
    table = torch.arange(9, dtype=I32, device=DEV).view(3, 3)
    starts, lens = torch.arange(4, dtype=I32, device=DEV), torch.tensor([1, 15, 30], dtype=I32, device=DEV)
    cos, sin = (t.to(DEV) for t in R64.tables(48, D))
    step = lambda a, b: pkg.kv_append_fp4(x[:, 2 * H:3 * H], x[:, 3 * H:], a, b, table, starts, lens, cos, sin, q=x[:, :2 * H], norm=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kc, vc)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = step(kc, vc)
    for i in range(6):
        x.normal_()
        lens += 1
        want = [kc.clone(), vc.clone()]
        wq = step(*want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1]) and torch.equal(q, wq)
