"""paged_sdpa against the definition in 64 bits.

Bounds (u = 2^-24).  A score is a sum of D <= 128 products in fp32: off by at
most 128 u of the sum of their sizes, times the scale; its place in the exponent is
rounded once more (4 u of its size and of one).  So a weight is off by a
relative delta = 128 u A + 4 u (1 + |s|), A and |s| the largest of a row, and
so are the sum of the weights and, twice (weight and sum), the weighted mean of |v|.
Sums of n weights or products add n u.  fp16 rounds the weights in the product
with v to half precision (2^-11 of each, 2^-25 for the smallest, whose number
is n) and the result once more."""
import ctypes

import pytest
import torch

import _heads as R64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
NAN, INF = float("nan"), float("inf")


def _dev(*ts):
    return [t.to(DEV) for t in ts]


class Batch:
    """Sequences over a cache whose pages lie in no order; every row of the
    cache that holds no token is NaN, columns behind the last page are no pages."""

    def __init__(self, T, new, lens, H_q, H_kv, D, D_v, page, behind=0, spread=1.0, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.T, self.new, self.lens, self.page, self.G = T, new, lens, page, H_q // H_kv
        used = [-(-l // page) for l in lens]
        width = max(max(used), 1)
        self.pages = sum(used) + 2
        order = torch.randperm(self.pages, generator=g).tolist()
        table, at = [], 0
        for u in used:
            table.append(order[at:at + u] + [-9] * (width - u))
            at += u
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32)
        self.table, self.starts, self.kv_lens = i32(table), i32(starts), i32(lens)
        n = starts[-1] + behind
        self.q = (torch.randn((n, H_q, D), generator=g) * spread).to(T)
        self.k = [torch.randn((l, H_kv, D), generator=g).to(T) for l in lens]
        self.v = [torch.randn((l, H_kv, D_v), generator=g).to(T) for l in lens]
        self.scale = D ** -0.5
        self.shape = (n, H_q, H_kv, D, D_v)

    def caches(self):
        _, _, H_kv, D, D_v = self.shape
        out = []
        for rows, d in ((self.k, D), (self.v, D_v)):
            c = torch.full((self.pages, H_kv, self.page, d), NAN, dtype=self.T)
            for s, x in enumerate(rows):
                for j in range(0, len(x), self.page):
                    part = x[j:j + self.page]
                    c[int(self.table[s, j // self.page]), :, :len(part)] = part.transpose(0, 1)
            out.append(c)
        return out

    def args(self):
        return _dev(self.q, *self.caches(), self.table, self.starts, self.kv_lens)

    def reference(self, causal):
        """o, stats and their bounds; NaN in rows of no sequence."""
        n, H_q, H_kv, D, D_v = self.shape
        u, G = R64.U32, self.G
        rel, tiny = R64.half_step(self.T)
        o, bo = (torch.full((n, H_q, D_v), NAN, dtype=torch.float64) for _ in range(2))
        st, bs = (torch.full((n, H_q), NAN, dtype=torch.float64) for _ in range(2))
        for s, (m, l) in enumerate(zip(self.new, self.lens)):
            for h in range(H_q if m else 0):
                rows = slice(int(self.starts[s]), int(self.starts[s]) + m)
                q, k, v = self.q[rows, h].double(), self.k[s][:, h // G].double(), self.v[s][:, h // G].double()
                z, size = q @ k.T * self.scale, q.abs() @ k.abs().T * abs(self.scale)
                seen = torch.ones((m, l), dtype=torch.bool)
                if causal:
                    seen = torch.arange(l)[None] <= torch.arange(m)[:, None] + l - m
                z = z.masked_fill(~seen, -INF)
                lse = torch.logsumexp(z, -1)
                w = torch.exp(z - lse[:, None]).nan_to_num(0)
                mean, mean_abs = w @ v, w @ v.abs()
                top = size.masked_fill(~seen, 0).amax(-1) if l else torch.zeros(m, dtype=torch.float64)
                delta = 128 * u * top + 4 * u * (1 + top)
                count = seen.sum(-1)
                o[rows, h], st[rows, h] = mean, lse
                bs[rows, h] = delta + (count + 8) * u + 2 * u * lse.abs().nan_to_num(0, posinf=0)
                b = (2 * delta + 2 * (count + 8) * u)[:, None] * mean_abs + rel * mean.abs() + tiny
                if self.T == F16:
                    vmax = v.abs().amax(0) if l else torch.zeros(D_v, dtype=torch.float64)
                    b = b + 2 ** -11 * mean_abs + count[:, None] * 2.0 ** -25 * vmax
                bo[rows, h] = b
        return o, st, bo, bs


def check(out, ref, live=slice(None)):
    o, stats = (t.double().cpu()[live] for t in out)
    ro, rs, bo, bs = (t[live] for t in ref)
    empty = torch.isinf(rs)
    assert torch.equal(torch.isneginf(stats), empty)
    assert R64.worst(stats.masked_fill(empty, 0), rs.masked_fill(empty, 0), bs) <= 1
    assert R64.worst(o, ro, bo) <= 1


# dtype, new, lens, H_q, H_kv, D_qk, D_v, page, causal, tokens behind the last, spread of the queries
CASES = [
    (F16, (1,), (1,), 1, 1, 64, 64, 16, True, 0, 1),
    (F16, (1, 1, 1, 1), (1, 33, 250, 64), 8, 8, 128, 128, 16, True, 0, 3),
    (F16, (1, 1, 0, 1), (700, 5, 90, 1300), 16, 2, 128, 128, 32, True, 2, 3),     # a sequence without tokens
    (F16, (3, 1, 2), (3, 17, 1111), 12, 4, 64, 64, 16, True, 0, 3),               # short drafts
    (F16, (1, 2, 40), (0, 1, 20), 4, 2, 64, 64, 16, True, 0, 3),                  # rows that see nothing
    (F16, (65, 1, 33), (200, 90, 33), 6, 2, 80, 96, 16, True, 1, 3),              # mixed, widths between
    (F16, (130, 257), (130, 700), 4, 4, 128, 32, 64, True, 0, 3),
    (F16, (129, 5), (300, 61), 8, 1, 32, 128, 128, True, 0, 3),                   # one key head
    (F16, (40, 150), (90, 333), 6, 3, 64, 64, 16, False, 0, 3),                   # no mask
    (F16, (300,), (3000,), 8, 2, 128, 128, 256, True, 0, 3),                      # a chunk of a long sequence
    (F16, (1,), (6000,), 2, 1, 128, 128, 16, True, 0, 3),                         # many parts
    (F16, (1,) * 70, tuple(range(1, 1400, 20)), 4, 1, 64, 64, 16, True, 0, 3),    # more sequences than lanes
    (F16, (2, 70) * 40, tuple(range(70, 870, 10)), 4, 1, 32, 32, 16, True, 0, 3),
    (F16, (7, 200), (50, 400), 2, 1, 8, 16, 16, True, 0, 2),                      # a quarter of a tile's width
    (F16, (90,), (90,), 5, 1, 40, 72, 32, True, 0, 3),
    (F16, (1, 2, 1), (777, 40, 300), 6, 2, 96, 80, 16, True, 0, 3),               # between the widths of tiles
    (F16, (200, 40), (500, 40), 4, 2, 88, 96, 64, True, 0, 3),
    (F16, (140,), (300,), 2, 1, 96, 128, 16, False, 0, 3),
    (F32, (1, 1), (900, 33), 6, 2, 96, 96, 32, True, 0, 3),
    (F32, (150, 33), (400, 100), 4, 2, 96, 96, 16, True, 0, 3),
    (F32, (140,), (300,), 2, 1, 128, 92, 16, True, 0, 3),
    (F32, (140,), (300,), 2, 1, 84, 24, 16, True, 0, 3),
    (F32, (1,), (1,), 1, 1, 64, 64, 16, True, 0, 1),
    (F32, (1, 1, 3), (300, 77, 1500), 8, 2, 128, 128, 16, True, 1, 3),
    (F32, (130, 1, 20), (400, 1111, 20), 6, 3, 64, 32, 64, True, 0, 3),
    (F32, (70, 3), (33, 0), 4, 1, 32, 128, 32, True, 0, 3),                       # rows that see nothing
    (F32, (33,), (200,), 2, 2, 36, 68, 16, False, 0, 3),
    (F32, (300, 140), (1000, 140), 4, 2, 128, 128, 128, True, 0, 3),
    (F32, (2, 150), (30, 600), 2, 1, 4, 12, 16, True, 0, 2),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c)[:80])
def test_against_definition(pkg, case):
    T, new, lens, H_q, H_kv, D, D_v, page, causal, behind, spread = case
    b = Batch(T, new, lens, H_q, H_kv, D, D_v, page, behind, spread)
    ref = b.reference(causal)
    live = slice(0, sum(new))
    args = b.args()
    kw = dict(scale=b.scale, causal_mask=causal)
    first = pkg.paged_sdpa(*args, **kw)
    check(first, ref, live)
    again = pkg.paged_sdpa(*args, **kw)
    assert torch.equal(first[0][live], again[0][live]) and torch.equal(first[1][live], again[1][live])
    # hints, right and wrong, choose kernels only
    for hint in (max(new), 1):
        check(pkg.paged_sdpa(*args, max_q_len=hint, **kw), ref, live)
    # without a workspace nothing is divided; rows behind the last sequence stay
    o = torch.full_like(first[0], 7)
    stats = torch.full_like(first[1], 7)
    n, width, pages = len(b.q), b.table.shape[1], b.pages
    rc = pkg.library().sdpa_hip_paged_fwd(
        int(T == F16), args[0].data_ptr(), None, args[1].data_ptr(), args[2].data_ptr(), o.data_ptr(), None,
        stats.data_ptr(), args[3].data_ptr(), width, args[4].data_ptr(), args[5].data_ptr(), None, 0, len(new), n, width,
        pages, page, H_q, H_kv, D, D_v, 0, b.scale, int(causal), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    check((o, stats), ref, live)
    assert bool((o[sum(new):] == 7).all()) and bool((stats[sum(new):] == 7).all())


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_scales(pkg, T, scale):
    b = Batch(T, (5, 140), (40, 300), 4, 2, 64, 64, 16)
    b.scale = scale
    check(pkg.paged_sdpa(*b.args(), scale=scale), b.reference(True))


@pytest.mark.parametrize("T", [F16, F32])
def test_strided_queries(pkg, T):
    """q as part of a projection's output, misaligned, and with features apart."""
    b = Batch(T, (3, 90), (30, 200), 4, 2, 64, 64, 16)
    q, *rest = b.args()
    want = pkg.paged_sdpa(q, *rest, scale=b.scale)
    wide = torch.randn((len(q), 9, 64), device=DEV).to(T)
    wide[:, 2:6] = q
    odd = torch.empty((q.numel() + 1,), device=DEV, dtype=T)[1:].view(q.shape).copy_(q)
    apart = q.transpose(1, 2).contiguous().transpose(1, 2)
    for x in (wide[:, 2:6], odd, apart):
        got = pkg.paged_sdpa(x, *rest, scale=b.scale)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("new,lens,page", [((60, 4), (100, 37), 16), ((300, 1), (700, 333), 64)])
def test_masked_places_have_no_influence(pkg, T, new, lens, page):
    """Infinite and NaN keys and values behind a row's last key leave it alone;
    an infinite value among its keys makes its feature infinite, a NaN one NaN."""
    b = Batch(T, new, lens, 4, 2, 64, 64, page)
    ref = b.reference(True)
    clean = pkg.paged_sdpa(*b.args(), scale=b.scale)
    check(clean, ref)
    m, l = new[0], lens[0]
    at = m // 2  # token `at` of sequence 0 is key j
    j = l - m + at
    b.v[0][j, 0, 5], b.v[0][j + 1, 0, 9] = INF, NAN
    b.k[0][j + 2, 1] = NAN
    b.k[0][j + 3, 1, 3] = INF
    o, stats = pkg.paged_sdpa(*b.args(), scale=b.scale)
    check((o[:at], stats[:at]), [t[:at] for t in ref])
    check((o[m:], stats[m:]), [t[m:] for t in ref])
    o, stats = o.cpu(), stats.cpu()
    assert bool((o[at:m, :2, 5] == INF).all())
    assert bool(torch.isnan(o[at + 1:m, :2, 9]).all()) and not torch.isnan(o[at, :2]).any()
    assert bool(torch.isnan(o[at + 2:m, 2:]).all()) and not torch.isnan(o[at:at + 2, 2:]).any()
    # the other features of rows that met the values are right
    others = [f for f in range(64) if f not in (5, 9)]
    check((o[at:m, :2][..., others], stats[at:m, :2]),
          [ref[0][at:m, :2][..., others], ref[1][at:m, :2], ref[2][at:m, :2][..., others], ref[3][at:m, :2]])


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("new,lens", [((3,), (300,)), ((150,), (400,))])
def test_infinite_keys_and_queries(pkg, T, new, lens):
    """A score of -inf weighs nothing, one of +inf or NaN makes its row NaN, and
    only rows that see it."""
    b = Batch(T, new, lens, 2, 1, 64, 64, 16)
    m, l = new[0], lens[0]
    b.q = b.q.abs() + T.itemsize / 8  # every product with a key of one sign has its sign
    b.k[0][7, 0, 11] = -INF            # seen by all
    ref = b.reference(True)
    out = pkg.paged_sdpa(*b.args(), scale=b.scale)
    # (the bound's sum of sizes is infinite for that key: it has no share in any sum)
    c = Batch(T, new, lens, 2, 1, 64, 64, 16)
    c.q, c.k, c.v = b.q, [b.k[0].clone()], b.v
    c.k[0][7] = 0
    bounds = c.reference(True)[2:]
    check(out, [ref[0], ref[1], bounds[0], bounds[1]])
    b.k[0][l - 2, 0, 3] = INF          # seen by the last two tokens
    o, stats = pkg.paged_sdpa(*b.args(), scale=b.scale)
    assert bool(torch.isnan(o[m - 2:]).all()) and bool(torch.isnan(stats[m - 2:]).all())
    check((o[:m - 2], stats[:m - 2]), [ref[0][:m - 2], ref[1][:m - 2], bounds[0][:m - 2], bounds[1][:m - 2]])
    b.q[0, 1, 5] = NAN
    o, _ = pkg.paged_sdpa(*b.args(), scale=b.scale)
    assert bool(torch.isnan(o[0, 1]).all()) and not torch.isnan(o[0, 0]).any()


@pytest.mark.parametrize("T", [F16, F32])
def test_pages_that_are_none(pkg, T):
    """A sequence with a missing page (past the cache, negative, or more tokens
    than columns) is NaN where rows may see it; the others are right."""
    new, lens = (2, 40, 3, 150), (60, 200, 33, 400)
    b = Batch(T, new, lens, 4, 2, 64, 64, 16)
    ref = b.reference(True)
    q, kc, vc, table, starts, kv_lens = b.args()
    for s, change in ((0, lambda t, l: t[0].__setitem__(0, b.pages)), (1, lambda t, l: t[1].__setitem__(3, -1)),
                      (3, lambda t, l: l.__setitem__(3, 16 * t.shape[1] + 1)),
                      (2, lambda t, l: t[2].__setitem__(1, 2 ** 31 - 1))):
        t, l = table.clone(), kv_lens.clone()
        change(t, l)
        o, stats = pkg.paged_sdpa(q, kc, vc, t, starts, l, scale=b.scale)
        rows = slice(int(starts[s]), int(starts[s + 1]))
        assert bool(torch.isnan(o[rows]).all()) and bool(torch.isnan(stats[rows]).all())
        keep = torch.ones(len(q), dtype=torch.bool)
        keep[rows] = False
        check((o[keep.to(DEV)], stats[keep.to(DEV)]), [x[keep] for x in ref])


def test_ranges_that_are_none(pkg):
    """Sequences whose range of tokens is not one are left out; no pages at all."""
    b = Batch(F16, (2, 3), (20, 30), 4, 2, 64, 64, 16)
    q, kc, vc, table, starts, kv_lens = b.args()
    out = (torch.full((5, 4, 64), 7.0, device=DEV, dtype=F16), torch.full((5, 4), 7.0, device=DEV))
    bad = torch.tensor([-2, 9, 3], dtype=torch.int32, device=DEV)
    pkg.paged_sdpa(q, kc, vc, table, bad, kv_lens, scale=b.scale, out=out)
    assert bool((out[0] == 7).all()) and bool((out[1] == 7).all())
    o, stats = pkg.paged_sdpa(q, kc[:0], vc[:0], table, starts, kv_lens, scale=b.scale)
    assert bool(torch.isnan(o).all())
    o, stats = pkg.paged_sdpa(q, kc[:0], vc[:0], table, starts, torch.zeros_like(kv_lens), scale=b.scale)
    assert not o.any() and bool(torch.isneginf(stats).all())
    o, stats = pkg.paged_sdpa(q[:0], kc, vc, table, torch.zeros_like(starts), kv_lens, scale=b.scale)
    assert o.shape == (0, 4, 64)


@pytest.mark.parametrize("T", [F16, F32])
def test_cache_past_32_bits(pkg, T):
    """Pages beyond 2^32 bytes of the cache."""
    H, D, page = 2, 64, 256
    pages = 2 ** 32 // (H * D * page * T.itemsize) + 3
    k = torch.zeros((pages, H, page, D), device=DEV, dtype=T)
    v = torch.zeros((pages, H, page, D), device=DEV, dtype=T)
    b = Batch(T, (1, 70), (300, 500), 4, H, D, D, page)
    ref = b.reference(True)
    q, kc, vc, table, starts, lens = b.args()
    far = pages - b.pages
    k[far:], v[far:] = kc, vc
    check(pkg.paged_sdpa(q, k, v, table + far, starts, lens, scale=b.scale), ref)


def test_captured_steps_share_memory(pkg):
    """Two captured calls, replayed in turn on their own streams with lengths that
    grow between replays and eager work in between."""
    b = Batch(F16, (1, 1, 1), (100, 900, 31), 8, 2, 128, 128, 16, spread=2)
    q, kc, vc, table, starts, lens = b.args()
    kc, vc = kc.nan_to_num(0.25), vc.nan_to_num(0.5)  # rows that later lengths reach
    lens -= 20
    run = lambda: pkg.paged_sdpa(q, kc, vc, table, starts, lens, scale=b.scale, max_q_len=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    for i in range(5):
        want = [t.clone() for t in run()]
        for g, out in zip(graphs, outs):
            out[0].zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        with torch.cuda.stream(side):
            other = run()
        side.synchronize()
        assert torch.equal(other[0], want[0])
        lens += 4


@pytest.mark.parametrize("T,tol", [(F16, 2 ** -7), (F32, 2 ** -16)])
def test_serving_matches_the_dense_path(pkg, T, tol):
    """A sequence taken in chunks and single tokens through kv_append and
    paged_sdpa, beside another, against qk_norm_rope and sdpa on all of it at
    once: the same model, so the same outputs, up to roundings of normed rows near 1
    to T (2^-11 each for q, k, the weights, v and o, at most 16 steps of 2^-11
    together in fp16; fp32 has 2^-24 and sums of 200 keys)."""
    L, H_q, H_kv, D, page = 200, 4, 2, 64, 16
    g = torch.Generator().manual_seed(4)
    qkv = [torch.randn((L, H_q + 2 * H_kv, D), generator=g).to(T).to(DEV) for _ in range(2)]
    w = [(1 + 0.2 * torch.randn((D,), generator=g)).to(DEV) for _ in range(2)]
    cos, sin = _dev(*R64.tables(L, D))
    dense = []
    for x in qkv:
        q, k = pkg.qk_norm_rope(x[None, :, :H_q], x[None, :, H_q:H_q + H_kv], cos, sin, *w)
        k, v = (t.repeat_interleave(H_q // H_kv, 0) for t in (k, x[:, H_q + H_kv:].transpose(0, 1).contiguous()))
        dense.append(pkg.sdpa(q, k, v, scale=D ** -0.5, causal_mask=True)[0].transpose(0, 1))
    kc, vc = (torch.full((2 * L // page + 2, H_kv, page, D), NAN, device=DEV, dtype=T) for _ in range(2))
    width = -(-L // page)
    table = torch.randperm(2 * width, generator=g).to(torch.int32).view(2, width).to(DEV)
    done = [0, 0]
    for step in [(70, 1), (1, 33), (64, 1), (1, 1), (40, 100), (1, 1), (1, 40), (22, 23)]:
        x = torch.cat([qkv[s][done[s]:done[s] + n] for s, n in enumerate(step)])
        done = [d + n for d, n in zip(done, step)]
        starts, lens = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, step[0], sum(step)], done))
        q = pkg.kv_append(x[:, H_q:H_q + H_kv], x[:, H_q + H_kv:], kc, vc, table, starts, lens, cos, sin, q=x[:, :H_q],
                          q_weight=w[0], k_weight=w[1], norm=True)
        o, _ = pkg.paged_sdpa(q, kc, vc, table, starts, lens, scale=D ** -0.5, max_q_len=max(step))
        for s, n in enumerate(step):
            got, want = o[sum(step[:s]):sum(step[:s]) + n], dense[s][done[s] - n:done[s]]
            assert float((got.double() - want.double()).abs().max()) <= tol
    assert done == [L, L]


def test_many_shared_heads(pkg):
    """64 query heads on one key head, 33 tokens a sequence and one."""
    for T in (F16, F32):
        for new, lens in (((1, 1), (300, 77)), ((33, 1), (200, 900))):
            b = Batch(T, new, lens, 64, 1, 64, 64, 16, spread=2)
            check(pkg.paged_sdpa(*b.args(), scale=b.scale), b.reference(True))


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("new", [(1, 2), (90, 2)])
def test_layouts_of_the_batch(pkg, T, new):
    """A table that is part of a wider one, a first sequence that does not begin at
    the first token, results that are part of a wider tensor (C entry)."""
    b = Batch(T, new, (150, 60), 4, 2, 64, 64, 16, behind=3)
    ref = b.reference(True)
    q, kc, vc, table, starts, lens = b.args()
    wide = torch.full((2, table.shape[1] + 5), -3, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + table.shape[1]] = table
    q = torch.cat([q[-2:], q[:-2]])
    starts = starts + 2
    n, m = len(q), sum(new)
    out = (torch.full((n, 4, 64), 7.0, device=DEV, dtype=T), torch.full((n, 4), 7.0, device=DEV))
    view = wide[:, 2:2 + table.shape[1]]
    pkg.paged_sdpa(q, kc, vc, view, starts, lens, scale=b.scale, out=out)
    check((out[0][2:2 + m], out[1][2:2 + m]), [t[:m] for t in ref])
    for t in out:
        assert bool((t[:2] == 7).all()) and bool((t[2 + m:] == 7).all())
    big = torch.full((n, 6, 80), 7.0, device=DEV, dtype=T)
    strides = (ctypes.c_int64 * 2)(big.stride(0), big.stride(1))
    o, stats = big[:, 1:5, 8:72], torch.empty((n, 4), device=DEV)
    rc = pkg.library().sdpa_hip_paged_fwd(
        int(T == F16), q.data_ptr(), None, kc.data_ptr(), vc.data_ptr(), o.data_ptr(), strides, stats.data_ptr(),
        view.data_ptr(), view.stride(0), starts.data_ptr(), lens.data_ptr(), None, 0, 2, n, view.shape[1], b.pages, 16, 4, 2,
        64, 64, max(new), b.scale, 1, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    check((o[2:2 + m], stats[2:2 + m]), [t[:m] for t in ref])
    o[2:2 + m] = 7
    assert bool((big == 7).all())


def test_calls_at_once(pkg):
    """Calls of several batches in flight together on streams of their own."""
    batches = [Batch(T, new, lens, 8, 2, 128, 128, 16, seed=i) for i, (T, new, lens) in enumerate((
        (F16, (1, 1, 1), (900, 40, 3000)), (F16, (200, 3), (700, 90)), (F32, (1, 2), (1500, 33)), (F32, (140,), (600,))))]
    refs, args = [b.reference(True) for b in batches], [b.args() for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    outs = []
    for _ in range(4):
        for s, a, b in zip(streams, args, batches):
            with torch.cuda.stream(s):
                outs.append(pkg.paged_sdpa(*a, scale=b.scale))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        check(out, refs[i % 4])


def test_lengths_of_zero(pkg):
    """No tokens, no keys, no sequences."""
    b = Batch(F16, (1, 1, 1), (0, 0, 5), 4, 2, 64, 64, 16)
    check(pkg.paged_sdpa(*b.args(), scale=b.scale), b.reference(True))
    q, kc, vc, table, starts, lens = b.args()
    out = (torch.full((3, 4, 64), 7.0, device=DEV, dtype=F16), torch.full((3, 4), 7.0, device=DEV))
    pkg.paged_sdpa(q, kc, vc, table[:0], starts[:1], lens[:0], scale=b.scale, out=out)
    assert bool((out[0] == 7).all()) and bool((out[1] == 7).all())
    o, stats = pkg.paged_sdpa(q, kc, vc, table[:, :0], starts, lens * 0, scale=b.scale)
    assert not o.any() and bool(torch.isneginf(stats).all())


@pytest.mark.parametrize("case", [
    (F16, (16,), (50000,), 8, 1, 64, 64, 16, 0),      # one tile of many parts
    (F16, (40, 1), (30000, 100), 8, 2, 96, 128, 64, 1),
    (F16, (600,), (9000,), 8, 4, 32, 64, 128, 0),
    (F32, (20,), (40000,), 8, 1, 64, 64, 64, 0),
    (F32, (300, 3), (20000, 70), 4, 2, 36, 128, 16, 2),
], ids=str)
def test_tiles_of_many_parts(pkg, case):
    T, new, lens, H_q, H_kv, D, D_v, page, behind = case
    b = Batch(T, new, lens, H_q, H_kv, D, D_v, page, behind, 3)
    args = b.args()
    out = pkg.paged_sdpa(*args, scale=b.scale)
    check(out, b.reference(True), slice(0, sum(new)))
    again = pkg.paged_sdpa(*args, scale=b.scale)
    assert all(torch.equal(x[:sum(new)], y[:sum(new)]) for x, y in zip(out, again))


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("new,lens,heads,D,page", [
    ((4,), (5000,), 4, 128, 16), ((1, 3), (2000, 2600), 4, 96, 32), ((90,), (6000,), 4, 128, 64), ((200, 30), (900, 3000), 4, 96, 16)])
def test_infinite_values_of_divided_tiles(pkg, T, new, lens, heads, D, page):
    """Infinities of both signs among a row's keys, in keys of other parts than the
    mask's edge, and NaN behind it."""
    b = Batch(T, new, lens, heads, 1, D, D, page)
    ref = b.reference(True)
    m, l = new[-1], lens[-1]
    first = sum(new) - m
    at = m // 2
    j = l - m + at                       # the key of token `at`
    v = b.v[-1]
    v[3, 0, 1], v[l // 3, 0, 2] = -INF, INF       # seen by all
    v[5, 0, 7], v[j, 0, 7] = INF, -INF            # of both signs from token `at` on
    v[j, 0, D - 1] = -INF
    if at + 1 < m:
        v[j + 1, 0, 11] = NAN
    o, stats = (t.cpu() for t in pkg.paged_sdpa(*b.args(), scale=b.scale))
    seq = o[first:]
    assert bool((seq[..., 1] == -INF).all()) and bool((seq[..., 2] == INF).all())
    assert bool((seq[:at, :, 7] == INF).all()) and bool(torch.isnan(seq[at:, :, 7]).all())
    assert bool((seq[at:, :, D - 1] == -INF).all()) and bool(torch.isfinite(seq[:at, :, D - 1]).all())
    assert bool(torch.isnan(seq[at + 1:, :, 11]).all()) and bool(torch.isfinite(seq[:at + 1, :, 11]).all())
    others = [f for f in range(D) if f not in (1, 2, 7, 11, D - 1)]
    check((o[..., others], stats), [ref[0][..., others], ref[1], ref[2][..., others], ref[3]])


def test_out_that_shares_memory(pkg):
    b = Batch(F16, (3, 1), (40, 9), 4, 2, 64, 64, 16)
    q, kc, vc, *batch = b.args()
    n = len(q)
    room = torch.zeros((3 * n, 4, 64), device=DEV, dtype=F16)
    stats = torch.empty((n, 4), device=DEV)
    x = room[:n].copy_(q)
    new = lambda o, s=stats: pkg.paged_sdpa(x, kc, vc, *batch, scale=b.scale, out=(o, s))
    for bad in (x, room[1:n + 1]):
        with pytest.raises(pkg.InvalidArgumentError, match="share memory with q"):
            new(bad)
    with pytest.raises(pkg.InvalidArgumentError, match="share memory with v_cache"):
        new(vc.view(-1, 64)[:4 * n].view(n, 4, 64))
    o = room[n:2 * n]
    with pytest.raises(pkg.InvalidArgumentError, match="tensors of out"):
        new(o, o.view(torch.float32).view(-1)[:4 * n].view(n, 4))
    check(new(o), b.reference(True))
