"""paged_sdpa_fp4 against the definition in 64 bits over the values that the cache holds.

Bounds (u = 2^-24) as in test_paged_gpu.py, but for: fp32 queries enter as three parts,
so that a score is a sum of up to 384 products; weights enter as two fp16 parts (or, in tiles of
128 rows of fp16 calls, one unless few keys carry a row: 2^-11 of each), off by 2^-22 of each, and
by 2^-25 where the largest of the row is at least 2^7: 2^-32 of it."""
import ctypes

import pytest
import torch

import _fp4 as F
import _heads as R64
from test_paged_gpu import Batch, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
I32 = torch.int32
NAN, INF = float("nan"), float("inf")


class Fp4Batch(Batch):
    """The same over a cache in 4 bits; rows that hold no token have NaN scales and any codes."""

    def __init__(self, T, new, lens, H_q, H_kv, D, D_v, page, behind=0, spread=1.0, seed=0):
        super().__init__(T, new, lens, H_q, H_kv, D, D_v, page, behind, spread, seed)
        self.codes = []
        for rows in (self.k, self.v):
            c = [F.encode(x) for x in rows]
            self.codes.append(c)
            rows[:] = [F.decode(*x) for x in c]

    def caches(self):
        _, _, H_kv, D, D_v = self.shape
        g = torch.Generator().manual_seed(7)
        out = []
        for rows, d, is_v in ((self.codes[0], D, False), (self.codes[1], D_v, True)):
            c = torch.randint(0, 16, (self.pages, H_kv, self.page, d), generator=g).byte()
            s = torch.full((self.pages, H_kv, self.page, d // 32), 0x7F, dtype=torch.uint8)
            for i, (codes, scales) in enumerate(rows):
                for j in range(0, len(codes), self.page):
                    n, pg = len(codes[j:j + self.page]), int(self.table[i, j // self.page])
                    c[pg, :, :n] = codes[j:j + self.page].transpose(0, 1)
                    s[pg, :, :n] = scales[j:j + self.page].transpose(0, 1)
            out.append(F.pack(c, s, is_v))
        return out

    def reference(self, causal):
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
                delta = (128 if self.T == F16 else 384) * u * top + 4 * u * (1 + top)
                count = seen.sum(-1)
                vmax = v.abs().amax(0) if l else torch.zeros(D_v, dtype=torch.float64)
                o[rows, h], st[rows, h] = mean, lse
                bs[rows, h] = delta + (count + 8) * u + 2 * u * lse.abs().nan_to_num(0, posinf=0)
                b = (2 * delta + 2 * (count + 8) * u + 4 * u)[:, None] * mean_abs + rel * mean.abs() + tiny
                if self.T == F16:
                    b = b + 2.0 ** -11 * mean_abs
                bo[rows, h] = b + count[:, None] * 2.0 ** -32 * vmax
        return o, st, bo, bs


# dtype, new, lens, H_q, H_kv, D_qk, D_v, page, causal, tokens behind the last, spread of the queries
CASES = [
    (F16, (1,), (1,), 1, 1, 64, 64, 16, True, 0, 1),
    (F16, (1, 1, 1, 1), (1, 33, 250, 64), 8, 8, 128, 128, 16, True, 0, 3),
    (F16, (1, 1, 0, 1), (700, 5, 90, 1300), 16, 2, 128, 128, 32, True, 2, 3),     # a sequence without tokens
    (F16, (3, 1, 2), (3, 17, 1111), 12, 4, 64, 64, 16, True, 0, 3),               # short drafts
    (F16, (1, 2, 40), (0, 1, 20), 4, 2, 64, 64, 16, True, 0, 3),                  # rows that see nothing
    (F16, (65, 1, 33), (200, 90, 33), 6, 2, 96, 96, 16, True, 1, 3),              # three words a lane
    (F16, (130, 257), (130, 700), 4, 4, 128, 32, 64, True, 0, 3),
    (F16, (129, 5), (300, 61), 8, 1, 32, 128, 128, True, 0, 3),                   # one key head
    (F16, (40, 150), (90, 333), 6, 3, 64, 64, 16, False, 0, 3),                   # no mask
    (F16, (300,), (3000,), 8, 2, 128, 128, 256, True, 0, 3),                      # a chunk of a long sequence
    (F16, (1,), (6000,), 2, 1, 128, 128, 16, True, 0, 3),                         # many parts
    (F16, (1,) * 70, tuple(range(1, 1400, 20)), 4, 1, 64, 64, 16, True, 0, 3),    # more sequences than lanes
    (F16, (2, 70) * 40, tuple(range(70, 870, 10)), 4, 1, 32, 32, 16, True, 0, 3),
    (F16, (1, 2, 1), (777, 40, 300), 6, 2, 96, 32, 16, True, 0, 3),
    (F16, (200, 40), (500, 40), 4, 2, 32, 96, 64, True, 0, 3),
    (F16, (140,), (300,), 2, 1, 96, 128, 16, False, 0, 3),
    (F16, (1, 7), (900, 500), 20, 1, 64, 128, 32, True, 0, 3),                    # more heads than a tile's rows
    (F32, (1, 1), (900, 33), 6, 2, 96, 96, 32, True, 0, 3),
    (F32, (150, 33), (400, 100), 4, 2, 96, 96, 16, True, 0, 3),
    (F32, (140,), (300,), 2, 1, 128, 96, 16, True, 0, 3),
    (F32, (140,), (300,), 2, 1, 32, 32, 16, True, 0, 3),
    (F32, (1,), (1,), 1, 1, 64, 64, 16, True, 0, 1),
    (F32, (1, 1, 3), (300, 77, 1500), 8, 2, 128, 128, 16, True, 1, 3),
    (F32, (130, 1, 20), (400, 1111, 20), 6, 3, 64, 32, 64, True, 0, 3),
    (F32, (70, 3), (33, 0), 4, 1, 32, 128, 32, True, 0, 3),                       # rows that see nothing
    (F32, (33,), (200,), 2, 2, 64, 64, 16, False, 0, 3),
    (F32, (300, 140), (1000, 140), 4, 2, 128, 128, 128, True, 0, 3),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c)[:80])
def test_against_definition(pkg, case):
    T, new, lens, H_q, H_kv, D, D_v, page, causal, behind, spread = case
    b = Fp4Batch(T, new, lens, H_q, H_kv, D, D_v, page, behind, spread)
    ref = b.reference(causal)
    live = slice(0, sum(new))
    args = b.args()
    kw = dict(scale=b.scale, causal_mask=causal)
    first = pkg.paged_sdpa_fp4(*args, **kw)
    check(first, ref, live)
    again = pkg.paged_sdpa_fp4(*args, **kw)
    assert torch.equal(first[0][live], again[0][live]) and torch.equal(first[1][live], again[1][live])
    # hints, right and wrong, choose kernels only
    for hint in (max(new), 1):
        check(pkg.paged_sdpa_fp4(*args, max_q_len=hint, **kw), ref, live)
    # without a workspace nothing is divided; rows behind the last sequence stay
    n, width, pages = len(b.q), b.table.shape[1], b.pages
    for hint in (0, 1):
        o, stats = torch.full_like(first[0], 7), torch.full_like(first[1], 7)
        rc = pkg.library().sdpa_hip_paged_fwd_fp4(
            int(T == F16), args[0].data_ptr(), None, args[1].data_ptr(), args[2].data_ptr(), o.data_ptr(), None,
            stats.data_ptr(), args[3].data_ptr(), width, args[4].data_ptr(), args[5].data_ptr(), None, 0, len(new), n, width,
            pages, page, H_q, H_kv, D, D_v, hint, b.scale, int(causal), torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        check((o, stats), ref, live)
        assert bool((o[sum(new):] == 7).all()) and bool((stats[sum(new):] == 7).all())


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("hint", [None, 1])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_scales(pkg, T, scale, hint):
    b = Fp4Batch(T, (5, 140), (40, 300), 4, 2, 64, 64, 16)
    b.scale = scale
    check(pkg.paged_sdpa_fp4(*b.args(), scale=scale, max_q_len=hint), b.reference(True))


@pytest.mark.parametrize("size", [1e30, 2.0 ** 90, 1e-30, 2.0 ** -110, 1e-3])
@pytest.mark.parametrize("hint", [None, 1])
def test_large_and_small_queries(pkg, size, hint):
    """fp32 queries far from 1, with a scale that brings the scores back; rows of very different size in a tile."""
    b = Fp4Batch(F32, (3, 140), (90, 300), 4, 2, 64, 64, 16)
    b.q *= size
    b.q[::2] *= 0.25
    b.scale = 0.125 / size
    # (the sums of sizes in the bounds scale back too)
    check(pkg.paged_sdpa_fp4(*b.args(), scale=b.scale, max_q_len=hint), b.reference(True))


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("hint", [None, 1])
def test_strided_queries(pkg, T, hint):
    b = Fp4Batch(T, (3, 90), (30, 200), 4, 2, 64, 64, 16)
    q, *rest = b.args()
    kw = dict(scale=b.scale, max_q_len=hint)
    want = pkg.paged_sdpa_fp4(q, *rest, **kw)
    wide = torch.randn((len(q), 9, 64), device=DEV).to(T)
    wide[:, 2:6] = q
    odd = torch.empty((q.numel() + 1,), device=DEV, dtype=T)[1:].view(q.shape).copy_(q)
    apart = q.transpose(1, 2).contiguous().transpose(1, 2)
    for x in (wide[:, 2:6], odd, apart):
        got = pkg.paged_sdpa_fp4(x, *rest, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("hint", [None, 1])
@pytest.mark.parametrize("new,lens,page,D", [((60, 4), (100, 37), 16, 64), ((300, 1), (700, 333), 64, 128), ((9,), (40,), 16, 96)])
def test_masked_places_have_no_influence(pkg, T, new, lens, page, D, hint):
    """Groups of NaN among keys and values behind a row's last key leave it alone;
    one among its values makes the group's features NaN, one among its keys the row."""
    b = Fp4Batch(T, new, lens, 4, 2, D, D, page)
    ref = b.reference(True)
    kw = dict(scale=b.scale, max_q_len=hint)
    check(pkg.paged_sdpa_fp4(*b.args(), **kw), ref)
    m, l = new[0], lens[0]
    at = m // 2  # token `at` of sequence 0 is key j
    j = l - m + at
    b.codes[1][0][1][j, 0, 1] = 0x7F            # values of key j, features 32 .. 63
    b.codes[0][0][1][j + 2, 1, 0] = 0x7D        # keys of key j + 2
    o, stats = pkg.paged_sdpa_fp4(*b.args(), **kw)
    check((o[:at], stats[:at]), [t[:at] for t in ref])
    check((o[m:], stats[m:]), [t[m:] for t in ref])
    assert bool(torch.isnan(o[at:m, :2, 32:64]).all()) and not torch.isnan(o[at:m, :2, :32]).any()
    assert bool(torch.isnan(o[at + 2:m, 2:]).all()) and not torch.isnan(o[at:at + 2, 2:]).any()
    others = [f for f in range(D) if not 32 <= f < 64]
    o, stats = o.cpu(), stats.cpu()
    check((o[at:m, :2][..., others], stats[at:m, :2]),
          [ref[0][at:m, :2][..., others], ref[1][at:m, :2], ref[2][at:m, :2][..., others], ref[3][at:m, :2]])


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("hint", [None, 1])
def test_nan_queries(pkg, T, hint):
    b = Fp4Batch(T, (3, 140), (90, 300), 4, 2, 64, 64, 16)
    ref = b.reference(True)
    b.q[1, 2, 5], b.q[100, 0, 60] = NAN, NAN
    o, stats = pkg.paged_sdpa_fp4(*b.args(), scale=b.scale, max_q_len=hint)
    keep = torch.ones((143, 4), dtype=torch.bool)
    keep[1, 2] = keep[100, 0] = False
    assert bool(torch.isnan(o.cpu()[~keep]).all()) and bool(torch.isnan(stats.cpu()[~keep]).all())
    check((o.cpu()[keep], stats.cpu()[keep]), [t[keep] for t in ref])


@pytest.mark.parametrize("T", [F16, F32])
def test_extreme_values(pkg, T):
    """Values at the ends of the scales' range: the largest, and below the normal fp16 numbers."""
    for size in (50000.0, 3e-5, 2e-6):
        b = Fp4Batch(T, (1, 140), (90, 300), 4, 2, 64, 64, 16)
        for i in range(2):
            codes = F.encode(torch.randn((b.lens[i], 2, 64)).clamp(-1.2, 1.2) * size)
            b.codes[1][i] = codes
            b.v[i] = F.decode(*codes)
        b_o = b.reference(True)
        for hint in (None, 1):
            check(pkg.paged_sdpa_fp4(*b.args(), scale=b.scale, max_q_len=hint), b_o)


@pytest.mark.parametrize("T", [F16, F32])
@pytest.mark.parametrize("hint", [None, 1])
def test_pages_that_are_none(pkg, T, hint):
    new, lens = (2, 40, 3, 150), (60, 200, 33, 400)
    b = Fp4Batch(T, new, lens, 4, 2, 64, 64, 16)
    ref = b.reference(True)
    q, kc, vc, table, starts, kv_lens = b.args()
    for s, change in ((0, lambda t, l: t[0].__setitem__(0, b.pages)), (1, lambda t, l: t[1].__setitem__(3, -1)),
                      (3, lambda t, l: l.__setitem__(3, 16 * t.shape[1] + 1)),
                      (2, lambda t, l: t[2].__setitem__(1, 2 ** 31 - 1))):
        t, l = table.clone(), kv_lens.clone()
        change(t, l)
        o, stats = pkg.paged_sdpa_fp4(q, kc, vc, t, starts, l, scale=b.scale, max_q_len=hint)
        rows = slice(int(starts[s]), int(starts[s + 1]))
        assert bool(torch.isnan(o[rows]).all()) and bool(torch.isnan(stats[rows]).all())
        keep = torch.ones(len(q), dtype=torch.bool)
        keep[rows] = False
        check((o[keep.to(DEV)], stats[keep.to(DEV)]), [x[keep] for x in ref])


@pytest.mark.parametrize("hint", [None, 1])
def test_ranges_that_are_none(pkg, hint):
    b = Fp4Batch(F16, (2, 3), (20, 30), 4, 2, 64, 64, 16)
    q, kc, vc, table, starts, kv_lens = b.args()
    out = (torch.full((5, 4, 64), 7.0, device=DEV, dtype=F16), torch.full((5, 4), 7.0, device=DEV))
    bad = torch.tensor([-2, 9, 3], dtype=I32, device=DEV)
    pkg.paged_sdpa_fp4(q, kc, vc, table, bad, kv_lens, scale=b.scale, out=out, max_q_len=hint)
    assert bool((out[0] == 7).all()) and bool((out[1] == 7).all())
    o, stats = pkg.paged_sdpa_fp4(q, kc[:0], vc[:0], table, starts, kv_lens, scale=b.scale, max_q_len=hint)
    assert bool(torch.isnan(o).all())
    o, stats = pkg.paged_sdpa_fp4(q, kc, vc, table, starts, torch.zeros_like(kv_lens), scale=b.scale, max_q_len=hint)
    assert not o.any() and bool(torch.isneginf(stats).all())
    o, stats = pkg.paged_sdpa_fp4(q[:0], kc, vc, table, torch.zeros_like(starts), kv_lens, scale=b.scale, max_q_len=hint)
    assert o.shape == (0, 4, 64)


def test_cache_past_32_bits(pkg):
    """Pages beyond 2^32 bytes of the cache."""
    H, D, page = 2, 64, 256
    pages = 2 ** 32 // (H * D * page * 17 // 32) + 3
    k, v = pkg.fp4_cache(pages, H, page, D, D, device=DEV)
    b = Fp4Batch(F16, (1, 70), (300, 500), 4, H, D, D, page)
    ref = b.reference(True)
    q, kc, vc, table, starts, lens = b.args()
    far = pages - b.pages
    k[far:], v[far:] = kc, vc
    for hint in (None, 1):
        check(pkg.paged_sdpa_fp4(q, k, v, table + far, starts, lens, scale=b.scale, max_q_len=hint), ref)
    # tokens appended and read there
    x = torch.randn((71, H, D), generator=torch.Generator().manual_seed(2)).half()
    pkg.kv_append_fp4(x.to(DEV), x.to(DEV), k, v, table + far, starts, lens)
    want = F.decode(*F.encode(x))
    for t in pkg.kv_read_fp4(k, v, table + far, starts, lens, 71):
        assert torch.equal(t.double().cpu(), want)


@pytest.mark.parametrize("T,new,lens,D", [(F16, (16,), (50000,), 64), (F16, (40, 1), (30000, 100), 128), (F32, (20,), (40000,), 96),
                                          (F32, (1,), (60000,), 128), (F16, (300, 3), (20000, 70), 128)])
def test_tiles_of_many_parts(pkg, T, new, lens, D):
    b = Fp4Batch(T, new, lens, 8, 2, D, D, 64)
    ref = b.reference(True)
    for hint in (None, 1):
        check(pkg.paged_sdpa_fp4(*b.args(), scale=b.scale, max_q_len=hint), ref)


def test_few_keys_that_carry_a_row(pkg):
    """One key of weight one beside many of 2^-25.25, whose sum is a hundredth: none is lost."""
    D, l = 64, 400000
    for T, m in ((F16, 1), (F16, 40), (F32, 1), (F32, 40)):
        b = Fp4Batch(T, (m,), (64,), 2, 1, D, D, 64)
        q = torch.zeros((m, 2, D))
        q[..., 0] = 1
        x = torch.zeros((l, 1, D))
        x[:, 0, 0], x[5, 0, 0] = -6, 0
        v = torch.ones((l, 1, D))
        v[5] = 6
        pages = -(-l // 64)
        rows = [F.encode(t) for t in (x, v)]
        pad = pages * 64 - l
        caches = []
        for (c, s), is_v in zip(rows, (False, True)):
            c, s = (torch.cat((t, t[:1].expand(pad, -1, -1))) for t in (c, s))
            caches.append(F.pack(c.reshape(pages, 64, 1, D).transpose(1, 2).contiguous(),
                                 s.reshape(pages, 64, 1, D // 32).transpose(1, 2).contiguous(), is_v))
        vd = F.decode(*rows[1])[:, 0]
        scale = 17.5 / 6
        o, stats = pkg.paged_sdpa_fp4(q.to(T).to(DEV), *(c.to(DEV) for c in caches), torch.arange(pages, dtype=I32, device=DEV)[None],
                                      *(torch.tensor(t, dtype=I32, device=DEV) for t in ([0, m], [l])), scale=scale, causal_mask=False)
        w = torch.exp(torch.tensor(-17.5, dtype=torch.float64))
        want = (vd[5] + w * (l - 1) * vd[0]) / (1 + w * (l - 1))
        # weights of 2^-25.25, in two parts of 11 bits and above 2^-25 - 7 of the largest: a thousandth of
        # their share of a hundredth, the sums' rounding (2^-24 a step, 400000 / 16 of them at most) and o's
        assert float((o.double().cpu() - want).abs().max()) <= 6 * (1e-5 + 25000 * 2.0 ** -24) + 2.0 ** -10 * 6 * (T == F16)


def test_out_that_shares_memory(pkg):
    b = Fp4Batch(F16, (1, 2), (30, 40), 4, 2, 64, 64, 16)
    q, *rest = b.args()
    stats = torch.empty((3, 4), device=DEV)
    for o in (q, rest[0].view(-1)[:3 * 4 * 64 * 2].view(F16).view(3, 4, 64)):
        with pytest.raises(pkg.InvalidArgumentError, match="share memory"):
            pkg.paged_sdpa_fp4(q, *rest, out=(o, stats))
    o = torch.empty_like(q)
    got = pkg.paged_sdpa_fp4(q, *rest, scale=b.scale, out=(o, stats))
    assert got[0] is o and torch.equal(pkg.paged_sdpa_fp4(q, *rest, scale=b.scale)[0], o)


def test_captured_steps_share_memory(pkg):
    """Two captured calls, replayed in turn with lengths that grow between replays and eager work
    in between, on another stream too."""
    b = Fp4Batch(F16, (1, 1, 1), (100, 900, 31), 8, 2, 128, 128, 16, spread=2)
    q, kc, vc, table, starts, lens = b.args()
    lens -= 20
    run = lambda hint=1: pkg.paged_sdpa_fp4(q, kc, vc, table, starts, lens, scale=b.scale, max_q_len=hint)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(), run(None)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for hint in (1, 1, None):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(hint))
        graphs.append((g, hint))
    for i in range(5):
        for (g, hint), out in zip(graphs, outs):
            want = [t.clone() for t in run(hint)]
            out[0].zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        with torch.cuda.stream(side):
            other = run()
        torch.cuda.synchronize()
        assert torch.equal(other[0], outs[0][0])
        lens += 4


def test_serving_steps(pkg):
    """Reserve, append in 4 bits, attend: whole steps, the last ones as one captured graph, against attention in
    64 bits over what the cache says it holds."""
    N, H_q, H_kv, D, page, width = 3, 8, 2, 64, 16, 8
    g = torch.Generator().manual_seed(3)
    i32 = lambda x: torch.tensor(x, dtype=I32, device=DEV)
    table, lens = torch.full((N, width), -1, dtype=I32, device=DEV), i32([0] * N)
    free, count, new = torch.randperm(24, generator=g).int().to(DEV), i32([24]), i32([0] * N)
    kc, vc = (c.fill_(0xFF) for c in pkg.fp4_cache(24, H_kv, page, D, D, device=DEV))
    cos, sin = (t.to(DEV) for t in R64.tables(128, D))
    x = torch.zeros((40, H_q + 2 * H_kv, D), device=DEV, dtype=F16)

    def step(total, longest):
        t = x[:total]
        r = pkg.kv_reserve(table, lens, new, free, count, page, total, in_place=True)
        q = pkg.kv_append_fp4(t[:, H_q:-H_kv], t[:, -H_kv:], kc, vc, table, r.q_starts, lens, cos, sin, q=t[:, :H_q], norm=True)
        return q, *pkg.paged_sdpa_fp4(q, kc, vc, table, r.q_starts, lens, scale=D ** -0.5, max_q_len=longest)

    def checked(more, q, o):
        ends = lens.tolist()
        all_starts = i32([0] + [sum(ends[:s + 1]) for s in range(N)])
        k, v = (t.double().cpu() for t in pkg.kv_read_fp4(kc, vc, table, all_starts, lens, sum(ends)))
        at = first = 0
        for m, l in zip(more, ends):
            K, V = (t[first:first + l].repeat_interleave(H_q // H_kv, 1).transpose(0, 1) for t in (k, v))
            first += l
            if m:
                z = q[at:at + m].double().transpose(0, 1).cpu() @ K.transpose(1, 2) * D ** -0.5
                z = z.masked_fill(torch.arange(l)[None] > torch.arange(m)[:, None] + l - m, -INF)
                want = (torch.softmax(z, -1) @ V).transpose(0, 1)
                # (fp16 weights and results: 2^-11 of values of up to some units, twice)
                assert float((o[at:at + m].double().cpu() - want).abs().max()) <= 2.0 ** -10 * float(V.abs().max())
            at += m

    for more in ((20, 0, 5), (1, 33, 1), (1, 1, 1)):
        new.copy_(i32(more))
        x.normal_()
        q, o, _ = step(sum(more), max(more))
        checked(more, q, o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, o, _ = step(3, 1)
    for _ in range(14):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        checked((1, 1, 1), q, o)
    assert lens.tolist() == [36, 48, 21] and count.tolist() == [24 - 3 - 3 - 2]
