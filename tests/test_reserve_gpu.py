"""kv_reserve against a loop over the sequences: whole numbers, equal."""
import random

import pytest
import torch

import _heads as R64
from _reserve import reserve

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = torch.int32


def _state(rng, lens, new, page, width, spare, finished=None, holes=False):
    used = [min(-(-max(l, 0) // page), width) for l in lens]
    need = sum(max(0, min(-(-(max(l, 0) + max(n, 0)) // page), width) - u) for l, n, u in zip(lens, new, used))
    free = max(0, need + spare)
    order = list(range(sum(used) + free))
    rng.shuffle(order)
    table, at = [], 0
    for u in used:
        table.append((order[at:at + u] + [-7] * width)[:width])
        at += u
    if holes:
        for row in table:
            row[rng.randrange(width)] = -1
    return dict(table=table, lens=list(lens), new=list(new), free=order[at:] + [-3] * at, count=free, page=page,
                total=sum(max(n, 0) for n in new), finished=finished)


def _both(pkg, st, in_place=False, wide=0, **change):
    """The library's results and the loop's, equal in every place."""
    st = dict(st, **change)
    i32 = lambda x: torch.tensor(x, dtype=I32, device=DEV)
    N, width = len(st["table"]), len(st["table"][0]) if st["table"] else 3
    big = torch.full((N, width + wide), -77, dtype=I32, device=DEV)
    table = big[:, :width]
    if N:
        table.copy_(i32(st["table"]))
    lens, new, free, count = i32(st["lens"]), i32(st["new"]), i32(st["free"]), i32([st["count"]])
    fin = None if st["finished"] is None else torch.tensor(st["finished"], dtype=torch.bool, device=DEV)
    got = pkg.kv_reserve(table, lens, new, free, count, st["page"], st["total"], finished=fin, in_place=in_place)
    rows, stack = [list(r) for r in st["table"]], list(st["free"])
    want = reserve(rows, st["lens"], st["new"], stack, st["count"], st["page"], st["total"], st["finished"])
    for g, w in zip(got, want):
        assert g.tolist() == (w if isinstance(w, list) else [w])
    assert table.tolist() == rows and free.tolist() == stack and bool((big[:, width:] == -77).all())
    assert new.tolist() == st["new"]
    if in_place:
        assert got.kv_lens is lens and got.free_count is count
    else:
        assert lens.tolist() == st["lens"] and count.tolist() == [st["count"]]
    return got


CASES = [  # lens, new, page, width, spare, finished
    ((0,), (1,), 16, 1, 0, None),
    ((16,), (1,), 16, 2, 3, None),                             # the token begins a page
    ((15, 16, 17, 0), (1, 1, 1, 1), 16, 4, 1, None),
    ((5, 0, 40, 31), (0, 33, 8, 1), 16, 8, 2, (False, False, False, True)),   # a finished one begins anew
    ((100, 20, 64), (0, 0, 200), 16, 20, 0, (True, True, False)),            # pages back and out again
    ((100, 20, 64), (40, 1, 200), 16, 20, -5, (True, False, False)),         # the pages run out
    ((10, 60), (100, 10), 16, 4, 0, None),                      # behind the table's columns
    ((0, 500, 3), (3000, 1, 700), 64, 64, 9, None),
    ((0, 33), (9000, 100), 128, 80, 1, (False, True)),          # tokens enough for the second kernel
    ((0,), (200000,), 16, 12600, 0, None),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c))[:80])
@pytest.mark.parametrize("in_place", (False, True))
def test_reserve(pkg, case, in_place):
    lens, new, page, width, spare, finished = case
    _both(pkg, _state(random.Random(1), lens, new, page, width, spare, finished), in_place, wide=2)


@pytest.mark.parametrize("N", (63, 64, 65, 1023, 1025, 2500))
def test_many_sequences(pkg, N):
    rng = random.Random(N)
    lens = [rng.choice([0, 1, 15, 16, 17, rng.randrange(400)]) for _ in range(N)]
    new = [rng.choice([0, 1, 1, 1, 2, 30]) for _ in range(N)]
    fin = [rng.random() < 0.2 for _ in range(N)]
    st = _state(rng, lens, new, 16, 30, 5, fin, holes=True)
    _both(pkg, st)
    _both(pkg, st, in_place=True, finished=None)


def test_lengths_that_are_none(pkg):
    """Negative and too large ones, a stack said to be larger than it is, rows for fewer tokens than there are."""
    st = _state(random.Random(2), (-4, 300, 2 ** 31 - 1, 20), (3, -9, 2, 5), 16, 4, 4, (False, False, True, False))
    _both(pkg, st)
    _both(pkg, st, count=99)
    _both(pkg, st, count=-1)
    _both(pkg, st, total=4)
    _both(pkg, st, total=0)
    _both(pkg, st, total=40)  # tokens of none behind the last
    _both(pkg, st, new=[3, 2 ** 31 - 1, 2 ** 31 - 1, 1], total=6000)
    _both(pkg, st, free=[], count=0)


def test_nothing(pkg):
    _both(pkg, dict(table=[], lens=[], new=[], free=[4, 2], count=2, page=16, total=3, finished=None))
    one = lambda *x: torch.tensor(x, dtype=I32, device=DEV)
    r = pkg.kv_reserve(torch.empty((2, 0), dtype=I32, device=DEV), one(0, 5), one(1, 0), one(), one(0), 16, 1)
    assert r.slots.tolist() == [-1] and r.q_starts.tolist() == [0, 1, 1] and r.positions.tolist() == [0]


def test_memory_of_its_own(pkg):
    buf = torch.zeros(40, dtype=I32, device=DEV)
    t, v = buf[:8].view(2, 4), lambda a, n: buf[a:a + n]
    ok = dict(kv_lens=v(8, 2), new_lens=v(10, 2), free_pages=v(12, 9), free_count=v(30, 1))
    pkg.kv_reserve(t, **ok, page_size=16, total=0)
    for change in (dict(free_pages=v(4, 9)), dict(kv_lens=v(7, 2)), dict(new_lens=v(12, 2)), dict(free_count=v(12, 1))):
        with pytest.raises(pkg.InvalidArgumentError, match="share memory"):
            pkg.kv_reserve(t, **dict(ok, **change), page_size=16, total=0)
    for change in (dict(new_lens=v(9, 2)), dict(free_count=v(8, 1))):
        with pytest.raises(pkg.InvalidArgumentError, match="memory of their own"):
            pkg.kv_reserve(t, **dict(ok, **change), page_size=16, total=0, in_place=True)


def test_captured_steps(pkg):
    """A captured step in place: sequences come, grow and go between its replays."""
    rng = random.Random(5)
    N, page, width, total = 6, 16, 8, 64
    st = _state(rng, [0] * N, [0] * N, page, width, 40)
    i32 = lambda x: torch.tensor(x, dtype=I32, device=DEV)
    table, lens, free, count = i32(st["table"]), i32(st["lens"]), i32(st["free"]), i32([st["count"]])
    new, fin = i32([0] * N), torch.zeros(N, dtype=torch.bool, device=DEV)
    step = lambda: pkg.kv_reserve(table, lens, new, free, count, page, total, finished=fin, in_place=True)
    step()  # (changes nothing)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    rows, stack, k, held = [list(r) for r in st["table"]], list(st["free"]), st["count"], [0] * N
    for _ in range(12):
        ended = [h > 0 and rng.random() < 0.2 for h in held]
        more = [rng.choice([1, 1, 1, 10]) if h and not e else rng.choice([0, 20]) for h, e in zip(held, ended)]
        new.copy_(i32(more))
        fin.copy_(torch.tensor(ended))
        graph.replay()
        torch.cuda.synchronize()
        starts, held, k, positions, slots = reserve(rows, held, more, stack, k, page, total, ended)
        assert out.q_starts.tolist() == starts and lens.tolist() == held and count.tolist() == [k]
        assert out.positions.tolist() == positions and out.slots.tolist() == slots
        assert table.tolist() == rows and free.tolist() == stack


def test_reserve_append_attend(pkg):
    """Steps of a server, whole: pages reserved, tokens with three positions appended, attention over
    the cache, against attention over dense tensors."""
    N, H_q, H_kv, D, page, width = 3, 4, 2, 64, 16, 6
    axes = (0, 1, 2, 2) * 8
    g = torch.Generator().manual_seed(3)
    table = torch.full((N, width), -1, dtype=I32, device=DEV)
    lens, free, count = torch.zeros(N, dtype=I32, device=DEV), torch.randperm(20, generator=g).int().to(DEV), torch.tensor(
        [20], dtype=I32, device=DEV)
    kc, vc = (torch.full((20, H_kv, page, D), float("nan"), device=DEV, dtype=torch.float32) for _ in range(2))
    cos, sin = (t.to(DEV) for t in R64.tables(90, D))
    held = [([], []) for _ in range(N)]
    for new in ((20, 0, 5), (1, 33, 1), (1, 1, 1), (16, 1, 0)):
        n = sum(new)
        x = torch.randn((n, H_q + 2 * H_kv, D), generator=g).to(DEV)
        pos = torch.randint(0, 90, (3, n), generator=g, dtype=I32).to(DEV)
        r = pkg.kv_reserve(table, lens, torch.tensor(new, dtype=I32, device=DEV), free, count, page, n, in_place=True)
        k, v = x[:, H_q:-H_kv], x[:, -H_kv:]
        q = pkg.kv_append(k, v, kc, vc, table, r.q_starts, lens, cos, sin, q=x[:, :H_q], positions=pos, axes=axes)
        o, _ = pkg.paged_sdpa(q, kc, vc, table, r.q_starts, lens, scale=D ** -0.5)
        rot = pkg.qk_norm_rope(x[None, :, :H_q], k[None], cos, sin, positions=pos, norm=False, fold_heads=False, axes=axes)
        assert torch.equal(rot[0][0], q)
        # (where each token went)
        assert torch.equal(kc.transpose(1, 2).reshape(-1, H_kv, D)[r.slots], rot[1][0])
        at = 0
        for s, m in enumerate(new):
            held[s][0].append(rot[1][0, at:at + m])
            held[s][1].append(v[at:at + m])
            if m:
                K, V = (torch.cat(t).double().repeat_interleave(H_q // H_kv, 1).transpose(0, 1).cpu() for t in held[s])
                z = q[at:at + m].double().transpose(0, 1).cpu() @ K.transpose(1, 2) * D ** -0.5
                l = K.shape[1]
                z = z.masked_fill(torch.arange(l)[None] > torch.arange(m)[:, None] + l - m, float("-inf"))
                want = (torch.softmax(z, -1) @ V).transpose(0, 1)
                # (fp32: sums of up to 70 keys and 64 features of values near 1)
                assert float((o[at:at + m].double().cpu() - want).abs().max()) <= 2000 * R64.U32
            at += m
    assert lens.tolist() == [38, 35, 7] and count.tolist() == [20 - 3 - 3 - 1]
