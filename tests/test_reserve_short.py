"""kv_reserve where the stack of pages runs out: what is reported, and how sequences recover without the
host, against a loop over the sequences."""
import ctypes
import random

import pytest
import torch

import _heads as R64
from _reserve import reserve

DEV = "cuda:0"
I32 = torch.int32


def _meta(*shape, dtype=I32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("short,message", [(_meta(2), "short must have shape"), (_meta(), "short must have shape"), ([0], "short must be"),
                                           (_meta(1, dtype=torch.int64), "short must be"), (_meta(1), "on the GPU")])
def test_refusals(pkg, short, message):
    with pytest.raises(pkg.InvalidArgumentError, match=message):
        pkg.kv_reserve(_meta(3, 4), _meta(3), _meta(3), _meta(9), _meta(1), 16, 5, short=short)


def test_abi_refusals(pkg):
    L, some = pkg.library(), ctypes.c_void_p(64)  # never read: every call fails its checks
    call = lambda N, T, page: L.sdpa_hip_kv_reserve_counted(some, 4, some, some, None, some, some, some, some, some, some, some, some,
                                                            N, T, 4, page, 9, None)
    assert call(-1, 5, 16) == 19 and call(3, 5, 24) == 27 and call(3, 1 << 30, 16) == 30


def _i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def _wanted(lens, new, page, width, total, finished):
    """Columns that the new tokens of each sequence are the first to need."""
    up = lambda x: min(-(-max(x, 0) // page), width)
    new = [min(max(n, 0), total) for n in new]
    old = [0 if f else min(max(l, 0), width * page) for l, f in zip(lens, finished)]
    return sum(up(o + n) - up(o) for o, n in zip(old, new))


@pytest.mark.gpu
@pytest.mark.parametrize("N,most,width", [(1, 40, 4), (3, 200, 20), (70, 40, 6), (1300, 1, 3), (2000, 3, 3)])
def test_count(pkg, N, most, width):
    """Enough pages, some too few, none at all; with and without sequences that end."""
    rng = random.Random(N)
    page = 16
    for free, fin_share in ((10 ** 9, 0), (3, 0), (N // 2, 0.3), (0, 0), (0, 0.5)):
        lens = [rng.choice([0, 15, 16, rng.randrange(width * page)]) for _ in range(N)]
        new = [rng.randrange(most + 1) for _ in range(N)]
        fin = [rng.random() < fin_share for _ in range(N)]
        total, capacity = sum(new) + rng.choice([0, 3]), N * width + 5
        used = [min(-(-l // page), width) for l in lens]
        table = [[1000 * s + c if c < u else -7 for c in range(width)] for s, u in enumerate(used)]
        stack = [10 ** 7 + i for i in range(capacity)]
        count = min(free, capacity)
        short, gt, gs = _i32([-5]), _i32(table), _i32(stack)
        got = pkg.kv_reserve(gt, _i32(lens), _i32(new), gs, _i32([count]), page, total,
                             finished=torch.tensor(fin, device=DEV), short=short)
        back = sum(u for u, f in zip(used, fin) if f)
        want = reserve(table, lens, new, stack, count, page, total, fin)
        for g, w in zip(got, want):
            assert g.tolist() == (w if isinstance(w, list) else [w])
        assert gt.tolist() == table and gs.tolist() == stack
        assert short.tolist() == [max(_wanted(lens, new, page, width, total, fin) - min(count + back, capacity), 0)]


@pytest.mark.gpu
def test_memory_of_its_own(pkg):
    buf = torch.zeros(60, dtype=I32, device=DEV)
    v = lambda a, n: buf[a:a + n]
    args = dict(page_table=v(0, 8).view(2, 4), kv_lens=v(8, 2), new_lens=v(10, 2), free_pages=v(12, 9), free_count=v(30, 1),
                page_size=16, total=0, finished=v(40, 2).view(torch.uint8)[:2])
    pkg.kv_reserve(**args, short=v(50, 1))
    for at in (0, 7, 8, 11, 12, 20, 30, 40):
        with pytest.raises(pkg.InvalidArgumentError, match="short must be memory of its own"):
            pkg.kv_reserve(**args, short=v(at, 1))


@pytest.mark.gpu
def test_a_call_made_again(pkg):
    """A call that was short, made again with the same lengths and count: as if it had not been made."""
    rng = random.Random(4)
    N, page, width, total = 5, 16, 6, 96
    lens, new = [30, 16, 0, 90, 5], [3, 1, 40, 1, 1]
    used = [-(-l // page) for l in lens]
    table, at = [], 0
    for u in used:
        table.append(list(range(at, at + u)) + [-1] * (width - u))
        at += u
    stack, count = [at + i for i in range(3)] + [-9] * 30, 3
    gt, gl, gs, gc = _i32(table), _i32(lens), _i32(stack), _i32([count])
    short = _i32([0])
    fin = torch.zeros(N, dtype=torch.bool, device=DEV)
    pkg.kv_reserve(gt, gl, _i32(new), gs, gc, page, total, finished=fin, short=short)
    assert short.tolist() == [2]  # one column each of 0 and 1, three of 2
    for more, ended in ((new, [False, False, False, True, False]), ([3, 1, 9, 1, 1], [False] * 5)):
        if ended[3]:
            more = more[:3] + [0] + more[4:]
        again = pkg.kv_reserve(gt, gl, _i32(more), gs, gc, page, total, finished=torch.tensor(ended, device=DEV), short=short)
        rows, st = [list(r) for r in table], list(stack)
        want = reserve(rows, lens, more, st, count, page, total, ended)
        for g, w in zip(again, want):
            assert g.tolist() == (w if isinstance(w, list) else [w])
        assert short.tolist() == [0]
        for s, l in enumerate(want[1]):
            n = -(-l // page)
            assert gt[s, :n].tolist() == rows[s][:n]


@pytest.mark.gpu
@pytest.mark.parametrize("fp4", (False, True))
def test_steps_that_run_out(pkg, fp4):
    """A captured step that is replayed without the host: pages run out, the sequences that lack one end and begin
    anew with their tokens as soon as there are pages, and attention is over all of their tokens at the end."""
    N, page, width, total, pages = 4, 16, 8, 256, 17
    H_q, H_kv, D = 4, 2, 64
    axis = torch.arange(width, device=DEV)
    table, free, count = torch.full((N, width), -1, dtype=I32, device=DEV), torch.arange(pages, dtype=I32, device=DEV), _i32([pages])
    lens, new, fin, short = _i32([0] * N), _i32([0] * N), torch.zeros(N, dtype=torch.bool, device=DEV), _i32([0])
    worst = _i32([0])
    if fp4:
        kc, vc = (c.fill_(0xFF) for c in pkg.fp4_cache(pages, H_kv, page, D, D, device=DEV))
        append, attend = pkg.kv_append_fp4, pkg.paged_sdpa_fp4
    else:
        kc, vc = (torch.full((pages, H_kv, page, D), float("nan"), device=DEV, dtype=torch.float16) for _ in range(2))
        append, attend = pkg.kv_append, pkg.paged_sdpa
    # token j of sequence s has the row j of its own
    g = torch.Generator().manual_seed(0)
    tokens = torch.randn((N, width * page, H_q + 2 * H_kv, D), generator=g).half().to(DEV)

    def step():
        # decided on the device: sequences with a column that is none end and begin anew with all of their tokens, the
        # others get a token more
        held = (lens + page - 1) // page
        lost = ((table < 0) & (axis < held[:, None])).any(1)
        torch.where(lost, lens + 1, torch.ones_like(lens), out=new)
        # the last sequence gives way (it ends, without tokens) as long as pages lack
        give = torch.zeros_like(lost)
        give[N - 1] = lost.any()
        fin.copy_(lost | give)
        new.masked_fill_(give, 0)
        r = pkg.kv_reserve(table, lens, new, free, count, page, total, finished=fin, in_place=True, short=short)
        worst.copy_(torch.maximum(worst, short))
        seq = (torch.searchsorted(r.q_starts, torch.arange(total, dtype=I32, device=DEV), right=True) - 1).clamp(0, N - 1)
        x = tokens[seq, r.positions.long().clamp_min(0)]
        q = append(x[:, H_q:-H_kv], x[:, -H_kv:], kc, vc, table, r.q_starts, lens, q=x[:, :H_q])
        o, _ = attend(q, kc, vc, table, r.q_starts, lens, scale=D ** -0.5)
        return r.q_starts, o

    # the same by a loop
    rows, stack, k, held = [[-1] * width for _ in range(N)], list(range(pages)), pages, [0] * N
    def loop():
        nonlocal k, held
        lost = [any(rows[s][c] < 0 for c in range(-(-held[s] // page))) for s in range(N)]
        more = [held[s] + 1 if lost[s] else 1 for s in range(N)]
        ended = list(lost)
        if any(lost):
            ended[N - 1], more[N - 1] = True, 0
        starts, held, k, _, _ = reserve(rows, held, more, stack, k, page, total, ended)
        return starts, any(lost)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    loop()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        starts, o = step()
    nan_seen = came_back = False
    for _ in range(79):  # (80 tokens each but for the last: 15 of the 17 pages, and its one)
        graph.replay()
        torch.cuda.synchronize()
        want, lost = loop()
        assert starts.tolist() == want and lens.tolist() == held and count.tolist() == [k]
        assert table.tolist() == rows
        lacks = [any(rows[s][c] < 0 for c in range(-(-held[s] // page))) for s in range(N)]
        assert (short.item() > 0) == any(lacks)
        for s in range(N):
            part = o[want[s]:want[s + 1]]
            assert bool(torch.isnan(part).any()) == (lacks[s] and len(part) > 0)
        nan_seen, came_back = nan_seen or any(lacks), came_back or (lost and not any(lacks))
    assert nan_seen and came_back and worst.item() > 0
    # all of the cached tokens, against attention in 64 bits
    ends = [0]
    for h in held:
        ends.append(ends[-1] + h)
    at = 0
    q = torch.cat([tokens[s, :h, :H_q] for s, h in enumerate(held)])
    o, _ = attend(q, kc, vc, table, _i32(ends), lens, scale=D ** -0.5)
    if fp4:
        k4, v4 = pkg.kv_read_fp4(kc, vc, table, _i32(ends), lens, ends[-1])
    for s, h in enumerate(held):
        if h == 0:
            continue
        K, V = (t[s, :h].double().cpu() for t in (tokens[:, :, H_q:-H_kv], tokens[:, :, -H_kv:]))
        if fp4:
            K, V = (t[ends[s]:ends[s + 1]].double().cpu() for t in (k4, v4))
        K, V = (t.repeat_interleave(H_q // H_kv, 1).transpose(0, 1) for t in (K, V))
        z = tokens[s, :h, :H_q].double().cpu().transpose(0, 1) @ K.transpose(1, 2) * D ** -0.5
        z = z.masked_fill(torch.arange(h)[None] > torch.arange(h)[:, None], float("-inf"))
        ref = (torch.softmax(z, -1) @ V).transpose(0, 1)
        # (fp16 weights and results: 2^-11 of the values, twice)
        assert float((o[ends[s]:ends[s + 1]].double().cpu() - ref).abs().max()) <= 2.0 ** -10 * float(V.abs().max())


@pytest.mark.gpu
def test_entry_without_a_count(pkg):
    """The C entry that reports nothing does the same."""
    page, width, total = 16, 4, 40
    lens, new, stack, count = [3, 0, 60], [14, 20, 3], [4, 7, 8, 9, 5], 4
    table = [[0, -1, -1, -1], [-1] * 4, [1, 2, 3, 6]]
    t, l, n, f, c = _i32(table), _i32(lens), _i32(new), _i32(stack), _i32([count])
    starts, out, left, places = _i32([0] * 4), _i32([0] * 3), _i32([0]), _i32([0] * total)
    slots = torch.zeros(total, dtype=torch.int64, device=DEV)
    rc = pkg.library().sdpa_hip_kv_reserve(t.data_ptr(), width, *(x.data_ptr() for x in (l, n)), None,
                                           *(x.data_ptr() for x in (f, c, starts, out, left, places, slots)), 3, total, width, page, 5,
                                           torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    want = reserve(table, lens, new, stack, count, page, total)
    for g, w in zip((starts, out, left, places, slots), want):
        assert g.tolist() == (w if isinstance(w, list) else [w])
    assert t.tolist() == table and f.tolist() == stack
