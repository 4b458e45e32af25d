"""Paths of the append in 4 bits and of the page tables that small calls do not take: windows of 8 tokens and
several rows of queries per group of lanes with positions of the tokens' own, sums carried over groups of 1024 sequences;
and the widths that kv_read_fp4 refuses."""
import random

import pytest
import torch

import _fp4 as F
import _heads as R64
from _reserve import reserve

DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
I32 = torch.int32


@pytest.mark.parametrize("k_row,v_row", [(64, 17), (17, 64), (102, 17), (34, 16), (85, 34)])
def test_widths_that_a_read_refuses(pkg, k_row, v_row):
    meta = lambda *s, dtype=I32: torch.empty(s, dtype=dtype, device="meta")
    with pytest.raises(pkg.InvalidArgumentError, match="bytes a token"):
        pkg.kv_read_fp4(meta(9, 2, 16, k_row, dtype=torch.uint8), meta(9, 2, 16, v_row, dtype=torch.uint8), meta(3, 4), meta(4),
                        meta(3), 6)


def _sections(*n):
    return tuple(a for a, m in enumerate(n) for _ in range(m))


# dtype, new, lens, H_q, H_kv, D, axes (a number: that many pairs, by one position), interleaved, norm, elements off alignment
CASES = [
    (F16, (600, 503), (700, 503), 40, 8, 128, _sections(16, 24, 24), False, True, 0),
    (F16, (600, 503), (700, 503), 40, 8, 128, _sections(16, 24, 24), True, True, 0),
    (F16, (1100,), (1203,), 40, 8, 128, (0, 1, 2) * 21 + (0,), False, False, 0),
    (F16, (1100,), (1203,), 40, 8, 64, (3, 1, 0, 0) * 8, True, True, 0),
    (F16, (1, 1100, 5), (9, 1203, 70), 33, 8, 96, _sections(5, 7, 8), False, True, 0),   # pairs in no whole chunks
    (F16, (1100,), (1103,), 40, 8, 64, _sections(8, 12, 12), False, True, 3),            # odd addresses
    (F16, (2600,), (2600,), 6, 4, 64, 32, True, False, 0),
    (F32, (600, 503), (700, 503), 20, 8, 128, _sections(16, 24, 24), False, True, 0),
    (F32, (1100,), (1203,), 20, 8, 64, (0, 1, 2) * 10 + (0, 1), True, True, 0),
    (F32, (1100,), (1203,), 20, 8, 32, (2, 0, 1) * 3, False, False, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c)[:60])
def test_large_appends_by_positions(pkg, case):
    T, new, lens, H_q, H_kv, D, axes, inter, norm, off = case
    page, n = 32, sum(new)
    by_one = type(axes) is int
    axes = (0,) * axes if by_one else axes
    R = 2 * len(axes)
    used = [-(-l // page) for l in lens]
    g = torch.Generator().manual_seed(1)
    order = torch.randperm(sum(used), generator=g).tolist()
    table, at = [], 0
    for u in used:
        table.append(order[at:at + u] + [-7] * (max(used) - u))
        at += u
    table, kv_lens = torch.tensor(table, dtype=I32), torch.tensor(lens, dtype=I32)
    starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=I32)
    x = torch.randn((n, H_q + 2 * H_kv, D), generator=g).to(T)
    w = [(1 + 0.3 * torch.randn((D,), generator=g)) for _ in range(2)] if norm else [None, None]
    cos, sin = R64.tables(200, R)
    A = 1 + max(axes)
    pos = torch.randint(0, 200, (A, n), generator=g, dtype=I32)
    kc, vc = F.random_cache(g, sum(used), H_kv, page, D, False), F.random_cache(g, sum(used), H_kv, page, D, True)
    dev = lambda t: None if t is None else t.to(DEV)
    gx = torch.empty((x.numel() + off,), dtype=T, device=DEV)[off:].view(x.shape).copy_(x)
    gkc, gvc = dev(kc), dev(vc)
    q = pkg.kv_append_fp4(gx[:, H_q:-H_kv], gx[:, -H_kv:], gkc, gvc, dev(table), dev(starts), dev(kv_lens), dev(cos), dev(sin),
                          q=gx[:, :H_q], q_weight=dev(w[0]), k_weight=dev(w[1]), norm=norm, interleaved=inter,
                          positions=dev(pos[0] if by_one else pos), axes=None if by_one else axes)
    c, s = (torch.stack([t.double()[pos[a].long(), i] for i, a in enumerate(axes)], -1)[:, None] for t in (cos, sin))
    # queries: bounds of test_norm_rope_gpu.py
    h = R64.norm(x[:, :H_q].double(), w[0].double(), 1e-6) if norm else x[:, :H_q].double()
    y = R64.turn(h, c, s, inter)
    rel, tiny = R64.half_step(T)
    assert R64.worst(q, y, rel * y.abs() + 32 * R64.U32 * R64.pair_size(h, R, inter) + tiny) <= 1
    # codes and scales of the new tokens, every other as it was
    h = R64.norm(x[:, H_q:-H_kv].double(), w[1].double(), 1e-6) if norm else x[:, H_q:-H_kv].double()
    seq = torch.cat([torch.full((m,), i) for i, m in enumerate(new)])
    place = torch.cat([torch.arange(l - m, l) for m, l in zip(new, lens)])
    pg, slot = table[seq, place // page].long(), place % page
    for before, cache, rows, is_v in ((kc, gkc, R64.turn(h, c, s, inter), False), (vc, gvc, x[:, -H_kv:], True)):
        want_c, want_s = F.unpack(before, is_v)
        codes, scales = F.encode(rows)
        want_c[pg, :, slot], want_s[pg, :, slot] = codes, scales
        got_c, got_s = F.unpack(cache, is_v)
        assert torch.equal(got_s, want_s) and torch.equal(got_c, want_c)


@pytest.mark.gpu
@pytest.mark.parametrize("N", (1025, 2000))
def test_single_tokens_of_many_sequences(pkg, N):
    """More than 1024 sequences and few tokens: one kernel writes positions and slots, with sums carried between
    groups of 1024."""
    rng = random.Random(N)
    page, width = 16, 5
    lens = [rng.choice([0, 1, 15, 16, 17, rng.randrange(79)]) for _ in range(N)]
    new = [rng.choice([0, 1, 1]) for _ in range(N)]
    fin = [rng.random() < 0.1 for _ in range(N)]
    total = sum(new) + 7
    assert total <= 2048
    used = [-(-l // page) for l in lens]
    table, at = [], 0
    for u in used:
        table.append(list(range(at, at + u)) + [-7] * (width - u))
        at += u
    i32 = lambda t: torch.tensor(t, dtype=I32, device=DEV)
    for spare in (N, 100):
        rows, stack = [list(r) for r in table], [at + i for i in range(spare)] + [-3] * (at + 5)
        gt, gs = i32(rows), i32(stack)
        got = pkg.kv_reserve(gt, i32(lens), i32(new), gs, i32([spare]), page, total, finished=torch.tensor(fin, device=DEV))
        want = reserve(rows, lens, new, stack, spare, page, total, fin)
        for a, b in zip(got, want):
            assert a.tolist() == (b if isinstance(b, list) else [b])
        assert gt.tolist() == rows and gs.tolist() == stack
