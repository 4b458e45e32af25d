"""Sequences that reach past the tokens of a call: append and attention leave them out, whole; their
tokens can be appended by a further call."""
import ctypes

import pytest
import torch

import _heads as R64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32
I32 = torch.int32


def _i32(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def _same(a, b):
    """To the bit (a NaN is its own like: some positions are outside of the tables)."""
    return torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def _caches(pkg, fp4, T, pages, H_kv, page, D):
    if fp4:
        return [c.fill_(0x11) for c in pkg.fp4_cache(pages, H_kv, page, D, D, device=DEV)]
    return [torch.full((pages, H_kv, page, D), 7.0, dtype=T, device=DEV) for _ in range(2)]


# new tokens, tokens that the call has: small calls, and those of the kernels of large ones
CASES = [((2, 5, 1), 5), ((3, 4), 6), ((9,), 8), ((700, 900, 3), 1500), ((40, 2000), 1100)]


@pytest.mark.parametrize("fp4", (False, True))
@pytest.mark.parametrize("T,axes", [(F16, None), (F32, None), (F16, (0, 1, 1, 0) * 8)])
@pytest.mark.parametrize("new,total", CASES, ids=str)
def test_append_leaves_out(pkg, fp4, T, axes, new, total):
    H_q, H_kv, D, page = 16, 8, 64, 64
    N, width = len(new), 2 + max(new) // page
    table = torch.arange(N * width, dtype=I32, device=DEV).view(N, width)
    lens = _i32([n + 11 for n in new])
    starts = [sum(new[:s]) for s in range(N + 1)]
    x = torch.randn((total, H_q + 2 * H_kv, D), device=DEV).to(T)
    cos, sin = (t.to(DEV) for t in R64.tables(max(new) + 11, D))
    pos = None if axes is None else torch.randint(0, 20, (2, total), dtype=I32, device=DEV)
    append = pkg.kv_append_fp4 if fp4 else pkg.kv_append
    outs = []
    # (a range that ends where the last whole sequence does, for comparison)
    for s in (starts, [min(b, max(a for a in starts if a <= total)) for b in starts]):
        kc, vc = _caches(pkg, fp4, T, N * width, H_kv, page, D)
        q = append(x[:, H_q:-H_kv], x[:, -H_kv:], kc, vc, table, _i32(s), lens, cos, sin, q=x[:, :H_q], norm=True, positions=pos,
                   axes=axes)
        outs.append((kc, vc, q[:s[-1] if s[-1] <= total else 0]))
    n = len(outs[1][2])
    assert _same(outs[0][0], outs[1][0]) and _same(outs[0][1], outs[1][1])
    assert n == max(a for a in starts if a <= total)


@pytest.mark.parametrize("fp4", (False, True))
@pytest.mark.parametrize("n", (5, 1500))
def test_rows_stay(pkg, fp4, n):
    """Rows of queries of a sequence that reaches past the tokens, or begins before them, stay as they were."""
    H, D, page = 8, 32, 16
    x = torch.randn((n, 3 * H, D), device=DEV).half()
    width = 200
    table = torch.arange(2 * width, dtype=I32, device=DEV).view(2, width)
    cos, sin = (t.to(DEV) for t in R64.tables(3200, D))
    for starts, live in (([0, 2, n + 1], slice(0, 2)), ([-1, 2, n], slice(2, n))):
        lens = _i32([40, n + 3])
        kc, vc = _caches(pkg, fp4, F16, 2 * width, H, page, D)
        before = kc.clone()
        y = torch.full((n, H, D), 5.0, device=DEV, dtype=F16)
        st = (ctypes.c_int64 * 2)(*x.stride()[:2])
        part = [x[:, i * H:(i + 1) * H].data_ptr() for i in range(3)]
        by = (None, None, 0) if fp4 else ()
        entry = pkg.library().sdpa_hip_kv_append_fp4 if fp4 else pkg.library().sdpa_hip_kv_append
        rc = entry(1, part[1], st, part[2], st, kc.data_ptr(), vc.data_ptr(), part[0], st, y.data_ptr(), None, None, None, 0,
                   cos.data_ptr(), sin.data_ptr(), 3200, *by, table.data_ptr(), width, _i32(starts).data_ptr(), lens.data_ptr(), 2, n,
                   width, 2 * width, page, H, H, D, D, D, 1e-6, 0, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        stay = torch.ones(n, dtype=torch.bool, device=DEV)
        stay[live] = False
        assert bool((y[stay] == 5).all()) and not (y[live] == 5).all(-1).any()
        changed = (kc != before).flatten(1).any(1).nonzero().flatten().tolist()
        # (pages of the sequence that is left out)
        out = range(width, 2 * width) if live.start == 0 else range(0, width)
        assert changed and not set(changed) & set(out)


@pytest.mark.parametrize("fp4", (False, True))
@pytest.mark.parametrize("few", (12, 22))
def test_reserve_with_too_few_rows(pkg, fp4, few):
    """A step whose tokens pass ``total``: the sequences that fit are served, the others' tokens appended by a further
    call, and then the cache is what a step with room for all makes of it.  (Of a sequence's new tokens ``total``
    count at most.)"""
    H_q, H_kv, D, page, width, new = 4, 2, 64, 16, 4, (3, 20, 2)
    x = torch.randn((25, H_q + 2 * H_kv, D), device=DEV).half()
    cos, sin = (t.to(DEV) for t in R64.tables(64, D))
    append, attend = (pkg.kv_append_fp4, pkg.paged_sdpa_fp4) if fp4 else (pkg.kv_append, pkg.paged_sdpa)
    m = min(20, few)  # of the second sequence
    starts = [0, 3, 3 + m, 5 + m]

    def run(total, new):
        table, lens, count = torch.full((3, width), -1, dtype=I32, device=DEV), _i32([0, 0, 0]), _i32([9])
        free = torch.arange(9, dtype=I32, device=DEV)
        kc, vc = _caches(pkg, fp4, F16, 9, H_kv, page, D)
        r = pkg.kv_reserve(table, lens, _i32(new), free, count, page, total, in_place=True)
        assert r.q_starts.tolist() == starts and lens.tolist() == [3, m, 2]
        rows = lambda t, starts: append(t[:, H_q:-H_kv], t[:, -H_kv:], kc, vc, table, starts, lens, cos, sin, q=t[:, :H_q])
        q = rows(x[:total], r.q_starts)[:5 + m]
        if total == few:
            out = (torch.full((total, H_q, D), 9.0, device=DEV, dtype=F16), torch.full((total, H_q), 9.0, device=DEV))
            attend(q, kc, vc, table, r.q_starts, lens, scale=0.125, out=out)
            assert bool((out[0][3:] == 9).all()) and bool((out[1][3:] == 9).all()) and not (out[0][:3] == 9).any()
            q = torch.cat((q[:3], rows(x[3:], _i32([0, 0, m, m + 2]))[:m + 2]))
        o, _ = attend(q, kc, vc, table, _i32(starts), lens, scale=0.125)
        return q, kc, vc, table, count, o

    for a, b in zip(run(few, new), run(25, (3, m, 2))):
        assert torch.equal(a, b)
