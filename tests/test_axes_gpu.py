"""Positions with several axes: qk_norm_rope, its gradient and kv_append
against the formulas in 64 bits (bounds: test_norm_rope_gpu.py)."""
import pytest
import torch

import _heads as R64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32


def _sections(*n):
    return tuple(a for a, m in enumerate(n) for _ in range(m))


# dtype, B, S, H_q, H_kv, D, axes of the pairs, interleaved, fold, norm, weight dtype, positions per batch
CASES = [
    (F16, 1, 1, 32, 8, 128, _sections(16, 24, 24), False, False, True, F16, False),       # one token
    (F16, 2, 37, 5, 3, 128, _sections(16, 24, 24), False, True, True, F32, True),         # whole chunks of an axis
    (F16, 2, 33, 4, 4, 64, (0, 1, 2) * 10 + (0, 1), False, True, True, F32, True),        # axes in turn
    (F16, 3, 50, 2, 1, 64, (2, 1, 0, 0) * 4, True, True, True, F16, False),               # neighbouring features
    (F16, 1, 130, 6, 2, 80, _sections(10, 15, 15), False, True, False, None, True),       # axes that change inside a chunk
    (F16, 2, 21, 3, 2, 36, (0, 3) * 5, False, True, True, F32, True),                     # no whole chunks; axes 0 and 3
    (F16, 1, 17, 2, 2, 33, (1,) * 5, True, False, True, F32, False),                      # one axis, not the first
    (F16, 2, 2100, 8, 8, 128, _sections(16, 16, 16, 16), False, True, True, F32, True),   # several rows per group of lanes
    (F32, 2, 65, 12, 12, 64, (0, 1, 2) * 10 + (0, 1), True, True, True, F32, True),
    (F32, 1, 40, 16, 2, 128, _sections(16, 24, 24), False, True, True, F32, True),
    (F32, 2, 23, 3, 3, 20, (0, 2, 1, 1, 0, 0), False, False, True, None, False),
    (F32, 1, 1000, 4, 2, 64, _sections(4, 6, 6), False, True, True, F32, True),
]


def _inputs(case, seed=0):
    T, B, S, H_q, H_kv, D, axes, inter, fold, norm, wt, per_batch = case
    g = torch.Generator().manual_seed(seed)
    qk = (torch.randn((B, S, H_q + H_kv, D), generator=g) * 1.5).to(T)
    w = [None, None] if wt is None else [(1 + 0.3 * torch.randn((D,), generator=g)).to(wt) for _ in range(2)]
    rows, A = 300, max(axes) + 1
    positions = torch.randint(0, rows, (A, B, S) if per_batch else (A, S), generator=g, dtype=torch.int32)
    # (an axis that no pair follows may hold anything)
    for a in set(range(A)) - set(axes):
        positions[a] = -5
    cos, sin = R64.tables(rows, 2 * len(axes))
    dy = [torch.randn((B, S, H, D), generator=g).to(T) for H in (H_q, H_kv)]
    return qk, w, positions, cos, sin, dy


def _angles(positions, axes, cos, sin, B, S):
    """cos and sin [B, S, 1, pairs] of every token."""
    at = positions.long().reshape(positions.shape[0], -1, S).expand(-1, B, S)
    return tuple(torch.stack([t.double()[at[a], i] for i, a in enumerate(axes)], -1)[:, :, None] for t in (cos, sin))


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c if type(x) is not tuple))
def test_forward_and_gradient(pkg, case):
    T, B, S, H_q, H_kv, D, axes, inter, fold, norm, wt, per_batch = case
    qk, w, positions, cos, sin, dy = _inputs(case)
    c, s = _angles(positions, axes, cos, sin, B, S)
    R = 2 * len(axes)
    gx = qk.to(DEV)
    dev = lambda t: None if t is None else t.to(DEV)
    kw = dict(q_weight=dev(w[0]), k_weight=dev(w[1]), positions=dev(positions), eps=1e-5, norm=norm, interleaved=inter,
              fold_heads=fold, axes=axes)
    outs = pkg.qk_norm_rope(gx[:, :, :H_q], gx[:, :, H_q:], dev(cos), dev(sin), **kw)
    lay = R64.fold if fold else lambda x: x
    grads = pkg.qk_norm_rope_grad(*(lay(d).contiguous().to(DEV) for d in dy), gx[:, :, :H_q], gx[:, :, H_q:], dev(cos), dev(sin),
                                  **kw)
    rel, tiny = R64.half_step(T)
    u = R64.U32
    for i, x in enumerate((qk[:, :, :H_q], qk[:, :, H_q:])):
        x = x.double()
        wd = torch.ones(D, dtype=torch.float64) if w[i] is None else w[i].double()
        n = R64.norm(x, wd, 1e-5) if norm else x
        y = R64.turn(n, c, s, inter)
        assert R64.worst(outs[i], lay(y), lay(rel * y.abs() + 32 * u * R64.pair_size(n, R, inter) + tiny)) <= 1
        g = dy[i].double()
        dn, size = R64.turn(g, c, -s, inter), R64.pair_size(g, R, inter)
        if norm:
            r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
            xr = x * r
            dx = r * (wd * dn - xr * (wd * dn * xr).mean(-1, keepdim=True))
            spread = r * (wd.abs() * size + xr.abs() * (wd.abs() * size * xr.abs()).mean(-1, keepdim=True))
            dw, dw_size = (dn * xr).sum((0, 1, 2)), (size * xr.abs()).sum((0, 1, 2))
        else:
            dx, spread = dn, size
        assert R64.worst(grads[i], dx, rel * dx.abs() + 96 * u * spread + tiny) <= 1
        if w[i] is not None:
            wrel, wtiny = R64.half_step(wt)
            assert R64.worst(grads[2 + i], dw, wrel * dw.abs() + 92 * u * dw_size + wtiny) <= 1


def test_gradient_against_differences(pkg):
    """The autograd form against central differences of the 64-bit forward (h = 1e-4: off by
    h^2 times third derivatives, below 1e-4 for values near 1)."""
    axes = (0, 1, 2, 1, 0, 2, 2, 1)
    case = (F32, 2, 6, 3, 2, 32, axes, False, True, True, F32, True)
    qk, w, positions, cos, sin, dy = _inputs(case, 3)
    c, s = _angles(positions, axes, cos, sin, 2, 6)
    base = [t.double() for t in (qk[:, :, :3], qk[:, :, 3:], *w)]

    def loss(q, k, w0, w1):
        return sum((R64.turn(R64.norm(x, ww, 1e-6), c, s, False) * d.double()).sum() for x, ww, d in ((q, w0, dy[0]), (k, w1, dy[1])))

    leaves = [t.float().to(DEV).requires_grad_(True) for t in base]
    q_out, k_out = pkg.qk_norm_rope_autograd(leaves[0], leaves[1], cos.to(DEV), sin.to(DEV), leaves[2], leaves[3],
                                             positions.to(DEV), axes=axes)
    ((q_out * R64.fold(dy[0]).to(DEV)).sum() + (k_out * R64.fold(dy[1]).to(DEV)).sum()).backward()
    g = torch.Generator().manual_seed(5)
    for i in range(4):
        for _ in range(4):
            v = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
            v /= v.norm()
            up, down = ([t + h * v if j == i else t for j, t in enumerate(base)] for h in (1e-4, -1e-4))
            want = float(loss(*up) - loss(*down)) / 2e-4
            part = leaves[i].grad.double().cpu() * v
            assert abs(float(part.sum()) - want) <= 1e-4 * max(1.0, float(part.abs().sum()))


def test_equal_axes_are_one_position(pkg):
    """Tokens that count alike on all axes come out, to the bit, as with one position."""
    x = torch.randn((2, 40, 6, 64), device=DEV).half()
    cos, sin = (t.to(DEV) for t in R64.tables(50, 64))
    pos = torch.randint(0, 50, (2, 40), dtype=torch.int32, device=DEV)
    dy = torch.randn((12, 40, 64), device=DEV).half()
    for axes in ((0,) * 32, (2, 1, 0, 1) * 8):
        for inter in (False, True):
            three = pos.expand(3, 2, 40).contiguous()
            a = pkg.qk_norm_rope(x, x, cos, sin, positions=pos, interleaved=inter)
            b = pkg.qk_norm_rope(x, x, cos, sin, positions=three, interleaved=inter, axes=axes)
            assert all(torch.equal(s, t) for s, t in zip(a, b))
            a = pkg.qk_norm_rope_grad(dy, dy, x, x, cos, sin, positions=pos, interleaved=inter)
            b = pkg.qk_norm_rope_grad(dy, dy, x, x, cos, sin, positions=three, interleaved=inter, axes=list(axes))
            assert all(torch.equal(s, t) for s, t in zip(a[:2], b[:2]))


def test_places_outside_the_tables(pkg):
    """A position outside the tables on an axis that some pair follows makes the token's
    rows NaN, others are untouched."""
    x = torch.ones((1, 4, 2, 32), device=DEV, dtype=F16)
    cos, sin = (t.to(DEV) for t in R64.tables(3, 32))
    pos = torch.tensor([[0, 1, 2, 0], [0, 3, 1, 1], [2, 0, 0, -1], [9, 9, 9, 9]], dtype=torch.int32, device=DEV)
    y = pkg.qk_norm_rope(x, x, cos, sin, positions=pos, fold_heads=False, axes=(0, 1, 2, 2) * 4)[0]
    assert torch.isnan(y).all(-1).all(-1)[0].tolist() == [False, True, False, True] and not torch.isnan(y[0, [0, 2]]).any()
    dq = pkg.qk_norm_rope_grad(y.nan_to_num(0), y.nan_to_num(0), x, x, cos, sin, positions=pos, fold_heads=False,
                               axes=(0, 1, 2, 2) * 4)[0]
    assert torch.isnan(dq[0, [1, 3]]).all() and not torch.isnan(dq[0, [0, 2]]).any()


def test_strided_and_empty(pkg):
    x = torch.randn((2, 12, 4, 64), device=DEV).half()
    cos, sin = (t.to(DEV) for t in R64.tables(20, 64))
    pos = torch.randint(0, 20, (2, 12, 3), dtype=torch.int32, device=DEV).permute(2, 0, 1)  # not dense
    axes = (0, 1, 2, 2) * 8
    want = pkg.qk_norm_rope(x, x, cos, sin, positions=pos.contiguous(), axes=axes)[0]
    assert torch.equal(pkg.qk_norm_rope(x, x, cos, sin, positions=pos, axes=axes)[0], want)
    turned = x.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)
    assert torch.equal(pkg.qk_norm_rope(turned, turned, cos, sin, positions=pos, axes=axes)[0], want)
    assert pkg.qk_norm_rope(x[:0], x[:0], cos, sin, positions=pos[:, :0], axes=axes)[0].shape == (0, 12, 64)
    none = pkg.qk_norm_rope(x, x, cos[:, :0], sin[:, :0], positions=pos, axes=())[0]
    assert torch.equal(none, pkg.qk_norm_rope(x, x, None, None)[0])


@pytest.mark.parametrize("T,axes,inter,norm", [(F16, _sections(16, 24, 24), False, True), (F16, (0, 1, 2) * 21 + (0,), True, False),
                                               (F32, _sections(8, 12, 12), False, True), (F16, None, False, True)])
def test_append(pkg, T, axes, inter, norm):
    """kv_append: rotated by given positions instead of the places in the sequences."""
    H_q, H_kv, D, page, n = 6, 2, 128, 16, 12
    R = 2 * len(axes) if axes else 64
    new, lens = (1, 9, 2), (20, 33, 2)
    table = torch.tensor([[4, 1, -1], [0, 2, 5], [3, -1, -1]], dtype=torch.int32)
    starts, kv = torch.tensor([0, 1, 10, 12], dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    x = torch.randn((n, H_q + 2 * H_kv, D), generator=g).to(T)
    w = [(1 + 0.3 * torch.randn((D,), generator=g)).to(F32) for _ in range(2)] if norm else [None, None]
    cos, sin = R64.tables(90, R)
    pos = torch.randint(0, 90, (3, n) if axes else (n,), generator=g, dtype=torch.int32)
    kc, vc = (torch.randn((7, H_kv, page, D), generator=g).to(T) for _ in range(2))
    dev = lambda t: None if t is None else t.to(DEV)
    gx, gkc, gvc = dev(x), dev(kc), dev(vc)
    q = pkg.kv_append(gx[:, H_q:-H_kv], gx[:, -H_kv:], gkc, gvc, dev(table), dev(starts), dev(kv), dev(cos), dev(sin),
                      q=gx[:, :H_q], q_weight=dev(w[0]), k_weight=dev(w[1]), norm=norm, interleaved=inter, positions=dev(pos),
                      axes=axes)
    c, s = _angles(pos if axes else pos[None], axes or (0,) * (R // 2), cos, sin, 1, n)
    u = R64.U32
    rel, tiny = R64.half_step(T)
    want = []
    for heads, ww in ((x[:, :H_q], w[0]), (x[:, H_q:-H_kv], w[1])):
        h = R64.norm(heads.double(), ww.double(), 1e-6) if norm else heads.double()
        y = R64.turn(h[None], c, s, inter)[0]
        want.append((y, rel * y.abs() + 32 * u * R64.pair_size(h, R, inter) + tiny))
    assert R64.worst(q, *want[0]) <= 1
    wk, bk, wv = kc.double(), torch.zeros_like(kc.double()), vc.clone()
    for i, (m, l) in enumerate(zip(new, lens)):
        for j in range(m):
            t, place = int(starts[i]) + j, l - m + j
            pg, slot = int(table[i, place // page]), place % page
            wk[pg, :, slot], bk[pg, :, slot], wv[pg, :, slot] = want[1][0][t], want[1][1][t], x[t, -H_kv:]
    assert R64.worst(gkc, wk, bk) <= 1 and torch.equal(gvc.cpu(), wv)


def test_captured(pkg):
    """A captured step follows positions that change between its replays."""
    x = torch.randn((1, 30, 6, 64), device=DEV).half()
    dy = torch.randn((6, 30, 64), device=DEV).half()
    cos, sin = (t.to(DEV) for t in R64.tables(60, 64))
    w = torch.rand(64, device=DEV) + 0.5
    pos = torch.zeros((3, 30), dtype=torch.int32, device=DEV)
    axes = _sections(8, 12, 12)
    step = lambda: (pkg.qk_norm_rope(x, x, cos, sin, w, w, pos, axes=axes) +
                    pkg.qk_norm_rope_grad(dy, dy, x, x, cos, sin, w, w, pos, axes=axes))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        pos.random_(0, 60)
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step()))


def test_axes_that_change_before_the_backward_pass(pkg):
    """The gradient is that of the call, whatever becomes of the list that the axes came in."""
    T, B, S, H_q, H_kv, D = F32, 1, 9, 2, 1, 64
    g = torch.Generator().manual_seed(3)
    q, k, dq, dk = (torch.randn(s, generator=g).to(DEV) for s in ((B, S, H_q, D), (B, S, H_kv, D), (H_q, S, D), (H_kv, S, D)))
    cos, sin = (t.to(DEV) for t in R64.tables(40, D))
    pos = torch.randint(0, 40, (3, S), generator=g, dtype=torch.int32).to(DEV)
    axes = [0, 1] * 16
    want = pkg.qk_norm_rope_grad(dq, dk, q, k, cos, sin, positions=pos, axes=tuple(axes))
    x = [t.clone().requires_grad_() for t in (q, k)]
    out = pkg.qk_norm_rope_autograd(*x, cos, sin, positions=pos, axes=axes)
    axes[:] = [2] * 32
    got = torch.autograd.grad(out, x, (dq, dk))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
