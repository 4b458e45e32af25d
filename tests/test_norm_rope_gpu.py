"""qk_norm_rope and its gradient against the formulas in 64 bits.

Bounds.  fp32 arithmetic: the mean of squares of D <= 128 features is summed
in chains of at most 32 + 6 additions (relative error 40 u, u = 2^-24), the root halves it
and adds 2 u, the products x r w add 3 u, the rotation two roundings of each
product and one of the sum: together below 32 u of the size of the pair; the
result is rounded once to T.  Gradient: dn as above (4 u of its pair), the
mean of w dn x r again 40 u of the mean of the sizes, the rest 4 u.  The
weight's gradient: chains below 64 additions and 28 u in each term."""
import ctypes

import pytest
import torch

import _heads as R64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32

# dtype, B, S, H_q, H_kv, D, R, interleaved, fold, norm, weight dtype (None: without), positions
CASES = [
    (F16, 1, 1, 1, 1, 8, 8, False, True, True, None, None),             # one row; R / 2 is half a chunk
    (F16, 4, 1, 32, 8, 128, 128, False, False, True, F16, "far"),       # single tokens
    (F16, 2, 37, 5, 3, 128, 64, False, True, True, F32, "batch"),       # heads that fill no wave
    (F16, 1, 130, 12, 12, 80, 80, False, True, True, F16, None),        # idle lanes
    (F16, 3, 50, 2, 1, 64, 32, True, True, True, F32, "shared"),        # several tokens a wave
    (F16, 2, 33, 4, 4, 96, 96, True, False, False, None, "batch"),      # rotation alone
    (F16, 2, 19, 3, 2, 40, 24, False, True, True, F16, None),           # five chunks a row
    (F16, 2, 21, 3, 2, 36, 20, False, True, True, F32, None),           # no whole chunks
    (F16, 1, 17, 2, 2, 33, 10, True, False, True, F32, None),           # odd width
    (F16, 2, 9, 3, 1, 64, 0, False, True, True, F32, None),             # norm alone
    (F32, 2, 65, 12, 12, 64, 32, False, True, True, F32, None),
    (F32, 1, 40, 16, 2, 128, 128, True, True, True, F32, "far"),
    (F32, 2, 23, 3, 3, 20, 12, False, False, True, None, "shared"),
    (F32, 1, 7, 1, 1, 127, 126, False, True, True, F32, None),
    (F32, 1, 5, 2, 1, 1, 0, False, True, True, F32, None),              # one feature
    (F16, 2, 2100, 8, 8, 128, 128, False, True, True, F32, None),       # four rows per group of lanes
    (F16, 1, 3000, 4, 2, 64, 64, True, True, True, F16, None),          # more rows than the gradient's workgroups
]


def _inputs(case, seed=0):
    T, B, S, H_q, H_kv, D, R, inter, fold, norm, wt, pos = case
    g = torch.Generator().manual_seed(seed)
    qk = (torch.randn((B, S, H_q + H_kv, D), generator=g) * 1.5).to(T)
    w = [None, None] if wt is None else [(1 + 0.3 * torch.randn((D,), generator=g)).to(wt) for _ in range(2)]
    rows = S + 5
    positions = None
    if pos == "far":
        rows = 9000
        positions = torch.arange(rows - S, rows, dtype=torch.int32)
    elif pos == "shared":
        positions = torch.randint(0, rows, (S,), generator=g, dtype=torch.int32)
    elif pos == "batch":
        positions = torch.randint(0, rows, (B, S), generator=g, dtype=torch.int32)
    cos, sin = R64.tables(rows, R) if R else (None, None)
    dy = [torch.randn((B, S, H, D), generator=g).to(T) for H in (H_q, H_kv)]
    return qk[:, :, :H_q], qk[:, :, H_q:], w, positions, cos, sin, dy


def _angles(case, positions, cos, sin):
    _, B, S, _, _, _, R = case[:7]
    at = torch.arange(S) if positions is None else positions.long()
    at = at.expand(B, S)
    if not R:
        z = torch.zeros((B, S, 1, 0), dtype=torch.float64)
        return z, z
    return cos.double()[at][:, :, None], sin.double()[at][:, :, None]


def _gpu(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _on_gpu_strided(q, k):
    """q and k as parts of one tensor on the GPU."""
    qk = torch.cat([q, k], 2).to(DEV)
    return qk[:, :, :q.shape[2]], qk[:, :, q.shape[2]:]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_forward_and_gradient(pkg, case):
    T, B, S, H_q, H_kv, D, R, inter, fold, norm, wt, pos = case
    q, k, w, positions, cos, sin, dy = _inputs(case)
    c, s = _angles(case, positions, cos, sin)
    gq, gk = _on_gpu_strided(q, k)
    gw0, gw1, gpos, gcos, gsin = _gpu(w[0], w[1], positions, cos, sin)
    kw = dict(q_weight=gw0, k_weight=gw1, positions=gpos, eps=1e-5, norm=norm, interleaved=inter, fold_heads=fold)
    outs = pkg.qk_norm_rope(gq, gk, gcos, gsin, **kw)
    lay = R64.fold if fold else lambda x: x
    gd = [lay(d).contiguous().to(DEV) for d in dy]
    grads = pkg.qk_norm_rope_grad(*gd, gq, gk, gcos, gsin, **kw)
    again = pkg.qk_norm_rope_grad(*gd, gq, gk, gcos, gsin, **kw)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(grads, again))  # repeats to the bit
    rel, tiny = R64.half_step(T)
    u = R64.U32
    for i, (x, H) in enumerate(((q, H_q), (k, H_kv))):
        x = x.double()
        wd = torch.ones(D, dtype=torch.float64) if w[i] is None else w[i].double()
        n = R64.norm(x, wd, 1e-5) if norm else x
        y = R64.turn(n, c, s, inter)
        bound = rel * y.abs() + 32 * u * R64.pair_size(n, R, inter) + tiny
        assert outs[i].shape == ((B * H, S, D) if fold else (B, S, H, D))
        assert R64.worst(outs[i], lay(y), lay(bound)) <= 1
        # gradient, by the formula
        g = dy[i].double()
        dn = R64.turn(g, c, -s, inter)
        size = R64.pair_size(g, R, inter)
        if norm:
            r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5)
            xr = x * r
            dx = r * (wd * dn - xr * (wd * dn * xr).mean(-1, keepdim=True))
            spread = r * (wd.abs() * size + xr.abs() * (wd.abs() * size * xr.abs()).mean(-1, keepdim=True))
            dw, dw_size = (dn * xr).sum((0, 1, 2)), (size * xr.abs()).sum((0, 1, 2))
        else:
            dx, spread = dn, size
        assert R64.worst(grads[i], dx, rel * dx.abs() + 96 * u * spread + tiny) <= 1
        if w[i] is None:
            assert grads[2 + i] is None
        else:
            wrel, wtiny = R64.half_step(wt)
            assert grads[2 + i].dtype == wt and grads[2 + i].shape == (D,)
            assert R64.worst(grads[2 + i], dw, wrel * dw.abs() + 92 * u * dw_size + wtiny) <= 1


def test_gradient_against_differences(pkg):
    """The autograd form, against central differences of the 64-bit forward:
    their step h leaves an error of h^2 times third derivatives (below 1e-4
    for values near 1 at h = 1e-4), far below fp32's share of the sum."""
    case = (F32, 2, 6, 3, 2, 32, 16, False, True, True, F32, "batch")
    q, k, w, positions, cos, sin, dy = _inputs(case, 3)
    c, s = _angles(case, positions, cos, sin)

    def loss(q, k, w0, w1):
        total = 0
        for x, ww, d in ((q, w0, dy[0]), (k, w1, dy[1])):
            total = total + (R64.turn(R64.norm(x, ww, 1e-6), c, s, False) * d.double()).sum()
        return total

    leaves = [t.clone().to(DEV).requires_grad_(True) for t in (q, k, w[0], w[1])]
    q_out, k_out = pkg.qk_norm_rope_autograd(leaves[0], leaves[1], cos.to(DEV), sin.to(DEV), leaves[2], leaves[3],
                                             positions.to(DEV))
    ((q_out * R64.fold(dy[0]).to(DEV)).sum() + (k_out * R64.fold(dy[1]).to(DEV)).sum()).backward()
    base = [t.double() for t in (q, k, w[0], w[1])]
    g = torch.Generator().manual_seed(5)
    for i in range(4):
        for _ in range(4):
            v = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
            v /= v.norm()
            up = [t + 1e-4 * v if j == i else t for j, t in enumerate(base)]
            down = [t - 1e-4 * v if j == i else t for j, t in enumerate(base)]
            want = float(loss(*up) - loss(*down)) / 2e-4
            got = float((leaves[i].grad.double().cpu() * v).sum())
            size = float((leaves[i].grad.double().cpu() * v).abs().sum())
            assert abs(got - want) <= 1e-4 * max(1.0, size)


def test_layouts_agree_and_inputs_broadcast(pkg):
    """Folded and token-major results hold the same values, and so do dense,
    strided, misaligned and broadcast inputs (which take other kernels)."""
    g = torch.Generator(device=DEV).manual_seed(1)
    B, S, H, D = 2, 40, 6, 64
    x = torch.randn((B, S, H, D), generator=g, device=DEV, dtype=F32).half()
    cos, sin = (t.to(DEV) for t in R64.tables(S, D))
    folded = pkg.qk_norm_rope(x, x, cos, sin)[0]
    plain = pkg.qk_norm_rope(x, x, cos, sin, fold_heads=False)[0]
    assert torch.equal(folded, R64.fold(plain))
    buf = torch.empty((x.numel() + 3,), device=DEV, dtype=torch.float16)
    odd = buf[3:].view(B, S, H, D).copy_(x)
    assert odd.data_ptr() % 16 != 0
    near = pkg.qk_norm_rope(odd, odd, cos, sin)[0]  # sums in another order: a step apart at most
    assert float((near.float() - folded.float()).abs().max()) <= float(folded.abs().max()) * 2 ** -10
    wide = x[:1, :, :1].expand(3, S, 4, D)
    got = pkg.qk_norm_rope(wide, x[:1, :, :1].expand(3, S, 2, D), cos, sin, fold_heads=False)[0]
    assert torch.equal(got, pkg.qk_norm_rope(wide.contiguous(), wide.contiguous(), cos, sin, fold_heads=False)[0])
    turned = x.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)  # features not dense
    assert torch.equal(pkg.qk_norm_rope(turned, turned, cos, sin)[0], folded)


def test_places_outside_the_tables(pkg):
    """Rows at positions outside the tables are NaN, others untouched by them."""
    x = torch.ones((1, 4, 2, 32), device=DEV, dtype=F16)
    cos, sin = (t.to(DEV) for t in R64.tables(3, 32))
    pos = torch.tensor([0, 3, -1, 2], dtype=torch.int32, device=DEV)
    y = pkg.qk_norm_rope(x, x, cos, sin, positions=pos, fold_heads=False)[0]
    bad = torch.isnan(y).all(-1).all(-1)[0].tolist()
    assert bad == [False, True, True, False] and not torch.isnan(y[0, [0, 3]]).any()
    dq = pkg.qk_norm_rope_grad(y.nan_to_num(0), y.nan_to_num(0), x, x, cos, sin, positions=pos, fold_heads=False)[0]
    assert torch.isnan(dq[0, 1:3]).all() and not torch.isnan(dq[0, [0, 3]]).any()


def test_infinities_stay_in_their_row(pkg):
    """An infinite or NaN feature spoils its own row (norm) or pair (rotation
    alone), and nothing else."""
    x = torch.randn((1, 8, 3, 64), device=DEV).half()
    cos, sin = (t.to(DEV) for t in R64.tables(8, 32))
    clean = pkg.qk_norm_rope(x, x, cos, sin, fold_heads=False)[0]
    turned = pkg.qk_norm_rope(x, x, cos, sin, norm=False, fold_heads=False)[0]
    x[0, 3, 1, 50] = float("inf")  # behind the rotated features
    x[0, 5, 2, 4] = float("nan")   # paired with feature 20
    y = pkg.qk_norm_rope(x, x, cos, sin, fold_heads=False)[0]
    keep = torch.ones((8, 3), dtype=torch.bool, device=DEV)
    keep[3, 1] = keep[5, 2] = False
    assert torch.equal(y[0][keep], clean[0][keep])
    z = pkg.qk_norm_rope(x, x, cos, sin, norm=False, fold_heads=False)[0]
    changed = (z != turned).nonzero().tolist()
    assert changed == [[0, 3, 1, 50], [0, 5, 2, 4], [0, 5, 2, 20]] and torch.isinf(z[0, 3, 1, 50])


def test_empty(pkg):
    cos, sin = (t.to(DEV) for t in R64.tables(4, 32))
    w = torch.ones(32, device=DEV)
    for B, S, H in ((0, 4, 2), (2, 0, 2), (2, 4, 0)):
        q = torch.empty((B, S, H, 32), device=DEV, dtype=F16)
        k = torch.empty((B, S, 2, 32), device=DEV, dtype=F16).zero_()
        a, b = pkg.qk_norm_rope(q, k, cos, sin, w, w)
        assert a.shape == (B * H, S, 32) and b.shape == (B * 2, S, 32)
        dq, dk, dw, _ = pkg.qk_norm_rope_grad(a, b, q, k, cos, sin, w, w)
        assert dq.shape == q.shape and dk.shape == k.shape and not dw.any()


def test_training_step_through_attention(pkg):
    """Projection output -> qk_norm_rope -> sdpa -> loss, as a layer runs it:
    results and gradients against the same layer in 64 bits on the CPU.  fp32
    throughout, sums of up to 48 keys and 32 features: errors stay below
    2000 u of values near 1 (1.2e-4)."""
    B, S, H, D = 2, 48, 4, 32
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn((B, S, 3 * H, D), generator=g)
    w = [1 + 0.2 * torch.randn((D,), generator=g) for _ in range(2)]
    d_o = torch.randn((B * H, S, D), generator=g)
    cos, sin = R64.tables(S, D)

    def layer(x, w0, w1, norm_rope, attend):
        q, k = norm_rope(x[:, :, :H], x[:, :, H:2 * H], w0, w1)
        return attend(q, k, R64.fold(x[:, :, 2 * H:]).contiguous())

    x64, a64, b64 = (t.double().requires_grad_(True) for t in (qkv, *w))

    def rope64(q, k, w0, w1):
        c, s = cos.double()[:, None], sin.double()[:, None]
        return (R64.fold(R64.turn(R64.norm(t, u, 1e-6), c, s, False)) for t, u in ((q, w0), (k, w1)))

    def attend64(q, k, v):
        z = q @ k.transpose(1, 2) * D ** -0.5
        z = z.masked_fill(torch.ones((S, S), dtype=torch.bool).triu(1), float("-inf"))
        return torch.softmax(z, -1) @ v

    o64 = layer(x64, a64, b64, rope64, attend64)
    (o64 * d_o.double()).sum().backward()

    x, a, b = (t.to(DEV).requires_grad_(True) for t in (qkv, *w))
    gcos, gsin = cos.to(DEV), sin.to(DEV)
    o = layer(x, a, b, lambda q, k, w0, w1: pkg.qk_norm_rope_autograd(q, k, gcos, gsin, w0, w1),
              lambda q, k, v: pkg.sdpa_autograd(q, k, v, scale=D ** -0.5, causal_mask=True)[0])
    (o * d_o.to(DEV)).sum().backward()
    for got, want in ((o, o64), (x.grad, x64.grad), (a.grad, a64.grad), (b.grad, b64.grad)):
        want = want.detach()
        assert float((got.detach().double().cpu() - want).abs().max()) <= 2000 * R64.U32 * float(want.abs().max().clamp_min(1))


def test_captured_forward_and_gradient(pkg):
    """A captured step replays on new inputs, with eager work in between, and
    on a stream of its own."""
    B, S, H, D = 2, 64, 4, 64
    x = torch.randn((B, S, 2 * H, D), device=DEV).half()
    dy = torch.randn((B * H, S, D), device=DEV).half()
    w = torch.rand(D, device=DEV) + 0.5
    cos, sin = (t.to(DEV) for t in R64.tables(S, D))

    def step():
        q, k = x[:, :, :H], x[:, :, H:]
        return (*pkg.qk_norm_rope(q, k, cos, sin, w, w), *pkg.qk_norm_rope_grad(dy, dy, q, k, cos, sin, w, w))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)).half())
        eager = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_in_place(pkg):
    """The C entry with the inputs as results, dense and as parts of one tensor."""
    B, S, H, D = 2, 70, 5, 64
    x = torch.randn((B, S, 2 * H, D), device=DEV).half()
    cos, sin = (t.to(DEV) for t in R64.tables(S, D))
    want = pkg.qk_norm_rope(x[:, :, :H], x[:, :, H:], cos, sin, fold_heads=False)
    q, k = x[:, :, :H], x[:, :, H:]
    st = (ctypes.c_int64 * 3)(*q.stride()[:3])
    rc = pkg.library().sdpa_hip_qk_norm_rope(1, q.data_ptr(), st, k.data_ptr(), st, q.data_ptr(), st, k.data_ptr(), st, None,
                                             None, 0, cos.data_ptr(), sin.data_ptr(), S, None, 0, B, S, H, H, D, D, 1e-6, 1,
                                             0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert torch.equal(x[:, :, :H], want[0]) and torch.equal(x[:, :, H:], want[1])


def test_one_weight_and_one_side(pkg):
    """A weight for the queries alone; keys without heads."""
    x = torch.randn((2, 9, 6, 32), device=DEV)
    w = torch.rand(32, device=DEV) + 0.5
    cos, sin = (t.to(DEV) for t in R64.tables(9, 32))
    both = pkg.qk_norm_rope(x, x, cos, sin, w, w)
    bare = pkg.qk_norm_rope(x, x, cos, sin)
    one = pkg.qk_norm_rope(x, x, cos, sin, w)
    assert torch.equal(one[0], both[0]) and torch.equal(one[1], bare[1])
    g = pkg.qk_norm_rope_grad(*both, x, x, cos, sin, w)
    assert torch.equal(g[2], pkg.qk_norm_rope_grad(*both, x, x, cos, sin, w, w)[2]) and g[3] is None
    q_only = pkg.qk_norm_rope(x, x[:, :, :0], cos, sin, w)
    assert torch.equal(q_only[0], both[0]) and q_only[1].shape == (0, 9, 32)


def test_captured_backward(pkg):
    """Forward and backward of the autograd form in one captured graph."""
    B, S, H, D = 2, 40, 3, 64
    x = torch.randn((B, S, 2 * H, D), device=DEV)
    w = torch.rand(D, device=DEV) + 0.5
    d = torch.randn((B * H, S, D), device=DEV)
    cos, sin = (t.to(DEV) for t in R64.tables(S, D))

    def step():
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        q, k = pkg.qk_norm_rope_autograd(a[:, :, :H], a[:, :, H:], cos, sin, b, b)
        return torch.autograd.grad((q, k), (a, b), (d, d))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_gradient_of_a_gradient_is_refused(pkg):
    x = torch.randn((1, 3, 2, 32), device=DEV, requires_grad=True)
    cos, sin = (t.to(DEV) for t in R64.tables(3, 32))
    q, k = pkg.qk_norm_rope_autograd(x, x, cos, sin)
    (g,) = torch.autograd.grad((q * q).sum() + k.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
