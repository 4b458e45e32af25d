"""CPU tests of the norm and rotation of queries and keys and of the paged
cache: what the entry points refuse, before any device work."""
import ctypes

import pytest
import torch

I64 = ctypes.c_int64


def _meta(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="meta")


def _refused(pkg, message, fn, *args, **kw):
    with pytest.raises(pkg.InvalidArgumentError, match=message):
        fn(*args, **kw)


QK = dict(q=(2, 5, 4, 32), k=(2, 5, 2, 32))
TABLE = (7, 16)


@pytest.mark.parametrize("change,message", [
    (dict(q=(2, 5, 32)), "batch, tokens, heads, features"),
    (dict(k=(2, 6, 2, 32)), "differ in batch, tokens or features"),
    (dict(k=(2, 5, 2, 30)), "differ in batch, tokens or features"),
    (dict(k_dtype=torch.float32), "same dtype T"),
    (dict(dtype=torch.float64), "T must be half or float"),
    (dict(cos=(7, 15)), "one shape"),
    (dict(cos=(4, 16), sin=(4, 16)), "4 positions, the sequence 5 tokens"),
    (dict(cos=None), "belong together"),
    (dict(table_dtype=torch.float16), "must be float32"),
    (dict(q_weight=(31,)), r"shape \[32\]"),
    (dict(q_weight=(32,), w_dtype=torch.float64), "dtype T or float32"),
    (dict(q_weight=(32,), norm=False), "needs the norm"),
    (dict(positions=(4,)), "must have shape"),
    (dict(positions=(5,), p_dtype=torch.int64), "int32"),
    ({}, "on the GPU"),
])
def test_norm_rope_refusals(pkg, change, message):
    c = dict(QK, cos=TABLE, sin=TABLE, dtype=torch.float16, table_dtype=torch.float32, w_dtype=torch.float32,
             p_dtype=torch.int32, norm=True, q_weight=None, positions=None, k_dtype=None)
    c.update(change)
    t = lambda s, d: None if s is None else _meta(*s, dtype=d)
    q, k = t(c["q"], c["dtype"]), t(c["k"], c["k_dtype"] or c["dtype"])
    args = (t(c["cos"], c["table_dtype"]), t(c["sin"], c["table_dtype"]))
    kw = dict(q_weight=t(c["q_weight"], c["w_dtype"]), positions=t(c["positions"], c["p_dtype"]), norm=c["norm"])
    _refused(pkg, message, pkg.qk_norm_rope, q, k, *args, **kw)
    d = _meta(8, 5, 32), _meta(4, 5, 32)
    _refused(pkg, message, pkg.qk_norm_rope_grad, *d, q, k, *args, **kw)


def test_norm_rope_abi_refusals(pkg):
    L = pkg.library()
    some = ctypes.c_void_p(64)  # never read: every call below fails its checks

    def call(dtype=1, D=32, R=16, B=1, S=4, H_q=2, H_kv=2, norm=1, w=None, wt=0, q=some, cos=some, grad=False, dw=None,
             ws=None, ws_bytes=0):
        tail = (B, S, H_q, H_kv, D, R, 1e-6, norm, 0, None)
        if grad:
            return L.sdpa_hip_qk_norm_rope_grad(dtype, some, None, some, None, q, None, some, None, some, None, some,
                                                None, dw, None, w, None, wt, cos, some, 8, None, 0, ws, ws_bytes, *tail)
        return L.sdpa_hip_qk_norm_rope(dtype, q, None, some, None, some, None, some, None, w, None, wt, cos, some, 8,
                                       None, 0, *tail)

    for grad in (False, True):
        for kw, code in ((dict(dtype=2), 18), (dict(D=-1), 19), (dict(B=-1), 19), (dict(H_kv=-1), 19), (dict(D=129), 16),
                         (dict(R=15), 26), (dict(R=34), 26), (dict(R=-2), 26), (dict(w=some, norm=0), 31),
                         (dict(w=some, wt=7), 31), (dict(q=None), 20), (dict(cos=None), 20),
                         (dict(B=1 << 20, S=1 << 12), 30)):
            assert call(grad=grad, **kw) == code, (grad, kw)
        assert call(grad=grad, B=0) == 0  # nothing to do
    need = L.sdpa_hip_qk_norm_rope_grad_workspace_bytes(32)
    assert need > 0 and L.sdpa_hip_qk_norm_rope_grad_workspace_bytes(129) == 0
    for ws, n in ((None, need), (some, need - 1), (ctypes.c_void_p(72), need)):
        assert call(grad=True, dw=some, ws=ws, ws_bytes=n) == 22
    assert "even" in pkg.status_string(26) and len({pkg.status_string(c) for c in range(26, 32)}) == 6


BATCH = dict(k=(6, 2, 32), v=(6, 2, 16), k_cache=(9, 2, 16, 32), v_cache=(9, 2, 16, 16), page_table=(3, 4),
             q_starts=(4,), kv_lens=(3,))


@pytest.mark.parametrize("change,message", [
    (dict(k=(6, 32)), "tokens, heads"),
    (dict(v=(5, 2, 16)), "differ in tokens or heads"),
    (dict(v_cache=(9, 2, 32, 16)), "differ in pages, heads or page size"),
    (dict(k_cache=(9, 2, 16, 24)), "do not hold rows"),
    (dict(k_cache=(9, 2, 32)), "must be .pages"),
    (dict(cache_dtype=torch.float32), "same dtype T"),
    (dict(q=(6, 4, 24)), "q must be"),
    (dict(q=(5, 4, 32)), "q has 5 tokens"),
    (dict(q_starts=(3,)), "q_starts must have shape"),
    (dict(kv_lens=(4,)), "kv_lens must have shape"),
    (dict(page_table=(12,)), "page_table must be"),
    (dict(i_dtype=torch.int64), "int32"),
    (dict(k_weight=(32,)), "needs the norm"),
    ({}, "on the GPU"),
])
def test_append_refusals(pkg, change, message):
    c = dict(BATCH, cache_dtype=torch.float16, i_dtype=torch.int32, q=None, k_weight=None)
    c.update(change)
    t = lambda name, d=torch.float16: None if c[name] is None else _meta(*c[name], dtype=d)
    _refused(pkg, message, pkg.kv_append, t("k"), t("v"), t("k_cache", c["cache_dtype"]), t("v_cache", c["cache_dtype"]),
             t("page_table", c["i_dtype"]), t("q_starts", c["i_dtype"]), t("kv_lens", c["i_dtype"]), q=t("q"),
             k_weight=t("k_weight", torch.float32))


def test_append_refuses_a_sliced_cache(pkg):
    cache = _meta(9, 2, 32, 32)[:, :, :16]
    _refused(pkg, "contiguous", pkg.kv_append, _meta(6, 2, 32), _meta(6, 2, 32), cache, cache,
             *(_meta(*s, dtype=torch.int32) for s in ((3, 4), (4,), (3,))))


def test_append_abi_refusals(pkg):
    L = pkg.library()
    some = ctypes.c_void_p(64)

    def call(dtype=1, N=3, T=6, width=4, pages=9, page=16, H_q=4, H_kv=2, D=32, D_v=16, R=16, k=some, q=some, table=some,
             w=None):
        return L.sdpa_hip_kv_append(dtype, k, None, some, None, some, some, q, None, some, None, w, None, 0, some, some, 8,
                                    table, width, some, some, N, T, width, pages, page, H_q, H_kv, D, D_v, R, 1e-6, 0, 0,
                                    None)

    for kw, code in ((dict(dtype=3), 18), (dict(N=-1), 19), (dict(T=-1), 19), (dict(pages=-1), 19), (dict(D_v=-1), 19),
                     (dict(page=8), 27), (dict(page=48), 27), (dict(page=1 << 17), 27), (dict(D=130), 16),
                     (dict(D_v=130), 16), (dict(R=34), 26), (dict(w=some), 31), (dict(k=None), 20), (dict(q=None), 20),
                     (dict(table=None), 20), (dict(width=1 << 27, page=16), 30), (dict(T=1 << 30), 30)):
        assert call(**kw) == code, kw
    assert call(T=0) == 0 and call(N=0) == 0


PAGED = dict(q=(6, 4, 32), k_cache=(9, 2, 16, 32), v_cache=(9, 2, 16, 16), page_table=(3, 4), q_starts=(4,), kv_lens=(3,))


@pytest.mark.parametrize("change,message", [
    (dict(q=(6, 4)), "q must be"),
    (dict(q=(6, 4, 24)), "q has 24 features"),
    (dict(dtype=torch.bfloat16), "T must be half or float"),
    (dict(cache_dtype=torch.float32), "same dtype T"),
    (dict(v_cache=(8, 2, 16, 16)), "differ in pages"),
    (dict(q_starts=(5,)), "q_starts must have shape"),
    (dict(out=((6, 4, 32), (6, 4))), "out must be"),
    (dict(out=((6, 4, 16), (6, 3))), "out must be"),
    ({}, "on the GPU"),
])
def test_paged_refusals(pkg, change, message):
    c = dict(PAGED, dtype=torch.float16, cache_dtype=None, out=None)
    c.update(change)
    t = lambda name, d: _meta(*c[name], dtype=d)
    d = c["cache_dtype"] or c["dtype"]
    out = None if c["out"] is None else (_meta(*c["out"][0]), _meta(*c["out"][1], dtype=torch.float32))
    _refused(pkg, message, pkg.paged_sdpa, t("q", c["dtype"]), t("k_cache", d), t("v_cache", d),
             *(t(n, torch.int32) for n in ("page_table", "q_starts", "kv_lens")), out=out)


def test_paged_abi_refusals(pkg):
    L = pkg.library()
    some = ctypes.c_void_p(64)

    def call(dtype=1, N=3, T=6, width=4, pages=9, page=16, H_q=4, H_kv=2, D=32, D_v=16, q=some, table=some, stats=some,
             k=some, strides=None):
        return L.sdpa_hip_paged_fwd(dtype, q, strides, k, some, some, None, stats, table, width, some, some, None, 0, N, T,
                                    width, pages, page, H_q, H_kv, D, D_v, 0, 0.5, 1, None)

    odd = (I64 * 2)(132, 32)
    for kw, code in ((dict(dtype=2), 18), (dict(N=-1), 19), (dict(width=-1), 19), (dict(H_q=-4), 19), (dict(D=136), 16),
                     (dict(D=0), 29), (dict(D_v=12), 29), (dict(dtype=0, D_v=14), 29), (dict(H_q=3), 28),
                     (dict(H_kv=0), 28), (dict(page=24), 27), (dict(q=None), 20), (dict(stats=None), 20),
                     (dict(table=None), 20), (dict(k=None), 20), (dict(q=ctypes.c_void_p(72)), 29),
                     (dict(k=ctypes.c_void_p(72)), 29), (dict(strides=odd), 29), (dict(T=1 << 30), 30)):
        assert call(**kw) == code, kw
    assert call(T=0) == 0 and call(N=0) == 0 and call(H_q=0) == 0
    need = lambda **k: L.sdpa_hip_paged_fwd_workspace_bytes(*dict(dict(dtype=1, N=3, T=6, width=400, page=16, H_q=4, H_kv=2,
                                                                       D=32, D_v=16, most=1), **k).values())
    assert need() > 0 and need(width=1) == 0 and need(H_q=3) == 0 and need(N=0) == 0


def test_sizes_that_pass_64_bits(pkg):
    """Products of sizes are not formed where they would wrap around."""
    L, some, most = pkg.library(), ctypes.c_void_p(64), 0x7FFFFFFF
    rope = lambda B, S, H_q, H_kv: L.sdpa_hip_qk_norm_rope(
        1, some, None, some, None, some, None, some, None, None, None, 0, some, some, 8, None, 0, B, S, H_q, H_kv, 64, 64,
        1e-6, 1, 0, None)
    append = lambda T, H_q, H_kv, N=3: L.sdpa_hip_kv_append(
        1, some, None, some, None, some, some, some, None, some, None, None, None, 0, some, some, 8, some, 4, some, some,
        N, T, 4, 9, 16, H_q, H_kv, 64, 64, 64, 1e-6, 0, 0, None)
    for sizes in ((most, 1, most, most), (1, 1, most, most), (2, 1, most, 1), (most, most, 1, 0)):
        assert rope(*sizes) == 30, sizes
    for sizes in ((most, most, most), (1, most, most), (3, 1, most), (1, 0, most)):
        assert append(*sizes) == 30, sizes
    assert append(1, 1, 1, N=most) == 30
    assert L.sdpa_hip_paged_fwd(1, some, None, some, some, some, None, some, some, 4, some, some, None, 0, most, 6, 4, 9, 16,
                                4, 2, 32, 16, 0, 0.5, 1, None) == 30


def test_spans_of_memory():
    from importlib import import_module
    share = import_module("tf-custom-flash-attention_amd.heads")._share_memory
    x = torch.empty((4, 6, 8))
    a, b = x[:2], x[2:]
    assert share(a, a) and share(a, x) and share(x, b) and not share(a, b) and not share(b, a)
    assert share(b, x[:, 1]) and not share(a, x[2:, ::2]) and share(b, x[1:3, ::2])
    assert not share(x[:0], x) and not share(x, torch.empty((4,)))
