"""CPU tests of the cache in 4 bits: what the entry points refuse, before any device work."""
import ctypes

import pytest
import torch

I32, U8 = torch.int32, torch.uint8


def _meta(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="meta")


def _refused(pkg, message, fn, *args, **kw):
    with pytest.raises(pkg.InvalidArgumentError, match=message):
        fn(*args, **kw)


BATCH = dict(k=(6, 2, 64), v=(6, 2, 32), k_cache=(9, 2, 16, 34), v_cache=(9, 2, 16, 17), page_table=(3, 4), q_starts=(4,),
             kv_lens=(3,))
CHANGES = [
    (dict(k_cache=(9, 2, 16, 64)), "do not hold rows|bytes a token"),
    (dict(k_cache=(9, 2, 16, 34 * 3), k=(6, 2, 192)), "do not hold rows|bytes a token"),
    (dict(k_cache=(9, 2, 16, 0), k=(6, 2, 0)), "do not hold rows|bytes a token"),
    (dict(v_cache=(9, 2, 32, 17)), "differ in pages, heads or page size"),
    (dict(k_cache=(9, 2, 34)), "must be .pages"),
    (dict(cache_dtype=torch.int8), "uint8"),
    (dict(cache_dtype=torch.float16), "uint8"),
    (dict(q_starts=(3,)), "q_starts must have shape"),
    (dict(kv_lens=(4,)), "kv_lens must have shape"),
    (dict(i_dtype=torch.int64), "int32"),
    ({}, "on the GPU"),
]


def _tensors(change):
    c = dict(BATCH, cache_dtype=U8, i_dtype=I32)
    c.update(change)
    kinds = dict(k_cache=c["cache_dtype"], v_cache=c["cache_dtype"], page_table=c["i_dtype"], q_starts=c["i_dtype"],
                 kv_lens=c["i_dtype"])
    return {n: _meta(*c[n], dtype=kinds.get(n, torch.float16)) for n in BATCH}


@pytest.mark.parametrize("change,message", CHANGES + [
    (dict(k=(6, 2, 32)), "do not hold rows"),
    (dict(k=(6, 3, 64), v=(6, 3, 32)), "do not hold rows"),
    (dict(v=(5, 2, 32)), "differ in tokens or heads"),
])
def test_append_refusals(pkg, change, message):
    _refused(pkg, message, pkg.kv_append_fp4, **_tensors(change))


@pytest.mark.parametrize("change,message", CHANGES)
def test_read_refusals(pkg, change, message):
    t = _tensors(change)
    if message != "on the GPU" and t["k_cache"].dim() == 4 and t["k_cache"].shape[3] in (64, 102, 0):
        message = "on the GPU|bytes a token"  # (the device is looked at first)
    del t["k"], t["v"]
    _refused(pkg, message, pkg.kv_read_fp4, **t, total=6)


def test_cache_refusals(pkg):
    for D in (0, 16, 48, 160, -32):
        _refused(pkg, "32, 64, 96 or 128", pkg.fp4_cache, 4, 2, 16, 64, D, device="cpu")
    for page in (8, 24, 1 << 17):
        _refused(pkg, "power of two", pkg.fp4_cache, 4, 2, page, 64, 64, device="cpu")
    k, v = pkg.fp4_cache(4, 2, 32, 128, 96, device="cpu")
    assert k.shape == (4, 2, 32, 68) and v.shape == (4, 2, 32, 51) and k.dtype == U8 and not k.any()


def test_abi_refusals(pkg):
    L = pkg.library()
    some, odd = ctypes.c_void_p(64), ctypes.c_void_p(72)  # never read: every call below fails its checks

    def append(dtype=1, N=3, T=6, width=4, pages=9, page=16, H_kv=2, D=64, D_v=32, R=16, k=some, cache=some, table=some):
        return L.sdpa_hip_kv_append_fp4(dtype, k, None, some, None, cache, some, some, None, some, None, None, None, 0, some,
                                        some, 8, None, None, 0, table, width, some, some, N, T, width, pages, page, 4, H_kv, D,
                                        D_v, R, 1e-6, 0, 0, None)

    def read(dtype=1, N=3, T=6, width=4, pages=9, page=16, H_kv=2, D=64, D_v=32, k=some, cache=some, table=some, R=0):
        return L.sdpa_hip_kv_read_fp4(dtype, cache, some, k, some, table, width, some, some, N, T, width, pages, page, H_kv, D,
                                      D_v, None)

    for fn in (append, read):
        for kw, code in ((dict(dtype=3), 18), (dict(N=-1), 19), (dict(T=-1), 19), (dict(H_kv=-1), 19), (dict(page=8), 27),
                         (dict(D=160), 16), (dict(D_v=160), 16), (dict(D=48), 33), (dict(D=0), 33), (dict(D_v=8), 33),
                         (dict(k=None), 20), (dict(cache=None), 20), (dict(table=None), 20), (dict(cache=odd), 29),
                         (dict(width=1 << 27), 30), (dict(T=1 << 30), 30)):
            kw = dict(kw, R=0) if "D" in kw else kw
            assert fn(**kw) == code, (fn, kw)
        assert fn(T=0) == 0 and fn(N=0) == 0
    assert read(k=odd) == 29 and "32" in pkg.status_string(33)


@pytest.mark.parametrize("change,message", CHANGES + [
    (dict(k=(6, 2, 32)), "q has 32 features, k_cache 64"),
    (dict(k=(6, 64)), "q must be"),
])
def test_paged_refusals(pkg, change, message):
    t = _tensors(change)
    q = t.pop("k")
    del t["v"]
    if t["k_cache"].dim() == 4 and t["k_cache"].shape[3] == 102:
        message = "bytes a token"
    _refused(pkg, message, pkg.paged_sdpa_fp4, q, **t)


def test_paged_abi_refusals(pkg):
    L = pkg.library()
    some, odd = ctypes.c_void_p(64), ctypes.c_void_p(72)

    def call(dtype=1, N=3, T=6, width=4, pages=9, page=16, H_q=4, H_kv=2, D=32, D_v=64, q=some, table=some, stats=some, k=some):
        return L.sdpa_hip_paged_fwd_fp4(dtype, q, None, k, some, some, None, stats, table, width, some, some, None, 0, N, T,
                                        width, pages, page, H_q, H_kv, D, D_v, 0, 0.5, 1, None)

    for kw, code in ((dict(dtype=2), 18), (dict(N=-1), 19), (dict(width=-1), 19), (dict(H_q=-4), 19), (dict(D=160), 16),
                     (dict(D=0), 33), (dict(D_v=16), 33), (dict(dtype=0, D_v=80), 33), (dict(H_q=3), 28), (dict(H_kv=0), 28),
                     (dict(page=24), 27), (dict(q=None), 20), (dict(stats=None), 20), (dict(table=None), 20), (dict(k=None), 20),
                     (dict(q=odd), 29), (dict(k=odd), 29), (dict(T=1 << 30), 30)):
        assert call(**kw) == code, kw
    assert call(T=0) == 0 and call(N=0) == 0 and call(H_q=0) == 0
    need = lambda **k: L.sdpa_hip_paged_fwd_fp4_workspace_bytes(*dict(dict(dtype=1, N=3, T=6, width=400, page=16, H_q=4, H_kv=2,
                                                                           D=32, D_v=64, most=1), **k).values())
    assert need() > 0 and need(width=1) == 0 and need(H_q=3) == 0 and need(D=48) == 0
