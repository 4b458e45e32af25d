"""CPU tests of positions with several axes and of page tables made on the GPU:
what the entry points refuse, before any device work."""
import ctypes

import pytest
import torch

I32 = torch.int32


def _meta(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="meta")


def _refused(pkg, message, fn, *args, **kw):
    with pytest.raises(pkg.InvalidArgumentError, match=message):
        fn(*args, **kw)


@pytest.mark.parametrize("axes,positions,dtype,tables,message", [
    ((0,) * 15, (3, 5), I32, True, "axes has 15 entries, the tables 16 pairs"),
    ((0,) * 15 + (4,), (5, 5), I32, True, "0, 1, 2 or 3"),
    ((0,) * 15 + (-1,), (5, 5), I32, True, "0, 1, 2 or 3"),
    ((0,) * 15 + (True,), (5, 5), I32, True, "0, 1, 2 or 3"),
    ((0,) * 15 + (2,), (2, 5), I32, True, "positions have 2 axes, axes names 2"),
    ((0,) * 15 + (2,), (3, 4), I32, True, "must have shape"),
    ((0,) * 15 + (2,), (3, 1, 5), I32, True, "must have shape"),
    ((0,) * 15 + (2,), (3, 2, 5), torch.int64, True, "int32"),
    ((0,) * 15 + (2,), (), I32, True, "must have shape"),
    ((0,) * 15 + (2,), None, I32, True, "axes need positions"),
    ((0,) * 15 + (2,), (3, 5), I32, False, "axes need cos and sin"),
    ([0, 1, 2, 3] * 4, (4, 2, 5), I32, True, "on the GPU"),
    ((0, 1, 2, 0) * 4, (3, 5), I32, True, "on the GPU"),
])
def test_axes_refusals(pkg, axes, positions, dtype, tables, message):
    q, k = _meta(2, 5, 4, 32), _meta(2, 5, 2, 32)
    cos = _meta(7, 16, dtype=torch.float32) if tables else None
    kw = dict(positions=None if positions is None else _meta(*positions, dtype=dtype), axes=axes)
    for fn, d in ((pkg.qk_norm_rope, ()), (pkg.qk_norm_rope_grad, (_meta(8, 5, 32), _meta(4, 5, 32))),
                  (pkg.qk_norm_rope_autograd, ())):
        _refused(pkg, message, fn, *d, q, k, cos, cos, **kw)


@pytest.mark.parametrize("one", [True, 1.0, [1], None])
def test_axes_that_equal_numbers(pkg, one):
    """What is no integer is refused, also where integers of its value came before it."""
    q, cos, pos = _meta(2, 5, 4, 32), _meta(7, 16, dtype=torch.float32), _meta(2, 5, dtype=I32)
    for axes, message in ((((0, 1) * 8), "on the GPU"), ((0, 1) * 7 + (0, one), "0, 1, 2 or 3")):
        _refused(pkg, message, pkg.qk_norm_rope, q, q, cos, cos, positions=pos, axes=axes)


def test_append_positions_need_whole_tables(pkg):
    cache, table = _meta(4, 2, 16, 32), _meta(7, dtype=torch.float32)
    batch = _meta(1, 3, dtype=I32), _meta(2, dtype=I32), _meta(1, dtype=I32)
    for axes in (None, (0,) * 16):
        _refused(pkg, "cos and sin must have one shape", pkg.kv_append, _meta(6, 2, 32), _meta(6, 2, 32), cache, cache, *batch, table,
                 table, positions=_meta(*((6,) if axes is None else (1, 6)), dtype=I32), axes=axes)


@pytest.mark.parametrize("axes,positions,message", [
    (None, (3, 6), "must have shape"),
    ((0, 1) * 8, (6,), "must have shape"),
    ((0, 1) * 8, (1, 6), "positions have 1 axes, axes names 1"),
    ((0, 1) * 7, (2, 6), "axes has 14 entries"),
    ((0, 1) * 8, (2, 6), "on the GPU"),
    (None, (6,), "on the GPU"),
])
def test_append_axes_refusals(pkg, axes, positions, message):
    cos = _meta(7, 16, dtype=torch.float32)
    cache, batch = _meta(9, 2, 16, 32), [_meta(*s, dtype=I32) for s in ((3, 4), (4,), (3,))]
    _refused(pkg, message, pkg.kv_append, _meta(6, 2, 32), _meta(6, 2, 32), cache, cache, *batch, cos, cos,
             positions=_meta(*positions, dtype=I32), axes=axes)
    _refused(pkg, "need cos and sin" if axes is None else "axes need cos and sin|on the GPU", pkg.kv_append, _meta(6, 2, 32),
             _meta(6, 2, 32), cache, cache, *batch, positions=_meta(*positions, dtype=I32), axes=axes)


def test_axes_abi_refusals(pkg):
    L = pkg.library()
    some = ctypes.c_void_p(64)  # never read: every call below fails its checks
    axes = lambda *a: (ctypes.c_uint8 * 16)(*(a * 16)[:16])

    def call(pairs=axes(0, 1, 2), n=3, positions=some, R=32, B=1, grad=False, D=32):
        tail = (B, 4, 2, 2, D, R, 1e-6, 1, 0, None)
        by = (positions, 0, pairs, n)
        if grad:
            return L.sdpa_hip_qk_norm_rope_axes_grad(1, some, None, some, None, some, None, some, None, some, None, some, None,
                                                     None, None, None, None, 0, some, some, 8, *by, None, 0, *tail)
        return L.sdpa_hip_qk_norm_rope_axes(1, some, None, some, None, some, None, some, None, None, None, 0, some, some, 8, *by,
                                            *tail)

    for grad in (False, True):
        for kw, code in ((dict(pairs=None), 20), (dict(positions=None), 20), (dict(n=-1), 19), (dict(n=2), 32),
                         (dict(pairs=axes(0, 4), n=5), 32), (dict(R=34), 26), (dict(D=129), 16)):
            assert call(grad=grad, **kw) == code, (grad, kw)
        assert call(grad=grad, B=0) == 0
    append = lambda pairs, n, positions=some: L.sdpa_hip_kv_append_axes(
        1, some, None, some, None, some, some, some, None, some, None, None, None, 0, some, some, 8, positions, pairs, n, some, 4,
        some, some, 3, 6, 4, 9, 16, 4, 2, 32, 32, 32, 1e-6, 0, 0, None)
    assert append(None, 3) == 20 and append(axes(0, 1), 1) == 32 and append(axes(0), 1, None) == 20
    assert "axes" in pkg.status_string(32)


def _call(pkg, **change):
    c = dict(page_table=(3, 4), kv_lens=(3,), new_lens=(3,), free_pages=(9,), free_count=(1,), finished=(3,), page=16, total=5,
             dtype=I32, f_dtype=torch.bool, in_place=False)
    c.update(change)
    t = lambda n, d: _meta(*c[n], dtype=d)
    return pkg.kv_reserve(*(t(n, c["dtype"]) for n in ("page_table", "kv_lens", "new_lens", "free_pages", "free_count")),
                          c["page"], c["total"], finished=t("finished", c["f_dtype"]), in_place=c["in_place"])


@pytest.mark.parametrize("change,message", [
    (dict(page_table=(12,)), "page_table must be"),
    (dict(kv_lens=(4,)), "kv_lens must have shape"),
    (dict(new_lens=(2,)), "new_lens must have shape"),
    (dict(free_pages=(3, 3)), "free_pages must have shape"),
    (dict(free_count=(2,)), "free_count must have shape"),
    (dict(finished=(1,)), "finished must have shape"),
    (dict(f_dtype=torch.int32), "finished must be"),
    (dict(dtype=torch.int64), "int32"),
    (dict(total=-1), "must be sizes"),
    (dict(total=2.0), "must be sizes"),
    (dict(page=0), "must be sizes"),
    ({}, "on the GPU"),
])
def test_reserve_refusals(pkg, change, message):
    with pytest.raises(pkg.InvalidArgumentError, match=message):
        _call(pkg, **change)


def test_reserve_refuses_rows_that_overlap(pkg):
    wide = torch.empty((1, 4), dtype=I32).expand(3, 4)
    v = lambda n: torch.empty((n,), dtype=I32)
    _refused(pkg, "memory of their own", pkg.kv_reserve, wide, v(3), v(3), v(9), v(1), 16, 5)
    _refused(pkg, "rows of page_table", pkg.kv_reserve, torch.empty((3, 8), dtype=I32)[:, ::2], v(3), v(3), v(9), v(1), 16, 5)
    _refused(pkg, "contiguous", pkg.kv_reserve, torch.empty((3, 4), dtype=I32), v(6)[::2], v(3), v(9), v(1), 16, 5)


def test_reserve_abi_refusals(pkg):
    L, some = pkg.library(), ctypes.c_void_p(64)

    def call(table=some, stride=4, lens=some, new=some, free=some, count=some, starts=some, out=some, positions=some, N=3, T=5,
             width=4, page=16, capacity=9):
        return L.sdpa_hip_kv_reserve(table, stride, lens, new, None, free, count, starts, out, count, positions, some, N, T,
                                     width, page, capacity, None)

    for kw, code in ((dict(N=-1), 19), (dict(T=-1), 19), (dict(width=-1), 19), (dict(capacity=-1), 19), (dict(page=24), 27),
                     (dict(page=8), 27), (dict(table=None), 20), (dict(lens=None), 20), (dict(new=None), 20),
                     (dict(free=None), 20), (dict(count=None), 20), (dict(starts=None), 20), (dict(out=None), 20),
                     (dict(positions=None), 20), (dict(stride=3), 29), (dict(T=1 << 30), 30), (dict(width=1 << 27), 30),
                     (dict(N=0x7FFFFFFF), 30)):
        assert call(**kw) == code, kw
