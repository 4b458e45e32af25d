"""CPU tests: sizes that pass the int of the C entries are refused, not cut off."""
import pytest
import torch

BIG = 2 ** 32 + 3  # as an int: 3


def _meta(*shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device="meta")


def _refused(pkg, fn, *args, **kw):
    with pytest.raises(pkg.InvalidArgumentError, match="too large for one call"):
        fn(*args, **kw)


@pytest.mark.parametrize("q,k", [((1, BIG, 1, 2), (1, BIG, 1, 2)), ((BIG, 1, 1, 2), (BIG, 1, 1, 2)), ((1, 1, BIG, 2), (1, 1, 1, 2)),
                                 ((1, 1, 1, 2), (1, 1, BIG, 2)), ((1, 1, 1, BIG), (1, 1, 1, BIG))])
def test_norm_rope(pkg, q, k):
    _refused(pkg, pkg.qk_norm_rope, _meta(*q), _meta(*k), None, None)
    _refused(pkg, pkg.qk_norm_rope_grad, _meta(q[0] * q[2], q[1], q[3]), _meta(k[0] * k[2], k[1], k[3]), _meta(*q), _meta(*k),
             None, None)


@pytest.mark.parametrize("shape", [(BIG, 1), (1, BIG)])
def test_tables(pkg, shape):
    t = _meta(*shape, dtype=torch.float32)
    _refused(pkg, pkg.qk_norm_rope, _meta(1, 1, 1, 2), _meta(1, 1, 1, 2), t, t)


CACHE, TABLE = (2, 1, 16, 8), (1, 2)


@pytest.mark.parametrize("T,cache,table,H_q", [(BIG, CACHE, TABLE, 1), (1, (BIG, 1, 16, 8), TABLE, 1), (1, CACHE, (1, BIG), 1),
                                               (1, CACHE, (BIG, 1), 1), (1, CACHE, TABLE, BIG)])
def test_paged(pkg, T, cache, table, H_q):
    i32 = lambda *s: _meta(*s, dtype=torch.int32)
    c, batch = _meta(*cache), (i32(*table), i32(table[0] + 1), i32(table[0]))
    _refused(pkg, pkg.paged_sdpa, _meta(T, H_q, 8), c, c, *batch)
    _refused(pkg, pkg.kv_append, _meta(T, 1, 8), _meta(T, 1, 8), c, c, *batch, q=_meta(T, H_q, 8))


def test_any_path(pkg):
    """The check by comparisons leaves such sizes to the checks one by one."""
    from importlib import import_module
    heads = import_module("tf-custom-flash-attention_amd.heads")
    with pytest.raises(Exception, match="too large for one call"):
        heads._sizes_fit(q=None, k=_meta(1, 2 ** 31))
    heads._sizes_fit(q=_meta(1, 2 ** 31 - 1), k=_meta(0, 4))
