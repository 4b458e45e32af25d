"""The steps around ``sdpa`` of a layer of a language model: norm and rotation
of queries and keys (with the gradient), and a paged cache of keys and values, in
fp16, fp32 or 4 bits.

As with the op itself, torch tensors are device memory and streams only; the
arithmetic runs in the HIP kernels behind ``include/sdpa_hip.h``, fp16 or fp32.
Arguments that the device alone knows (lengths, page tables, positions) are
checked there, where they are used.
"""
from __future__ import annotations

import collections
import ctypes
import functools

import torch

from . import (DTYPE_F16, DTYPE_F32, InvalidArgumentError, _dtype_code, _raise_for, _stream_handle, _workspace,
               library)

_Strides3 = ctypes.c_int64 * 3
_Strides2 = ctypes.c_int64 * 2


_F32, _I32, _U8 = torch.float32, torch.int32, torch.uint8
_MOST = 0x7FFFFFFF  # of any size: the C entries take them as int
_CODES = {torch.float16: DTYPE_F16, torch.float32: DTYPE_F32}


# (a ctypes array costs a third of a microsecond, and programs have few layouts)
@functools.lru_cache(maxsize=512)
def _strides3(strides):
    """The first three strides of a [batch, tokens, heads, features] tensor for the C entries."""
    return _Strides3(*strides[:3])


@functools.lru_cache(maxsize=512)
def _strides2(strides):
    """The first two strides of a [tokens, heads, features] tensor for the C entries."""
    return _Strides2(*strides[:2])


def _fail(message):
    raise InvalidArgumentError(message)


def _on_device(device, **tensors):
    """Every tensor lies on one GPU."""
    if device.type != "cuda":
        _fail("tensors must be on the GPU (the op's HIP kernel)")
    for name, t in tensors.items():
        if t is not None and t.device != device:
            _fail(f"{name} is on {t.device}, not on {device}")


_current_device = torch.cuda.current_device


def _call(entry, device, *args):
    """``entry(*args, stream)`` with ``device`` current."""
    if _current_device() == device.index:
        code = entry(*args, _stream_handle(device))
    else:
        with torch.cuda.device(device):
            code = entry(*args, _stream_handle(device))
    if code:
        _raise_for(code)


def _dense_features(t):
    """``t`` with its features next to each other."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _int32(name, t, *shape):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        _fail(f"{name} must be an int32 tensor")
    if tuple(t.shape) != shape:
        _fail(f"{name} must have shape {list(shape)}, got {list(t.shape)}")


def _tables(cos, sin):
    """Rows and rotated features of the rotation tables (0, 0 without)."""
    if cos is None and sin is None:
        return 0, 0
    if cos is None or sin is None:
        _fail("cos and sin belong together")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        _fail("cos and sin must be float32")
    if cos.dim() != 2 or cos.shape != sin.shape:
        _fail("cos and sin must have one shape [positions, rotated features / 2]")
    _sizes_fit(cos=cos)
    return cos.shape[0], 2 * cos.shape[1]


def _weight_dtype(T, D, q_weight, k_weight, norm):
    code = None
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if not norm:
            _fail(f"{name} needs the norm")
        if tuple(w.shape) != (D,):
            _fail(f"{name} must have shape [{D}], got {list(w.shape)}")
        if w.dtype not in (T, torch.float32):
            _fail(f"{name} must be of dtype T or float32, got {w.dtype}")
        c = DTYPE_F32 if w.dtype == torch.float32 else DTYPE_F16
        if code is not None and c != code:
            _fail("q_weight and k_weight must have the same dtype")
        code = c
    return DTYPE_F32 if code is None else code


def _sizes_fit(**tensors):
    for name, t in tensors.items():
        if t is not None and t.dim() and max(t.shape) > _MOST:
            _fail(f"{name} {list(t.shape)} is too large for one call")


def _check_qk(q, k):
    if q.dim() != 4 or k.dim() != 4:
        _fail("q and k must be [batch, tokens, heads, features]")
    if q.dtype != k.dtype:
        _fail("q and k must have the same dtype T")
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        _fail(f"q {list(q.shape)} and k {list(k.shape)} differ in batch, tokens or features")
    _sizes_fit(q=q, k=k)


def _pair_axes(axes, pairs):
    """The axis of every rotated pair, for the C entries, and the largest."""
    axes = tuple(axes)
    # (before the numbers are looked up, among which 1, True and 1.0 are one key)
    if set(map(type, axes)) - {int}:
        _fail("axes are 0, 1, 2 or 3")
    return _axes_bytes(axes, pairs)


@functools.lru_cache(maxsize=64)
def _axes_bytes(axes, pairs):
    if len(axes) != pairs:
        _fail(f"axes has {len(axes)} entries, the tables {pairs} pairs")
    if any(not 0 <= a < 4 for a in axes):
        _fail("axes are 0, 1, 2 or 3")
    return (ctypes.c_uint8 * max(1, pairs))(*axes), max(axes, default=-1)


def _axes_args(axes, positions, cos, *shape):
    """(axes of the pairs, number of axes) for the C entries; positions [axes, *shape]."""
    if cos is None:
        _fail("axes need cos and sin")
    if not isinstance(positions, torch.Tensor):
        _fail("axes need positions")
    if cos.dim() != 2:
        _fail("cos and sin must have one shape [positions, rotated features / 2]")
    pairs, top = _pair_axes(axes, cos.shape[1])
    n = positions.shape[0] if positions.dim() else 0
    _int32("positions", positions, n, *shape)
    if top >= n:
        _fail(f"positions have {n} axes, axes names {top}")
    _sizes_fit(positions=positions)
    return pairs, n


def _plain_rope(q, k, cos, sin, q_weight, k_weight, positions, norm, axes):
    """What ``_rope_args`` returns, of arguments that pass its checks by a few
    comparisons and need no copies; None of others, which go through them (the
    checks one by one took half of a small call's host time)."""
    sq, sk = q.shape, k.shape
    if cos is None or sin is None or len(sq) != 4 or len(sk) != 4:
        return None
    T, device, sc = q.dtype, q.device, cos.shape
    B, S, H_q, D = sq
    code = _CODES.get(T)
    w = q_weight
    if not (code is not None and k.dtype is T and device.type == "cuda" and k.device == device and cos.device == device
            and sin.device == device and sk[0] == B and sk[1] == S and sk[3] == D and len(sc) == 2 and sin.shape == sc
            and cos.dtype is _F32 and sin.dtype is _F32 and B + S + H_q + sk[2] + D + sc[0] + sc[1] <= _MOST and cos.is_contiguous()
            and sin.is_contiguous()):
        return None
    per_batch = 0
    if positions is None:
        if S > sc[0] or axes is not None:
            return None
    else:
        sp = positions.shape
        if axes is not None:
            pairs, top = _pair_axes(axes, sc[1])
            if not 2 <= len(sp) <= 3 or not top < sp[0] <= _MOST:
                return None
            n_axes, sp = sp[0], sp[1:]
        per_batch = int(len(sp) == 2)
        if (sp != ((B, S) if per_batch else (S,)) or positions.dtype is not _I32 or positions.device != device
                or not positions.is_contiguous()):
            return None
        if axes is not None:
            per_batch = (per_batch, pairs, n_axes)
    w_code = DTYPE_F32
    if w is not None or k_weight is not None:
        if (not norm or w is None or k_weight is None or w.dtype is not k_weight.dtype or w.dtype not in (T, _F32)
                or w.shape != (D,) or k_weight.shape != (D,) or w.device != device or k_weight.device != device
                or not w.is_contiguous() or not k_weight.is_contiguous()):
            return None
        w_code = _CODES[w.dtype]
    return code, (B, S, H_q, sk[2], D, 2 * sc[1]), (cos, sin, sc[0]), (w, k_weight, w_code), positions, per_batch


def _rope_args(q, k, cos, sin, q_weight, k_weight, positions, norm, axes=None):
    """Checks of what the forward and the gradient have in common."""
    plain = _plain_rope(q, k, cos, sin, q_weight, k_weight, positions, norm, axes)
    if plain is not None:
        return plain
    _check_qk(q, k)
    code = _dtype_code(q)
    B, S, H_q, D = q.shape
    rows, R = _tables(cos, sin)
    w_code = _weight_dtype(q.dtype, D, q_weight, k_weight, norm)
    per_batch = 0
    if axes is not None:
        per_batch = int(isinstance(positions, torch.Tensor) and positions.dim() == 3)
        per_batch = (per_batch,) + _axes_args(axes, positions, cos, *((B, S) if per_batch else (S,)))
        positions = positions.contiguous()
    elif positions is not None:
        per_batch = int(positions.dim() == 2)
        _int32("positions", positions, *((B, S) if per_batch else (S,)))
        positions = positions.contiguous()
    elif R and S > rows:
        _fail(f"the rotation tables have {rows} positions, the sequence {S} tokens")
    _on_device(q.device, k=k, cos=cos, sin=sin, q_weight=q_weight, k_weight=k_weight, positions=positions)
    cos, sin, q_weight, k_weight = _dense(cos), _dense(sin), _dense(q_weight), _dense(k_weight)
    return code, (B, S, H_q, k.shape[2], D, R), (cos, sin, rows), (q_weight, k_weight, w_code), positions, per_batch


def _out_rows(like, B, S, H, D, fold_heads):
    """A result [B H, S, D] (folded) or [B, S, H, D], and its strides {batch, token, head}."""
    if fold_heads:
        return torch.empty((B * H, S, D), dtype=like.dtype, device=like.device), _strides3((H * S * D, D, S * D))
    return torch.empty((B, S, H, D), dtype=like.dtype, device=like.device), None


def qk_norm_rope(q, k, cos, sin, q_weight=None, k_weight=None, positions=None, eps: float = 1e-6,
                 norm: bool = True, interleaved: bool = False, fold_heads: bool = True, axes=None):
    """RMS norm of every head of q and k, and its rotation by position: ``(q_out, k_out)``.

    q [B, S, H_q, D] and k [B, S, H_kv, D] (fp16 or fp32; any strides, so both may be parts of one
    projection's output; D <= 128).  ``norm``: each row divided by sqrt(mean of its squares + eps)
    and multiplied by its weight [D] (dtype T or float32), if there is one.  The first R features,
    R = 2 * cos.shape[1], are rotated by row ``positions`` (int32 [S] or [B, S]; None: 0 .. S - 1) of the float32 tables
    cos and sin [P, R / 2]: pairs (i, i + R/2), or (2i, 2i + 1) if ``interleaved``; without tables
    (None) nothing is.  A position outside the tables makes its rows NaN.

    ``axes``: tokens with several positions (time, height, width): the axis that each of the R/2 pairs
    follows, as a sequence of numbers below 4 ((0,) * 16 + (1,) * 24 + (2,) * 24: the first 16 pairs time, and so on);
    positions are then int32 [axes, S] or [axes, B, S].

    ``fold_heads``: results [B * H, S, D], the layout of ``sdpa``; else [B, S, H, D].
    """
    code, (B, S, H_q, H_kv, D, R), tables, weights, positions, per_batch = _rope_args(
        q, k, cos, sin, q_weight, k_weight, positions, norm, axes)
    q, k = _dense_features(q), _dense_features(k)
    q_out, qos = _out_rows(q, B, S, H_q, D, fold_heads)
    k_out, kos = _out_rows(k, B, S, H_kv, D, fold_heads)
    L = library()
    entry = L.sdpa_hip_qk_norm_rope if axes is None else L.sdpa_hip_qk_norm_rope_axes
    by = (per_batch,) if axes is None else per_batch
    _call(entry, q.device, code, q.data_ptr(), _strides3(q.stride()), k.data_ptr(), _strides3(k.stride()),
          q_out.data_ptr(), qos, k_out.data_ptr(), kos, _ptr(weights[0]), _ptr(weights[1]), weights[2],
          _ptr(tables[0]), _ptr(tables[1]), tables[2], _ptr(positions), *by, B, S, H_q, H_kv, D, R, float(eps),
          int(bool(norm)), int(bool(interleaved)))
    return q_out, k_out


def qk_norm_rope_grad(d_q_out, d_k_out, q, k, cos, sin, q_weight=None, k_weight=None, positions=None,
                      eps: float = 1e-6, norm: bool = True, interleaved: bool = False, fold_heads: bool = True, axes=None):
    """Gradient of ``qk_norm_rope``: ``(dq, dk, dq_weight, dk_weight)``.

    ``d_q_out`` and ``d_k_out`` are laid out as its results; dq and dk come as
    dense [B, S, H, D], the weights' gradients in their dtype, None for a
    weight that was not given.
    """
    code, (B, S, H_q, H_kv, D, R), tables, weights, positions, per_batch = _rope_args(
        q, k, cos, sin, q_weight, k_weight, positions, norm, axes)
    L = library()
    _on_device(q.device, d_q_out=d_q_out, d_k_out=d_k_out)
    grads = []
    for name, d, H in (("d_q_out", d_q_out, H_q), ("d_k_out", d_k_out, H_kv)):
        shape = (B * H, S, D) if fold_heads else (B, S, H, D)
        if tuple(d.shape) != shape or d.dtype != q.dtype:
            _fail(f"{name} must be {q.dtype} of shape {list(shape)}, got {d.dtype} {list(d.shape)}")
        d = _dense_features(d)
        # (batch and head of a folded row are H rows and one row apart)
        grads.append((d, _strides3((H * d.stride(0), d.stride(1), d.stride(0)) if fold_heads else d.stride())))
    q, k = _dense_features(q), _dense_features(k)
    dq = torch.empty((B, S, H_q, D), dtype=q.dtype, device=q.device)
    dk = torch.empty((B, S, H_kv, D), dtype=q.dtype, device=q.device)
    dw = [None if w is None else torch.empty_like(w) for w in weights[:2]]
    ws, ws_bytes = None, 0
    if dw[0] is not None or dw[1] is not None:
        ws_bytes = L.sdpa_hip_qk_norm_rope_grad_workspace_bytes(D)
        ws = torch.empty((ws_bytes,), dtype=torch.uint8, device=q.device)
    entry = L.sdpa_hip_qk_norm_rope_grad if axes is None else L.sdpa_hip_qk_norm_rope_axes_grad
    by = (per_batch,) if axes is None else per_batch
    _call(entry, q.device, code, grads[0][0].data_ptr(), grads[0][1], grads[1][0].data_ptr(),
          grads[1][1], q.data_ptr(), _strides3(q.stride()), k.data_ptr(), _strides3(k.stride()), dq.data_ptr(), None, dk.data_ptr(),
          None, _ptr(dw[0]), _ptr(dw[1]), _ptr(weights[0]), _ptr(weights[1]), weights[2], _ptr(tables[0]),
          _ptr(tables[1]), tables[2], _ptr(positions), *by, _ptr(ws), ws_bytes, B, S, H_q, H_kv, D, R,
          float(eps), int(bool(norm)), int(bool(interleaved)))
    return dq, dk, dw[0], dw[1]


def _make_function():

    class QkNormRopeFunction(torch.autograd.Function):
        """``qk_norm_rope`` with its gradient for q, k and the weights."""

        @staticmethod
        def forward(ctx, q, k, cos, sin, q_weight, k_weight, positions, eps, norm, interleaved, fold_heads, axes):
            ctx.save_for_backward(q, k, cos, sin, q_weight, k_weight, positions)
            ctx.attrs = dict(eps=eps, norm=norm, interleaved=interleaved, fold_heads=fold_heads, axes=axes)
            return qk_norm_rope(q, k, cos, sin, q_weight, k_weight, positions, **ctx.attrs)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, d_q_out, d_k_out):
            dq, dk, dqw, dkw = qk_norm_rope_grad(d_q_out, d_k_out, *ctx.saved_tensors, **ctx.attrs)
            return dq, dk, None, None, dqw, dkw, None, None, None, None, None, None

    return QkNormRopeFunction


_fn = None


def qk_norm_rope_autograd(q, k, cos, sin, q_weight=None, k_weight=None, positions=None, eps: float = 1e-6,
                          norm: bool = True, interleaved: bool = False, fold_heads: bool = True, axes=None):
    """Differentiable ``qk_norm_rope`` (once; no gradient for the tables)."""
    global _fn
    if _fn is None:
        _fn = _make_function()
    if axes is not None:
        axes = tuple(axes)  # (a list may change before the backward pass)
    return _fn.apply(q, k, cos, sin, q_weight, k_weight, positions, eps, norm, interleaved, fold_heads, axes)


def _check_cache(k_cache, v_cache, T):
    if k_cache.dim() != 4 or v_cache.dim() != 4:
        _fail("k_cache and v_cache must be [pages, heads, tokens per page, features]")
    if k_cache.shape[:3] != v_cache.shape[:3]:
        _fail(f"k_cache {list(k_cache.shape)} and v_cache {list(v_cache.shape)} differ in pages, heads or page size")
    if k_cache.dtype != T or v_cache.dtype != T:
        _fail("a cache in 4 bits is uint8 (fp4_cache)" if T is _U8 else "the caches must have the same dtype T as the tokens")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        _fail("k_cache and v_cache must be contiguous")
    _sizes_fit(k_cache=k_cache, v_cache=v_cache)


def _check_batch(page_table, q_starts, kv_lens):
    """(N, width) of a batch over the cache."""
    if page_table.dim() != 2:
        _fail("page_table must be [sequences, pages per sequence]")
    N, width = page_table.shape
    _int32("page_table", page_table, N, width)
    _int32("q_starts", q_starts, N + 1)
    _int32("kv_lens", kv_lens, N)
    if width > 1 and page_table.stride(1) != 1:
        _fail("the rows of page_table must be contiguous")
    if (N > 0 and q_starts.stride(0) != 1) or (N > 1 and kv_lens.stride(0) != 1):
        _fail("q_starts and kv_lens must be contiguous")
    _sizes_fit(page_table=page_table)
    return N, width


def _plain_batch(device, T, k_cache, v_cache, page_table, q_starts, kv_lens):
    """(N, width) of arguments that pass ``_check_cache``, ``_check_batch`` and
    ``_on_device`` by a few comparisons, None of others."""
    st, sk, sv = page_table.shape, k_cache.shape, v_cache.shape
    if (device.type == "cuda" and k_cache.dtype is T and v_cache.dtype is T and k_cache.device == device
            and v_cache.device == device and len(sk) == 4 and len(sv) == 4 and sk[:3] == sv[:3]
            and sum(sk) + sv[3] + sum(st) <= _MOST and k_cache.is_contiguous() and v_cache.is_contiguous() and len(st) == 2 and page_table.dtype is _I32
            and q_starts.dtype is _I32 and kv_lens.dtype is _I32 and page_table.device == device
            and q_starts.device == device and kv_lens.device == device and q_starts.shape == (st[0] + 1,)
            and kv_lens.shape == (st[0],) and page_table.is_contiguous() and q_starts.is_contiguous()
            and kv_lens.is_contiguous()):
        return st
    return None


def _check_tokens(name, t, T, features=None):
    if t.dim() != 3 or (features is not None and t.shape[2] != features):
        _fail(f"{name} must be [tokens, heads{'' if features is None else f', {features}'}], got {list(t.shape)}")
    if t.dtype != T:
        _fail(f"{name} must have dtype {T}, got {t.dtype}")
    if sum(t.shape) > _MOST:
        _sizes_fit(**{name: t})


def _check_append(k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos, sin, q, q_weight, k_weight, norm, fp4):
    """Checks of ``kv_append``: (N, width) and (dtype code, table rows, rotated features, weights' code)."""
    T = k.dtype
    _check_tokens("k", k, T)
    _check_tokens("v", v, T)
    code = _dtype_code(k)
    _check_cache(k_cache, v_cache, _U8 if fp4 else T)
    batch = _check_batch(page_table, q_starts, kv_lens)
    n, H_kv, D_qk = k.shape
    if v.shape[:2] != k.shape[:2]:
        _fail(f"k {list(k.shape)} and v {list(v.shape)} differ in tokens or heads")
    row_k, row_v = (_fp4_bytes(D_qk), _fp4_bytes(v.shape[2])) if fp4 else (D_qk, v.shape[2])
    if k_cache.shape[1] != H_kv or k_cache.shape[3] != row_k or v_cache.shape[3] != row_v or (fp4 and not (row_k and row_v)):
        _fail(f"the caches {list(k_cache.shape)}, {list(v_cache.shape)} do not hold rows of k {list(k.shape)} and v "
              f"{list(v.shape)}")
    if q is not None:
        _check_tokens("q", q, T, D_qk)
        if q.shape[0] != n:
            _fail(f"q has {q.shape[0]} tokens, k {n}")
    rows, R = _tables(cos, sin)
    w_code = _weight_dtype(T, D_qk, q_weight, k_weight, norm)
    _on_device(k.device, v=v, cos=cos, sin=sin, q=q, q_weight=q_weight, k_weight=k_weight, k_cache=k_cache,
               v_cache=v_cache, page_table=page_table, q_starts=q_starts, kv_lens=kv_lens)
    return batch, (code, rows, R, w_code)


def _plain_append(k, v, sk_cache, sv_cache, cos, sin, q, q_weight, k_weight, norm, fp4):
    """What ``_check_append`` returns second, of usual arguments that pass its
    checks by a few comparisons; None of others."""
    sk, sv, T, device = k.shape, v.shape, k.dtype, k.device
    code = _CODES.get(T)
    if (code is None or q is None or cos is None or sin is None or len(sk) != 3 or len(sv) != 3 or v.dtype is not T
            or q.dtype is not T or v.device != device or q.device != device or cos.device != device or sin.device != device):
        return None
    n, H_kv, D = sk
    sq, sc = q.shape, cos.shape
    row_k, row_v = (_fp4_bytes(D), _fp4_bytes(sv[2])) if fp4 else (D, sv[2])
    if not (sv[0] == n and sv[1] == H_kv == sk_cache[1] and sk_cache[3] == row_k and sv_cache[3] == row_v and len(sq) == 3
            and sq[0] == n and sq[2] == D and len(sc) == 2 and sin.shape == sc and cos.dtype is _F32 and sin.dtype is _F32
            and sum(sq) + sum(sc) <= _MOST):
        return None
    if q_weight is not None or k_weight is not None:
        if (not norm or q_weight is None or k_weight is None or q_weight.dtype is not k_weight.dtype
                or q_weight.dtype not in (T, _F32) or q_weight.shape != (D,) or k_weight.shape != (D,)
                or q_weight.device != device or k_weight.device != device):
            return None
        return code, sc[0], 2 * sc[1], _CODES[q_weight.dtype]
    return code, sc[0], 2 * sc[1], DTYPE_F32


Reserved = collections.namedtuple("Reserved", "q_starts kv_lens free_count positions slots")


def _vector(name, t, n, *dtypes):
    """``t`` is a dense vector of n entries (None: of any number) of one of the dtypes."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        _fail(f"{name} must be a tensor of {' or '.join(str(d) for d in dtypes)}")
    if t.dim() != 1 or (n is not None and t.shape[0] != n):
        _fail(f"{name} must have shape [{'entries' if n is None else n}], got {list(t.shape)}")
    if not t.is_contiguous():
        _fail(f"{name} must be contiguous")


def kv_reserve(page_table, kv_lens, new_lens, free_pages, free_count, page_size: int, total: int, finished=None,
               in_place: bool = False, short=None):
    """Pages for the new tokens of a batch, and where each token goes, all on the GPU.

    page_table int32 [N, pages per sequence] and kv_lens int32 [N] say what the N sequences hold,
    new_lens int32 [N] how many tokens each of them gets, free_pages int32 [capacity] is a stack of pages that
    none holds: its first free_count (int32 [1]) entries.  Sequences with ``finished`` (bool or uint8 [N])
    first give the pages of their tokens back; their length is 0 then (new tokens begin a new sequence there).
    Every column that the new tokens are the first to need gets the page on top of the stack, in the order
    sequence, column; once the stack is empty -1.  page_table and free_pages are changed in place.

    Returns ``Reserved``: q_starts [N + 1] and kv_lens [N], as ``kv_append`` and ``paged_sdpa`` take them;
    free_count [1]; and for the ``total`` packed tokens positions (int32, the place in the sequence) and
    slots (int64, page * page_size + row; -1 without a page), -1 behind the last.  ``in_place``: kv_lens
    and free_count are the tensors given, changed (for a captured step that is replayed).

    ``short`` (int32 [1]) receives how many pages the stack lacked.  A column that got -1 for want of one stays so, and
    what sees its tokens is NaN, until its sequence is finished: that gives back the pages it has, and it
    can begin anew at once.  Where not ``in_place``, the call can also be made again, with the same kv_lens and free_count,
    fewer new_lens or more of ``finished``, as long as no sequence that was finished got new tokens.

    More tokens than ``total`` have no rows: ``kv_append`` and ``paged_sdpa`` leave out the sequences that reach past it, whole.
    Those have their pages and lengths all the same (of a sequence's new tokens ``total`` count at most), so that their new
    tokens are to be appended, by a further call with q_starts of its own, before anything is attended over them.
    """
    N, width, capacity, device = _check_reserve(page_table, kv_lens, new_lens, free_pages, free_count, page_size, total, finished,
                                                short)
    table, lens, fresh, pages, count, ended = (page_table.data_ptr(), kv_lens.data_ptr(), new_lens.data_ptr(), free_pages.data_ptr(),
                                               free_count.data_ptr(), _ptr(finished))
    # what is written shares memory with nothing else
    stride = page_table.stride(0)
    reads = [(lens, 4 * N), (fresh, 4 * N), (count, 4)]
    if ended is not None:
        reads.append((ended, N))
    table_bytes = 4 * ((N - 1) * stride + width) if N and width else 0
    for start, size in reads:
        if (start < table + table_bytes and table < start + size) or (start < pages + 4 * capacity and pages < start + size):
            _fail("page_table, free_pages, kv_lens and free_count must not share memory")
    if pages < table + table_bytes and table < pages + 4 * capacity:
        _fail("page_table, free_pages, kv_lens and free_count must not share memory")
    lack = None
    if short is not None:
        lack = short.data_ptr()
        for start, size in reads + [(table, table_bytes), (pages, 4 * capacity)]:
            if start < lack + 4 and lack < start + size:
                _fail("short must be memory of its own")
    new = kv_lens.new_empty
    if in_place:
        for start, size in reads[1:]:
            if start < lens + 4 * N and lens < start + size:
                _fail("kv_lens and free_count must be memory of their own")
        for start, size in reads[1:2] + reads[3:]:
            if start < count + 4 and count < start + size:
                _fail("kv_lens and free_count must be memory of their own")
        out = Reserved(new(N + 1), kv_lens, free_count, new(total), new(total, dtype=torch.int64))
    else:
        out = Reserved(new(N + 1), new(N), new(1), new(total), new(total, dtype=torch.int64))
    _call(library().sdpa_hip_kv_reserve_counted, device, table, stride, lens, fresh, ended, pages, count, out[0].data_ptr(),
          out[1].data_ptr(), out[2].data_ptr(), lack, out[3].data_ptr(), out[4].data_ptr(), N, total, width, page_size, capacity)
    return out


def _check_reserve(page_table, kv_lens, new_lens, free_pages, free_count, page_size, total, finished, short):
    """Checks of ``kv_reserve`` but for shared memory: (N, width, capacity, device)."""
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2:
        _fail("page_table must be [sequences, pages per sequence]")
    N, width = page_table.shape
    device = page_table.device
    if short is not None:
        _vector("short", short, 1, _I32)
    one, sizes = (N,), type(page_size) is int and type(total) is int and 0 <= total <= _MOST and 0 < page_size <= _MOST
    # (usual arguments by a few comparisons, others one by one)
    if (sizes and page_table.dtype is _I32 and page_table.is_contiguous() and device.type == "cuda"
            and isinstance(kv_lens, torch.Tensor) and isinstance(new_lens, torch.Tensor) and isinstance(free_pages, torch.Tensor)
            and isinstance(free_count, torch.Tensor)
            and kv_lens.dtype is _I32 and new_lens.dtype is _I32 and free_pages.dtype is _I32 and free_count.dtype is _I32
            and kv_lens.shape == one and new_lens.shape == one and free_count.shape == (1,) and free_pages.dim() == 1
            and kv_lens.is_contiguous() and new_lens.is_contiguous() and free_pages.is_contiguous()
            and kv_lens.device == device and new_lens.device == device and free_pages.device == device and free_count.device == device
            and (finished is None or (isinstance(finished, torch.Tensor) and finished.dtype in (torch.bool, _U8)
                                      and finished.shape == one and finished.is_contiguous() and finished.device == device))
            and (short is None or short.device == device)):
        capacity = free_pages.shape[0]
        if N + width + capacity <= _MOST:
            return N, width, capacity, device
    _int32("page_table", page_table, N, width)
    if (width > 1 and page_table.stride(1) != 1) or (N > 1 and page_table.stride(0) < width):
        _fail("the rows of page_table must be contiguous and memory of their own")
    _vector("kv_lens", kv_lens, N, _I32)
    _vector("new_lens", new_lens, N, _I32)
    _vector("free_pages", free_pages, None, _I32)
    _vector("free_count", free_count, 1, _I32)
    if finished is not None:
        _vector("finished", finished, N, torch.bool, _U8)
    if not sizes:
        _fail("page_size and total must be sizes")
    _sizes_fit(page_table=page_table, free_pages=free_pages)
    _on_device(device, kv_lens=kv_lens, new_lens=new_lens, free_pages=free_pages, free_count=free_count, finished=finished,
               short=short)
    return N, width, free_pages.shape[0], device


def _append_positions(positions, axes, cos, n, device):
    """Positions [axes, n] of the new tokens, the axes of the pairs and their number; [n]
    without ``axes``: one axis."""
    if axes is None:
        if cos is None:
            _fail("positions need cos and sin")
        if cos.dim() != 2:
            _fail("cos and sin must have one shape [positions, rotated features / 2]")
        _int32("positions", positions, n)
        positions, axes = positions[None], (0,) * cos.shape[1]
    pairs, n_axes = _axes_args(axes, positions, cos, n)
    _on_device(device, positions=positions)
    return positions.contiguous(), pairs, n_axes


def kv_append(k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos=None, sin=None, q=None, q_weight=None,
              k_weight=None, norm: bool = False, eps: float = 1e-6, interleaved: bool = False, positions=None, axes=None):
    """Appends new tokens to a paged cache, in place, and returns their rotated queries.

    k [T, H_kv, D_qk] and v [T, H_kv, D_v] are the packed new tokens of N sequences (any strides):
    those of sequence s are q_starts[s] .. q_starts[s + 1] - 1 (int32 [N + 1]).  kv_lens (int32 [N])
    counts its cached tokens with the new ones, which are the last.  Token j of s goes to row j % page of page
    page_table[s, j // page] (int32 [N, pages per sequence]) of the caches [pages, H_kv, page, D],
    page a power of two of at least 16.  On the way k is normed (``norm``, ``k_weight``) and rotated
    by j as in ``qk_norm_rope`` (cos and sin None: not), and so is q [T, H_q, D_qk], where given:
    the result is [T, H_q, D_qk], else None.  ``positions``: what the tokens are rotated by instead of their
    places j: int32 [T], or [axes, T] with ``axes``, the axis of each rotated pair, as in ``qk_norm_rope``.

    Tokens behind the last sequence are skipped (their rows of the result are not written), and so are those of a
    sequence that reaches past the T tokens.  A token
    without a place in the table or the cache is not appended and its query row is NaN.  No two tokens
    of a call may have the same place.  D_qk or D_v may be 0 (a cache of keys or of values alone).
    Any width up to 128 can be cached; ``paged_sdpa`` reads multiples of 8 (fp16) or 4 (fp32).
    """
    return _append(False, k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos, sin, q, q_weight, k_weight, norm, eps,
                   interleaved, positions, axes)


def _append(fp4, k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos, sin, q, q_weight, k_weight, norm, eps, interleaved,
            positions, axes):
    T, device = k.dtype, k.device
    L = library()
    entry, by = (L.sdpa_hip_kv_append_fp4, (None, None, 0)) if fp4 else (L.sdpa_hip_kv_append, ())
    if positions is not None or axes is not None:
        positions, pairs, n_axes = _append_positions(positions, axes, cos, k.shape[0], device)
        by = (positions.data_ptr(), pairs, n_axes)
        if not fp4:
            entry = L.sdpa_hip_kv_append_axes
    batch = _plain_batch(device, _U8 if fp4 else T, k_cache, v_cache, page_table, q_starts, kv_lens)
    checked = None
    if batch is not None:
        checked = _plain_append(k, v, k_cache.shape, v_cache.shape, cos, sin, q, q_weight, k_weight, norm, fp4)
    if checked is None:
        batch, checked = _check_append(k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos, sin, q, q_weight,
                                       k_weight, norm, fp4)
    N, width = batch
    code, rows, R, w_code = checked
    n, H_kv, D_qk = k.shape
    D_v = v.shape[2]
    pages, _, page, _ = k_cache.shape
    H_q = 0 if q is None else q.shape[1]
    k, v = _dense_features(k), _dense_features(v)
    cos, sin, q_weight, k_weight = _dense(cos), _dense(sin), _dense(q_weight), _dense(k_weight)
    q_out = None
    if q is not None:
        q = _dense_features(q)
        q_out = torch.empty((n, H_q, D_qk), dtype=T, device=device)
    _call(entry, device, code, k.data_ptr(), _strides2(k.stride()), v.data_ptr(), _strides2(v.stride()),
          k_cache.data_ptr(), v_cache.data_ptr(), _ptr(q), None if q is None else _strides2(q.stride()), _ptr(q_out), None,
          _ptr(q_weight), _ptr(k_weight), w_code, _ptr(cos), _ptr(sin), rows, *by, page_table.data_ptr(),
          page_table.stride(0), q_starts.data_ptr(), kv_lens.data_ptr(), N, n, width, pages, page, H_q, H_kv, D_qk,
          D_v, R, float(eps), int(bool(norm)), int(bool(interleaved)))
    return q_out


def _fp4_bytes(D):
    """Bytes of a token's D features in a cache in 4 bits (0: no such width)."""
    return D // 2 + D // 32 if D % 32 == 0 and 0 < D <= 128 else 0


def _fp4_features(cache):
    """Features of a cache in 4 bits."""
    D = cache.shape[3] // 17 * 32
    if not cache.shape[3] or _fp4_bytes(D) != cache.shape[3]:
        _fail(f"a cache in 4 bits has 17, 34, 51 or 68 bytes a token and head, not {cache.shape[3]}")
    return D


def fp4_cache(pages: int, heads: int, page_size: int, D_qk: int, D_v: int, device="cuda"):
    """An empty cache in 4 bits: ``(k_cache, v_cache)``, uint8 [pages, heads, page_size, 17 * D / 32].

    32 neighbouring features of a token and head share a scale (8 bits), so a value takes 4.25 bits; D_qk and
    D_v are 32, 64, 96 or 128.  What a value becomes, and where the bytes of a page lie, stands in
    ``include/sdpa_hip.h``.  ``kv_append_fp4`` fills it, ``paged_sdpa_fp4`` attends over it, ``kv_read_fp4`` reads it.
    """
    for D in (D_qk, D_v):
        if not _fp4_bytes(D):
            _fail(f"feature sizes of a cache in 4 bits must be 32, 64, 96 or 128, got {D}")
    if page_size < 16 or page_size > 65536 or page_size & (page_size - 1):
        _fail("tokens per page must be a power of two from 16 to 65536")
    return tuple(torch.zeros((pages, heads, page_size, _fp4_bytes(D)), dtype=_U8, device=device) for D in (D_qk, D_v))


def kv_append_fp4(k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos=None, sin=None, q=None, q_weight=None,
                  k_weight=None, norm: bool = False, eps: float = 1e-6, interleaved: bool = False, positions=None, axes=None):
    """``kv_append`` into a cache in 4 bits (``fp4_cache``), with the same arguments and result.

    The keys are rounded after norm and rotation, which are formed in fp64 for them, so that a token's codes do
    not depend on what else is in the call.  Groups of 32 features that hold an infinity or a NaN become
    NaN, values beyond 61440 in size become that.  No two sequences of a call may append to the same 8 tokens (8 i .. 8 i + 7) of a page.
    """
    return _append(True, k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos, sin, q, q_weight, k_weight, norm, eps,
                   interleaved, positions, axes)


def kv_read_fp4(k_cache, v_cache, page_table, q_starts, kv_lens, total: int, dtype=torch.float16):
    """The values of a batch's tokens out of a cache in 4 bits: ``(k, v)``, [total, H_kv, D] in ``dtype``.

    The batch as in ``kv_append``: of sequence s its last q_starts[s + 1] - q_starts[s] cached tokens (all of them where that
    is kv_lens[s]; those that lie in the first ``total`` rows).  The values are exact (fp16 or fp32).  Rows of a token
    without a place are NaN, those behind the last sequence arbitrary.
    """
    batch = _plain_batch(k_cache.device, _U8, k_cache, v_cache, page_table, q_starts, kv_lens)
    plain = batch is not None
    if not plain:
        _check_cache(k_cache, v_cache, _U8)
        batch = _check_batch(page_table, q_starts, kv_lens)
    D_qk, D_v = _fp4_features(k_cache), _fp4_features(v_cache)
    if not plain:
        _on_device(k_cache.device, v_cache=v_cache, page_table=page_table, q_starts=q_starts, kv_lens=kv_lens)
    if type(total) is not int or not 0 <= total <= _MOST:
        _fail("total must be a size")
    if dtype not in _CODES:
        _fail(f"T must be half or float, got {dtype}")
    N, width = batch
    pages, H_kv, page, _ = k_cache.shape
    k, v = (torch.empty((total, H_kv, D), dtype=dtype, device=k_cache.device) for D in (D_qk, D_v))
    _call(library().sdpa_hip_kv_read_fp4, k_cache.device, _CODES[dtype], k_cache.data_ptr(), v_cache.data_ptr(), k.data_ptr(),
          v.data_ptr(), page_table.data_ptr(), page_table.stride(0), q_starts.data_ptr(), kv_lens.data_ptr(), N, total, width,
          pages, page, H_kv, D_qk, D_v)
    return k, v


def _whole_chunks(t):
    """``t`` with rows of whole 16-byte chunks (as far as its features allow)."""
    e = t.element_size()
    if t.stride(-1) != 1 or t.stride(0) * e % 16 or t.stride(1) * e % 16:
        t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _share_memory(a, b):
    """The spans of ``a`` (contiguous) and ``b`` overlap."""
    if not a.numel() or not b.numel():
        return False
    end = b.data_ptr() + b.element_size() * (1 + sum((n - 1) * s for n, s in zip(b.shape, b.stride())))
    return a.data_ptr() < end and b.data_ptr() < a.data_ptr() + a.numel() * a.element_size()


def paged_sdpa(q, k_cache, v_cache, page_table, q_starts, kv_lens, scale: float = 1.0, causal_mask: bool = True,
               max_q_len=None, out=None):
    """Attention of new tokens over a paged cache that holds them already: ``(o, stats)``.

    q [T, H_q, D_qk] and the batch as in ``kv_append``; H_q is a multiple of the caches' heads, and
    query head h reads key head h // (H_q // H_kv).  Token i of a sequence's n new ones sees its keys
    j <= kv_len - n + i (``causal_mask``; else all of them).  o [T, H_q, D_v] in T; stats [T, H_q]
    float32 is the logarithm of the sum of the exponentials of the scaled scores.  A row that sees
    nothing has o = 0 and stats = -inf.  What the pages hold behind a row's last key has no influence.

    ``max_q_len``: the most new tokens of a sequence, where it is known (1 in generation); it chooses
    kernels only.  ``out``: (o, stats) to write into, memory of their own; rows of tokens of no sequence stay as they were
    (in new ones they are arbitrary).  Feature sizes are multiples of 8 (fp16) or 4 (fp32), up to 128.
    """
    return _paged(False, q, k_cache, v_cache, page_table, q_starts, kv_lens, scale, causal_mask, max_q_len, out)


def paged_sdpa_fp4(q, k_cache, v_cache, page_table, q_starts, kv_lens, scale: float = 1.0, causal_mask: bool = True,
                   max_q_len=None, out=None):
    """``paged_sdpa`` over a cache in 4 bits (``fp4_cache``, ``kv_append_fp4``): ``(o, stats)``.

    Arguments and results as there; the queries are fp16 or fp32, and the cache's values exact in either.  The weights
    enter the product with the values in 22 bits, but in 11 for fp16 queries of more than 32 rows (tokens times the
    query heads of a key head; unless few keys carry a row), as with ``paged_sdpa``.
    """
    return _paged(True, q, k_cache, v_cache, page_table, q_starts, kv_lens, scale, causal_mask, max_q_len, out)


def _paged(fp4, q, k_cache, v_cache, page_table, q_starts, kv_lens, scale, causal_mask, max_q_len, out):
    T = q.dtype
    _check_tokens("q", q, T)
    code = _dtype_code(q)
    of = _U8 if fp4 else T
    plain = _plain_batch(q.device, of, k_cache, v_cache, page_table, q_starts, kv_lens)
    known = plain is not None
    if not known:
        _check_cache(k_cache, v_cache, of)
        plain = _check_batch(page_table, q_starts, kv_lens)
    N, width = plain
    n, H_q, D_qk = q.shape
    pages, H_kv, page, D_v = v_cache.shape
    D_k = k_cache.shape[3]
    if fp4:
        D_k, D_v = _fp4_features(k_cache), _fp4_features(v_cache)
    if D_k != D_qk:
        _fail(f"q has {D_qk} features, k_cache {D_k}")
    if out is None:
        if not known:
            _on_device(q.device, k_cache=k_cache, v_cache=v_cache, page_table=page_table, q_starts=q_starts, kv_lens=kv_lens)
        o = torch.empty((n, H_q, D_v), dtype=T, device=q.device)
        stats = torch.empty((n, H_q), dtype=torch.float32, device=q.device)
    else:
        o, stats = out
        if o.dtype != T or tuple(o.shape) != (n, H_q, D_v) or stats.dtype != torch.float32 or tuple(stats.shape) != (n, H_q):
            _fail(f"out must be ({T} {[n, H_q, D_v]}, float32 {[n, H_q]})")
        if not (o.is_contiguous() and stats.is_contiguous()):
            _fail("out must be contiguous")
        _on_device(q.device, k_cache=k_cache, v_cache=v_cache, page_table=page_table, q_starts=q_starts, kv_lens=kv_lens,
                   o=o, stats=stats)
        for name, t in (("q", q), ("k_cache", k_cache), ("v_cache", v_cache)):
            if _share_memory(o, t) or _share_memory(stats, t):
                _fail(f"out must not share memory with {name}")
        if _share_memory(o, stats):
            _fail("the tensors of out must not share memory")
    L = library()
    size, entry = ((L.sdpa_hip_paged_fwd_fp4_workspace_bytes, L.sdpa_hip_paged_fwd_fp4) if fp4 else
                   (L.sdpa_hip_paged_fwd_workspace_bytes, L.sdpa_hip_paged_fwd))
    longest = 0 if max_q_len is None else int(max_q_len)
    ws_bytes = size(code, N, n, width, page, H_q, H_kv, D_qk, D_v, longest)
    ws = _workspace(torch, ws_bytes, q.device) if ws_bytes else None
    q = _whole_chunks(q)
    _call(entry, q.device, code, q.data_ptr(), _strides2(q.stride()), k_cache.data_ptr(), v_cache.data_ptr(),
          o.data_ptr(), None, stats.data_ptr(), page_table.data_ptr(), page_table.stride(0), q_starts.data_ptr(),
          kv_lens.data_ptr(), _ptr(ws), ws_bytes if ws is not None else 0, N, n, width, pages, page, H_q, H_kv, D_qk,
          D_v, longest, float(scale), int(bool(causal_mask)))
    return o, stats
