"""The steps around ``sdpa`` of a layer of a language model: norm and rotation
of queries and keys (with the gradient), and a paged cache of keys and values.

As with the op itself, torch tensors are device memory and streams only; the
arithmetic runs in the HIP kernels behind ``include/sdpa_hip.h``, fp16 or fp32.
Arguments that the device alone knows (lengths, page tables, positions) are
checked there, where they are used.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import (DTYPE_F16, DTYPE_F32, InvalidArgumentError, _dtype_code, _raise_for, _stream_handle, _workspace,
               library)

_Strides3 = ctypes.c_int64 * 3
_Strides2 = ctypes.c_int64 * 2


_F32, _I32 = torch.float32, torch.int32
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


def _call(entry, device, *args):
    """``entry(*args, stream)`` with ``device`` current."""
    if torch.cuda.current_device() == device.index:
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


def _plain_rope(q, k, cos, sin, q_weight, k_weight, positions, norm):
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
        if S > sc[0]:
            return None
    else:
        sp = positions.shape
        per_batch = int(len(sp) == 2)
        if (sp != ((B, S) if per_batch else (S,)) or positions.dtype is not _I32 or positions.device != device
                or not positions.is_contiguous()):
            return None
    w_code = DTYPE_F32
    if w is not None or k_weight is not None:
        if (not norm or w is None or k_weight is None or w.dtype is not k_weight.dtype or w.dtype not in (T, _F32)
                or w.shape != (D,) or k_weight.shape != (D,) or w.device != device or k_weight.device != device
                or not w.is_contiguous() or not k_weight.is_contiguous()):
            return None
        w_code = _CODES[w.dtype]
    return code, (B, S, H_q, sk[2], D, 2 * sc[1]), (cos, sin, sc[0]), (w, k_weight, w_code), positions, per_batch


def _rope_args(q, k, cos, sin, q_weight, k_weight, positions, norm):
    """Checks of what the forward and the gradient have in common."""
    plain = _plain_rope(q, k, cos, sin, q_weight, k_weight, positions, norm)
    if plain is not None:
        return plain
    _check_qk(q, k)
    code = _dtype_code(q)
    B, S, H_q, D = q.shape
    rows, R = _tables(cos, sin)
    w_code = _weight_dtype(q.dtype, D, q_weight, k_weight, norm)
    per_batch = 0
    if positions is not None:
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
                 norm: bool = True, interleaved: bool = False, fold_heads: bool = True):
    """RMS norm of every head of q and k, and its rotation by position: ``(q_out, k_out)``.

    q [B, S, H_q, D] and k [B, S, H_kv, D] (fp16 or fp32; any strides, so both may be parts of one
    projection's output; D <= 128).  ``norm``: each row divided by sqrt(mean of its squares + eps)
    and multiplied by its weight [D] (dtype T or float32), if there is one.  The first R features,
    R = 2 * cos.shape[1], are rotated by row ``positions`` (int32 [S] or [B, S]; None: 0 .. S - 1) of the float32 tables
    cos and sin [P, R / 2]: pairs (i, i + R/2), or (2i, 2i + 1) if ``interleaved``; without tables
    (None) nothing is.  A position outside the tables makes its rows NaN.

    ``fold_heads``: results [B * H, S, D], the layout of ``sdpa``; else [B, S, H, D].
    """
    code, (B, S, H_q, H_kv, D, R), tables, weights, positions, per_batch = _rope_args(
        q, k, cos, sin, q_weight, k_weight, positions, norm)
    q, k = _dense_features(q), _dense_features(k)
    q_out, qos = _out_rows(q, B, S, H_q, D, fold_heads)
    k_out, kos = _out_rows(k, B, S, H_kv, D, fold_heads)
    _call(library().sdpa_hip_qk_norm_rope, q.device, code, q.data_ptr(), _strides3(q.stride()), k.data_ptr(), _strides3(k.stride()),
          q_out.data_ptr(), qos, k_out.data_ptr(), kos, _ptr(weights[0]), _ptr(weights[1]), weights[2],
          _ptr(tables[0]), _ptr(tables[1]), tables[2], _ptr(positions), per_batch, B, S, H_q, H_kv, D, R, float(eps),
          int(bool(norm)), int(bool(interleaved)))
    return q_out, k_out


def qk_norm_rope_grad(d_q_out, d_k_out, q, k, cos, sin, q_weight=None, k_weight=None, positions=None,
                      eps: float = 1e-6, norm: bool = True, interleaved: bool = False, fold_heads: bool = True):
    """Gradient of ``qk_norm_rope``: ``(dq, dk, dq_weight, dk_weight)``.

    ``d_q_out`` and ``d_k_out`` are laid out as its results; dq and dk come as
    dense [B, S, H, D], the weights' gradients in their dtype, None for a
    weight that was not given.
    """
    code, (B, S, H_q, H_kv, D, R), tables, weights, positions, per_batch = _rope_args(
        q, k, cos, sin, q_weight, k_weight, positions, norm)
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
    _call(L.sdpa_hip_qk_norm_rope_grad, q.device, code, grads[0][0].data_ptr(), grads[0][1], grads[1][0].data_ptr(),
          grads[1][1], q.data_ptr(), _strides3(q.stride()), k.data_ptr(), _strides3(k.stride()), dq.data_ptr(), None, dk.data_ptr(),
          None, _ptr(dw[0]), _ptr(dw[1]), _ptr(weights[0]), _ptr(weights[1]), weights[2], _ptr(tables[0]),
          _ptr(tables[1]), tables[2], _ptr(positions), per_batch, _ptr(ws), ws_bytes, B, S, H_q, H_kv, D, R,
          float(eps), int(bool(norm)), int(bool(interleaved)))
    return dq, dk, dw[0], dw[1]


def _make_function():

    class QkNormRopeFunction(torch.autograd.Function):
        """``qk_norm_rope`` with its gradient for q, k and the weights."""

        @staticmethod
        def forward(ctx, q, k, cos, sin, q_weight, k_weight, positions, eps, norm, interleaved, fold_heads):
            ctx.save_for_backward(q, k, cos, sin, q_weight, k_weight, positions)
            ctx.attrs = dict(eps=eps, norm=norm, interleaved=interleaved, fold_heads=fold_heads)
            return qk_norm_rope(q, k, cos, sin, q_weight, k_weight, positions, **ctx.attrs)

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, d_q_out, d_k_out):
            dq, dk, dqw, dkw = qk_norm_rope_grad(d_q_out, d_k_out, *ctx.saved_tensors, **ctx.attrs)
            return dq, dk, None, None, dqw, dkw, None, None, None, None, None

    return QkNormRopeFunction


_fn = None


def qk_norm_rope_autograd(q, k, cos, sin, q_weight=None, k_weight=None, positions=None, eps: float = 1e-6,
                          norm: bool = True, interleaved: bool = False, fold_heads: bool = True):
    """Differentiable ``qk_norm_rope`` (once; no gradient for the tables)."""
    global _fn
    if _fn is None:
        _fn = _make_function()
    return _fn.apply(q, k, cos, sin, q_weight, k_weight, positions, eps, norm, interleaved, fold_heads)


def _check_cache(k_cache, v_cache, T):
    if k_cache.dim() != 4 or v_cache.dim() != 4:
        _fail("k_cache and v_cache must be [pages, heads, tokens per page, features]")
    if k_cache.shape[:3] != v_cache.shape[:3]:
        _fail(f"k_cache {list(k_cache.shape)} and v_cache {list(v_cache.shape)} differ in pages, heads or page size")
    if k_cache.dtype != T or v_cache.dtype != T:
        _fail("the caches must have the same dtype T as the tokens")
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


def _check_append(k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos, sin, q, q_weight, k_weight, norm):
    """Checks of ``kv_append``: (N, width) and (dtype code, table rows, rotated features, weights' code)."""
    T = k.dtype
    _check_tokens("k", k, T)
    _check_tokens("v", v, T)
    code = _dtype_code(k)
    _check_cache(k_cache, v_cache, T)
    batch = _check_batch(page_table, q_starts, kv_lens)
    n, H_kv, D_qk = k.shape
    if v.shape[:2] != k.shape[:2]:
        _fail(f"k {list(k.shape)} and v {list(v.shape)} differ in tokens or heads")
    if k_cache.shape[1] != H_kv or k_cache.shape[3] != D_qk or v_cache.shape[3] != v.shape[2]:
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


def _plain_append(k, v, sk_cache, sv_cache, cos, sin, q, q_weight, k_weight, norm):
    """What ``_check_append`` returns second, of usual arguments that pass its
    checks by a few comparisons; None of others."""
    sk, sv, T, device = k.shape, v.shape, k.dtype, k.device
    code = _CODES.get(T)
    if (code is None or q is None or cos is None or sin is None or len(sk) != 3 or len(sv) != 3 or v.dtype is not T
            or q.dtype is not T or v.device != device or q.device != device or cos.device != device or sin.device != device):
        return None
    n, H_kv, D = sk
    sq, sc = q.shape, cos.shape
    if not (sv[0] == n and sv[1] == H_kv == sk_cache[1] and sk_cache[3] == D and sv_cache[3] == sv[2] and len(sq) == 3
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


def kv_append(k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos=None, sin=None, q=None, q_weight=None,
              k_weight=None, norm: bool = False, eps: float = 1e-6, interleaved: bool = False):
    """Appends new tokens to a paged cache, in place, and returns their rotated queries.

    k [T, H_kv, D_qk] and v [T, H_kv, D_v] are the packed new tokens of N sequences (any strides):
    those of sequence s are q_starts[s] .. q_starts[s + 1] - 1 (int32 [N + 1]).  kv_lens (int32 [N])
    counts its cached tokens with the new ones, which are the last.  Token j of s goes to row j % page of page
    page_table[s, j // page] (int32 [N, pages per sequence]) of the caches [pages, H_kv, page, D],
    page a power of two of at least 16.  On the way k is normed (``norm``, ``k_weight``) and rotated
    by j as in ``qk_norm_rope`` (cos and sin None: not), and so is q [T, H_q, D_qk], where given:
    the result is [T, H_q, D_qk], else None.

    Tokens behind the last sequence are skipped (their rows of the result are not written).  A token
    without a place in the table or the cache is not appended and its query row is NaN.  No two tokens
    of a call may have the same place.  D_qk or D_v may be 0 (a cache of keys or of values alone).
    Any width up to 128 can be cached; ``paged_sdpa`` reads multiples of 8 (fp16) or 4 (fp32).
    """
    T, device = k.dtype, k.device
    batch = _plain_batch(device, T, k_cache, v_cache, page_table, q_starts, kv_lens)
    checked = None
    if batch is not None:
        checked = _plain_append(k, v, k_cache.shape, v_cache.shape, cos, sin, q, q_weight, k_weight, norm)
    if checked is None:
        batch, checked = _check_append(k, v, k_cache, v_cache, page_table, q_starts, kv_lens, cos, sin, q, q_weight,
                                       k_weight, norm)
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
    _call(library().sdpa_hip_kv_append, device, code, k.data_ptr(), _strides2(k.stride()), v.data_ptr(), _strides2(v.stride()),
          k_cache.data_ptr(), v_cache.data_ptr(), _ptr(q), None if q is None else _strides2(q.stride()), _ptr(q_out), None,
          _ptr(q_weight), _ptr(k_weight), w_code, _ptr(cos), _ptr(sin), rows, page_table.data_ptr(),
          page_table.stride(0), q_starts.data_ptr(), kv_lens.data_ptr(), N, n, width, pages, page, H_q, H_kv, D_qk,
          D_v, R, float(eps), int(bool(norm)), int(bool(interleaved)))
    return q_out


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
    T = q.dtype
    _check_tokens("q", q, T)
    code = _dtype_code(q)
    plain = _plain_batch(q.device, T, k_cache, v_cache, page_table, q_starts, kv_lens)
    known = plain is not None
    if not known:
        _check_cache(k_cache, v_cache, T)
        plain = _check_batch(page_table, q_starts, kv_lens)
    N, width = plain
    n, H_q, D_qk = q.shape
    pages, H_kv, page, D_v = v_cache.shape
    if k_cache.shape[3] != D_qk:
        _fail(f"q has {D_qk} features, k_cache {k_cache.shape[3]}")
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
    longest = 0 if max_q_len is None else int(max_q_len)
    ws_bytes = L.sdpa_hip_paged_fwd_workspace_bytes(code, N, n, width, page, H_q, H_kv, D_qk, D_v, longest)
    ws = _workspace(torch, ws_bytes, q.device) if ws_bytes else None
    q = _whole_chunks(q)
    _call(L.sdpa_hip_paged_fwd, q.device, code, q.data_ptr(), _strides2(q.stride()), k_cache.data_ptr(), v_cache.data_ptr(),
          o.data_ptr(), None, stats.data_ptr(), page_table.data_ptr(), page_table.stride(0), q_starts.data_ptr(),
          kv_lens.data_ptr(), _ptr(ws), ws_bytes if ws is not None else 0, N, n, width, pages, page, H_q, H_kv, D_qk,
          D_v, longest, float(scale), int(bool(causal_mask)))
    return o, stats
