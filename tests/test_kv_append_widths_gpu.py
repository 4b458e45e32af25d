"""kv_append of keys or values without features: that side is left out (an empty
tensor has no address), the other is appended as beside a side with features."""
import ctypes

import pytest
import torch

import _heads as R64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H_Q, H_KV, PAGE, N_TOK = 4, 2, 16, 23


def _batch():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    return i32([[4, 0, 2], [1, 3, 5]]), i32([0, 20, 22]), i32([40, 17])  # the last token is behind the sequences


def _side(d, T, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((N_TOK, H_KV, d), generator=g).to(T).to(DEV),
            torch.randn((6, H_KV, PAGE, d), generator=g).to(T).to(DEV))


@pytest.mark.parametrize("T", [torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 33])  # rows of whole chunks, and not
@pytest.mark.parametrize("empty", ["k", "v", "both"])
def test_sides_without_features(pkg, T, D, empty):
    D_qk, D_v = (0 if empty in (x, "both") else D for x in ("k", "v"))
    (k, kc), (v, vc) = _side(D, T, 1), _side(D, T, 2)
    q = _side(D, T, 3)[0].repeat(1, H_Q // H_KV, 1)
    cos, sin = (t.to(DEV) for t in R64.tables(64, 32))
    batch = _batch()
    want_k, want_v = kc.clone(), vc.clone()
    want_q = pkg.kv_append(k, v, want_k, want_v, *batch, cos, sin, q=q)
    got_k, got_v = kc[..., :D_qk].contiguous(), vc[..., :D_v].contiguous()
    turn = (cos, sin) if D_qk else (None, None)
    got_q = pkg.kv_append(k[..., :D_qk], v[..., :D_v], got_k, got_v, *batch, *turn, q=q[..., :D_qk])
    torch.cuda.synchronize()
    assert got_q.shape == (N_TOK, H_Q, D_qk)
    if D_qk:
        assert torch.equal(got_k, want_k) and torch.equal(got_q[:22], want_q[:22])
    if D_v:
        assert torch.equal(got_v, want_v)


@pytest.mark.parametrize("empty", ["k", "v", "both"])
def test_null_pointers_of_sides_without_features(pkg, empty):
    """The C entry takes NULL for what has no features."""
    D_qk, D_v = (0 if empty in (x, "both") else 64 for x in ("k", "v"))
    (k, kc), (v, vc) = _side(64, torch.float16, 1), _side(64, torch.float16, 2)
    want_k, want_v = kc.clone(), vc.clone()
    batch = _batch()
    pkg.kv_append(k, v, want_k, want_v, *batch)
    at = lambda t, d: t.data_ptr() if d else None
    dense = (ctypes.c_int64 * 2)(H_KV * 64, 64)
    rc = pkg.library().sdpa_hip_kv_append(
        1, at(k, D_qk), dense, at(v, D_v), dense, at(kc, D_qk), at(vc, D_v), None, None, None, None, None, None, 0, None, None,
        0, batch[0].data_ptr(), 3, batch[1].data_ptr(), batch[2].data_ptr(), 2, N_TOK, 3, 6, PAGE, 0, H_KV, D_qk, D_v, 0, 1e-6,
        0, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    if D_qk:
        assert torch.equal(kc, want_k)
    if D_v:
        assert torch.equal(vc, want_v)
