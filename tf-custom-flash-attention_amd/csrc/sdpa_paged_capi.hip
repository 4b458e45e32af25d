// sdpa_paged_capi.hip -- the extern "C" entry points of include/sdpa_hip.h for
// the norm and rotation of queries and keys and for the paged cache: argument
// checks and dispatch.
#include <stdint.h>

#include "sdpa_checks.h"
#include "sdpa_hip.h"
#include "sdpa_kv_append.h"
#include "sdpa_norm_rope.h"
#include "sdpa_paged.h"

namespace {

using sdpa::hip_status;

// Whether rows can be taken in 16-byte chunks: address and strides (of those
// dimensions that have more than one entry).
struct Chunks {
    int epc;
    bool ok = true;
    void address(const void* p) { ok = ok && ((uintptr_t)p & 15u) == 0; }
    void stride(int64_t s) { ok = ok && s % epc == 0; }
    void features(int d) { ok = ok && d % epc == 0; }
    void rotated(int R, int interleaved) { ok = ok && (interleaved ? R : R / 2) % epc == 0; }
};

// a (b + c), of sizes, fits into an int
bool rows_fit(long long a, long long b, long long c) { return a == 0 || b + c <= 0x7FFFFFFFLL / a; }

int check_rows(int dtype, int weight_dtype, const void* w0, const void* w1, const float* cos, const float* sin,
               int table_rows, int D, int R, int norm) {
    if (dtype != SDPA_DTYPE_F32 && dtype != SDPA_DTYPE_F16) return SDPA_ERR_DTYPE;
    if (D < 0 || table_rows < 0) return SDPA_ERR_NEGATIVE_DIM;
    if (D > 128) return SDPA_ERR_FEATURE_TOO_LARGE;
    if (R < 0 || R % 2 != 0 || R > D) return SDPA_ERR_ROTARY;
    if ((w0 || w1) && (!norm || (weight_dtype != dtype && weight_dtype != SDPA_DTYPE_F32))) return SDPA_ERR_WEIGHT;
    if (R > 0 && table_rows > 0 && (!cos || !sin)) return SDPA_ERR_NULL_POINTER;
    return SDPA_OK;
}

// Strides of a [B, S, H, D] tensor; those of dimensions of one entry are dropped.
sdpa::RowStrides row_strides(const int64_t* s, int B, int S, int H, int D) {
    if (!s) return sdpa::RowStrides{(long long)S * H * D, (long long)H * D, D};
    return sdpa::RowStrides{B > 1 ? s[0] : 0, S > 1 ? s[1] : 0, H > 1 ? s[2] : 0};
}

void add_rows(Chunks& c, const void* p, const sdpa::RowStrides& s) {
    c.address(p);
    c.stride(s.b);
    c.stride(s.s);
    c.stride(s.h);
}

int norm_rope_entry(bool grad, int dtype, const void* const (&x)[2], const int64_t* const (&xs)[2],
                    const void* const (&dy)[2], const int64_t* const (&dys)[2], void* const (&y)[2],
                    const int64_t* const (&ys)[2], const void* const (&w)[2], void* const (&dw)[2], int weight_dtype,
                    const float* cos, const float* sin, int table_rows, const int32_t* positions,
                    int positions_per_batch, void* workspace, size_t workspace_bytes, int B, int S, int H_q, int H_kv,
                    int D, int R, float eps, int norm, int interleaved, hipStream_t stream) {
    if (B < 0 || S < 0 || H_q < 0 || H_kv < 0) return SDPA_ERR_NEGATIVE_DIM;
    const bool any_dw = dw[0] || dw[1];
    int st = check_rows(dtype, weight_dtype, any_dw ? (dw[0] ? dw[0] : dw[1]) : w[0], w[1] ? w[1] : w[0], cos, sin,
                        table_rows, D, R, norm);
    if (st != SDPA_OK) return st;
    if (!rows_fit(B, S, 0) || !rows_fit((long long)B * S, H_q, H_kv)) return SDPA_ERR_TOO_LARGE;
    if (D == 0) return SDPA_OK;
    const bool rows = B > 0 && S > 0;
    sdpa::NormRopeParams p{};
    Chunks ch{dtype == SDPA_DTYPE_F16 ? 8 : 4};
    ch.features(D);
    ch.rotated(R, interleaved);
    ch.address(cos);
    ch.address(sin);
    ch.address(w[0]);
    ch.address(w[1]);
    for (int i = 0; i < 2; ++i) {
        sdpa::NormRopeSide& s = p.side[i];
        s.H = i == 0 ? H_q : H_kv;
        s.w = w[i];
        s.dw = dw[i];
        if (!rows || s.H == 0) continue;
        if (!x[i] || !y[i] || (grad && !dy[i])) return SDPA_ERR_NULL_POINTER;
        s.x = x[i];
        s.y = y[i];
        s.xs = row_strides(xs[i], B, S, s.H, D);
        s.ys = row_strides(ys[i], B, S, s.H, D);
        add_rows(ch, s.x, s.xs);
        add_rows(ch, s.y, s.ys);
        if (grad) {
            s.dy = dy[i];
            s.dys = row_strides(dys[i], B, S, s.H, D);
            add_rows(ch, s.dy, s.dys);
        }
    }
    if (any_dw) {
        if (!workspace || ((uintptr_t)workspace & 15u) ||
            workspace_bytes < sdpa_hip_qk_norm_rope_grad_workspace_bytes(D))
            return SDPA_ERR_WORKSPACE;
        p.part_dw = static_cast<float*>(workspace);
    }
    p.r = sdpa::RopeArgs{cos, sin, table_rows, R, norm != 0, eps, 1.f / (float)D};
    p.positions = positions;
    p.positions_stride = positions_per_batch ? S : 0;
    p.B = B;
    p.S = S;
    p.D = D;
    p.interleaved = interleaved != 0;
    p.w32 = weight_dtype == SDPA_DTYPE_F32;
    p.vec = ch.ok;
    const sdpa::DType dt = (sdpa::DType)dtype;
    return hip_status(grad ? sdpa::launch_norm_rope_grad(p, dt, stream) : sdpa::launch_norm_rope(p, dt, stream));
}

// Checks of a batch over a paged cache and its description.
int make_batch(sdpa::PagedBatch& b, const int32_t* page_table, int64_t page_table_stride, const int32_t* q_starts,
               const int32_t* kv_lens, int N, int T, int width, int pages, int page_size) {
    if (N < 0 || T < 0 || width < 0 || pages < 0) return SDPA_ERR_NEGATIVE_DIM;
    if (page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)) != 0) return SDPA_ERR_PAGE_SIZE;
    // token numbers of a sequence, and those of sequences a wave ahead, stay below 2^31
    if (N > 0x7FFFFFFF - 65536 || (long long)width * page_size > 0x7FFFFFFFLL - 65536) return SDPA_ERR_TOO_LARGE;
    if (N > 0 && T > 0 && (!q_starts || !kv_lens || (width > 0 && !page_table))) return SDPA_ERR_NULL_POINTER;
    int l2 = 4;
    while ((1 << l2) < page_size) ++l2;
    b = sdpa::PagedBatch{page_table, q_starts, kv_lens, page_table_stride, N, T, width, pages, l2};
    return SDPA_OK;
}

sdpa::TokenStrides token_strides(const int64_t* s, int T, int H, int D) {
    if (!s) return sdpa::TokenStrides{(long long)H * D, D};
    return sdpa::TokenStrides{T > 1 ? s[0] : 0, H > 1 ? s[1] : 0};
}

void add_tokens(Chunks& c, const void* p, const sdpa::TokenStrides& s) {
    c.address(p);
    c.stride(s.t);
    c.stride(s.h);
}

}  // namespace

extern "C" {

int sdpa_hip_qk_norm_rope(int dtype, const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                          void* q_out, const int64_t* q_out_strides, void* k_out, const int64_t* k_out_strides,
                          const void* q_weight, const void* k_weight, int weight_dtype, const float* cos,
                          const float* sin, int table_rows, const int32_t* positions, int positions_per_batch, int B,
                          int S, int H_q, int H_kv, int D, int R, float eps, int norm, int interleaved,
                          hipStream_t stream) {
    return norm_rope_entry(false, dtype, {q, k}, {q_strides, k_strides}, {nullptr, nullptr}, {nullptr, nullptr},
                           {q_out, k_out}, {q_out_strides, k_out_strides}, {q_weight, k_weight}, {nullptr, nullptr},
                           weight_dtype, cos, sin, table_rows, positions, positions_per_batch, nullptr, 0, B, S, H_q,
                           H_kv, D, R, eps, norm, interleaved, stream);
}

size_t sdpa_hip_qk_norm_rope_grad_workspace_bytes(int D) {
    return D <= 0 || D > 128 ? 0 : 2 * (size_t)sdpa::kGradBlocks * (size_t)D * sizeof(float);
}

int sdpa_hip_qk_norm_rope_grad(int dtype, const void* d_q_out, const int64_t* d_q_out_strides, const void* d_k_out,
                               const int64_t* d_k_out_strides, const void* q, const int64_t* q_strides, const void* k,
                               const int64_t* k_strides, void* dq, const int64_t* dq_strides, void* dk,
                               const int64_t* dk_strides, void* dq_weight, void* dk_weight, const void* q_weight,
                               const void* k_weight, int weight_dtype, const float* cos, const float* sin,
                               int table_rows, const int32_t* positions, int positions_per_batch, void* workspace,
                               size_t workspace_bytes, int B, int S, int H_q, int H_kv, int D, int R, float eps,
                               int norm, int interleaved, hipStream_t stream) {
    return norm_rope_entry(true, dtype, {q, k}, {q_strides, k_strides}, {d_q_out, d_k_out},
                           {d_q_out_strides, d_k_out_strides}, {dq, dk}, {dq_strides, dk_strides},
                           {q_weight, k_weight}, {dq_weight, dk_weight}, weight_dtype, cos, sin, table_rows, positions,
                           positions_per_batch, workspace, workspace_bytes, B, S, H_q, H_kv, D, R, eps, norm,
                           interleaved, stream);
}

int sdpa_hip_kv_append(int dtype, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                       void* k_cache, void* v_cache, const void* q, const int64_t* q_strides, void* q_out,
                       const int64_t* q_out_strides, const void* q_weight, const void* k_weight, int weight_dtype,
                       const float* cos, const float* sin, int table_rows, const int32_t* page_table,
                       int64_t page_table_stride, const int32_t* q_starts, const int32_t* kv_lens, int N, int T,
                       int width, int pages, int page_size, int H_q, int H_kv, int D_qk, int D_v, int R, float eps,
                       int norm, int interleaved, hipStream_t stream) {
    int st = check_rows(dtype, weight_dtype, q_weight, k_weight, cos, sin, table_rows, D_qk, R, norm);
    if (st != SDPA_OK) return st;
    if (H_q < 0 || H_kv < 0 || D_v < 0) return SDPA_ERR_NEGATIVE_DIM;
    if (D_v > 128) return SDPA_ERR_FEATURE_TOO_LARGE;
    sdpa::AppendParams p{};
    st = make_batch(p.batch, page_table, page_table_stride, q_starts, kv_lens, N, T, width, pages, page_size);
    if (st != SDPA_OK) return st;
    if (!rows_fit(T, H_q, 2LL * H_kv)) return SDPA_ERR_TOO_LARGE;
    if (N == 0 || T == 0) return SDPA_OK;
    const bool has_k = H_kv > 0 && D_qk > 0, has_v = H_kv > 0 && D_v > 0, has_q = H_q > 0 && D_qk > 0;
    if ((has_k && (!k || (pages > 0 && !k_cache))) || (has_v && (!v || (pages > 0 && !v_cache))) ||
        (has_q && (!q || !q_out)))
        return SDPA_ERR_NULL_POINTER;
    p.q = q;
    p.q_out = q_out;
    p.k = k;
    p.v = v;
    p.k_cache = k_cache;
    p.v_cache = v_cache;
    p.q_weight = q_weight;
    p.k_weight = k_weight;
    p.qs = token_strides(q_strides, T, H_q, D_qk);
    p.qos = token_strides(q_out_strides, T, H_q, D_qk);
    p.ks = token_strides(k_strides, T, H_kv, D_qk);
    p.vs = token_strides(v_strides, T, H_kv, D_v);
    p.r = sdpa::RopeArgs{cos, sin, table_rows, R, norm != 0, eps, D_qk > 0 ? 1.f / (float)D_qk : 0.f};
    p.H_q = has_q ? H_q : 0;
    p.H_kv = H_kv;
    p.H_k = has_k ? H_kv : 0;
    p.H_v = has_v ? H_kv : 0;
    p.D_qk = D_qk;
    p.D_v = D_v;
    p.interleaved = interleaved != 0;
    p.w32 = weight_dtype == SDPA_DTYPE_F32;
    Chunks ch{dtype == SDPA_DTYPE_F16 ? 8 : 4};
    ch.features(D_qk);
    ch.features(D_v);
    ch.rotated(R, interleaved);
    ch.address(cos);
    ch.address(sin);
    ch.address(k_cache);
    ch.address(v_cache);
    ch.address(q_weight);
    ch.address(k_weight);
    if (has_q) {
        add_tokens(ch, q, p.qs);
        add_tokens(ch, q_out, p.qos);
    }
    if (has_k) add_tokens(ch, k, p.ks);
    if (has_v) add_tokens(ch, v, p.vs);
    p.vec = ch.ok;
    return hip_status(sdpa::launch_kv_append(p, (sdpa::DType)dtype, stream));
}

}  // extern "C"

namespace {

// Whether the parts of divided tiles can come up at all, and their bytes.
size_t paged_workspace(bool small, int width, int page_size, int D_v) {
    if ((long long)width * page_size <= 128) return 0;  // (one block of the smallest kind)
    return sdpa::paged_part_bytes(D_v, small ? sdpa::kPagedSmallBM : sdpa::kPagedBM);
}

int check_paged(int dtype, int H_q, int H_kv, int D_qk, int D_v) {
    if (dtype != SDPA_DTYPE_F32 && dtype != SDPA_DTYPE_F16) return SDPA_ERR_DTYPE;
    if (H_q < 0 || H_kv < 0 || D_qk < 0 || D_v < 0) return SDPA_ERR_NEGATIVE_DIM;
    if (D_qk > 128 || D_v > 128) return SDPA_ERR_FEATURE_TOO_LARGE;
    const int epc = dtype == SDPA_DTYPE_F16 ? 8 : 4;
    if (D_qk == 0 || D_v == 0 || D_qk % epc != 0 || D_v % epc != 0) return SDPA_ERR_LAYOUT;
    if (H_q > 0 && (H_kv == 0 || H_q % H_kv != 0)) return SDPA_ERR_HEADS;
    return SDPA_OK;
}

}  // namespace

extern "C" {

size_t sdpa_hip_paged_fwd_workspace_bytes(int dtype, int N, int T, int width, int page_size, int H_q, int H_kv,
                                          int D_qk, int D_v, int max_q_len) {
    if (check_paged(dtype, H_q, H_kv, D_qk, D_v) != SDPA_OK || N <= 0 || T <= 0 || width <= 0 || page_size <= 0 || H_q == 0)
        return 0;
    return paged_workspace(sdpa::paged_small(dtype == SDPA_DTYPE_F16, sdpa::paged_most_rows(T, H_q / H_kv, max_q_len)), width, page_size, D_v);
}

int sdpa_hip_paged_fwd(int dtype, const void* q, const int64_t* q_strides, const void* k_cache, const void* v_cache,
                       void* o, const int64_t* o_strides, float* stats, const int32_t* page_table,
                       int64_t page_table_stride, const int32_t* q_starts, const int32_t* kv_lens, void* workspace,
                       size_t workspace_bytes, int N, int T, int width, int pages, int page_size, int H_q, int H_kv,
                       int D_qk, int D_v, int max_q_len, float scale, int causal_mask, hipStream_t stream) {
    int st = check_paged(dtype, H_q, H_kv, D_qk, D_v);
    if (st != SDPA_OK) return st;
    sdpa::PagedParams p{};
    // without pages no column of the table holds any
    st = make_batch(p.batch, page_table, page_table_stride, q_starts, kv_lens, N, T, pages > 0 ? width : (width < 0 ? -1 : 0),
                    pages, page_size);
    if (st != SDPA_OK) return st;
    if (N == 0 || T == 0 || H_q == 0) return SDPA_OK;
    if (!q || !o || !stats || (p.batch.width > 0 && (!k_cache || !v_cache))) return SDPA_ERR_NULL_POINTER;
    p.q = q;
    p.k_cache = k_cache;
    p.v_cache = v_cache;
    p.o = o;
    p.stats = stats;
    p.qs = token_strides(q_strides, T, H_q, D_qk);
    p.os = token_strides(o_strides, T, H_q, D_v);
    Chunks ch{dtype == SDPA_DTYPE_F16 ? 8 : 4};
    ch.address(k_cache);
    ch.address(v_cache);
    add_tokens(ch, q, p.qs);
    add_tokens(ch, o, p.os);
    if (!ch.ok) return SDPA_ERR_LAYOUT;
    p.H_kv = H_kv;
    p.G = H_q / H_kv;
    p.D_qk = D_qk;
    p.D_v = D_v;
    p.scale = scale;
    p.causal = causal_mask != 0;
    if ((long long)T * p.G > 0x7FFFFFFFLL - 65536) return SDPA_ERR_TOO_LARGE;
    // sequences of few rows, as far as is known here (either kernel takes any)
    p.most_rows = (int)sdpa::paged_most_rows(T, p.G, max_q_len);
    const bool small = sdpa::paged_small(dtype == SDPA_DTYPE_F16, p.most_rows);
    if (sdpa::paged_max_tiles(p, sdpa::kPagedSmallBM) > 0x7FFFFFFFLL - 65536) return SDPA_ERR_TOO_LARGE;
    const size_t need = paged_workspace(small, p.batch.width, page_size, D_v);
    p.target_log2 = sdpa::kPagedTargetLog2;
    if (need > 0 && workspace && ((uintptr_t)workspace & 15u) == 0 && workspace_bytes >= need) {
        p.part_o = static_cast<float*>(workspace);
        p.part_ml = p.part_o + ((size_t)2 << p.target_log2) * (small ? sdpa::kPagedSmallBM : sdpa::kPagedBM) * D_v;
    }
    if (dtype == SDPA_DTYPE_F32)
        return hip_status(small ? sdpa::launch_paged_f32_small(p, stream) : sdpa::launch_paged_f32(p, stream));
    return hip_status(small ? sdpa::launch_paged_f16_small(p, stream) : sdpa::launch_paged_f16(p, stream));
}

}  // extern "C"
