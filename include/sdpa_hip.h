/*
 * sdpa_hip.h -- C ABI of the MI355X (gfx950) implementation of the Sdpa /
 * SdpaGrad TensorFlow custom ops of gravytrain777/tf-custom-flash-attention.
 *
 * This library replaces the reference's device seam
 *     functor::FlashAttnFunctor<GPUDevice, T>       (sdpa/sdpa.h:11-18)
 *     functor::FlashAttnGradFunctor<GPUDevice, T>   (sdpa/sdpa.h:20-34)
 * with plain-pointer entry points, plus the input validation the reference
 * performs in SdpaFwdOp::Compute / SdpaBwdOp::Compute (sdpa/sdpa_cpu.cc:29-87,
 * 105-192) so that every host binding reports the same errors.
 *
 * Conventions
 *   - Every tensor is dense row-major: q [B,S_q,D_qk], k [B,S_kv,D_qk],
 *     v [B,S_kv,D_v], o / do [B,S_q,D_v], stats [B,S_q] (fp32, natural log).
 *   - dtype: SDPA_DTYPE_F32 (float) or SDPA_DTYPE_F16 (IEEE binary16).
 *   - Pointers are device pointers; the caller owns every buffer (the
 *     library allocates nothing and keeps no per-call state).
 *   - Launches are asynchronous on `stream`; nothing synchronises.
 *   - Return value: SDPA_OK or an sdpa_status_t; sdpa_hip_status_string()
 *     gives the message (argument errors use the reference's wording).
 */
#ifndef SDPA_HIP_H_
#define SDPA_HIP_H_

#include <stddef.h>
#include <stdint.h>

/* The stream handle type of the HIP runtime (hip/hip_runtime_api.h declares
 * the same typedef), so that a host binding written in plain C or C++ needs
 * neither the HIP headers nor a HIP platform macro to include this file. */
typedef struct ihipStream_t* hipStream_t;

#ifdef __cplusplus
extern "C" {
#endif

#define SDPA_HIP_ABI_VERSION 1

typedef enum {
    SDPA_DTYPE_F32 = 0,
    SDPA_DTYPE_F16 = 1
} sdpa_dtype_t;

typedef enum {
    SDPA_OK = 0,
    /* argument errors, reference OP_REQUIRES order (sdpa/sdpa_cpu.cc:37-69, 116-168) */
    SDPA_ERR_SEED_NOT_SCALAR = 1,
    SDPA_ERR_OFFSET_NOT_SCALAR = 2,
    SDPA_ERR_K_BATCH = 3,
    SDPA_ERR_K_FEATURE = 4,
    SDPA_ERR_V_BATCH = 5,
    SDPA_ERR_V_SEQ = 6,
    SDPA_ERR_O_BATCH = 7,
    SDPA_ERR_O_SEQ = 8,
    SDPA_ERR_O_FEATURE = 9,
    SDPA_ERR_DO_BATCH = 10,
    SDPA_ERR_DO_SEQ = 11,
    SDPA_ERR_DO_FEATURE = 12,
    SDPA_ERR_S_BATCH = 13,
    SDPA_ERR_S_SEQ = 14,
    SDPA_ERR_CAUSAL_SEQ = 15,
    SDPA_ERR_FEATURE_TOO_LARGE = 16,
    /* shape-function error (sdpa/sdpa_ops.cc:22-25, 55-57) */
    SDPA_ERR_RANK = 17,
    /* errors of this library's own ABI */
    SDPA_ERR_DTYPE = 18,
    SDPA_ERR_NEGATIVE_DIM = 19,
    SDPA_ERR_NULL_POINTER = 20,
    SDPA_ERR_DROPOUT_RANGE = 21,
    SDPA_ERR_WORKSPACE = 22,
    SDPA_ERR_HIP = 23,
    SDPA_ERR_SCRATCH_LIMIT = 24,
    SDPA_ERR_DS_PATH = 25,
    SDPA_ERR_ROTARY = 26,
    SDPA_ERR_PAGE_SIZE = 27,
    SDPA_ERR_HEADS = 28,
    SDPA_ERR_LAYOUT = 29,
    SDPA_ERR_TOO_LARGE = 30,
    SDPA_ERR_WEIGHT = 31,
    SDPA_ERR_AXES = 32,
    SDPA_ERR_FP4_WIDTH = 33
} sdpa_status_t;

/* Message for a status code (static storage, never NULL). */
const char* sdpa_hip_status_string(int status);

/* HIP error of the most recent SDPA_ERR_HIP returned on this thread. */
int sdpa_hip_last_hip_error(void);

/* ---- validation (host only, no device work) -------------------------------
 * Mirrors SdpaFwdOp::Compute (sdpa/sdpa_cpu.cc:37-69) plus the Sdpa shape fn
 * (sdpa/sdpa_ops.cc:22-25): shapes are given as rank + dims; a scalar has
 * rank 0.  Returns the first failing check in the reference's order.       */
int sdpa_hip_check_fwd(int q_rank, const int64_t* q_shape, int k_rank, const int64_t* k_shape,
                       int v_rank, const int64_t* v_shape, int seed_rank, int offset_rank,
                       int causal_mask);

/* Mirrors SdpaBwdOp::Compute (sdpa/sdpa_cpu.cc:116-168) and the SdpaGrad
 * shape fn (sdpa/sdpa_ops.cc:55-57).                                        */
int sdpa_hip_check_bwd(int q_rank, const int64_t* q_shape, int k_rank, const int64_t* k_shape,
                       int v_rank, const int64_t* v_shape, int o_rank, const int64_t* o_shape,
                       int stats_rank, const int64_t* stats_shape, int do_rank,
                       const int64_t* do_shape, int seed_rank, int offset_rank, int causal_mask);

/* ---- forward: replaces FlashAttnFunctor<GPUDevice,T> (sdpa/sdpa_fwd.cu.cc:176-240)
 * o     = softmax(scale * q k^T [causal]) (dropout) v     [B,S_q,D_v], dtype
 * stats = m + log(l + 1e-6)                               [B,S_q] fp32
 * Requires max(D_qk, D_v) <= 128 and, with causal_mask, S_q == S_kv.
 * dropout <= 1e-6 disables dropout (as the reference GPU); dropout > 1 drops
 * every element as the reference does (o = 0, the usual stats; in the
 * backward dV = 0 and dS = -P delta); dropout == 1 returns
 * SDPA_ERR_DROPOUT_RANGE (the reference would scale by 1 / 0).  */
int sdpa_hip_fwd(int dtype, const void* q, const void* k, const void* v, void* o, float* stats,
                 int B, int S_q, int S_kv, int D_qk, int D_v, float scale, float dropout,
                 int causal_mask, uint64_t seed, uint64_t offset, hipStream_t stream);

/* The same with a workspace.  Where the query side has too few tiles to fill
 * the GPU (token generation, a few queries against a long memory) the keys
 * of a tile are divided over several workgroups, which needs
 * sdpa_hip_fwd_workspace_bytes(...) bytes of device memory, 16-byte aligned,
 * for their partial results; 0 where nothing is divided.  With less (or
 * none) the call runs undivided, as sdpa_hip_fwd does.  The sums of a divided
 * row are added in another order: its last bits differ between the two forms,
 * and, as the division goes by the number of tiles, between batch sizes.  Each
 * call repeats to the bit.                                                  */
size_t sdpa_hip_fwd_workspace_bytes(int dtype, int B, int S_q, int S_kv, int D_qk, int D_v,
                                    int causal_mask);

int sdpa_hip_fwd_ws(int dtype, const void* q, const void* k, const void* v, void* o, float* stats,
                    void* workspace, size_t workspace_bytes, int B, int S_q, int S_kv, int D_qk,
                    int D_v, float scale, float dropout, int causal_mask, uint64_t seed,
                    uint64_t offset, hipStream_t stream);

/* ---- backward: replaces FlashAttnGradFunctor<GPUDevice,T> (sdpa/sdpa_bwd.cu.cc:347-453)
 * Needs a device workspace of sdpa_hip_bwd_workspace_bytes(B, S_q) bytes
 * (two fp32 values per query row: stats * log2(e) and delta = sum_d dO * O),
 * provided by the caller as the TF op does with allocate_temp.              */
size_t sdpa_hip_bwd_workspace_bytes(int B, int S_q);

int sdpa_hip_bwd(int dtype, const void* q, const void* k, const void* v, const void* o,
                 const float* stats, const void* d_o, void* dq, void* dk, void* dv,
                 void* workspace, size_t workspace_bytes, int B, int S_q, int S_kv, int D_qk,
                 int D_v, float scale, float dropout, int causal_mask, uint64_t seed,
                 uint64_t offset, hipStream_t stream);

/* The two launches of sdpa_hip_bwd as separate calls, same arguments, same
 * stream order required (the reference launches its two backward kernels
 * back to back, sdpa/sdpa_bwd.cu.cc:402-405):
 *   sdpa_hip_bwd_dq   -- dQ, and the per-row values into the workspace;
 *   sdpa_hip_bwd_dkdv -- dK and dV, reading the values left in the workspace
 *                        by a preceding sdpa_hip_bwd_dq with the same inputs.
 * sdpa_hip_bwd == sdpa_hip_bwd_dq followed by sdpa_hip_bwd_dkdv.            */
int sdpa_hip_bwd_dq(int dtype, const void* q, const void* k, const void* v, const void* o,
                    const float* stats, const void* d_o, void* dq, void* workspace,
                    size_t workspace_bytes, int B, int S_q, int S_kv, int D_qk, int D_v,
                    float scale, float dropout, int causal_mask, uint64_t seed, uint64_t offset,
                    hipStream_t stream);

int sdpa_hip_bwd_dkdv(int dtype, const void* q, const void* k, const void* v, const float* stats,
                      const void* d_o, void* dk, void* dv, const void* workspace,
                      size_t workspace_bytes, int B, int S_q, int S_kv, int D_qk, int D_v,
                      float scale, float dropout, int causal_mask, uint64_t seed,
                      uint64_t offset, hipStream_t stream);

/* ---- backward, dS path --------------------------------------------------
 * No counterpart in the reference (an MI355X choice of how its two backward
 * kernels divide the work).  For float16 and float32 with a feature size
 * over 64, the dK/dV kernel can store the dS it forms (in T, every visited
 * score: about B * S_q * S_kv * sizeof(T) / 2 bytes under the causal mask,
 * twice that without) and dQ is then one product with it, instead of a
 * kernel that forms S, P, dP and dS again.  sdpa_hip_bwd takes this path whenever the shape qualifies, the
 * tensors are 16-byte aligned and workspace_bytes is at least
 * sdpa_hip_bwd_workspace_bytes_ds(...); with a smaller workspace (at least
 * sdpa_hip_bwd_workspace_bytes(B, S_q)) it takes the other one.  For shapes
 * that do not qualify the function returns sdpa_hip_bwd_workspace_bytes. */
size_t sdpa_hip_bwd_workspace_bytes_ds(int dtype, int B, int S_q, int S_kv, int D_qk, int D_v,
                                       int causal_mask);

/* The largest workspace sdpa_hip_bwd makes use of: that of the dS path; or,
 * for shapes without one that have few tiles, the per-row workspace plus the
 * partial sums of the workgroups that then share a tile: dQ of a tile's keys
 * (a few queries against a long memory) and, float32, dK and dV of a tile's
 * queries; elsewhere the per-row workspace.  Any smaller workspace works as
 * described above (with the note on divided sums at sdpa_hip_fwd_ws).       */
size_t sdpa_hip_bwd_workspace_bytes_full(int dtype, int B, int S_q, int S_kv, int D_qk, int D_v,
                                         int causal_mask);

/* The three launches of the dS path as separate calls (same arguments as
 * sdpa_hip_bwd; each phase reads what the previous one left in the workspace,
 * in stream order):
 *   phase 0 -- the per-row values (stats * log2(e), delta) into the workspace;
 *   phase 1 -- dK, dV and the stored dS;
 *   phase 2 -- dQ from the stored dS.
 * Returns SDPA_ERR_DS_PATH where sdpa_hip_bwd would not take the dS path.  */
int sdpa_hip_bwd_ds_phase(int phase, int dtype, const void* q, const void* k, const void* v,
                          const void* o, const float* stats, const void* d_o, void* dq, void* dk,
                          void* dv, void* workspace, size_t workspace_bytes, int B, int S_q,
                          int S_kv, int D_qk, int D_v, float scale, float dropout, int causal_mask,
                          uint64_t seed, uint64_t offset, hipStream_t stream);

/* ---- backward that allocates nothing ---------------------------------------
 * No counterpart in the reference.  For callers that cannot allocate device
 * memory or pass a workspace: code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc.  Same arguments and results as
 * sdpa_hip_bwd without the workspace: the per-query-row values live in a
 * static device array of SDPA_HIP_NOALLOC_SCRATCH_BYTES per GPU (8 bytes per
 * query row, so B * S_q <= 2,097,152; larger problems return
 * SDPA_ERR_SCRATCH_LIMIT).  Calls no hipMalloc / hipFree; its first call on
 * a device looks up that device's copy of the array (hipGetSymbolAddress).
 * Every call on one GPU shares that GPU's array: calls that overlap on one
 * GPU (different streams, or host threads without ordering) race.          */
#define SDPA_HIP_NOALLOC_SCRATCH_BYTES (16u << 20)

int sdpa_hip_bwd_noalloc(int dtype, const void* q, const void* k, const void* v, const void* o,
                         const float* stats, const void* d_o, void* dq, void* dk, void* dv, int B,
                         int S_q, int S_kv, int D_qk, int D_v, float scale, float dropout,
                         int causal_mask, uint64_t seed, uint64_t offset, hipStream_t stream);

/* ---- dropout hash (sdpa/sdpa_utils.cuh:13-19, sdpa/sdpa_cpu.cc:198-211) ----
 * Integer form of the reference's predicate (float)(st >> 32) / 2^32 < p:
 * element dropped iff (st >> 32) < T(p).  Returns T(p) as a 64-bit value
 * (2^32 means "every element dropped"; only reachable for p > 1).           */
uint64_t sdpa_hip_drop_threshold(float dropout);

/* Device dump of the keep mask the kernels apply (1 = kept), uint8
 * [B, S_q, S_kv], computed by the kernels' own hash code.  For tests.       */
int sdpa_hip_dropout_mask(uint8_t* keep, int B, int S_q, int S_kv, float dropout, uint64_t seed,
                          uint64_t offset, hipStream_t stream);

/* ---- norm and rotation of queries and keys ---------------------------------
 * No counterpart in the reference: what a layer does to its queries and keys
 * before Sdpa, in one launch for both.  For every head row x of D features
 *   n = weight x / sqrt(mean(x^2) + eps)   (norm; else n = x)
 *   y = n with its first R features turned by the row's position: the pairs
 *       (i, i + R/2), or (2i, 2i + 1) if interleaved, to
 *       (a c - b s, b c + a s), c = cos[position][i], s = sin[position][i]
 * in fp32, rounded once.  q is [B, S, H_q, D], k [B, S, H_kv, D] with dense
 * features and any other strides ({batch, token, head}, in elements); the
 * results go where their strides say: {H S D, D, S D} is the [B H, S, D] that
 * sdpa_hip_fwd reads.  A result may be the input itself (same strides).
 * cos, sin: float [table_rows, R / 2]; positions: int32 [S] (or [B, S] with
 * positions_per_batch), NULL for 0 .. S - 1; a position outside the tables
 * makes its rows NaN.  Weights: [D] of weight_dtype (that of q or
 * SDPA_DTYPE_F32) or NULL.  H_q or H_kv may be 0.  D <= 128.                  */
int sdpa_hip_qk_norm_rope(int dtype, const void* q, const int64_t* q_strides, const void* k,
                          const int64_t* k_strides, void* q_out, const int64_t* q_out_strides, void* k_out,
                          const int64_t* k_out_strides, const void* q_weight, const void* k_weight,
                          int weight_dtype, const float* cos, const float* sin, int table_rows,
                          const int32_t* positions, int positions_per_batch, int B, int S, int H_q, int H_kv,
                          int D, int R, float eps, int norm, int interleaved, hipStream_t stream);

/* Its gradient: d_q_out and d_k_out as the results were laid out, dq and dk
 * as their strides say, dq_weight and dk_weight [D] of weight_dtype (NULL: not
 * wanted; they need no weight in the forward call).  The weights' gradients are
 * summed in a fixed order, in fp32 over the rows of a workgroup and in fp64 over
 * the workgroups' sums in the workspace,
 * sdpa_hip_qk_norm_rope_grad_workspace_bytes(D) bytes, 16-byte aligned; without
 * them it may be NULL.                                                        */
size_t sdpa_hip_qk_norm_rope_grad_workspace_bytes(int D);

int sdpa_hip_qk_norm_rope_grad(int dtype, const void* d_q_out, const int64_t* d_q_out_strides,
                               const void* d_k_out, const int64_t* d_k_out_strides, const void* q,
                               const int64_t* q_strides, const void* k, const int64_t* k_strides, void* dq,
                               const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dq_weight,
                               void* dk_weight, const void* q_weight, const void* k_weight, int weight_dtype,
                               const float* cos, const float* sin, int table_rows, const int32_t* positions,
                               int positions_per_batch, void* workspace, size_t workspace_bytes, int B, int S,
                               int H_q, int H_kv, int D, int R, float eps, int norm, int interleaved,
                               hipStream_t stream);

/* The same where the pairs follow several positions of a token (time, height,
 * width of image and video patches): pair i, of the R / 2 rotated ones, is turned
 * by row positions[pair_axes[i]] of the tables.  positions: int32 [n_axes, S] (or
 * [n_axes, B, S] with positions_per_batch) on the device, dense; pair_axes: R / 2
 * bytes on the host, read before the call returns, each below n_axes and 4.  A
 * position outside the tables, on an axis that some pair follows, makes its rows NaN. */
int sdpa_hip_qk_norm_rope_axes(int dtype, const void* q, const int64_t* q_strides, const void* k,
                               const int64_t* k_strides, void* q_out, const int64_t* q_out_strides, void* k_out,
                               const int64_t* k_out_strides, const void* q_weight, const void* k_weight,
                               int weight_dtype, const float* cos, const float* sin, int table_rows,
                               const int32_t* positions, int positions_per_batch, const uint8_t* pair_axes, int n_axes,
                               int B, int S, int H_q, int H_kv, int D, int R, float eps, int norm, int interleaved,
                               hipStream_t stream);

int sdpa_hip_qk_norm_rope_axes_grad(int dtype, const void* d_q_out, const int64_t* d_q_out_strides,
                                    const void* d_k_out, const int64_t* d_k_out_strides, const void* q,
                                    const int64_t* q_strides, const void* k, const int64_t* k_strides, void* dq,
                                    const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dq_weight,
                                    void* dk_weight, const void* q_weight, const void* k_weight, int weight_dtype,
                                    const float* cos, const float* sin, int table_rows, const int32_t* positions,
                                    int positions_per_batch, const uint8_t* pair_axes, int n_axes, void* workspace,
                                    size_t workspace_bytes, int B, int S, int H_q, int H_kv, int D, int R, float eps,
                                    int norm, int interleaved, hipStream_t stream);

/* ---- paged cache -------------------------------------------------------------
 * No counterpart in the reference.  Keys and values of N sequences lie in pages
 * of page_size tokens (a power of two, 16 .. 65536): k_cache [pages, H_kv, page_size,
 * D_qk], v_cache [pages, H_kv, page_size, D_v], dense, so that a page's head is a
 * dense matrix as the op's k and v are.  T new tokens are packed, sequence after
 * sequence; device arrays of int32 say what belongs where:
 *   q_starts [N + 1]    sequence s has the new tokens q_starts[s] ..
 *                       q_starts[s + 1] - 1 (none, or not all of them among the
 *                       T: append and attention leave the sequence out);
 *   kv_lens [N]         its cached tokens, the new ones among them, last;
 *   page_table [N, width] (rows page_table_stride apart): token j of s is row
 *                       j % page_size of page page_table[s][j / page_size].
 * They are read on the device only, so a captured call follows them.  Nothing
 * outside of the T tokens, the width columns and the pages is touched whatever
 * they hold.                                                                  */

/* Pages for the new tokens of a batch, and where each token goes: what a server
 * does between two steps, on the device.  free_pages [capacity] is a stack of pages
 * that no sequence holds, its first *free_count entries.
 *   1. Sequences with finished[s] != 0 (NULL: none) give back the pages of their
 *      kv_lens[s] tokens, in the order sequence, column (entries below 0 are left
 *      out, and what would pass capacity), and have no tokens then; their rows of the
 *      table are left as they are.
 *   2. new_lens[s] tokens are added to every sequence (a finished one begins
 *      anew).  Each column that they are the first to need gets the top page of the
 *      stack, in the order sequence, column; -1 once the stack is empty, and what
 *      lies behind the table's columns gets none.
 * Out: q_starts [N + 1] and kv_lens_out [N] as below (kv_lens_out may be kv_lens);
 * free_count_out (may be free_count); for every one of the T packed tokens its
 * place in the sequence, positions [T], and slots [T], page * page_size + row, -1 for
 * a token without a page; both -1 behind the last sequence.  (With fewer than q_starts[N] tokens T
 * the sequences that reach past them have their pages and lengths all the same.)  Lengths below 0 count as
 * 0, cached ones above width * page_size and new ones above T as those.  No two
 * rows of the table may overlap.  T <= 2^30 - 1, width * page_size + T below 2^31.  */
int sdpa_hip_kv_reserve(int32_t* page_table, int64_t page_table_stride, const int32_t* kv_lens,
                        const int32_t* new_lens, const uint8_t* finished, int32_t* free_pages,
                        const int32_t* free_count, int32_t* q_starts, int32_t* kv_lens_out, int32_t* free_count_out,
                        int32_t* positions, int64_t* slots, int N, int T, int width, int page_size, int capacity,
                        hipStream_t stream);

/* The same, and *pages_short (NULL: not wanted): the pages that the stack lacked, that is the columns
 * that got -1 for want of one.  A column that got -1 stays so (tokens that belong there are in no
 * page, and rows that see them NaN) until its sequence is finished, which gives back the pages it has.
 * Where kv_lens_out and free_count_out are memory of their own, a call may also be taken back, by a call with the
 * same kv_lens and free_count: with other new_lens, with more sequences finished, but with none
 * that was finished and got new tokens.                                         */
int sdpa_hip_kv_reserve_counted(int32_t* page_table, int64_t page_table_stride, const int32_t* kv_lens,
                                const int32_t* new_lens, const uint8_t* finished, int32_t* free_pages,
                                const int32_t* free_count, int32_t* q_starts, int32_t* kv_lens_out,
                                int32_t* free_count_out, int32_t* pages_short, int32_t* positions, int64_t* slots, int N,
                                int T, int width, int page_size, int capacity, hipStream_t stream);

/* Keys and values of the new tokens into their places, k normed (norm) and
 * rotated by its place in the sequence on the way as above (R = 0: not
 * rotated), and the queries of the same tokens, normed and rotated, to q_out
 * (H_q = 0: none).  q, k, v, q_out: [T, H, D] with dense features and strides
 * {token, head} in elements.  q_out may be q.  Tokens of no sequence leave
 * everything as it was; a token whose place is outside of the table's columns or
 * of the pages is not appended, and its row of q_out is NaN.  Two tokens of one
 * call must not have the same place.  D_qk or D_v may be 0: nothing of that width
 * is read or written, and its pointers may be NULL.  Widths up to 128 need not be
 * whole 16-byte chunks here; attention over the cache asks that of them.      */
int sdpa_hip_kv_append(int dtype, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                       void* k_cache, void* v_cache, const void* q, const int64_t* q_strides, void* q_out,
                       const int64_t* q_out_strides, const void* q_weight, const void* k_weight, int weight_dtype,
                       const float* cos, const float* sin, int table_rows, const int32_t* page_table,
                       int64_t page_table_stride, const int32_t* q_starts, const int32_t* kv_lens, int N, int T,
                       int width, int pages, int page_size, int H_q, int H_kv, int D_qk, int D_v, int R, float eps,
                       int norm, int interleaved, hipStream_t stream);

/* The same, rotated by positions [n_axes, T] instead of the places in the
 * sequences (as in sdpa_hip_qk_norm_rope_axes).                               */
int sdpa_hip_kv_append_axes(int dtype, const void* k, const int64_t* k_strides, const void* v,
                            const int64_t* v_strides, void* k_cache, void* v_cache, const void* q,
                            const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, const void* q_weight,
                            const void* k_weight, int weight_dtype, const float* cos, const float* sin, int table_rows,
                            const int32_t* positions, const uint8_t* pair_axes, int n_axes, const int32_t* page_table,
                            int64_t page_table_stride, const int32_t* q_starts, const int32_t* kv_lens, int N, int T,
                            int width, int pages, int page_size, int H_q, int H_kv, int D_qk, int D_v, int R, float eps,
                            int norm, int interleaved, hipStream_t stream);

/* Attention of the new tokens over the cache (after their append): for query
 * head h of token i of the n new ones of sequence s, over the keys of head
 * h / (H_q / H_kv),
 *   o     = softmax(scale q k^T) v      [T, H_q, D_v], strides {token, head}
 *   stats = log(sum(exp(scale q k^T)))  [T, H_q] fp32, dense
 * over the cached tokens j < kv_lens[s]; with causal_mask over those with
 * j <= kv_lens[s] - n + i.  A row that sees no key has o = 0 and stats =
 * -infinity.  Rows of tokens of no sequence stay as they were.  Where a key that some
 * row of a sequence may see has no place in the table or on a page, rows of that
 * sequence are NaN.  What lies in the cache behind a row's last key has no
 * influence on it, infinities and NaN included; an infinite or NaN value
 * among its keys makes its feature of o infinite or NaN.
 * o, stats and the workspace share no memory with each other or with the inputs.
 * H_q is a multiple of H_kv; feature sizes, strides and addresses must be whole
 * 16-byte chunks; D_qk, D_v <= 128.
 * max_q_len: the most new tokens of a sequence, where the caller knows it (1 in
 * generation), else 0.  It helps to choose kernels; results are right
 * whatever it is.
 * The workspace (device memory, 16-byte aligned) holds the parts of tiles whose
 * keys are divided over workgroups; with less than
 * sdpa_hip_paged_fwd_workspace_bytes(...), or none, nothing is divided.  (At
 * D_v = 128 it is 17 MB for calls of few new tokens a sequence and 68 MB for others,
 * whatever their lengths.)  The
 * division goes by all lengths of the call: the last bits of a sequence's
 * results may differ between batches.  Each call repeats to the bit.         */
size_t sdpa_hip_paged_fwd_workspace_bytes(int dtype, int N, int T, int width, int page_size, int H_q, int H_kv,
                                          int D_qk, int D_v, int max_q_len);

int sdpa_hip_paged_fwd(int dtype, const void* q, const int64_t* q_strides, const void* k_cache,
                       const void* v_cache, void* o, const int64_t* o_strides, float* stats,
                       const int32_t* page_table, int64_t page_table_stride, const int32_t* q_starts,
                       const int32_t* kv_lens, void* workspace, size_t workspace_bytes, int N, int T, int width,
                       int pages, int page_size, int H_q, int H_kv, int D_qk, int D_v, int max_q_len, float scale,
                       int causal_mask, hipStream_t stream);

/* ---- paged cache in 4 bits -------------------------------------------------------
 * No counterpart in the reference.  A value is s c, c one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a
 * sign (a code: sign 8, then the place in this list) and s a scale that 32 neighbouring
 * features of a token and head share (a byte: the upper one of an fp16, e5m2).  s is the
 * largest |x| of the 32 over 6, rounded to nearest even, at most 10240; c is x / s, rounded
 * to nearest even, at most 6 in size (so what passes 61440 comes back as that).  Every
 * value is exact in fp16.  32 features with an infinity or a NaN among them are NaN.
 * k_cache and v_cache: bytes [pages, H_kv, page_size * 17 D / 32], 16-byte aligned, a page's
 * head its codes, then its scales:
 *   k  codes [page_size][D / 2], the feature before in the lower half; scales [page_size][D / 32]
 *   v  codes [page_size / 8][D][4]: 8 tokens of a feature, the token before in the lower
 *      half; scales [page_size / 8][D / 32][8]
 * D_qk and D_v are 32, 64, 96 or 128.                                          */

/* As sdpa_hip_kv_append (pair_axes NULL) or sdpa_hip_kv_append_axes, into such a cache.
 * The keys' norm and rotation are formed in fp64 and rounded to fp32 before they are
 * rounded to 4 bits.  The tokens 8 i .. 8 i + 7 of a page share words: no two sequences of
 * a call may append to the same 8.  Other tokens of the 8 keep their values.       */
int sdpa_hip_kv_append_fp4(int dtype, const void* k, const int64_t* k_strides, const void* v,
                           const int64_t* v_strides, void* k_cache, void* v_cache, const void* q,
                           const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, const void* q_weight,
                           const void* k_weight, int weight_dtype, const float* cos, const float* sin, int table_rows,
                           const int32_t* positions, const uint8_t* pair_axes, int n_axes, const int32_t* page_table,
                           int64_t page_table_stride, const int32_t* q_starts, const int32_t* kv_lens, int N, int T,
                           int width, int pages, int page_size, int H_q, int H_kv, int D_qk, int D_v, int R, float eps,
                           int norm, int interleaved, hipStream_t stream);

/* The values of the T tokens of a batch out of such a cache: k [T, H_kv, D_qk] and v
 * [T, H_kv, D_v] of dtype, dense, 16-byte aligned.  Rows of a token without a place are NaN,
 * those of no sequence stay as they were; of a sequence that reaches past the T tokens those
 * that lie among them are read.                                                 */
int sdpa_hip_kv_read_fp4(int dtype, const void* k_cache, const void* v_cache, void* k, void* v,
                         const int32_t* page_table, int64_t page_table_stride, const int32_t* q_starts,
                         const int32_t* kv_lens, int N, int T, int width, int pages, int page_size, int H_kv, int D_qk,
                         int D_v, hipStream_t stream);

/* Attention of new tokens over such a cache: as sdpa_hip_paged_fwd, with queries and o
 * of dtype, over the values.  A value is NaN where its scale is.                  */
size_t sdpa_hip_paged_fwd_fp4_workspace_bytes(int dtype, int N, int T, int width, int page_size, int H_q, int H_kv,
                                              int D_qk, int D_v, int max_q_len);

int sdpa_hip_paged_fwd_fp4(int dtype, const void* q, const int64_t* q_strides, const void* k_cache,
                           const void* v_cache, void* o, const int64_t* o_strides, float* stats,
                           const int32_t* page_table, int64_t page_table_stride, const int32_t* q_starts,
                           const int32_t* kv_lens, void* workspace, size_t workspace_bytes, int N, int T, int width,
                           int pages, int page_size, int H_q, int H_kv, int D_qk, int D_v, int max_q_len, float scale,
                           int causal_mask, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* SDPA_HIP_H_ */
