// sdpa_reserve.hip -- pages for the new tokens of a batch, and where each token
// goes, from the requests' lengths, for gfx950.
//
// Sequences that have finished give the pages of their tokens back to a stack, in the
// order sequence, column; then the columns that the new tokens need are taken off its
// top in that order: page number k of the call is entry count - 1 - k.  So the
// result is that of a loop over the sequences, whatever runs first.  q_starts are
// the sums of the new tokens before each sequence.
//
// 64 sequences, 60 new tokens, four finished: 5.9 us; 24147 tokens of 10 sequences: 5.4 and the fill 3.3.
// A chain of dependent loads (lengths, stack, table), which nothing but fewer steps
// shortens: one workgroup forms the sums over 1024 sequences at a time, in lanes
// and then over its 16 waves, and hands out the pages.  Up to kReserveFill tokens it also
// writes positions and slots; of more, a second kernel does, a thread a token.
#include "sdpa_reserve.h"
#include "sdpa_scan.h"

namespace sdpa {
namespace {

constexpr int kReserveThreads = 1024, kReserveWaves = kReserveThreads / 64;
// us a call by one kernel and by two: one sequence, 4096 tokens 13.8 and 15.8, 8192 24 and 15.8; 8
// sequences, 4096 15.6 and 15.8, 16384 45 and 15.7; 1024 sequences of one token 13.3 and 15.7, of four
// 29.8 and 16.4.  (13.3 is the host's time of a call.)
constexpr int kReserveFill = 2048;

// Sums over the workgroup: x becomes the sum over the threads before, the sum over
// all is returned.  Two barriers; `lds` is free again after the next ones.
__device__ __forceinline__ long long block_scan(long long& x, long long* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long up_to = wave_scan(x);
    __syncthreads();
    if (lane == 63) lds[wave] = up_to;
    __syncthreads();
    const long long sums = wave_scan(lane < kReserveWaves ? lds[lane] : 0);
    const long long before = wave == 0 ? 0 : readlane64(sums, wave - 1);
    x = before + up_to - x;
    return readlane64(sums, kReserveWaves - 1);
}

// Columns of a row that hold so many tokens.
__device__ __forceinline__ int columns_of(const ReserveParams& p, long long tokens) {
    const long long c = (tokens + (1 << p.page_log2) - 1) >> p.page_log2;
    return c < p.width ? (int)c : p.width;
}

__device__ __forceinline__ void put_token(const ReserveParams& p, long long t, int seq, long long place) {
    const long long c = place >> p.page_log2;
    const int page = c < p.width ? p.page_table[seq * p.table_stride + c] : -1;
    p.positions[t] = (int32_t)place;
    p.slots[t] = page < 0 ? -1 : ((long long)page << p.page_log2) + (place & ((1 << p.page_log2) - 1));
}

__global__ __launch_bounds__(kReserveThreads) void reserve_kernel(const ReserveParams p) {
    __shared__ long long lds[kReserveWaves];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cap = p.width << p.page_log2;
    const auto old_len = [&](int s) { return min(max(p.kv_lens[s], 0), cap); };
    long long count = min(max(*p.free_count, 0), p.capacity);

    // pages of finished sequences back
    if (p.finished)
        for (int n0 = 0; n0 < p.N; n0 += kReserveThreads) {
            const int s = n0 + tid;
            const int columns = s < p.N && p.finished[s] ? columns_of(p, old_len(s)) : 0;
            const uint64_t ended = __builtin_amdgcn_ballot_w64(columns > 0);
            // f(page, its number among the sequence's pages that are some) of sequence l of the wave; how many there are
            const auto each_page = [&](int l, auto&& f) {
                const int n = __builtin_amdgcn_readlane(columns, l);
                const int32_t* row = p.page_table + (long long)(n0 + 64 * wave + l) * p.table_stride;
                int found = 0;
                for (int c0 = 0; c0 < n; c0 += 64) {
                    const int page = c0 + lane < n ? row[c0 + lane] : -1;
                    const uint64_t some = __builtin_amdgcn_ballot_w64(page >= 0);
                    if (page >= 0) f(page, found + __popcll(some & ((1ull << lane) - 1)));
                    found += __popcll(some);
                }
                return found;
            };
            long long mine = 0;
            for (uint64_t todo = ended; todo != 0; todo &= todo - 1) {
                const int l = __builtin_ctzll(todo), n = each_page(l, [](int, int) {});
                if (lane == l) mine = n;
            }
            const long long all = block_scan(mine, lds);
            for (uint64_t todo = ended; todo != 0; todo &= todo - 1) {
                const int l = __builtin_ctzll(todo);
                const long long at = count + readlane64(mine, l);
                each_page(l, [&](int page, int i) {
                    if (at + i < p.capacity) p.free_pages[at + i] = page;
                });
            }
            count = min(count + all, (long long)p.capacity);
        }

    // pages for the new tokens
    long long tokens = 0, taken = 0;
    __syncthreads();  // (the pages that came back are there)
    for (int n0 = 0; n0 < p.N; n0 += kReserveThreads) {
        const int s = n0 + tid;
        int n = 0, old = 0;
        if (s < p.N) {
            n = min(max(p.new_lens[s], 0), p.T);
            old = p.finished && p.finished[s] ? 0 : old_len(s);
        }
        const int c0 = columns_of(p, old), need = n > 0 ? columns_of(p, (long long)old + n) - c0 : 0;
        long long start = n, k = need;
        const long long all_tokens = block_scan(start, lds), all_pages = block_scan(k, lds);
        start += tokens;
        k += taken;
        tokens += all_tokens;
        taken += all_pages;
        if (s < p.N) {
            p.q_starts[s] = (int32_t)min(start, 0x7FFFFFFFLL);
            p.kv_lens_out[s] = old + n;
        }
        const auto page_of = [&](long long number) {
            const long long at = count - 1 - number;
            return at >= 0 ? p.free_pages[at] : -1;
        };
        if (need > 0) p.page_table[s * p.table_stride + c0] = page_of(k);
        for (uint64_t todo = __builtin_amdgcn_ballot_w64(need > 1); todo != 0; todo &= todo - 1) {
            const int l = __builtin_ctzll(todo), m = __builtin_amdgcn_readlane(need, l);
            const long long kl = readlane64(k, l);
            int32_t* row = p.page_table + (long long)(n0 + 64 * wave + l) * p.table_stride + __builtin_amdgcn_readlane(c0, l);
            for (int j = 1 + lane; j < m; j += 64) row[j] = page_of(kl + j);
        }
        if (!p.fill) continue;
        // (a sequence's pages have been written by its own wave)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
        if (n > 0 && start < p.T) put_token(p, start, s, old);
        for (uint64_t todo = __builtin_amdgcn_ballot_w64(n > 1); todo != 0; todo &= todo - 1) {
            const int l = __builtin_ctzll(todo), m = __builtin_amdgcn_readlane(n, l), o = __builtin_amdgcn_readlane(old, l);
            const long long t0 = readlane64(start, l);
            const long long most = min((long long)m, p.T - t0);
            for (int i = 1 + lane; i < most; i += 64) put_token(p, t0 + i, n0 + 64 * wave + l, (long long)o + i);
        }
    }
    if (tid == 0) {
        p.q_starts[p.N] = (int32_t)min(tokens, 0x7FFFFFFFLL);
        *p.free_count_out = (int32_t)max(count - taken, 0LL);
        if (p.pages_short) *p.pages_short = (int32_t)min(max(taken - count, 0LL), 0x7FFFFFFFLL);
    }
    if (p.fill)
        for (long long t = tokens + tid; t < p.T; t += kReserveThreads) {
            p.positions[t] = -1;
            p.slots[t] = -1;
        }
}

// Positions and slots, a thread a token: its sequence is the last that begins at or before it.
__global__ __launch_bounds__(256) void reserve_fill_kernel(const ReserveParams p) {
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    if (t >= p.T) return;
    int lo = 0, hi = p.N;  // sequences [0, lo) begin at or before it, [hi, N) behind
    while (lo < hi) {
        const int m = (int)(((unsigned)lo + (unsigned)hi) / 2);
        if (p.q_starts[m] <= t) lo = m + 1;
        else hi = m;
    }
    const int s = lo - 1;
    if (s < 0 || t >= p.q_starts[s + 1]) {
        p.positions[t] = -1;
        p.slots[t] = -1;
        return;
    }
    const int start = p.q_starts[s], n = p.q_starts[s + 1] - start;
    put_token(p, t, s, (long long)p.kv_lens_out[s] - n + (t - start));
}

}  // namespace

hipError_t launch_kv_reserve(const ReserveParams& args, hipStream_t stream) {
    ReserveParams p = args;
    p.fill = p.T <= kReserveFill;
    const hipError_t e = launch_kernel<reserve_kernel>(dim3(1), kReserveThreads, 0, stream, p);
    if (e != hipSuccess || p.fill) return e;
    return launch_kernel<reserve_fill_kernel>(dim3((unsigned)(((long long)p.T + 255) / 256)), 256, 0, stream, p);
}

}  // namespace sdpa
