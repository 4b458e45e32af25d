// CPU check of the division of a paged batch over workgroups (csrc/sdpa_paged.h),
// over random batches, garbage ones among them:
//   - the items of a launch fit its grid, the parts of divided tiles the
//     workspace, and the divided tiles the merge's grid;
//   - every sequence whose range is one is in the plan, and no other;
//   - tiles cover the rows, and parts of a tile its blocks, once each;
//   - tokens and lengths stay inside the batch, whatever the arrays hold;
//   - shares are in order and equal to one block, and every block has its owner;
//   - workgroup ids map one to one onto the items.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "sdpa_paged_device.h"
#include "sdpa_parts.h"

using namespace sdpa;

#define CHECK(c)                                             \
    do {                                                     \
        if (!(c)) {                                          \
            printf("line %d: %s (case %d)\n", __LINE__, #c, cs); \
            return 1;                                        \
        }                                                    \
    } while (0)

int main() {
    std::mt19937 rng(7);
    const auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    for (int cs = 0; cs < 4000; ++cs) {
        const bool garbage = cs % 4 == 3;
        const int N = pick(1, cs % 10 == 0 ? 300 : 40), G = pick(1, 16), H_kv = pick(1, 16), log2 = pick(4, 9);
        const int big = pick(0, 3);
        std::vector<int> starts{0}, lens;
        int most = 0;
        for (int s = 0; s < N; ++s) {
            const int n = pick(0, 4) == 0 ? pick(0, big == 0 ? 3000 : 200) : pick(0, 2);
            starts.push_back(starts.back() + n);
            lens.push_back(n + (pick(0, 2) ? pick(0, big == 1 ? 100000 : 3000) : 0));
            if (pick(0, 30) == 0) lens.back() = 0;
            most = lens.back() > most ? lens.back() : most;
        }
        PagedParams p{};
        p.batch = PagedBatch{nullptr, nullptr, nullptr, 0, N, starts.back() + pick(0, 3), (most >> log2) + pick(0, 1), 100, log2};
        if (garbage)
            for (int i = 0; i < 5; ++i) {
                starts[pick(0, N)] = (int)rng() >> pick(0, 28);
                lens[pick(0, N - 1)] = (int)rng() >> pick(0, 28);
            }
        p.H_kv = H_kv;
        p.G = G;
        p.causal = pick(0, 1);
        p.target_log2 = kPagedTargetLog2;
        p.divide = pick(0, 5) != 0;
        const int target = 1 << p.target_log2;
        const int cap = p.batch.width << log2;
        for (int kernel = 0; kernel < 2; ++kernel) {
            const int BM = kernel ? kPagedBM : kPagedSmallBM, BN = kernel ? 64 : 32;
            std::vector<int> seen(N, 0);
            long long cost = 0, items = 0, slots = 0, divided = 0;
            std::vector<SeqPlan> plans;
            const auto plan = [&](int s, int chunk) {
                return seq_plan(starts[s], starts[s + 1], lens[s], p.batch, G, p.causal != 0, BM, BN, chunk);
            };
            for (int s = 0; s < N; ++s) cost += (long long)plan(s, 0).tiles * plan(s, 0).blocks;
            const int one = pick(0, 1) ? kPagedOnePerCu : 0;
            const int chunk = p.divide ? plan_chunk(cost * H_kv, p.target_log2, kPagedMinChunk * 64 / BN, one) : 0;
            for (int s = 0; s < N; ++s) {
                const SeqPlan q = plan(s, chunk);
                if (q.tiles == 0) continue;
                ++seen[s];
                CHECK(q.q0 >= 0 && q.n > 0 && q.q0 + q.n <= p.batch.T);
                CHECK(q.len >= 0 && q.len <= cap && q.parts >= 1 && q.parts <= kPagedMaxParts && q.blocks >= 1);
                CHECK(q.bad == (lens[s] > cap));
                CHECK((long long)q.tiles * BM >= (long long)q.n * G && (long long)(q.tiles - 1) * BM < (long long)q.n * G);
                CHECK(p.divide || q.parts == 1);
                items += (long long)q.tiles * q.parts * H_kv;
                if (q.parts > 1) {
                    slots += (long long)q.tiles * q.parts * H_kv;
                    divided += (long long)q.tiles * H_kv;
                }
                const int nblk = pick(0, 2 * q.blocks);
                CHECK(part_begin(nblk, 0, q.parts) == 0 && part_begin(nblk, q.parts, q.parts) == nblk);
                for (int i = 0; i < q.parts; ++i) CHECK(part_begin(nblk, i, q.parts) <= part_begin(nblk, i + 1, q.parts));
            }
            CHECK(slots <= 2 * target && divided <= target);
            if (!garbage) CHECK(items <= paged_max_tiles(p, BM) + (p.divide ? target : 0));
            if (cost > 0) {
                const long long total = cost * H_kv;
                const int n = (int)(total < target ? total : target), l2 = p.target_log2;
                CHECK(share_begin(total, 0, n, l2) == 0 && share_begin(total, n, n, l2) == total);
                for (int w = 0; w < n; ++w) {
                    const long long a = share_begin(total, w, n, l2), b = share_begin(total, w + 1, n, l2);
                    CHECK(b - a >= total / n && b - a <= total / n + 1);
                    CHECK(share_owner(total, a, n, l2) == w && share_owner(total, b - 1, n, l2) == w);
                }
            }
            if (cs % 50 == 0) {
                const int n = (int)items;
                std::vector<char> hit(n, 0);
                for (int id = 0; id < xcd_grid(n); ++id) {
                    const int at = xcd_item(id, n);
                    CHECK(at >= -1 && at < n);
                    if (at >= 0) CHECK(!hit[at]++);
                }
                for (int i = 0; i < n; ++i) CHECK(hit[i]);
            }
            for (int s = 0; s < N; ++s) {
                const long long n = (long long)starts[s + 1] - starts[s];
                const bool valid = starts[s] >= 0 && n > 0 && starts[s + 1] <= p.batch.T;
                CHECK(seen[s] == (valid ? 1 : 0));
            }
        }
    }
    printf("ok\n");
    return 0;
}
