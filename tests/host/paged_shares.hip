// CPU check of the plan by shares (csrc/sdpa_paged.h), over random batches, with the
// blocks, targets and masks of the kernels of few rows:
//   - every block of every tile is walked once, in order, by the workgroup that holds it;
//   - slots of parts are inside the workspace and have one part each;
//   - every divided tile is merged by one workgroup, from the slots its parts were
//     written to, in their order, and no other tile is;
//   - without a workspace every tile is walked whole, by one workgroup.
#include <cstdio>
#include <map>
#include <random>
#include <vector>

#include "sdpa_paged.h"

using namespace sdpa;

#define CHECK(c)                                             \
    do {                                                     \
        if (!(c)) {                                          \
            printf("line %d: %s (case %d)\n", __LINE__, #c, cs); \
            return 1;                                        \
        }                                                    \
    } while (0)

struct Tile {
    long long first;
    int blocks;
};
struct Part {
    int u0, u1, slot;
};

int main() {
    std::mt19937 rng(11);
    const auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    constexpr int BM = kPagedSmallBM, BN = 128;
    for (int cs = 0; cs < 3000; ++cs) {
        // more sequences than lanes, many short ones, few of many blocks
        const int kind = cs % 4, N = kind == 0 ? pick(65, 300) : kind == 1 ? pick(1, 3) : pick(1, 64);
        const int G = pick(1, 16), H_kv = pick(1, 16), log2 = pick(4, 9);
        std::vector<int> starts{0}, lens;
        int most = 0;
        for (int s = 0; s < N; ++s) {
            const int n = pick(0, 9) == 0 ? pick(0, 40) : pick(0, 2);
            starts.push_back(starts.back() + n);
            lens.push_back(pick(0, 9) == 0 ? 0 : pick(0, kind == 1 ? 300000 : kind == 2 ? 300 : 9000));
            most = lens.back() > most ? lens.back() : most;
        }
        PagedBatch b{nullptr, nullptr, nullptr, 0, N, starts.back(), (most >> log2) + 1, 100, log2};
        std::vector<Tile> tiles;
        long long total = 0;
        for (int s = 0; s < N; ++s) {
            const SeqPlan q = seq_plan(starts[s], starts[s + 1], lens[s], b, G, false, BM, BN, 0);
            for (int t = 0; t < q.tiles * H_kv; ++t) {
                CHECK(q.blocks >= 1 && (long long)q.blocks * BN >= lens[s]);
                tiles.push_back({total, q.blocks});
                total += q.blocks;
            }
        }
        if (total == 0) continue;
        const auto holds = [&](long long at) {  // the last tile that begins at or before it
            size_t lo = 0, hi = tiles.size();
            while (hi - lo > 1) (tiles[(lo + hi) / 2].first <= at ? lo : hi) = (lo + hi) / 2;
            return lo;
        };
        const int l2 = kPagedTargetLog2 - cs / 4 % 2, n = (int)(total < (1LL << l2) ? total : 1LL << l2);
        for (int divide = 0; divide < 2; ++divide) {
            std::vector<std::vector<Part>> parts(tiles.size());
            std::map<int, int> used;
            for (int w = 0; w < n; ++w) {
                const long long end = share_begin(total, w + 1, n, l2);
                for (long long at = share_begin(total, w, n, l2); at < end;) {
                    const size_t i = holds(at);
                    const Tile t = tiles[i];
                    const ShareStep s = share_step(at, end, t.first, t.first + t.blocks, w, divide != 0);
                    CHECK(s.stop > at && s.u0 >= 0 && s.u0 < s.u1 && s.u1 <= t.blocks);
                    CHECK(t.first + s.u0 == at && t.first + s.u1 == s.stop);
                    if (!s.skip) {
                        CHECK(s.divided == (s.u0 != 0 || s.u1 != t.blocks));
                        if (s.divided) CHECK(s.slot >= 0 && s.slot < 2 << l2 && used[s.slot]++ == 0);
                        parts[i].push_back({s.u0, s.u1, s.slot});
                    }
                    at = s.stop;
                }
            }
            std::vector<int> merged(tiles.size(), 0);
            if (divide)
                for (int w = 0; w + 1 < n; ++w) {
                    const long long at = share_begin(total, w + 1, n, l2);
                    const size_t i = holds(at);
                    const int np = share_merge(total, at, tiles[i].first, tiles[i].blocks, w, n, l2);
                    if (np == 0) continue;
                    ++merged[i];
                    CHECK(np == (int)parts[i].size());
                    for (int k = 0; k < np; ++k) CHECK(share_slot(w, k) == parts[i][k].slot);
                }
            for (size_t i = 0; i < tiles.size(); ++i) {
                int u = 0;
                for (const Part& x : parts[i]) {
                    CHECK(x.u0 == u);
                    u = x.u1;
                }
                CHECK(u == tiles[i].blocks);
                CHECK(divide ? merged[i] == (parts[i].size() > 1) : parts[i].size() == 1);
            }
        }
    }
    printf("ok\n");
    return 0;
}
