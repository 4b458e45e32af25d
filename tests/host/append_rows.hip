// CPU check of how rows of queries alone are dealt to waves (csrc/sdpa_kv_append_device.h): the rows of
// every token and head are taken once, and four per group of lanes only where the waves are many and no more than an
// eighth of their rows are idle.
#include <cstdio>
#include <vector>

#include "sdpa_kv_append_device.h"

using namespace sdpa;

#define CHECK(c)                                                                 \
    do {                                                                         \
        if (!(c)) {                                                              \
            printf("line %d: %s (T %d, H %d, LPR %d)\n", __LINE__, #c, T, H, LPR); \
            return false;                                                        \
        }                                                                        \
    } while (0)

template <int LPR, int KU>
bool covers(int T, int H) {
    const AppendMap m = append_map<LPR, KU>(T, H);
    std::vector<int> seen((size_t)T * H, 0);
    for (long long u = 0; u < m.units; ++u)
        for (int group = 0; group < 64 / LPR; ++group)
            for (int i = 0; i < KU; ++i) {
                const long long tok = u / m.splits * m.tpw + group / m.gpt;
                const int h = (int)(u % m.splits) * m.gpt * KU + group % m.gpt + i * m.gpt;
                if (tok < T && h < H) ++seen[(size_t)tok * H + h];
            }
    for (int n : seen) CHECK(n == 1);
    return true;
}

template <int LPR>
bool check() {
    for (int H = 1; H <= 130; ++H) {
        for (int T : {1, 3, 17})
            if (!covers<LPR, 1>(T, H) || !covers<LPR, 4>(T, H)) return false;
        for (int T : {100, 1024, 2047, 2048, 9000, 100000}) {
            const AppendMap one = append_map<LPR, 1>(T, H), four = append_map<LPR, 4>(T, H);
            // idle rows of a full wave of heads
            const long long rows = 4LL * (64 / LPR) * four.units, used = (long long)T * H;
            const bool taken = append_four_rows<LPR>(T, H);
            CHECK(!taken || four.units >= 2048);
            CHECK(!taken || 8 * used >= 7 * rows - 8 * 256);
            CHECK(taken || four.units < 2048 || 8 * used < 7 * rows);
            CHECK(one.units >= four.units);
        }
    }
    return true;
}

int main() {
    if (!check<4>() || !check<8>() || !check<16>() || !check<64>()) return 1;
    printf("ok\n");
    return 0;
}
