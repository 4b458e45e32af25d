// CPU check of what the C entries of norm and rotation hand to their kernels (the launches are
// recorded here, none runs): without rotated features no position is read, as
// the array of positions on no axis has no entries.
#include <cstdio>

#include "sdpa_paged_capi.hip"

namespace sdpa {
namespace {
NormRopeParams seen;
int calls = 0;
hipError_t take(const NormRopeParams& p) {
    seen = p;
    ++calls;
    return hipSuccess;
}
}  // namespace
int hip_status(hipError_t e) { return e == hipSuccess ? SDPA_OK : SDPA_ERR_HIP; }
hipError_t launch_norm_rope(const NormRopeParams& p, DType, hipStream_t) { return take(p); }
hipError_t launch_norm_rope_grad(const NormRopeParams& p, DType, hipStream_t) { return take(p); }
hipError_t launch_kv_append(const AppendParams&, DType, hipStream_t) { return hipErrorUnknown; }
hipError_t launch_kv_append_fp4(const AppendParams&, DType, hipStream_t) { return hipErrorUnknown; }
hipError_t launch_kv_read_fp4(const Fp4ReadParams&, DType, hipStream_t) { return hipErrorUnknown; }
hipError_t launch_kv_reserve(const ReserveParams&, hipStream_t) { return hipErrorUnknown; }
hipError_t launch_paged_fp4_small(const PagedParams&, DType, hipStream_t) { return hipErrorUnknown; }
hipError_t launch_paged_fp4(const PagedParams&, DType, hipStream_t) { return hipErrorUnknown; }
hipError_t launch_paged_f16_small(const PagedParams&, hipStream_t) { return hipErrorUnknown; }
hipError_t launch_paged_f16(const PagedParams&, hipStream_t) { return hipErrorUnknown; }
hipError_t launch_paged_f32_small(const PagedParams&, hipStream_t) { return hipErrorUnknown; }
hipError_t launch_paged_f32(const PagedParams&, hipStream_t) { return hipErrorUnknown; }
}  // namespace sdpa

#define CHECK(c)                                     \
    do {                                             \
        if (!(c)) {                                  \
            printf("line %d: %s\n", __LINE__, #c);   \
            return 1;                                \
        }                                            \
    } while (0)

int main() {
    // (addresses that are never read)
    void* some = reinterpret_cast<void*>(64);
    float* table = static_cast<float*>(some);
    int32_t* positions = static_cast<int32_t*>(some);
    const uint8_t pairs[16] = {1, 0, 1, 0};
    for (int R : {0, 8})
        for (int grad = 0; grad < 2; ++grad) {
            const int n_axes = R ? 2 : 0, before = sdpa::calls;
            const int st =
                grad ? sdpa_hip_qk_norm_rope_axes_grad(1, some, nullptr, some, nullptr, some, nullptr, some, nullptr, some, nullptr,
                                                       some, nullptr, nullptr, nullptr, nullptr, nullptr, 0, table, table, 9,
                                                       positions, 0, pairs, n_axes, nullptr, 0, 2, 5, 4, 2, 32, R, 1e-6f, 1, 0,
                                                       nullptr)
                     : sdpa_hip_qk_norm_rope_axes(1, some, nullptr, some, nullptr, some, nullptr, some, nullptr, nullptr, nullptr, 0,
                                                  table, table, 9, positions, 0, pairs, n_axes, 2, 5, 4, 2, 32, R, 1e-6f, 1, 0,
                                                  nullptr);
            CHECK(st == SDPA_OK && sdpa::calls == before + 1);
            CHECK(sdpa::seen.positions == (R ? positions : nullptr));
            CHECK(sdpa::seen.axes.used == (R ? 3 : 0));
        }
    printf("ok\n");
    return 0;
}
