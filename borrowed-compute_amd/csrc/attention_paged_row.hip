// attn_paged_row: launches whose items all have at most 16 query rows a KV head (paged_row.hpp).
#include "internal.hpp"
#include "paged_launch.hpp"
#include "paged_row.hpp"

namespace bchip {

namespace {

template <typename KVT, int NB, bool PK, int WAVES>
__global__ __launch_bounds__(64 * WAVES, NB > 4 ? 1 : 2) void attn_paged_row(const PgParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[PG_ROW_LDS<KVT, NB, WAVES>];
    row_block<KVT, NB, PK, WAVES>(p, blockIdx.x, lds);
}

template <typename KVT, int NB>
void launch(const PgParams& p, bool brief, hipStream_t s) {
    const dim3 grid((p.blocks + 7) / 8 * 8 * p.nkv);
    const bool few = pg_few(p);
    constexpr bool F16 = sizeof(KVT) == 2;
    constexpr int W = NB <= 4 ? 8 : 4;
    if (F16 && few) {
        if (brief) hipLaunchKernelGGL((attn_paged_row<KVT, NB, F16, W>), grid, dim3(64 * W), 0, s, p);
        else hipLaunchKernelGGL((attn_paged_row<KVT, NB, F16, 4>), grid, dim3(256), 0, s, p);
    } else {
        if (brief) hipLaunchKernelGGL((attn_paged_row<KVT, NB, false, W>), grid, dim3(64 * W), 0, s, p);
        else hipLaunchKernelGGL((attn_paged_row<KVT, NB, false, 4>), grid, dim3(256), 0, s, p);
    }
}

}  // namespace

void paged_rows_launch(const PgParams& p, bool f16_cache, bool brief, hipStream_t s) {
#define PG_ROW(NB) (f16_cache ? launch<f16, NB>(p, brief, s) : launch<float, NB>(p, brief, s))
    PG_BY_DIM(p.hd, PG_ROW)
#undef PG_ROW
}

}  // namespace bchip
