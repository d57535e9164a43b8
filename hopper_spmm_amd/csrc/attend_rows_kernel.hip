// Attention of a few rows of queries - single new tokens, and the heads that share their keys - over the pages of a cache.
#include "attend_rows.hpp"

namespace hspmm {

namespace {

template <class K, bool Whole, int DP>
__global__ __launch_bounds__(64 * kRowWaves, DP <= 64 ? 3 : DP <= 128 ? 2 : 1) void attend_rows_kernel(const AttendArgs aa)
{
    __shared__ __attribute__((aligned(16))) char lds[rows_lds(DP)];
    attend_rows<K, Whole, DP, kSpanAll>(aa, lds, blockIdx.x, blockIdx.y);
}

template <class K, int DP>
void launch(const AttendArgs &aa, hipStream_t s)
{
    const dim3 grid(aa.tiles * aa.heads.d, aa.splits);
    if (aa.pages.page_tokens.d % 16u == 0u) attend_rows_kernel<K, true, DP><<<grid, dim3(64 * kRowWaves), 0, s>>>(aa);
    else attend_rows_kernel<K, false, DP><<<grid, dim3(64 * kRowWaves), 0, s>>>(aa);
}

template <bool BF, bool Past>
void launch16(const AttendArgs &aa, hipStream_t s)
{
    const uint32_t D = aa.pages.head_dim;
    if (D <= 64u) launch<Rows16<BF, 64, Past>, 64>(aa, s);
    else if (D <= 128u) launch<Rows16<BF, 128, Past>, 128>(aa, s);
    else launch<Rows16<BF, 256, Past>, 256>(aa, s);
}

}  // namespace

hipError_t launch_attend_rows(int dtype, const AttendArgs &aa, bool past, hipStream_t s)
{
    const uint32_t D = aa.pages.head_dim;
    if (dtype == kDtypeF16) {
        if (past) launch16<false, true>(aa, s);
        else launch16<false, false>(aa, s);
    } else if (dtype == kDtypeBf16) {
        if (past) launch16<true, true>(aa, s);
        else launch16<true, false>(aa, s);
    } else {
        if (D <= 64u) launch<Rows32<64>, 64>(aa, s);
        else if (D <= 128u) launch<Rows32<128>, 128>(aa, s);
        else launch<Rows32<256>, 256>(aa, s);
    }
    return hipGetLastError();
}

}  // namespace hspmm
