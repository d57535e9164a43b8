// Attention of a few rows of queries - single new tokens, and the heads that share their keys - over the pages of a cache.
#include "attend_rows.hpp"

namespace hspmm {

namespace {

// kSpanBoth: small calls over shared prefixes, whose keys are looked up one by one (8 beams of a prompt of 1000, 32 heads on 8, fp16: 13.2 us, 12.8 without prefixes).
template <class K, bool Whole, int DP, AttendSpan Span>
__global__ __launch_bounds__(64 * kRowWaves, DP <= 64 ? 3 : DP <= 128 ? 2 : 1) void attend_rows_kernel(const AttendArgs aa)
{
    __shared__ __attribute__((aligned(16))) char lds[rows_lds(DP)];
    attend_rows<K, Whole, DP, Span>(aa, lds, blockIdx.x, blockIdx.y);
}

template <class K, int DP, AttendSpan Span>
void launch(const AttendArgs &aa, hipStream_t s)
{
    const dim3 grid(aa.tiles * aa.heads.d, aa.splits);
    if constexpr (Span == kSpanAll) {
        if (aa.pages.page_tokens.d % 16u == 0u) return attend_rows_kernel<K, true, DP, Span><<<grid, dim3(64 * kRowWaves), 0, s>>>(aa);
    }
    attend_rows_kernel<K, false, DP, Span><<<grid, dim3(64 * kRowWaves), 0, s>>>(aa);
}

template <bool BF, bool Past, AttendSpan Span>
void launch16(const AttendArgs &aa, hipStream_t s)
{
    const uint32_t D = aa.pages.head_dim;
    if (D <= 64u) launch<Rows16<BF, 64, Past>, 64, Span>(aa, s);
    else if (D <= 128u) launch<Rows16<BF, 128, Past>, 128, Span>(aa, s);
    else launch<Rows16<BF, 256, Past>, 256, Span>(aa, s);
}

template <AttendSpan Span>
void launch32(const AttendArgs &aa, hipStream_t s)
{
    const uint32_t D = aa.pages.head_dim;
    if (D <= 64u) launch<Rows32<64>, 64, Span>(aa, s);
    else if (D <= 128u) launch<Rows32<128>, 128, Span>(aa, s);
    else launch<Rows32<256>, 256, Span>(aa, s);
}

template <bool BF>
void launch_type(const AttendArgs &aa, bool past, bool both, hipStream_t s)
{
    if (both) launch16<BF, false, kSpanBoth>(aa, s);
    else if (past) launch16<BF, true, kSpanAll>(aa, s);
    else launch16<BF, false, kSpanAll>(aa, s);
}

}  // namespace

hipError_t launch_attend_rows(int dtype, const AttendArgs &aa, bool past, bool both, hipStream_t s)
{
    if (dtype == kDtypeF16) launch_type<false>(aa, past, both, s);
    else if (dtype == kDtypeBf16) launch_type<true>(aa, past, both, s);
    else if (both) launch32<kSpanBoth>(aa, s);
    else launch32<kSpanAll>(aa, s);
    return hipGetLastError();
}

}  // namespace hspmm
