// Attention of many rows of queries - chunks of a prompt - over the pages of a cache, 16-bit types.
#include "attend_chunk.hpp"

namespace hspmm {

namespace {

template <bool BF, int DP, int W, bool Whole, AttendSpan Span>
__global__ __launch_bounds__(64 * W, DP <= 128 ? 2 : 1) void attend_chunk_kernel(const AttendArgs aa)
{
    attend_chunk<BF, DP, W, Whole, Span, chunk_lds(DP, W)>(aa, blockIdx.x, gridDim.x, blockIdx.y);
}

template <bool BF, int DP, int W, AttendSpan Span>
void launch_span(const AttendArgs &aa, hipStream_t s)
{
    const dim3 grid(aa.tiles * aa.heads.d, aa.splits);
    if (aa.pages.page_tokens.d % 16u == 0u) attend_chunk_kernel<BF, DP, W, true, Span><<<grid, dim3(64 * W), 0, s>>>(aa);
    else attend_chunk_kernel<BF, DP, W, false, Span><<<grid, dim3(64 * W), 0, s>>>(aa);
}

template <bool BF, int DP, int W>
void launch(const AttendArgs &aa, bool both, hipStream_t s)
{
    if (both) launch_span<BF, DP, W, kSpanBoth>(aa, s);
    else launch_span<BF, DP, W, kSpanAll>(aa, s);
}

template <bool BF>
void launch_type(const AttendArgs &aa, bool both, uint32_t rows_log, hipStream_t s)
{
    const uint32_t D = aa.pages.head_dim;
    if (rows_log == 8u) launch<BF, 128, 8>(aa, both, s);
    else if (D <= 64u) launch<BF, 64, 4>(aa, both, s);
    else if (D <= 96u) launch<BF, 96, 4>(aa, both, s);
    else if (D <= 128u) launch<BF, 128, 4>(aa, both, s);
    else if (D <= 160u) launch<BF, 160, 4>(aa, both, s);
    else launch<BF, 256, 4>(aa, both, s);
}

}  // namespace

hipError_t launch_attend_chunk(int dtype, const AttendArgs &aa, bool both, uint32_t rows_log, hipStream_t s)
{
    if (dtype == kDtypeF16) launch_type<false>(aa, both, rows_log, s);
    else launch_type<true>(aa, both, rows_log, s);
    return hipGetLastError();
}

}  // namespace hspmm
