// Attention of new tokens over the pages of a cache: out = softmax(scale q k) v.
#include "cache_device.h"
#include "spmm_tile_common.hpp"

namespace hspmm {

namespace {

template <int DT> struct Elem;
template <> struct Elem<kDtypeF16> { typedef _Float16 T; };
template <> struct Elem<kDtypeBf16> { typedef __bf16 T; };
template <> struct Elem<kDtypeF32> { typedef float T; };

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// A wave has a token and a head of queries: 64 keys at a time, a lane each, then a lane has elements of the values.
template <int DT>
__global__ __launch_bounds__(64) void attend_simple_kernel(const AttendArgs aa)
{
    typedef typename Elem<DT>::T T;
    constexpr uint32_t kPiece = 16u / sizeof(T);
    struct alignas(16) Piece { T e[kPiece]; };
    __shared__ float q[256], p[64];
    __shared__ int64_t rows[64];
    const uint32_t t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, D = aa.pages.head_dim;
    const TokenPlace place = token_place(aa.batch, aa.pages, t);
    if (!place.there) return;
    const uint32_t head = aa.shared.quotient(h);
    const T *qg = reinterpret_cast<const T *>(aa.q.data) + int64_t(t) * aa.q.token_stride + int64_t(h) * aa.q.head_stride;
    for (uint32_t d = lane; d < D; d += 64u) q[d] = float(qg[d]);
    __syncthreads();
    const int32_t length = tokens_held(aa.pages, place.sequence);
    const int32_t end = aa.causal ? place.position + 1 : length;
    const int32_t begin = aa.window && int64_t(end) > int64_t(aa.window) ? end - int32_t(aa.window) : 0;
    float most = -INFINITY, total = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    const T *keys = reinterpret_cast<const T *>(aa.pages.keys), *values = reinterpret_cast<const T *>(aa.pages.values);
    for (int32_t j0 = begin; j0 < end; j0 += 64) {
        const int32_t j = j0 + int32_t(lane);
        const int64_t at = j < end ? row_offset(aa.pages, place.sequence, j, head) : -1;
        float s = -INFINITY;
        if (at >= 0) {
            float dot = 0.f;
            for (uint32_t d = 0; d < D; d += kPiece) {
                const Piece k = *reinterpret_cast<const Piece *>(keys + at + d);
#pragma unroll
                for (uint32_t e = 0; e < kPiece; ++e) dot += q[d + e] * float(k.e[e]);
            }
            s = dot * aa.scale;
        }
        const float now = fmaxf(most, wave_max(s));
        const float base = now > -INFINITY ? now : 0.f;
        const float w = at >= 0 ? expf(s - base) : 0.f, keep = expf(most - base);
        total = total * keep + wave_sum(w);
        most = now;
        __syncthreads();
        p[lane] = w;
        rows[lane] = at;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t d = lane + 64u * i;
            if (d >= D) break;
            float sum = o[i] * keep;
            for (uint32_t k = 0; k < 64u; ++k)
                if (rows[k] >= 0) sum += p[k] * float(values[rows[k] + d]);
            o[i] = sum;
        }
    }
    T *og = reinterpret_cast<T *>(aa.out.data) + int64_t(t) * aa.out.token_stride + int64_t(h) * aa.out.head_stride;
    const float by = total > 0.f || total != total ? 1.f / total : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t d = lane + 64u * i;
        if (d < D) og[int64_t(d) * aa.out.dim_stride] = T(o[i] * by);
    }
    if (aa.lse && lane == 0u) aa.lse[size_t(t) * aa.q_heads + h] = most + logf(total);
}

}  // namespace

hipError_t launch_attend_simple(int dtype, const AttendArgs &aa, hipStream_t s)
{
    const dim3 grid(aa.batch.tokens, aa.q_heads);
    if (dtype == kDtypeF16) attend_simple_kernel<kDtypeF16><<<grid, dim3(64), 0, s>>>(aa);
    else if (dtype == kDtypeBf16) attend_simple_kernel<kDtypeBf16><<<grid, dim3(64), 0, s>>>(aa);
    else attend_simple_kernel<kDtypeF32><<<grid, dim3(64), 0, s>>>(aa);
    return hipGetLastError();
}

}  // namespace hspmm
