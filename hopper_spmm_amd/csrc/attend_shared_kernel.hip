// Attention of sequences that begin with the same tokens: a group's prefix by tiles of rows of all its sequences, the keys behind it by each sequence's own, in one launch, and another one
// that adds up a row's sums.
//
// out_r = (sum over parts p of 2^(m_p - m) o_p) / (sum of 2^(m_p - m) l_p), m the largest reference m_p of the row's parts, l_p and o_p their totals and sums of values relative to it.
// Prefixes are bound by matrix instructions or by the L2, what is behind them by memory, so both run at a time: workgroups of the prefixes come first, as they are the longer ones.
// A token for each of 64 sequences of up to 1500 keys behind 8000, 32 heads on 8 of 128, bf16: 57.6 us, and 10.7 to add up 17 MB of sums (one behind the other 94; by attention alone, which reads the prefix 64 times, from the L2 as far as it goes, 232);
// drafts of up to 12 tokens over 5 prompts of up to 6000, 12 heads on 4 of 64, fp32, 60 + 7.6.
// Registers are short with heads of 161 to 256 elements, whose one wave a SIMD has 512: of 16-bit types 50 to 131 of them lie in memory where either kind of tile is of 128 rows, of fp32 94 to 98.
#include "attend_rows.hpp"
#include "attend_chunk.hpp"

namespace hspmm {

namespace {

constexpr uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }

// PrefixChunk, RestChunk: tiles of 128 rows, else of 16.  DR, DC: of the rows and the chunk kernel.  Workgroups: tiles and heads of the prefixes, part by part, then the others.
template <class K, bool BF, int DR, int DC, bool Whole, bool PrefixChunk, bool RestChunk>
__global__ __launch_bounds__(256, DC <= 64 && !PrefixChunk && !RestChunk ? 3 : DC <= 128 ? 2 : 1) void attend_shared_kernel(const AttendArgs prefix, const AttendArgs rest)
{
    constexpr uint32_t kLds = larger(PrefixChunk || RestChunk ? chunk_lds(DC, 4) : 0u, rows_lds(DR));
    const uint32_t of_prefix = prefix.tiles * prefix.heads.d, of_rest = rest.tiles * rest.heads.d, n_prefix = of_prefix * prefix.splits;
    if (blockIdx.x < n_prefix) {
        const uint32_t part = blockIdx.x / of_prefix, number = blockIdx.x - part * of_prefix;
        if constexpr (PrefixChunk) attend_chunk<BF, DC, 4, Whole, kSpanPrefix, kLds>(prefix, number, of_prefix, part);
        else attend_rows<K, Whole, DR, kSpanPrefix>(prefix, Lds<kLds>::bytes, number, part);
    } else {
        const uint32_t part = (blockIdx.x - n_prefix) / of_rest, number = blockIdx.x - n_prefix - part * of_rest;
        if constexpr (RestChunk) attend_chunk<BF, DC, 4, Whole, kSpanRest, kLds>(rest, number, of_rest, part);
        else attend_rows<K, Whole, DR, kSpanRest>(rest, Lds<kLds>::bytes, number, part);
    }
}

// A workgroup has a head of sixteen tokens, sixteen lanes each; kAtOnce parts of a row's sums on their way at a time, added in order.
template <class T, int DP>
__global__ __launch_bounds__(256) void attend_merge_kernel(const AttendArgs aa)
{
    constexpr uint32_t kEach = DP / 64u, kAtOnce = 8u, kPitch = DP + 2u;
    __shared__ T turned[16u * kPitch];
    const uint32_t row_here = threadIdx.x / 16u, token0 = blockIdx.x * 16u, token = token0 + row_here, head = blockIdx.y, d0 = threadIdx.x % 16u * 4u, D = aa.pages.head_dim;
    const BatchArgs &ba = aa.batch;
    // (tokens of no sequence are nobody's; a wave looks for its four tokens together)
    bool there = false;
#pragma unroll
    for (uint32_t k = 0; k < 4u; ++k) {
        const uint32_t t = token0 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64u) * 4u + k;
        const uint32_t b = last_at_most(ba.sequences, t, [&](uint32_t i) __attribute__((always_inline)) { return uint32_t(clamp_i32(ba.starts[i], 0, int32_t(ba.tokens))); });
        const bool is = place_in(ba, aa.pages, b, t).there;
        there = row_here % 4u == k ? is : there;
    }
    const bool by_tokens = aa.out.dim_stride != 1;
    if (!__syncthreads_or(there)) return;
    if (there) {
        const float *const row = aa.prefix.sums + int64_t(size_t(token) * aa.q_heads + head) * (D + kPrefixExtra);
        const float *const own = row + int64_t(aa.prefix.splits) * aa.prefix.part_stride;
        const f32x4 header = *reinterpret_cast<const f32x4 *>(own + D);
        const uint32_t rests = min(__builtin_bit_cast(uint32_t, float(header[2])), aa.splits), others = min(__builtin_bit_cast(uint32_t, float(header[3])), aa.prefix.splits), all = rests + others;
        float ref = -INFINITY, total = 0.f;
        f32x4 acc[kEach];
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (uint32_t p0 = 0; p0 < all; p0 += kAtOnce) {
            f32x4 x[kAtOnce][kEach], h[kAtOnce];
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
                const uint32_t p = p0 + k < all ? p0 + k : p0;
                const float *const from = row + int64_t(p < others ? p : aa.prefix.splits + p - others) * aa.prefix.part_stride;
                h[k] = *reinterpret_cast<const f32x4 *>(from + D);
#pragma unroll
                for (uint32_t e = 0; e < kEach; ++e) x[k][e] = *reinterpret_cast<const f32x4 *>(from + (d0 + 64u * e < D ? d0 + 64u * e : 0u));
            }
#pragma unroll
            for (uint32_t k = 0; k < kAtOnce; ++k) {
                if (p0 + k >= all) break;
                const float other = h[k][0], top = fmaxf(ref, other);
                const float keep = ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - top), by = other == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(other - top);
                total = total * keep + h[k][1] * by;
#pragma unroll
                for (uint32_t e = 0; e < kEach; ++e) acc[e] = acc[e] * keep + x[k][e] * by;
                ref = top;
            }
        }
        const bool any = !(total == 0.f);
        const float by = any ? 1.f / total : 0.f;
        T *const to = reinterpret_cast<T *>(aa.out.data) + int64_t(token) * aa.out.token_stride + int64_t(head) * aa.out.head_stride;
        const bool side_by_side = !by_tokens && (reinterpret_cast<uintptr_t>(to) & (4u * sizeof(T) - 1u)) == 0u;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) {
            const uint32_t d = d0 + 64u * e;
            if (d >= D) continue;
            typedef T four __attribute__((ext_vector_type(4)));
            const four x{T(acc[e][0] * by), T(acc[e][1] * by), T(acc[e][2] * by), T(acc[e][3] * by)};
            if (side_by_side) *reinterpret_cast<four *>(to + d) = x;
            else
#pragma unroll
                for (uint32_t c = 0; c < 4u; ++c) (by_tokens ? turned[row_here * kPitch + d + c] : to[d + c]) = x[c];
        }
        if (aa.lse && d0 == 0u) aa.lse[size_t(token) * aa.q_heads + head] = any ? (ref + __builtin_amdgcn_logf(total)) * kLn2 : -INFINITY;
    }
    if (!by_tokens) return;
    // elements apart, features x tokens for one: sixteen tokens of an element side by side (a lane its own token's, as in `there`)
    __shared__ bool theres[16];
    if (threadIdx.x % 16u == 0u) theres[row_here] = there;
    __syncthreads();
    const uint32_t r = threadIdx.x % 16u;
    if (!theres[r]) return;
    T *const to = reinterpret_cast<T *>(aa.out.data) + int64_t(token0 + r) * aa.out.token_stride + int64_t(head) * aa.out.head_stride;
    for (uint32_t d = threadIdx.x / 16u; d < D; d += 16u) to[int64_t(d) * aa.out.dim_stride] = turned[r * kPitch + d];
}

template <class K, bool BF, int DR, int DC, bool Whole>
void launch_kinds(const AttendArgs &prefix, const AttendArgs &rest, bool prefix_chunk, bool rest_chunk, hipStream_t s)
{
    const dim3 grid(prefix.tiles * prefix.heads.d * prefix.splits + rest.tiles * rest.heads.d * rest.splits), threads(256);
    if constexpr (K::kElem == 2) {
        if (prefix_chunk && rest_chunk) return attend_shared_kernel<K, BF, DR, DC, Whole, true, true><<<grid, threads, 0, s>>>(prefix, rest);
        if (prefix_chunk) return attend_shared_kernel<K, BF, DR, DC, Whole, true, false><<<grid, threads, 0, s>>>(prefix, rest);
    }
    // (heads that the chunk kernel's part has a form of its own for come here with tiles of it only)
    if constexpr (DR == DC) attend_shared_kernel<K, BF, DR, DC, Whole, false, false><<<grid, threads, 0, s>>>(prefix, rest);
}

template <class K, bool BF, int DR, int DC>
void launch(const AttendArgs &prefix, const AttendArgs &rest, bool prefix_chunk, bool rest_chunk, hipStream_t s)
{
    if (prefix.pages.page_tokens.d % 16u == 0u) launch_kinds<K, BF, DR, DC, true>(prefix, rest, prefix_chunk, rest_chunk, s);
    else launch_kinds<K, BF, DR, DC, false>(prefix, rest, prefix_chunk, rest_chunk, s);
}

template <bool BF>
void launch16(const AttendArgs &prefix, const AttendArgs &rest, bool prefix_chunk, bool rest_chunk, hipStream_t s)
{
    const uint32_t D = prefix.pages.head_dim;
    if (D <= 64u) launch<Rows16<BF, 64, false>, BF, 64, 64>(prefix, rest, prefix_chunk, rest_chunk, s);
    else if (D <= 96u && prefix_chunk) launch<Rows16<BF, 128, false>, BF, 128, 96>(prefix, rest, prefix_chunk, rest_chunk, s);
    else if (D <= 128u) launch<Rows16<BF, 128, false>, BF, 128, 128>(prefix, rest, prefix_chunk, rest_chunk, s);
    // (160 / 256 elements, heads of 160, 16 heads on 4, us: 16 x 40 tokens behind 6000 122 / 270, 16 x 100 224 / 603)
    else if (D <= 160u && prefix_chunk) launch<Rows16<BF, 256, false>, BF, 256, 160>(prefix, rest, prefix_chunk, rest_chunk, s);
    else launch<Rows16<BF, 256, false>, BF, 256, 256>(prefix, rest, prefix_chunk, rest_chunk, s);
}

template <class T>
void merge(const AttendArgs &aa, hipStream_t s)
{
    const dim3 grid((aa.batch.tokens + 15u) / 16u, aa.q_heads), threads(256);
    const uint32_t D = aa.pages.head_dim;
    if (D <= 64u) attend_merge_kernel<T, 64><<<grid, threads, 0, s>>>(aa);
    else if (D <= 128u) attend_merge_kernel<T, 128><<<grid, threads, 0, s>>>(aa);
    else attend_merge_kernel<T, 256><<<grid, threads, 0, s>>>(aa);
}

}  // namespace

hipError_t launch_attend_shared(int dtype, const AttendArgs &prefix, const AttendArgs &rest, bool prefix_chunk, bool rest_chunk, hipStream_t s)
{
    const uint32_t D = prefix.pages.head_dim;
    if (dtype == kDtypeF16) launch16<false>(prefix, rest, prefix_chunk, rest_chunk, s);
    else if (dtype == kDtypeBf16) launch16<true>(prefix, rest, prefix_chunk, rest_chunk, s);
    else if (D <= 64u) launch<Rows32<64>, false, 64, 64>(prefix, rest, false, false, s);
    else if (D <= 128u) launch<Rows32<128>, false, 128, 128>(prefix, rest, false, false, s);
    else launch<Rows32<256>, false, 256, 256>(prefix, rest, false, false, s);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (dtype == kDtypeF16) merge<_Float16>(rest, s);
    else if (dtype == kDtypeBf16) merge<__bf16>(rest, s);
    else merge<float>(rest, s);
    return hipGetLastError();
}

}  // namespace hspmm
