// Rotary positions, and new keys and values into the pages of a cache.
//   y_a = x_a cos - x_b sin, y_b = x_a sin + x_b cos for the pairs (a, b) of a head's first `dims` elements, in fp32
// from 16-bit or fp32 elements, rounded once.  Every element is read and written once: memory bounds it.
#include "cache_device.h"
#include "spmm_tile_common.hpp"

namespace hspmm {

namespace {

template <int DT> struct Elem;
template <> struct Elem<kDtypeF16> { typedef _Float16 T; };
template <> struct Elem<kDtypeBf16> { typedef __bf16 T; };
template <> struct Elem<kDtypeF32> { typedef float T; };

// A pair turned, the same bits from every kernel: which product joins the sum is written down, and a sum does not become one instruction
// with its conversion to fp16, which rounds otherwise.
__device__ __forceinline__ float2 turn(float a, float b, const float2 cs, float sign)
{
    const float sn = sign * cs.y;
    float2 y{__builtin_fmaf(a, cs.x, -(b * sn)), __builtin_fmaf(a, sn, b * cs.x)};
    asm("" : "+v"(y.x), "+v"(y.y));
    return y;
}

// Which of a launch's heads this is: queries, then keys, then values.
struct HeadRole { const HeadsArgs *from; uint32_t head; bool query, key; };
__device__ __forceinline__ HeadRole head_role(const RotaryArgs &ra, uint32_t h)
{
    if (h < ra.q_heads) return HeadRole{&ra.q, h, true, false};
    h -= ra.q_heads;
    if (h < ra.k_heads) return HeadRole{&ra.k, h, false, true};
    return HeadRole{&ra.v, h - ra.k_heads, false, false};
}

__device__ __forceinline__ const float2 *angle_row(const RotaryArgs &ra, int32_t position)
{
    return reinterpret_cast<const float2 *>(ra.table) + size_t(clamp_i32(position, 0, int32_t(ra.positions) - 1)) * (ra.dims / 2u);
}

// Heads whose elements lie side by side in x and in y: a lane moves V of them at a time, with their partners where those are
// V elements of their own (HALF).  A token's items: per turned head and, HALF, pair of pieces (else piece) one, per piece that only is copied one.
template <int DT, int V, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs ra, const Divisor by_items, const Divisor by_turned, const Divisor by_copied,
                                                     const uint32_t turned_items, const uint64_t all)
{
    typedef typename Elem<DT>::T T;
    struct alignas(V * sizeof(T)) Piece { T e[V]; };
    const uint32_t pairs = HALF && ra.table ? ra.dims / 2u / V : 0u;                 // items of a turned head that are two pieces
    for (uint64_t i = uint64_t(blockIdx.x) * 256u + threadIdx.x; i < all; i += uint64_t(gridDim.x) * 256u) {
        const uint32_t t = by_items.quotient(uint32_t(i));
        uint32_t item = uint32_t(i) - t * by_items.d;
        uint32_t h, c;
        if (item < turned_items) {
            h = by_turned.quotient(item);
            c = item - h * by_turned.d;
        } else {
            item -= turned_items;
            const uint32_t v = by_copied.quotient(item);
            h = ra.q_heads + ra.k_heads + v;
            c = item - v * by_copied.d;
        }
        const HeadRole role = head_role(ra, h);
        TokenPlace place{0u, 0, true};
        if (ra.batch.starts) place = token_place(ra.batch, ra.pages, t);
        if (!place.there) continue;
        const T *x = reinterpret_cast<const T *>(role.from->data) + int64_t(t) * role.from->token_stride + int64_t(role.head) * role.from->head_stride;
        T *y;
        if (role.query) {
            y = reinterpret_cast<T *>(ra.q_out.data) + int64_t(t) * ra.q_out.token_stride + int64_t(role.head) * ra.q_out.head_stride;
        } else {
            const int64_t at = row_offset(ra.pages, place.sequence, place.position, role.head);
            if (at < 0) continue;
            y = reinterpret_cast<T *>(role.key ? ra.pages.keys : ra.pages.values) + at;
        }
        const bool turns = ra.table && (role.query || role.key);
        const float2 *angles = turns ? angle_row(ra, ra.at ? ra.at[t] : place.position) : nullptr;
        if (turns && HALF && c < pairs) {
            const uint32_t a = c * V, b = a + ra.dims / 2u;
            const Piece p = *reinterpret_cast<const Piece *>(x + a), q = *reinterpret_cast<const Piece *>(x + b);
            Piece r, s;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 y2 = turn(float(p.e[e]), float(q.e[e]), angles[a + e], ra.sign);
                r.e[e] = T(y2.x);
                s.e[e] = T(y2.y);
            }
            *reinterpret_cast<Piece *>(y + a) = r;
            *reinterpret_cast<Piece *>(y + b) = s;
            continue;
        }
        if (turns && HALF) c += pairs;
        Piece p = *reinterpret_cast<const Piece *>(x + c * V);
        if constexpr (!HALF && V > 1) {
            if (turns) {
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    if (c * V + e >= ra.dims) break;
                    const float2 y2 = turn(float(p.e[e]), float(p.e[e + 1]), angles[(c * V + e) / 2u], ra.sign);
                    p.e[e] = T(y2.x);
                    p.e[e + 1] = T(y2.y);
                }
            }
        }
        *reinterpret_cast<Piece *>(y + c * V) = p;
    }
}

// Any strides: a workgroup has tt (up to 64, a power of two) tokens of one head and 32 of its pairs (all elements count in pairs here, those that do not turn, too).
// Lanes lie along tokens where x is read or y is written with tokens side by side, along pairs else; between the two the elements go through LDS.
template <int DT>
__global__ __launch_bounds__(256) void rotary_strided_kernel(const RotaryArgs ra, const uint32_t tt_log)
{
    typedef typename Elem<DT>::T T;
    constexpr uint32_t kPairs = 32u;
    __shared__ T image[64u * (2u * kPairs + 2u)];
    const uint32_t tt = 1u << tt_log, t0 = blockIdx.x << tt_log, pair0 = blockIdx.y * kPairs;
    const HeadRole role = head_role(ra, blockIdx.z);
    const uint32_t all_pairs = ra.head_dim / 2u + (ra.head_dim & 1u), dims = ra.table && (role.query || role.key) ? ra.dims : 0u;
    const bool by_token = role.from->dim_stride != 1;
    // element of pair p's first or second half
    auto element = [&](uint32_t p, uint32_t second) __attribute__((always_inline)) {
        if (ra.interleaved || 2u * p >= dims) return 2u * p + second;
        return p + second * (dims / 2u);
    };
    for (uint32_t i = threadIdx.x; i < tt * kPairs; i += 256u) {
        const uint32_t ti = by_token ? i & (tt - 1u) : i / kPairs, pi = by_token ? i >> tt_log : i % kPairs, t = t0 + ti, p = pair0 + pi;
        if (t >= ra.tokens || p >= all_pairs) continue;
        const T *x = reinterpret_cast<const T *>(role.from->data) + int64_t(t) * role.from->token_stride + int64_t(role.head) * role.from->head_stride;
        const uint32_t a = element(p, 0u), b = element(p, 1u);
        T u = x[int64_t(a) * role.from->dim_stride], w = T(0.f);
        if (b < ra.head_dim) w = x[int64_t(b) * role.from->dim_stride];
        if (2u * p < dims) {
            int32_t at;
            if (ra.at) at = ra.at[t];
            else {
                const TokenPlace place = token_place(ra.batch, ra.pages, t);
                if (!place.there) continue;
                at = place.position;
            }
            const float2 y2 = turn(float(u), float(w), angle_row(ra, at)[p], ra.sign);
            u = T(y2.x);
            w = T(y2.y);
        }
        image[ti * (2u * kPairs + 2u) + 2u * pi] = u;
        image[ti * (2u * kPairs + 2u) + 2u * pi + 1u] = w;
    }
    __syncthreads();
    const bool out_by_token = role.query && ra.q_out.dim_stride != 1;
    for (uint32_t i = threadIdx.x; i < tt * 2u * kPairs; i += 256u) {
        uint32_t ti, pi, second;
        if (out_by_token) { ti = i & (tt - 1u); pi = (i >> tt_log) / 2u; second = (i >> tt_log) & 1u; }
        else if (ra.interleaved || 2u * (pair0 + kPairs) > dims) { ti = i / (2u * kPairs); pi = i / 2u % kPairs; second = i & 1u; }
        else { ti = i / (2u * kPairs); second = i / kPairs & 1u; pi = i % kPairs; }
        const uint32_t t = t0 + ti, p = pair0 + pi, e = element(p, second);
        if (t >= ra.tokens || p >= all_pairs || e >= ra.head_dim) continue;
        TokenPlace place{0u, 0, true};
        if (ra.batch.starts) place = token_place(ra.batch, ra.pages, t);
        if (!place.there) continue;
        const T v = image[ti * (2u * kPairs + 2u) + 2u * pi + second];
        if (role.query) {
            reinterpret_cast<T *>(ra.q_out.data)[int64_t(t) * ra.q_out.token_stride + int64_t(role.head) * ra.q_out.head_stride + int64_t(e) * ra.q_out.dim_stride] = v;
        } else {
            const int64_t at = row_offset(ra.pages, place.sequence, place.position, role.head);
            if (at >= 0) reinterpret_cast<T *>(role.key ? ra.pages.keys : ra.pages.values)[at + e] = v;
        }
    }
}

template <int DT, int V, bool HALF>
void launch_pieces(const RotaryArgs &ra, hipStream_t s)
{
    const uint32_t pieces = ra.head_dim / V, turned = HALF && ra.table ? pieces - ra.dims / 2u / V : pieces;
    const uint32_t turned_items = (ra.q_heads + ra.k_heads) * turned, items = turned_items + ra.k_heads * pieces;
    // (numbers of items stay below 2^31: tokens in several launches beyond)
    const uint32_t most = 0x7FFFFFFFu / items;
    for (uint32_t t = 0; t < ra.tokens; t += most) {
        RotaryArgs part = ra;
        if (ra.tokens > most) {
            part.tokens = ra.tokens - t < most ? ra.tokens - t : most;
            // (only rotations of whole tensors are that large: a batch's tokens are numbered as a whole)
            const int64_t el = DT == kDtypeF32 ? 4 : 2;
            part.q.data += int64_t(t) * ra.q.token_stride * el;
            part.q_out.data += int64_t(t) * ra.q_out.token_stride * el;
            part.at += t;
        }
        const uint64_t all = uint64_t(part.tokens) * items, groups = (all + 255u) / 256u;
        rotary_kernel<DT, V, HALF><<<dim3(uint32_t(groups < (1u << 20) ? groups : 1u << 20)), dim3(256), 0, s>>>(
            part, Divisor::of(items), Divisor::of(turned), Divisor::of(pieces), turned_items, all);
    }
}

template <int DT>
hipError_t launch_type(const RotaryArgs &ra, uint32_t vec, hipStream_t s)
{
    const bool half = !ra.interleaved && ra.table;
    switch (vec) {
    case 8: if constexpr (DT != kDtypeF32) { if (half) launch_pieces<DT, 8, true>(ra, s); else launch_pieces<DT, 8, false>(ra, s); } break;
    case 4: if (half) launch_pieces<DT, 4, true>(ra, s); else launch_pieces<DT, 4, false>(ra, s); break;
    case 2: if (half) launch_pieces<DT, 2, true>(ra, s); else launch_pieces<DT, 2, false>(ra, s); break;
    case 1: launch_pieces<DT, 1, true>(ra, s); break;
    default: {
        uint32_t tt_log = 0;
        while (tt_log < 6u && (1u << tt_log) < ra.tokens) ++tt_log;
        const uint32_t all_pairs = (ra.head_dim + 1u) / 2u;
        rotary_strided_kernel<DT><<<dim3((ra.tokens + (1u << tt_log) - 1u) >> tt_log, (all_pairs + 31u) / 32u, ra.q_heads + 2u * ra.k_heads), dim3(256), 0, s>>>(ra, tt_log);
    }
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rotary(int dtype, const RotaryArgs &ra, uint32_t vec, hipStream_t s)
{
    if (dtype == kDtypeF16) return launch_type<kDtypeF16>(ra, vec, s);
    if (dtype == kDtypeBf16) return launch_type<kDtypeBf16>(ra, vec, s);
    return launch_type<kDtypeF32>(ra, vec, s);
}

}  // namespace hspmm
