// Rotary positions, and new keys and values into the pages of a cache.
//   y_a = x_a cos - x_b sin, y_b = x_a sin + x_b cos for the pairs (a, b) of a head's first `dims` elements, in fp32
// from 16-bit or fp32 elements, rounded once.  Every element is read and written once: memory bounds it (a large copy: 4.8 TB/s).  us: 16384 tokens of 32
// heads of 128, fp16, 52, 5.2 TB/s; 12000 tokens of 50 heads of 80, fp32, into pages of 24, 87, 4.4 TB/s; 4096 tokens of 48 heads of 128, bf16, into pages
// 20, from features x tokens 37, 2.7 TB/s, where a lane moves an element of 2 bytes at a time (fp32 50, 4.0 TB/s); few tokens 7, which is the host's call.
#include "cache_device.h"
#include "spmm_tile_common.hpp"
#include <algorithm>

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

// A store that does not stay in the L2: what a launch writes is not read again in it (gradient of 16384 tokens 65 -> 51 us, 4096 tokens of 48 heads
// 29 -> 20).
template <class T, class P> __device__ __forceinline__ void store_past(T *to, const P &p)
{
    if constexpr (sizeof(P) >= 4u) {
        typedef uint32_t words __attribute__((ext_vector_type(sizeof(P) / 4u)));
        __builtin_nontemporal_store(__builtin_bit_cast(words, p), reinterpret_cast<words *>(to));
    } else {
        *reinterpret_cast<P *>(to) = p;
    }
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

// Where token t of a batch stands, t the same in every lane: the wave looks at 64 batch rows at a time.
__device__ __forceinline__ TokenPlace wave_token_place(const BatchArgs &ba, const PagesArgs &pg, uint32_t t)
{
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t lo = 0, n = ba.sequences;
    while (n > 1u) {
        const uint32_t step = (n + 63u) / 64u, b = lane * step;
        const uint32_t below = uint32_t(__popcll(__ballot(b < n && ba.starts[lo + (b < n ? b : 0u)] <= int32_t(t))));
        const uint32_t skip = (below ? below - 1u : 0u) * step;
        lo += skip;
        n = n - skip < step ? n - skip : step;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    return place_in(ba, pg, lo, t);
}

// Heads whose elements lie side by side in x and in y: a lane moves V of them at a time, with their partners where those are V elements of their
// own (HALF).  A wave has a token and a range of its heads, so that where the token stands is found once; its lanes lie along a head's pieces (a pair of pieces
// that turn, else a piece) and along heads, and keep their angles from head to head.  kAhead pieces of a lane are asked for before the first is turned.
template <int DT, int V, bool HALF>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs ra, const uint32_t heads_each, const uint32_t turned_items, const uint32_t copied_items)
{
    typedef typename Elem<DT>::T T;
    struct alignas(V * sizeof(T)) Piece { T e[V]; };
    constexpr int kAhead = 4;
    const uint32_t lane = threadIdx.x & 63u, t = __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6));
    if (t >= ra.tokens) return;
    const uint32_t h0 = blockIdx.y * heads_each, all = ra.q_heads + 2u * ra.k_heads, h1 = h0 + heads_each < all ? h0 + heads_each : all;
    TokenPlace place{0u, 0, true};
    int64_t at = -1;                                                             // of head 0 in the pages
    if (ra.batch.starts) {
        place = wave_token_place(ra.batch, ra.pages, t);
        if (!place.there) return;
        at = row_offset(ra.pages, place.sequence, place.position, 0u);
    }
    const uint32_t pairs = HALF && ra.table ? ra.dims / 2u / V : 0u;            // items of a turned head that are two pieces
    const float2 *angles = ra.table ? angle_row(ra, ra.at ? ra.at[t] : place.position) : nullptr;
    const uint32_t turned = ra.q_heads + ra.k_heads;
    auto source = [&](uint32_t h) __attribute__((always_inline)) {
        const HeadRole role = head_role(ra, h);
        return reinterpret_cast<const T *>(role.from->data) + int64_t(t) * role.from->token_stride + int64_t(role.head) * role.from->head_stride;
    };
    // null: the token is not stored
    auto target = [&](uint32_t h) __attribute__((always_inline)) -> T * {
        if (h < ra.q_heads) return reinterpret_cast<T *>(ra.q_out.data) + int64_t(t) * ra.q_out.token_stride + int64_t(h) * ra.q_out.head_stride;
        if (at < 0) return nullptr;
        const bool key = h < turned;
        return reinterpret_cast<T *>(key ? ra.pages.keys : ra.pages.values) + at + int64_t(h - (key ? ra.q_heads : turned)) * ra.pages.head_stride;
    };
    // heads [first, end) of `items` items each
    auto walk = [&](uint32_t first, uint32_t end, uint32_t items, auto turns) __attribute__((always_inline)) {
        constexpr bool kTurns = decltype(turns)::value;
        const uint32_t abreast = items < 64u ? 64u / items : 1u, mine = items < 64u ? lane / items : 0u;
        for (uint32_t c = items < 64u ? lane - mine * items : lane; c < items; c += 64u) {
            if (mine >= abreast) break;
            const bool pair = kTurns && HALF && c < pairs;
            const uint32_t a = pair ? c * V : (c + (kTurns ? pairs : 0u)) * V, b = a + ra.dims / 2u;
            float2 cs[V];
            if constexpr (kTurns) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    cs[e] = float2{1.f, 0.f};
                    if constexpr (HALF) {
                        if (pair) cs[e] = angles[a + e];
                    } else if (e % 2 == 0) {
                        if (ra.table && a + e < ra.dims) cs[e] = angles[(a + e) / 2u];
                    }
                }
            }
            for (uint32_t h = first + mine; h < end; h += kAhead * abreast) {
                Piece p[kAhead], q[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const uint32_t hk = h + k * abreast;
                    if (hk >= end) break;
                    const T *x = source(hk);
                    p[k] = *reinterpret_cast<const Piece *>(x + a);
                    if (pair) q[k] = *reinterpret_cast<const Piece *>(x + b);
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const uint32_t hk = h + k * abreast;
                    if (hk >= end) break;
                    T *y = target(hk);
                    if (!y) continue;
                    if constexpr (kTurns && HALF) {
                        if (pair) {
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                const float2 y2 = turn(float(p[k].e[e]), float(q[k].e[e]), cs[e], ra.sign);
                                p[k].e[e] = T(y2.x);
                                q[k].e[e] = T(y2.y);
                            }
                            store_past(y + b, q[k]);
                        }
                    }
                    if constexpr (kTurns && !HALF && V > 1) {
#pragma unroll
                        for (int e = 0; e < V; e += 2) {
                            if (!ra.table || a + e >= ra.dims) break;
                            const float2 y2 = turn(float(p[k].e[e]), float(p[k].e[e + 1]), cs[e], ra.sign);
                            p[k].e[e] = T(y2.x);
                            p[k].e[e + 1] = T(y2.y);
                        }
                    }
                    store_past(y + a, p[k]);
                }
            }
        }
    };
    if (h0 < turned) walk(h0, h1 < turned ? h1 : turned, turned_items, std::true_type{});
    if (h1 > turned) walk(h0 > turned ? h0 : turned, h1, copied_items, std::false_type{});
}

// Any strides: a workgroup has tt (up to 64, a power of two) tokens of one head and 32 of its pairs (all elements count in pairs here, those that do not turn, too).
// Lanes lie along tokens where x is read, or y is written, with tokens side by side, along pairs else; between the two the elements go through LDS.  Pairs
// turn on their way out, so that lanes along pairs read angles side by side.  A small batch's starts are asked for first, then the elements: where tokens stand is
// found while those are on their way.
constexpr uint32_t kStridedThreads = 512u;
template <int DT>
__global__ __launch_bounds__(kStridedThreads) void rotary_strided_kernel(const RotaryArgs ra, const uint32_t tt_log)
{
    typedef typename Elem<DT>::T T;
    constexpr uint32_t kPairs = 32u, kMine = 64u * kPairs / kStridedThreads, kPitch = 2u * kPairs + 2u;
    __shared__ T image[64u * kPitch];
    __shared__ int64_t rows[64];                    // a token's row in the pages (head 0), -1: not stored
    __shared__ int32_t position_of[64], starts[256], held[256];
    __shared__ uint32_t sequence_of[64], sequences[256];
    __shared__ bool there[64];
    const uint32_t tt = 1u << tt_log, t0 = blockIdx.x << tt_log, pair0 = blockIdx.y * kPairs, tid = threadIdx.x;
    const HeadRole role = head_role(ra, blockIdx.z);
    const uint32_t all_pairs = ra.head_dim / 2u + (ra.head_dim & 1u), dims = ra.table && (role.query || role.key) ? ra.dims : 0u;
    const BatchArgs batch = ra.batch;
    // (a small batch: a thread has a batch row, thread batch.sequences the end of the last one)
    const bool near = batch.starts && batch.sequences < 256u;
    int32_t my_start = 0, my_held = 0;
    uint32_t my_sequence = kIdxMax;
    if (near && tid <= batch.sequences) {
        my_start = batch.starts[tid];
        if (tid < batch.sequences) {
            my_sequence = batch.rows ? uint32_t(batch.rows[tid]) : tid;
            if (my_sequence < ra.pages.sequences) my_held = tokens_held(ra.pages, my_sequence);
        }
    }
    // element of pair p's first or second half
    auto element = [&](uint32_t p, uint32_t second) __attribute__((always_inline)) {
        if (ra.interleaved || 2u * p >= dims) return 2u * p + second;
        return p + second * (dims / 2u);
    };
    auto token_and_pair = [&](uint32_t i, bool by_token, uint32_t *ti, uint32_t *pi) __attribute__((always_inline)) {
        *ti = by_token ? i & (tt - 1u) : i / kPairs;
        *pi = by_token ? i >> tt_log : i % kPairs;
        return i < tt * kPairs && t0 + *ti < ra.tokens && pair0 + *pi < all_pairs;
    };
    const bool in_by_token = role.from->dim_stride != 1, out_by_token = role.query && ra.q_out.dim_stride != 1;
    T u[kMine], w[kMine];
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
        uint32_t ti, pi;
        u[k] = w[k] = T(0.f);
        if (!token_and_pair(tid + kStridedThreads * k, in_by_token, &ti, &pi)) continue;
        const T *x = reinterpret_cast<const T *>(role.from->data) + int64_t(t0 + ti) * role.from->token_stride + int64_t(role.head) * role.from->head_stride;
        const uint32_t a = element(pair0 + pi, 0u), b = element(pair0 + pi, 1u);
        u[k] = x[int64_t(a) * role.from->dim_stride];
        if (b < ra.head_dim) w[k] = x[int64_t(b) * role.from->dim_stride];
    }
    if (near) {
        if (tid <= batch.sequences) {
            starts[tid] = my_start;
            held[tid] = my_held;
            sequences[tid] = my_sequence;
        }
        __syncthreads();
    }
    if (tid < tt) {
        const uint32_t t = t0 + tid;
        TokenPlace place{0u, 0, t < ra.tokens};
        if (batch.starts && t < ra.tokens) {
            uint32_t lo = 0, hi = batch.sequences;
            while (hi - lo > 1u) {
                const uint32_t mid = (lo + hi) / 2u;
                if ((near ? starts[mid] : batch.starts[mid]) <= int32_t(t)) lo = mid; else hi = mid;
            }
            if (near) {
                const int32_t first = starts[lo], end = starts[lo + 1u];
                place.there = first <= int32_t(t) && end > int32_t(t) && end <= int32_t(batch.tokens) && sequences[lo] < ra.pages.sequences;
                place.sequence = sequences[lo];
                place.position = held[lo] - end + int32_t(t);
            } else {
                place = place_in(batch, ra.pages, lo, t);
            }
        }
        there[tid] = place.there;
        sequence_of[tid] = place.sequence;
        position_of[tid] = ra.at && t < ra.tokens ? ra.at[t] : place.position;
    }
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
        uint32_t ti, pi;
        if (!token_and_pair(tid + kStridedThreads * k, in_by_token, &ti, &pi)) continue;
        image[ti * kPitch + 2u * pi] = u[k];
        image[ti * kPitch + 2u * pi + 1u] = w[k];
    }
    __syncthreads();
    // (its page's number and the angles, side by side)
    if (tid < tt) rows[tid] = batch.starts && !role.query && there[tid] ? row_offset(ra.pages, sequence_of[tid], position_of[tid], 0u) : -1;
    float2 cs[kMine];
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
        uint32_t ti, pi;
        cs[k] = float2{1.f, 0.f};
        if (token_and_pair(tid + kStridedThreads * k, out_by_token, &ti, &pi) && 2u * (pair0 + pi) < dims && there[ti]) cs[k] = angle_row(ra, position_of[ti])[pair0 + pi];
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < kMine; ++k) {
        uint32_t ti, pi;
        if (!token_and_pair(tid + kStridedThreads * k, out_by_token, &ti, &pi) || !there[ti]) continue;
        const uint32_t t = t0 + ti, p = pair0 + pi, a = element(p, 0u), b = element(p, 1u);
        T first = image[ti * kPitch + 2u * pi], second = image[ti * kPitch + 2u * pi + 1u];
        if (2u * p < dims) {
            const float2 y2 = turn(float(first), float(second), cs[k], ra.sign);
            first = T(y2.x);
            second = T(y2.y);
        }
        T *y;
        int64_t stride = 1;
        if (role.query) {
            stride = ra.q_out.dim_stride;
            y = reinterpret_cast<T *>(ra.q_out.data) + int64_t(t) * ra.q_out.token_stride + int64_t(role.head) * ra.q_out.head_stride;
        } else {
            if (rows[ti] < 0) continue;
            y = reinterpret_cast<T *>(role.key ? ra.pages.keys : ra.pages.values) + rows[ti] + int64_t(role.head) * ra.pages.head_stride;
        }
        __builtin_nontemporal_store(first, y + int64_t(a) * stride);
        if (b < ra.head_dim) __builtin_nontemporal_store(second, y + int64_t(b) * stride);
    }
}

template <int DT, int V, bool HALF>
void launch_pieces(const RotaryArgs &ra, hipStream_t s)
{
    const uint32_t pieces = ra.head_dim / V, turned = HALF && ra.table ? pieces - ra.dims / 2u / V : pieces, heads = ra.q_heads + 2u * ra.k_heads;
    // Few tokens: their heads are shared out to several waves, as long as each has a round of its lanes.  Many heads, too, as soon as each has 500 pieces,
    // about two rounds of kAhead: shorter waves leave less of the chip idle at the end, but each finds its token's place.  us in 1 / 2 / 3 shares: 1000 pieces
    // (12000 tokens of 50 heads of 80, fp32) 96 / 87 / 90, 1536 (8192 tokens of 48 heads of 128, fp32) 86 / 84 / 83.5, 768 (16384 tokens, bf16)
    // 82 / 84 / 84, 512 (16384 tokens of 32 heads) 54 / 56 / 60.
    const uint32_t groups = (ra.tokens + 3u) / 4u, round = turned < 64u ? 64u / turned : 1u;
    uint32_t shares = std::max(groups < 512u ? 512u / groups : 1u, uint32_t(std::min<uint64_t>(uint64_t(heads) * pieces / 500u, 4096u)));
    if (shares > (heads + round - 1u) / round) shares = (heads + round - 1u) / round;
    const uint32_t each = (heads + shares - 1u) / shares;
    rotary_kernel<DT, V, HALF><<<dim3(groups, (heads + each - 1u) / each), dim3(256), 0, s>>>(ra, each, turned, pieces);
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
        rotary_strided_kernel<DT><<<dim3((ra.tokens + (1u << tt_log) - 1u) >> tt_log, (all_pairs + 31u) / 32u, ra.q_heads + 2u * ra.k_heads), dim3(kStridedThreads), 0, s>>>(ra, tt_log);
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
