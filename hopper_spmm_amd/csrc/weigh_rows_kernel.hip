// Accumulated attention weights of cached keys by a few rows of queries - single new tokens, the last ones of a prompt -, and by any rows in fp32.
#include "weigh_common.hpp"

namespace hspmm {

namespace {

// A tile's keys in a wave's registers, kKeys at a time; a lane (g, i) = (lane / 16, lane % 16).
//   scores: S^T = K Q^T by matrix instructions of 16 keys x 16 rows; register r of part t: key 16 t + 4 g + r, row i
// so that a row's lse and its range of keys are a lane's own, and a key's weights are summed over rows in its register, over lanes once at the end.
template <bool BF, int DP>
struct Keys16 {
    typedef typename HalfOps<BF>::elem_t T;
    static constexpr int kKeys = 32, kParts = 2, kElem = 2, kSteps = DP / 32, kPiece = 8;
    u32x4 k[kParts][kSteps];
    struct Query { u32x4 q[kSteps]; };
    __device__ static __forceinline__ uint32_t element(int s, uint32_t lane) { return 32u * s + 8u * (lane >> 4); }
    __device__ static __forceinline__ void load_query(Query &Q, const char *row, bool there, uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = element(s, lane);
            Q.q[s] = there && d < D ? *reinterpret_cast<const u32x4 *>(row + d * 2u) : u32x4{0u, 0u, 0u, 0u};
        }
    }
    __device__ __forceinline__ void load(int t, const char *keys, int64_t at, uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = element(s, lane);
            k[t][s] = *reinterpret_cast<const u32x4 *>(keys + (at + (d < D ? d : 0u)) * 2);
        }
    }
    // elements behind the last one
    __device__ __forceinline__ void clear(uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int t = 0; t < kParts; ++t)
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                if (element(s, lane) >= D) k[t][s] = u32x4{0u, 0u, 0u, 0u};
    }
    __device__ __forceinline__ void scores(const Query &Q, f32x4 (&s)[kParts]) const
    {
#pragma unroll
        for (int t = 0; t < kParts; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < kSteps; ++c) s[t] = HalfOps<BF>::mfma(k[t][c], Q.q[c], s[t]);
        }
    }
};

// fp32: products in fp32, four elements a matrix instruction; element 16 s + 4 g + e is step (s, e)'s.
template <int DP>
struct Keys32 {
    typedef float T;
    static constexpr int kKeys = 32, kParts = 2, kElem = 4, kSteps = DP / 16, kPiece = 4;
    f32x4 k[kParts][kSteps];
    struct Query { f32x4 q[kSteps]; };
    __device__ static __forceinline__ uint32_t element(int s, uint32_t lane) { return 16u * s + 4u * (lane >> 4); }
    __device__ static __forceinline__ void load_query(Query &Q, const char *row, bool there, uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = element(s, lane);
            Q.q[s] = there && d < D ? *reinterpret_cast<const f32x4 *>(row + d * 4u) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ void load(int t, const char *keys, int64_t at, uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = element(s, lane);
            k[t][s] = *reinterpret_cast<const f32x4 *>(keys + (at + (d < D ? d : 0u)) * 4);
        }
    }
    __device__ __forceinline__ void clear(uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int t = 0; t < kParts; ++t)
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                if (element(s, lane) >= D) k[t][s] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void scores(const Query &Q, f32x4 (&s)[kParts]) const
    {
#pragma unroll
        for (int t = 0; t < kParts; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < kSteps; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][c][e], Q.q[c][e], s[t], 0, 0, 0);
        }
    }
};

constexpr int kWeighWaves = 4;

// A wave has tiles of 32 keys in turn and all rows that count, sixteen at a time.
template <class K, int DP>
__global__ __launch_bounds__(64 * kWeighWaves) void weigh_rows_kernel(const WeighArgs wa)
{
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, i = lane & 15u, D = wa.pages.head_dim;
    const uint32_t b = wa.heads.quotient(blockIdx.x), head = blockIdx.x - b * wa.heads.d;
    const WeighRows w = weigh_rows(wa, b);
    if (!w.there) return;
    constexpr int32_t kKeys = K::kKeys;
    const float scale = wa.scale * kLog2e;
    const int32_t *table = wa.pages.table + size_t(w.sequence) * wa.pages.table_pages;
    const int64_t head_offset = int64_t(head) * wa.pages.head_stride;
    float *const weights = wa.weights + int64_t(w.sequence) * wa.sequence_stride + int64_t(head) * wa.head_stride;
    const int32_t n_tiles = (w.keys + kKeys - 1) / kKeys;
    for (int32_t tile = int32_t(blockIdx.y) * kWeighWaves + int32_t(wave); tile < n_tiles; tile += int32_t(gridDim.y) * kWeighWaves) {
        const int32_t key0 = tile * kKeys, mine = key0 + int32_t(lane % kKeys);
        const int64_t at = mine < w.keys ? key_offset(wa.pages, table, head_offset, mine) : -1;
        const uint32_t stored = uint32_t(__ballot(at >= 0));
        K k;
#pragma unroll
        for (int t = 0; t < K::kParts; ++t) {
            const int a = int(16u * t + i);
            const int64_t from = int64_t(uint64_t(uint32_t(__shfl(int(uint32_t(uint64_t(at))), a))) | uint64_t(uint32_t(__shfl(int(uint32_t(uint64_t(at) >> 32)), a))) << 32);
            k.load(t, wa.pages.keys, from < 0 ? 0 : from, lane, D);
        }
        if (D < uint32_t(DP)) k.clear(lane, D);
        const RowRange range = rows_that_see(wa, w, key0, kKeys);
        f32x4 sums[K::kParts];
#pragma unroll
        for (int t = 0; t < K::kParts; ++t) sums[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (uint32_t m0 = range.first & ~15u; m0 < range.end; m0 += 16u) {
            const RowOf row = weigh_row(wa, w, head, m0 + i);
            typename K::Query Q;
            K::load_query(Q, wa.q.data + (int64_t(row.token) * wa.q.token_stride + int64_t(row.head) * wa.q.head_stride) * K::kElem, m0 + i < w.rows, lane, D);
            const float lse = wa.lse[size_t(row.token) * wa.q_heads + row.head] * kLog2e;
            f32x4 s[K::kParts];
            k.scores(Q, s);
            const int32_t low = row.lo - key0 - int32_t(4u * g), high = row.hi - key0 - int32_t(4u * g);
            const uint32_t there = stored >> (4u * g);
#pragma unroll
            for (int t = 0; t < K::kParts; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int a = 16 * t + r;
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], scale, -lse));
                    sums[t][r] += select(bool(int(a < low) | int(a >= high) | int(!(there >> a & 1u))), 0.f, p);
                }
        }
        // lane i < 8 of a quarter writes key 16 (i / 4) + 4 g + i % 4
        float mine_sum = 0.f;
#pragma unroll
        for (int t = 0; t < K::kParts; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float s = sum_row(sums[t][r]);
                mine_sum = i == uint32_t(4 * t + r) ? s : mine_sum;
            }
        const int32_t key = key0 + int32_t(16u * (i / 4u) + 4u * g + i % 4u);
        if (i < 8u && key < w.keys) weights[key] = key < w.old ? weights[key] * wa.decay + mine_sum : mine_sum;
    }
}

template <class K, int DP>
void launch(const WeighArgs &wa, hipStream_t s)
{
    weigh_rows_kernel<K, DP><<<dim3(wa.batch.sequences * wa.heads.d, wa.parts), dim3(64 * kWeighWaves), 0, s>>>(wa);
}

template <bool BF>
void launch16(const WeighArgs &wa, hipStream_t s)
{
    const uint32_t D = wa.pages.head_dim;
    if (D <= 64u) launch<Keys16<BF, 64>, 64>(wa, s);
    else if (D <= 128u) launch<Keys16<BF, 128>, 128>(wa, s);
    else launch<Keys16<BF, 256>, 256>(wa, s);
}

}  // namespace

hipError_t launch_weigh_rows(int dtype, const WeighArgs &wa, hipStream_t s)
{
    const uint32_t D = wa.pages.head_dim;
    if (dtype == kDtypeF16) launch16<false>(wa, s);
    else if (dtype == kDtypeBf16) launch16<true>(wa, s);
    else if (D <= 64u) launch<Keys32<64>, 64>(wa, s);
    else if (D <= 128u) launch<Keys32<128>, 128>(wa, s);
    else launch<Keys32<256>, 256>(wa, s);
    return hipGetLastError();
}

}  // namespace hspmm
