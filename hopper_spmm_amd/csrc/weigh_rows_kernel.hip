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
    // the same from LDS
    __device__ static __forceinline__ void load_rows(Query &Q, const char *row, uint32_t lane)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) Q.q[s] = *reinterpret_cast<const u32x4 *>(row + element(s, lane) * 2u);
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
    __device__ static __forceinline__ void load_rows(Query &Q, const char *row, uint32_t lane)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) Q.q[s] = *reinterpret_cast<const f32x4 *>(row + element(s, lane) * 4u);
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
constexpr uint32_t kWeighBatch = 128u;                         // rows in LDS at a time

// A wave has tiles of 32 keys in turn, each loaded once for up to sixteen rows, which it has in registers (Few), or for 128, which the workgroup has in LDS; of more rows there is another
// turn of all tiles.  Keys of the next tile are asked for when the last scores of this one are made, its page numbers and weights a tile ahead.
// Per key and row 2 D operations and one exponential, and a key's bytes once: memory bounds it where rows are few.  A token for each of 48 sequences of up to 16000 keys, 32 heads on 8 of 128, bf16:
// 175 to 180 us, the rate of a copy (4.8 TB/s); 3 sequences of up to 300, fp32: 7.2, of which 6.8 are the host's call.  Rows in LDS: the last 32 tokens of 17 prompts of up to 5700, 12 heads
// on 4 of 96, fp16, 18 us, where its keys alone would be 8: reads of 96 rows from LDS for each 32 keys, their exponentials, and 4 us until the first keys are there.
// Waves share nothing (no barrier but those around the rows): a key's weights are one wave's, read ahead and written once, so no atomics and one result.
template <class K, int DP, bool Few>
__global__ __launch_bounds__(64 * kWeighWaves) void weigh_rows_kernel(const WeighArgs wa)
{
    constexpr uint32_t kBatch = Few ? 16u : kWeighBatch, kPitch = DP * K::kElem + 16u, kRowPieces = DP / K::kPiece;
    constexpr int32_t kKeys = K::kKeys;
    __shared__ __attribute__((aligned(16))) char rows_of[Few ? 16 : kBatch * kPitch];
    __shared__ float by_of[kBatch];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, i = lane & 15u, D = wa.pages.head_dim;
    const uint32_t b = wa.heads.quotient(blockIdx.x), head = blockIdx.x - b * wa.heads.d;
    const WeighRows w = weigh_rows(wa, b);
    if (!w.there) return;
    const float scale = wa.scale * kLog2e;
    const int32_t *table = wa.pages.table + size_t(w.sequence) * wa.pages.table_pages;
    const int64_t head_offset = int64_t(head) * wa.pages.head_stride;
    float *const weights = wa.weights + int64_t(w.sequence) * wa.sequence_stride + int64_t(head) * wa.head_stride;
    const int32_t n_tiles = (w.keys + kKeys - 1) / kKeys, step = int32_t(gridDim.y) * kWeighWaves, first_tile = int32_t(blockIdx.y) * kWeighWaves + int32_t(wave);
    if (int32_t(blockIdx.y) * kWeighWaves >= n_tiles) return;
    // where a lane's key of a tile lies, below 0: it is not stored
    auto locate = [&](int32_t tile) __attribute__((always_inline)) {
        const int32_t key = tile * kKeys + int32_t(lane % kKeys);
        return tile < n_tiles && key < w.keys ? key_offset(wa.pages, table, head_offset, key) : int64_t(-1);
    };
    // lane i < 8 of a quarter has the weight of key 16 (i / 4) + 4 g + i % 4
    auto my_key = [&](int32_t tile) __attribute__((always_inline)) { return tile * kKeys + int32_t(16u * (i / 4u) + 4u * g + i % 4u); };
    auto load_weight = [&](int32_t tile) __attribute__((always_inline)) { return weights[tile < n_tiles && i < 8u && my_key(tile) < w.keys ? my_key(tile) : 0]; };
    for (uint32_t base = 0; base < w.rows; base += kBatch) {
        const uint32_t end = min(w.rows, base + kBatch);
        RowOf row{};
        typename K::Query Q;
        float by = 0.f;
        if constexpr (Few) {
            row = weigh_row(wa, w, head, base + i);
            K::load_query(Q, wa.q.data + (int64_t(row.token) * wa.q.token_stride + int64_t(row.head) * wa.q.head_stride) * K::kElem, base + i < end, lane, D);
            by = moved_by(wa.lse[size_t(row.token) * wa.q_heads + row.head]);
        } else {
            __syncthreads();
            // (of rows behind the last one the first is read, and not used; behind a row's last element there are zeros: those of the keys do not undo an infinity)
            for (uint32_t p = tid; p < ((end - base + 15u) & ~15u) * kRowPieces; p += 64u * kWeighWaves) {
                const uint32_t m = p / kRowPieces, c = p % kRowPieces * K::kPiece;
                const RowOf r = weigh_row(wa, w, head, base + m);
                const u32x4 x = *reinterpret_cast<const u32x4 *>(wa.q.data + (int64_t(r.token) * wa.q.token_stride + int64_t(r.head) * wa.q.head_stride + (c < D ? c : 0u)) * K::kElem);
                *reinterpret_cast<u32x4 *>(rows_of + m * kPitch + c * K::kElem) = x & (c < D ? ~0u : 0u);
            }
            if (tid < kBatch) {
                const RowOf r = weigh_row(wa, w, head, base + tid);
                by_of[tid] = wa.lse[size_t(r.token) * wa.q_heads + r.head] * -kLog2e;
            }
            __syncthreads();
        }
        K k;
        auto request = [&](int64_t at) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < K::kParts; ++t) {
                const int a = int(16u * t + i);
                const int64_t from = int64_t(uint64_t(uint32_t(__shfl(int(uint32_t(uint64_t(at))), a))) | uint64_t(uint32_t(__shfl(int(uint32_t(uint64_t(at) >> 32)), a))) << 32);
                k.load(t, wa.pages.keys, from < 0 ? 0 : from, lane, D);
            }
        };
        int64_t at = locate(first_tile), at_next = locate(first_tile + step);
        request(at);
        float weight = load_weight(first_tile);
#pragma unroll 1
        for (int32_t tile = first_tile; tile < n_tiles; tile += step) {
            const int32_t key0 = tile * kKeys;
            const uint32_t stored = uint32_t(__ballot(at >= 0));
            const RowRange range = rows_that_see(wa, w, key0, kKeys);
            const uint32_t m_first = max(range.first, base) & ~15u, m_end = min(range.end, end);
            at = at_next;
            at_next = locate(tile + 2 * step);
            const float weight_next = load_weight(tile + step);
            if (D < uint32_t(DP)) {
                asm volatile("");
                k.clear(lane, D);
            }
            f32x4 sums[K::kParts];
#pragma unroll
            for (int t = 0; t < K::kParts; ++t) sums[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            auto add = [&](const f32x4 (&s)[K::kParts], uint32_t m0) __attribute__((always_inline)) {
                // keys that all of the rows see
                const int32_t p0 = w.position + int32_t(wa.shared.quotient(m0)), p1 = w.position + int32_t(wa.shared.quotient(min(m0 + 15u, w.rows - 1u)));
                const bool all_see = stored == ~0u && m0 + 16u <= end && key0 + kKeys <= (wa.causal ? p0 + 1 : w.length) && (!wa.window || int64_t(p1) + 1 - int64_t(wa.window) <= key0);
                if (all_see) {
#pragma unroll
                    for (int t = 0; t < K::kParts; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) sums[t][r] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], scale, by));
                } else {
                    if constexpr (!Few) row = weigh_row(wa, w, head, m0 + i < end ? m0 + i : w.rows);
                    const int32_t low = row.lo - key0 - int32_t(4u * g), high = row.hi - key0 - int32_t(4u * g);
                    const uint32_t there = stored >> (4u * g);
#pragma unroll
                    for (int t = 0; t < K::kParts; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int a = 16 * t + r;
                            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], scale, by));
                            sums[t][r] += select(bool(int(a < low) | int(a >= high) | int(!(there >> a & 1u))), 0.f, p);
                        }
                }
            };
            if constexpr (Few) {
                f32x4 s[K::kParts];
                k.scores(Q, s);
                request(at);
                if (m_first < m_end) add(s, base);
            } else {
#pragma unroll 1
                for (uint32_t m0 = m_first; m0 < m_end; m0 += 16u) {
                    K::load_rows(Q, rows_of + (m0 - base + i) * kPitch, lane);
                    by = by_of[m0 - base + i];
                    by = by == INFINITY ? -INFINITY : by;      // (as moved_by, but here: where it is put, 18.5 -> 20.5 us for the last 32 tokens of 17 prompts)
                    f32x4 s[K::kParts];
                    k.scores(Q, s);
                    if (m0 + 16u >= m_end) request(at);
                    add(s, m0);
                }
                if (m_first >= m_end) request(at);
            }
            float mine = 0.f;
#pragma unroll
            for (int t = 0; t < K::kParts; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float s = sum_row(sums[t][r]);
                    mine = i == uint32_t(4 * t + r) ? s : mine;
                }
            const int32_t key = my_key(tile);
            if (i < 8u && key < w.keys) weights[key] = base ? weight + mine : key < w.old ? weight * wa.decay + mine : mine;
            weight = weight_next;
        }
    }
}

template <class K, int DP>
void launch(const WeighArgs &wa, bool few, hipStream_t s)
{
    const dim3 grid(wa.batch.sequences * wa.heads.d, wa.parts);
    if (few) weigh_rows_kernel<K, DP, true><<<grid, dim3(64 * kWeighWaves), 0, s>>>(wa);
    else weigh_rows_kernel<K, DP, false><<<grid, dim3(64 * kWeighWaves), 0, s>>>(wa);
}

template <bool BF>
void launch16(const WeighArgs &wa, bool few, hipStream_t s)
{
    const uint32_t D = wa.pages.head_dim;
    if (D <= 64u) launch<Keys16<BF, 64>, 64>(wa, few, s);
    else if (D <= 128u) launch<Keys16<BF, 128>, 128>(wa, few, s);
    else launch<Keys16<BF, 256>, 256>(wa, few, s);
}

}  // namespace

hipError_t launch_weigh_rows(int dtype, const WeighArgs &wa, bool few, hipStream_t s)
{
    const uint32_t D = wa.pages.head_dim;
    if (dtype == kDtypeF16) launch16<false>(wa, few, s);
    else if (dtype == kDtypeBf16) launch16<true>(wa, few, s);
    else if (D <= 64u) launch<Keys32<64>, 64>(wa, few, s);
    else if (D <= 128u) launch<Keys32<128>, 128>(wa, few, s);
    else launch<Keys32<256>, 256>(wa, few, s);
    return hipGetLastError();
}

}  // namespace hspmm
