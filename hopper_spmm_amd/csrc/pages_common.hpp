// What the kernels that work on a cache's pages share: sums over a workgroup, the free pages, a list's entries.
#pragma once
#include "cache_device.h"

namespace hspmm {

namespace {

typedef uint32_t pg_u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kScanThreads = 1024u, kScanWaves = kScanThreads / 64u;

__device__ __forceinline__ uint64_t lanes_below() { return (uint64_t(1) << (threadIdx.x & 63u)) - 1u; }

// Sum of `value` over the threads in front of this one, of a workgroup of kScanThreads; *total: over all.  waves: 2 x kScanWaves
// words, `turn` 0 and 1 in turn (a thread may be a call ahead of another).
__device__ __forceinline__ uint32_t scan(uint32_t value, uint32_t *waves, uint32_t turn, uint32_t *total)
{
    uint32_t sum = value;
#pragma unroll
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t other = __shfl_up(sum, d);
        if ((threadIdx.x & 63u) >= d) sum += other;
    }
    uint32_t *w = waves + turn * kScanWaves;
    if ((threadIdx.x & 63u) == 63u) w[threadIdx.x / 64u] = sum;
    __syncthreads();
    uint32_t before = 0u, every = 0u;
    for (uint32_t i = 0; i < kScanWaves; ++i) {
        const uint32_t v = w[i];
        before += i < threadIdx.x / 64u ? v : 0u;
        every += v;
    }
    *total = every;
    return before + sum - value;
}

constexpr uint32_t kEach = 8u;                 // pages a thread looks at at a time

// Eight references from page p on, 1 behind the last one.
struct Eight { int32_t r[kEach]; };
__device__ __forceinline__ Eight load_references(const int32_t *references, uint32_t pages, uint32_t p)
{
    Eight v;
    if (p + kEach <= pages && (reinterpret_cast<uintptr_t>(references) & 15u) == 0u) {
        const int4 a = reinterpret_cast<const int4 *>(references + p)[0], b = reinterpret_cast<const int4 *>(references + p)[1];
        v.r[0] = a.x; v.r[1] = a.y; v.r[2] = a.z; v.r[3] = a.w; v.r[4] = b.x; v.r[5] = b.y; v.r[6] = b.z; v.r[7] = b.w;
    } else {
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) v.r[e] = p + e < pages ? references[p + e] : 1;
    }
    return v;
}

// The first `need` free pages, ascending, into list; how many there were.  A workgroup of kScanThreads, eight pages a thread at a time; ahead: a thread's first
// eight, asked for before it was known how many are needed.
__device__ uint32_t find_free(const int32_t *references, uint32_t pages, uint32_t need, int32_t *list, uint32_t *waves, uint32_t turn, const Eight &ahead)
{
    uint32_t found = 0u;
    for (uint32_t p0 = 0; p0 < pages && found < need; p0 += kScanThreads * kEach) {
        const uint32_t p = p0 + threadIdx.x * kEach;
        const Eight v = p0 ? load_references(references, pages, p) : ahead;
        uint32_t count = 0u;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) count += v.r[e] <= 0;
        uint32_t total, at = found + scan(count, waves, turn, &total);
        turn ^= 1u;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e)
            if (v.r[e] <= 0) {
                if (at < need) list[at] = int32_t(p + e);
                ++at;
            }
        found += total;
    }
    return found < need ? found : need;
}

__device__ __forceinline__ uint32_t row_of(const PoolArgs &pa, const int32_t *rows, uint32_t i)
{
    const uint32_t r = rows ? uint32_t(rows[i]) : i;
    return r < pa.sequences ? r : kIdxMax;
}

// Tokens of a sequence, more than its row has places for where it was extended past them.
__device__ __forceinline__ int32_t held(const PoolArgs &pa, uint32_t sequence) { return max(pa.lengths[sequence], 0); }
// Pages of so many tokens; places_for: of them, those that a row has places for.
__device__ __forceinline__ uint32_t pages_for(const PoolArgs &pa, int32_t tokens)
{
    return tokens ? pa.page_tokens.quotient(uint32_t(tokens) - 1u) + 1u : 0u;
}
__device__ __forceinline__ uint32_t places_for(const PoolArgs &pa, int32_t tokens) { return min(pages_for(pa, tokens), pa.table_pages); }
__device__ __forceinline__ int32_t extended(int32_t have, int32_t add) { return add > 0x7FFFFFFF - have ? 0x7FFFFFFF : have + max(add, 0); }

template <class F>
void by_unit(const PoolArgs &pa, F f)
{
    if (pa.unit == 16u) f(pg_u32x4{});
    else if (pa.unit == 4u) f(uint32_t{});
    else f(uint16_t{});
}

}  // namespace

}  // namespace hspmm
