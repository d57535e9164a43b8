// What the kernels that accumulate attention weights share: which rows of queries count, which keys they see.
//
// W[j] <- decay W[j] + sum over the rows r that see key j of e^(scale q_r k_j - lse_r), lse_r the logarithm of the softmax's denominator of row r.  As in the
// attention's kernels a row is a token and one of the query heads that share a head of keys, and weights are 2^(score') with score' = (scale q k - lse) / ln 2:
// lse is the reference, so nothing is carried from key to key, and no workgroup needs another one's keys.
#pragma once
#include "attend_common.hpp"

namespace hspmm {

// A sequence of the batch: its counted rows are those of the last tokens of its chunk.
struct WeighRows {
    uint32_t sequence, first_token, rows;                        // the first counted token, of the batch
    int32_t length, old, position;                               // tokens held; those in front of the chunk; the first counted token's position
    int32_t keys;                                                // that there are places for
    bool there;
};

__device__ __forceinline__ WeighRows weigh_rows(const WeighArgs &wa, uint32_t b)
{
    WeighRows w{};
    const BatchArgs &ba = wa.batch;
    const int32_t first = ba.starts[b], end = ba.starts[b + 1u];
    w.sequence = batch_sequence(ba, b);
    if (first < 0 || end <= first || end > int32_t(ba.tokens) || w.sequence >= wa.pages.sequences) return w;
    const int32_t chunk = end - first, count = wa.last && uint32_t(chunk) > wa.last ? int32_t(wa.last) : chunk;
    w.length = tokens_held(wa.pages, w.sequence);
    w.old = w.length - chunk;
    w.position = w.length - count;
    w.first_token = uint32_t(end - count);
    w.rows = uint32_t(count) * wa.shared.d;
    w.keys = min(w.length, keys_of_row(wa.pages));
    w.there = true;
    return w;
}

// Row m of them: its token of the batch, head and the keys [lo, hi) that it sees; a row behind the last one sees none.
__device__ __forceinline__ RowOf weigh_row(const WeighArgs &wa, const WeighRows &w, uint32_t head, uint32_t m)
{
    const uint32_t at = m < w.rows ? m : 0u, i = wa.shared.quotient(at);
    RowOf r;
    r.token = w.first_token + i;
    r.head = head * wa.shared.d + at - i * wa.shared.d;
    const int32_t p = w.position + int32_t(i);
    r.hi = m >= w.rows ? 0 : wa.causal ? p + 1 : w.length;
    r.lo = wa.window && int64_t(p) + 1 > int64_t(wa.window) ? p + 1 - int32_t(wa.window) : 0;
    return r;
}

// -lse in units of ln 2: what a row's scores are moved by.  Of a row whose lse says that it sees nothing every key receives 0.
__device__ __forceinline__ float moved_by(float lse) { return lse == -INFINITY ? -INFINITY : lse * -kLog2e; }

// The rows [first, end) that may see a key of [key0, key0 + n).
struct RowRange { uint32_t first, end; };
__device__ __forceinline__ RowRange rows_that_see(const WeighArgs &wa, const WeighRows &w, int32_t key0, int32_t n)
{
    RowRange r{0u, w.rows};
    if (wa.causal && key0 > w.position) {
        const int64_t first = int64_t(key0 - w.position) * wa.shared.d;
        r.first = first < int64_t(w.rows) ? uint32_t(first) : w.rows;
    }
    if (wa.window) {
        // (the last position that sees key0 + n - 1 is window - 1 behind it)
        const int64_t tokens = int64_t(key0) + n - 1 + int64_t(wa.window) - w.position, end = tokens > 0 ? tokens * wa.shared.d : 0;
        if (end < int64_t(r.end)) r.end = uint32_t(end);
    }
    return r;
}

// The sum over 16 lanes side by side, in all of them.
__device__ __forceinline__ float sum_row(float v)
{
#define HSPMM_ROTATED(n) __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + n, 0xF, 0xF, false))
    v += HSPMM_ROTATED(8);
    v += HSPMM_ROTATED(4);
    v += HSPMM_ROTATED(2);
    v += HSPMM_ROTATED(1);
#undef HSPMM_ROTATED
    return v;
}

}  // namespace hspmm
