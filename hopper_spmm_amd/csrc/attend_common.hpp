// What the attention kernels share: which rows of queries a workgroup has, which keys they see, sums of several workgroups.
//
// A row is a token and one of the query heads that share a head of keys: row m of a sequence's chunk is token m / shared, head
// m % shared of the group, so that a tile of rows reads its keys and values once for all heads that share them.
// Long spans of keys are cut into parts, a workgroup each.  A part leaves per row its reference, its total and its sums of values, all relative to the
// reference; the workgroup that leaves the last one adds them up in the parts' order, so the result does not depend on who that is.
// Scores are kept in units of ln 2 (scale' = scale / ln 2): weights are 2^(score - reference), one instruction each.
#pragma once
#include "cache_device.h"
#include "spmm_tile_common.hpp"

namespace hspmm {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// A reference is moved (and sums multiplied) only where a score is that far above the largest one when it was set: weights are up to 2^8 of what the largest
// had then, far inside every type.
constexpr float kReferenceSlack = 8.f;
// Weights are rounded to the elements' type, as matrix instructions of 16-bit types take no others; their total is of unrounded ones.  A reference is set that far
// below the largest score: fp16's weights are 2^7 there and up to 2^15, so that they keep eleven bits down to 2^-21 of the largest and 2^-32 of it is the most that
// a smaller one is off (from 1 on these would be 2^-14 and 2^-25, and 20000 keys of 2^-26 each had counted in the total and not in the sums).  bf16 has fp32's range.
template <class T> constexpr float kReferenceLead = sizeof(T) == 2 && !__is_same(T, __bf16) ? 7.f : 0.f;

struct RowTile {
    uint32_t sequence, first_row, rows, first_token, chunk;      // first_token of the batch; rows from first_row on
    int32_t length, position;                                    // tokens the cache holds; the position of the chunk's first token
    int32_t lo, hi;                                              // keys that any of the rows may see, as far as there are places for them
    bool there;
};

// Tile number `tile` of (1 << ROWS_LOG) rows.  Batch row b has the tiles from (starts[b] * shared >> ROWS_LOG) + b on: more than it needs at most by
// one, so that no list of tiles is made.  A wave looks at 64 batch rows at a time.
template <int ROWS_LOG>
__device__ __forceinline__ RowTile find_tile(const AttendArgs &aa, uint32_t tile)
{
    const BatchArgs &ba = aa.batch;
    const uint32_t lane = threadIdx.x & 63u;
    auto base = [&](uint32_t b) __attribute__((always_inline)) {
        return (uint32_t(clamp_i32(ba.starts[b], 0, int32_t(ba.tokens))) * aa.shared.d >> ROWS_LOG) + b;
    };
    uint32_t lo = 0, n = ba.sequences;
    while (n > 1u) {
        const uint32_t step = (n + 63u) / 64u, b = lane * step;
        const uint32_t below = uint32_t(__popcll(__ballot(b < n && base(lo + b) <= tile)));
        const uint32_t skip = (below ? below - 1u : 0u) * step;
        lo += skip;
        n = n - skip < step ? n - skip : step;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    RowTile t{};
    const int32_t first = ba.starts[lo], end = ba.starts[lo + 1u];
    t.sequence = ba.rows ? uint32_t(ba.rows[lo]) : lo;
    if (first < 0 || end <= first || end > int32_t(ba.tokens) || t.sequence >= aa.pages.sequences) return t;
    const uint32_t rows = uint32_t(end - first) * aa.shared.d;
    const uint32_t from = (tile - base(lo)) << ROWS_LOG;
    if (tile < base(lo) || from >= rows) return t;
    t.first_row = from;
    t.rows = rows - from < (1u << ROWS_LOG) ? rows - from : 1u << ROWS_LOG;
    t.first_token = uint32_t(first);
    t.chunk = uint32_t(end - first);
    t.length = tokens_held(aa.pages, t.sequence);
    t.position = t.length - (end - first);
    const int32_t p0 = t.position + int32_t(aa.shared.quotient(from)), p1 = t.position + int32_t(aa.shared.quotient(from + t.rows - 1u));
    t.hi = clamp_i32(aa.causal ? p1 + 1 : t.length, 0, keys_of_row(aa.pages));
    t.lo = aa.window && int64_t(p0) + 1 > int64_t(aa.window) ? min(p0 + 1 - int32_t(aa.window), t.hi) : 0;
    t.there = true;
    return t;
}

// The keys [begin, end) of part `part` of a tile's: parts begin a multiple of 32 keys apart.  Where aa.splits parts of aa.part_keys do not reach (long spans,
// or a sequence longer than the call said) all are longer, by the same: one token over 2^18 keys, 8 heads of 128, 1810 -> 192 us, 2^20 keys of one head 11500 -> 107.
struct KeyPart { int32_t begin, end, parts; };
__device__ __forceinline__ KeyPart key_part(const AttendArgs &aa, const RowTile &t, uint32_t part)
{
    const int32_t lo = t.lo & ~31;
    const uint32_t span = t.hi > lo ? uint32_t(t.hi - lo) : 0u;
    uint32_t each = aa.part_keys;
    if (uint64_t(each) * aa.splits < span) each = ((span + aa.splits - 1u) / aa.splits + 31u) & ~31u;
    const uint32_t parts = span ? (span + each - 1u) / each : 1u;
    const int32_t begin = lo + int32_t(part < parts ? part * each : 0u);
    return KeyPart{begin, part + 1u < parts ? begin + int32_t(each) : t.hi, int32_t(parts)};
}

// The tile and the head of a workgroup: heads side by side, as they are of one length, then tiles, then parts.  Workgroups go to the eight L2 domains and,
// there, to groups of compute units in turn, whatever they have to do, so what repeats in the numbers must not repeat in time: where chunks fill their
// tiles every (k + 1)th number is empty, so each eight tiles are turned by one against those in front (40 chunks of 32 tokens, 16 heads on 4: 69 -> 43 us);
// where a sequence is long all its parts are there, so the rows kernel's tiles move on by one from part to part (`moved`; the chunk kernel, whose parts
// are few, loses by it: 512 tokens over 8512 keys 40 -> 45 us).  48 sequences of up to 8000 keys, 16 rows each: 358 us by tiles, then heads, then
// parts, 178 so; 4 rows 173, 163.
struct Cell { uint32_t tile, head; };
__device__ __forceinline__ Cell cell_of(const AttendArgs &aa, uint32_t number, uint32_t moved)
{
    const uint32_t column = aa.heads.quotient(number), at = moved ? (column + moved) % aa.tiles : column;
    return Cell{(at | 7u) < aa.tiles ? (at & ~7u) | ((at + (at >> 3)) & 7u) : at, number - column * aa.heads.d};
}

// A row's token (of the batch), head and the keys [lo, hi) that it may see; a row behind the last one sees none.
struct RowOf { uint32_t token, head; int32_t lo, hi; };
__device__ __forceinline__ RowOf row_of_tile(const AttendArgs &aa, const RowTile &t, uint32_t head, uint32_t m)
{
    const uint32_t at = t.first_row + (m < t.rows ? m : 0u), i = aa.shared.quotient(at);
    RowOf r;
    r.token = t.first_token + i;
    r.head = head * aa.shared.d + at - i * aa.shared.d;
    const int32_t p = t.position + int32_t(i);
    r.hi = m >= t.rows ? 0 : aa.causal ? p + 1 : t.length;
    r.lo = aa.window && int64_t(p) + 1 > int64_t(aa.window) ? p + 1 - int32_t(aa.window) : 0;
    return r;
}

// Element offset of the row of a key (kv head `head`), -1: not stored.
__device__ __forceinline__ int64_t key_offset(const PagesArgs &pg, const int32_t *table_row, int64_t head_offset, int32_t key)
{
    const uint32_t place = pg.page_tokens.quotient(uint32_t(key));
    if (place >= pg.table_pages) return -1;
    const uint32_t id = uint32_t(table_row[place]);
    if (id >= pg.pages) return -1;
    return int64_t(id) * pg.page_stride + head_offset + int64_t(uint32_t(key) - place * pg.page_tokens.d) * pg.token_stride;
}

// yes or no by the condition, in one instruction.  (Elements of a matrix instruction's result are never written in a branch that some lanes take: where
// results lie in accumulation registers the compiler has been seen to write the neighbouring elements there, too.)
__device__ __forceinline__ float select(bool condition, float yes, float no)
{
    asm("" : "+v"(no));
    return condition ? yes : no;
}

// The larger of the values of two (four) lanes 32 (and 16) apart, in all of them.
__device__ __forceinline__ float max_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, uint32_t(r[0])), __builtin_bit_cast(float, uint32_t(r[1])));
}
__device__ __forceinline__ float max_quarters(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return max_halves(fmaxf(__builtin_bit_cast(float, uint32_t(r[0])), __builtin_bit_cast(float, uint32_t(r[1]))));
}

// Two floats rounded to a word of 16-bit elements (nearest, ties to even), in one instruction.
template <bool BF> __device__ __forceinline__ uint32_t pack_two(float lo, float hi)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef typename HalfOps<BF>::elem_t pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, pair));
}

// Whether a word holds a 16-bit element that is not finite.
template <bool BF> __device__ __forceinline__ bool word_not_finite(uint32_t w)
{
    constexpr uint32_t kE = BF ? 0x7F80u : 0x7C00u;
    return (~w & kE) == 0u || (~w & (kE << 16)) == 0u;
}

}  // namespace hspmm
