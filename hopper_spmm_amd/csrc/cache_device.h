// Shared between the kernels of rotary positions, cache pages and attention and their entry points (hspmm_cache.hip).
#pragma once
#include "hspmm_device.h"
#include "divisor.hpp"

namespace hspmm {

// One layer of a cache (strides in elements).
struct PagesArgs {
    char *keys, *values;
    const int32_t *table, *lengths;
    uint32_t pages, sequences, table_pages, heads, head_dim;
    Divisor page_tokens;
    int64_t page_stride, head_stride, token_stride;
};

struct BatchArgs {
    const int32_t *starts, *rows;
    uint32_t sequences, tokens;
};

struct HeadsArgs {
    char *data;
    int64_t token_stride, head_stride, dim_stride;
};

// What a rotation's launch turns and copies: `q_heads` heads from q to q_out, turned; k_heads heads from k, turned, and from v into pages.
struct RotaryArgs {
    HeadsArgs q, q_out, k, v;
    uint32_t q_heads, k_heads;
    uint32_t head_dim, dims, interleaved, positions;
    float sign;                          // of the sines
    const float *table;                  // null: nothing turns
    const int32_t *at;                   // positions of tokens; null: where they stand in the cache
    uint32_t tokens;
    PagesArgs pages;
    BatchArgs batch;
};
// vec: elements that a lane moves at a time where a head's elements lie side by side everywhere, 0: through LDS, any strides
hipError_t launch_rotary(int dtype, const RotaryArgs &ra, uint32_t vec, hipStream_t s);

// Groups of a batch's rows that begin with the same tokens (hspmm_prefix).
struct PrefixArgs {
    const int32_t *firsts, *tokens;
    uint32_t groups;
    uint32_t splits, part_keys;          // of the prefixes
    float *sums;                         // per part - of the prefixes, then of what is behind -, token and head of queries: sums over the part (kPrefixExtra floats more than head_dim)
    int64_t part_stride;                 // from a part to the next
};
constexpr uint32_t kPrefixExtra = 4u;    // reference, total, parts
// Which keys a workgroup of an attention has: all; those of a group's prefix; those behind it; all, those of the prefix by its first sequence's pages.
enum AttendSpan { kSpanAll, kSpanPrefix, kSpanRest, kSpanBoth };

struct AttendArgs {
    PagesArgs pages;
    BatchArgs batch;
    HeadsArgs q, out;
    float *lse;
    uint32_t q_heads;
    Divisor shared, heads;               // heads of queries to one of keys; heads of keys
    uint32_t tiles;                      // attend_tiles
    float scale;
    uint32_t causal, window;
    uint32_t splits, part_keys;          // parts that a tile's keys are cut into at most; keys of a part (a multiple of 32)
    float *sums;                         // of more than one part: their sums
    uint32_t *arrive;                    // and how many have left them (zero between launches)
    PrefixArgs prefix;
};
// Tiles of (1 << rows_log) rows that a batch has at most (find_tile numbers them).
constexpr uint32_t kAttendRowsLog = 4u;
inline uint32_t attend_tiles(uint32_t tokens, uint32_t sequences, uint32_t shared, uint32_t rows_log)
{
    return uint32_t((uint64_t(tokens) * shared >> rows_log) + sequences);
}
constexpr uint32_t kAttendCounters = 16384u;
// floats of a part of a tile's sums
inline uint32_t attend_slot(uint32_t rows_log, uint32_t head_dim) { return (1u << rows_log) * ((head_dim <= 64u ? 64u : head_dim <= 128u ? 128u : 256u) + 4u); }
// past: 16-bit keys and values are not kept in the L2
hipError_t launch_attend_rows(int dtype, const AttendArgs &aa, bool past, bool both, hipStream_t s);
// 16-bit types; tiles of 1 << rows_log rows: 128, or 256 for heads of up to 128 elements
// both: with prefixes, by the pages of their first sequences
hipError_t launch_attend_chunk(int dtype, const AttendArgs &aa, bool both, uint32_t rows_log, hipStream_t s);
// Attention over shared prefixes: `prefix` has the prefixes' tiles, `rest` those of what is behind them, by the rows kernel or the chunk kernel (tiles of 128 rows) each.
hipError_t launch_attend_shared(int dtype, const AttendArgs &prefix, const AttendArgs &rest, bool prefix_chunk, bool rest_chunk, hipStream_t s);

// Attention weights that cached keys have received.
struct WeighArgs {
    PagesArgs pages;
    BatchArgs batch;
    HeadsArgs q;
    const float *lse;
    uint32_t q_heads;
    Divisor shared, heads;               // heads of queries to one of keys; heads of keys
    float scale, decay;
    uint32_t causal, window, last;       // last: tokens of a chunk that count, 0: all
    float *weights;                      // of the layer
    int64_t sequence_stride, head_stride;
    uint32_t parts;                      // rows kernel: workgroups that share out a sequence's keys; chunk kernel: parts of the rows, at most
    Divisor blocks;                      // chunk kernel: of kWeighKeys keys, of the longest sequence that the call speaks of
    uint32_t part_rows;                  // rows of a part
    float *sums;                         // of more than one part: their sums
    uint32_t *arrive;                    // and how many have left them (zero between launches)
};
// few: up to 16 rows at a time
hipError_t launch_weigh_rows(int dtype, const WeighArgs &wa, bool few, hipStream_t s);
constexpr uint32_t kWeighKeys = 128u;    // of a workgroup of the chunk kernel
// 16-bit types
hipError_t launch_weigh_chunk(int dtype, const WeighArgs &wa, hipStream_t s);

// Page work: all layers.
struct PoolArgs {
    char *keys, *values;
    int32_t *table, *lengths, *references, *scratch;
    uint32_t layers, pages, heads, sequences, table_pages;
    Divisor page_tokens;
    uint32_t token_bytes;                // of one head
    uint32_t heads_first;
    uint32_t unit;                       // bytes moved at a time: 16, 4 or 2
    int64_t page_bytes, layer_bytes;     // from one to the next
};
hipError_t launch_pages_extend(const PoolArgs &pa, uint32_t n, const int32_t *rows, const int32_t *add, int32_t *status, hipStream_t s);
hipError_t launch_pages_fork(const PoolArgs &pa, uint32_t n, const int32_t *parents, const int32_t *children, int32_t *status, hipStream_t s);
hipError_t launch_pages_free(const PoolArgs &pa, uint32_t n, const int32_t *rows, hipStream_t s);
hipError_t launch_pages_compact(const PoolArgs &pa, int32_t *table_out, int32_t *references_out, int32_t *live, hipStream_t s);
// What an eviction is asked for, and where it notes things between its launches.
struct EvictArgs {
    uint32_t n;
    const int32_t *parents, *children;
    uint32_t keep, first, last;
    float *weights;
    int64_t weights_layer, weights_sequence, weights_head;       // strides
    int32_t *kept, *status;
    uint32_t *arrive;                    // zero between calls
    int32_t *entries;                    // of every entry of the list: EvictEntry
    int32_t *rows;                       // its parent's row of the table
    int32_t *to;                         // the pages its tokens go to: a page, or below 0, -1 - k: the k-th of its new ones
    int32_t *free;                       // free pages
    float *kept_weights;                 // layers x entries x heads x keep
    uint32_t keep_pages;                 // of `keep` tokens
};
constexpr uint32_t kEvictEntry = 8u;     // words of an entry
// Workgroups that share out keys, and values, of a layer, an entry and a head: as many as give a small call some thousand, of 64 bytes of a token at least.
inline uint32_t evict_shares(const PoolArgs &pa, uint64_t cells)
{
    const uint64_t wanted = cells < 4096u ? 4096u / (cells ? cells : 1u) : 1u, most = pa.token_bytes / 64u;
    return uint32_t(wanted < most ? wanted : most ? most : 1u);
}
hipError_t launch_evict(const PoolArgs &pa, const EvictArgs &ea, hipStream_t s);
hipError_t launch_pages_copy(const PoolArgs &pa, uint32_t n, const int32_t *from, const int32_t *to, hipStream_t s);

#ifdef __HIPCC__
// Where a token of a batch stands: its sequence and position (below 0: in front of the cache); not there: outside every chunk.
struct TokenPlace { uint32_t sequence; int32_t position; bool there; };

__device__ __forceinline__ int32_t clamp_i32(int32_t v, int32_t lo, int32_t hi) { return v < lo ? lo : v > hi ? hi : v; }

// Tokens a sequence has.  Where that is more than its row of the table has places for, those behind are like tokens without a page: a length that was
// cut to the row's would put a batch's tokens over stored ones.
__device__ __forceinline__ int32_t tokens_held(const PagesArgs &pg, uint32_t sequence) { return max(pg.lengths[sequence], 0); }

// Keys that a row of the table has places for (numbers a few tiles behind the last one are 31 bits, too).
__device__ __forceinline__ int32_t keys_of_row(const PagesArgs &pg)
{
    const int64_t most = int64_t(pg.table_pages) * pg.page_tokens.d;
    return most > 0x7FFF0000 ? 0x7FFF0000 : int32_t(most);
}

// Token t as one of batch row b's, if it is.
__device__ __forceinline__ TokenPlace place_in(const BatchArgs &ba, const PagesArgs &pg, uint32_t b, uint32_t t)
{
    const int32_t first = ba.starts[b], end = ba.starts[b + 1u];
    const uint32_t sequence = ba.rows ? uint32_t(ba.rows[b]) : b;
    if (first > int32_t(t) || end <= int32_t(t) || end > int32_t(ba.tokens) || sequence >= pg.sequences) return TokenPlace{0u, -1, false};
    return TokenPlace{sequence, tokens_held(pg, sequence) - end + int32_t(t), true};
}

// Element offset of a position's row in the pages, -1: it is not stored.
__device__ __forceinline__ int64_t row_offset(const PagesArgs &pg, uint32_t sequence, int32_t position, uint32_t head)
{
    if (position < 0) return -1;
    const uint32_t place = pg.page_tokens.quotient(uint32_t(position));
    if (place >= pg.table_pages) return -1;
    const uint32_t id = uint32_t(pg.table[size_t(sequence) * pg.table_pages + place]);
    if (id >= pg.pages) return -1;
    return int64_t(id) * pg.page_stride + int64_t(head) * pg.head_stride + int64_t(uint32_t(position) - place * pg.page_tokens.d) * pg.token_stride;
}
#endif

}  // namespace hspmm
