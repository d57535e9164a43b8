// Entry points of rotary positions, the paged cache and the attention over it (include/hspmm.h): checks of arguments, the rules
// that choose kernels, launches.  They keep nothing: what a call uses is the caller's.
#include "hspmm_plan.hpp"
#include "cache_device.h"

using namespace hspmm_host;
using namespace hspmm;

namespace {

uint32_t element_bytes(int dtype) { return dtype == HSPMM_TF32 ? 4u : 2u; }

int check_dtype(int dtype)
{
    if (dtype != HSPMM_FP16 && dtype != HSPMM_BF16 && dtype != HSPMM_TF32)
        return fail(HSPMM_ERR_INVALID, "dtype %d: HSPMM_FP16, HSPMM_TF32 or HSPMM_BF16", dtype);
    return HSPMM_OK;
}

// The current device has to be a gfx950 (asked for once per device).
int check_device()
{
    static std::atomic<bool> known[64];
    int dev = -1;
    HSPMM_HIP(hipGetDevice(&dev));
    if (dev >= 0 && dev < 64 && known[dev].load(std::memory_order_relaxed)) return HSPMM_OK;
    hipDeviceProp_t prop;
    HSPMM_HIP(hipGetDeviceProperties(&prop, dev));
    if (strncmp(prop.gcnArchName, "gfx950", 6) != 0)
        return fail(HSPMM_ERR_UNSUPPORTED, "device %d is %s; this library is built for gfx950 only", dev, prop.gcnArchName);
    if (dev >= 0 && dev < 64) known[dev].store(true, std::memory_order_relaxed);
    return HSPMM_OK;
}

int check_heads(const char *name, const hspmm_heads *x, int dtype)
{
    if (!x || !x->data) return fail(HSPMM_ERR_INVALID, "null %s", name);
    if (reinterpret_cast<uintptr_t>(x->data) % element_bytes(dtype)) return fail(HSPMM_ERR_INVALID, "%s is not aligned to the element size", name);
    if (x->token_stride < 0 || x->head_stride < 0 || x->dim_stride < 1) return fail(HSPMM_ERR_INVALID, "%s: strides below 0, or of elements below 1", name);
    return HSPMM_OK;
}

int check_rotary(const hspmm_rotary *r, uint32_t head_dim)
{
    if (r->dims % 2u || r->dims > head_dim) return fail(HSPMM_ERR_INVALID, "%u of %u elements turn: an even number, at most all", r->dims, head_dim);
    if (r->dims && (!r->table || reinterpret_cast<uintptr_t>(r->table) % 8u)) return fail(HSPMM_ERR_INVALID, "the table of rotary positions is null or not aligned to 8 bytes");
    if (r->dims && (r->positions == 0 || r->positions > 0x7FFFFFFFu)) return fail(HSPMM_ERR_INVALID, "a table of %u positions", r->positions);
    return HSPMM_OK;
}

int check_cache(const hspmm_cache *c)
{
    if (!c) return fail(HSPMM_ERR_INVALID, "null cache");
    if (const int rc = check_dtype(c->dtype)) return rc;
    if (c->order != HSPMM_HEADS_FIRST && c->order != HSPMM_TOKENS_FIRST) return fail(HSPMM_ERR_INVALID, "order %d of a page", c->order);
    if (!c->layers || !c->pages || !c->page_tokens || !c->heads || !c->head_dim || !c->sequences || !c->table_pages)
        return fail(HSPMM_ERR_INVALID, "a cache of %u layers, %u pages of %u tokens, %u heads of %u elements, %u sequences of %u pages", c->layers, c->pages,
                    c->page_tokens, c->heads, c->head_dim, c->sequences, c->table_pages);
    // (numbers that kernels multiply in 32 bits; a page is far below)
    const uint64_t page = uint64_t(c->heads) * c->page_tokens;
    if (c->pages > 0x3FFFFFFFu || c->page_tokens > 0x7FFFFFFFu || c->heads > 32768u || c->head_dim > 32768u || page > (1u << 30) || page * c->head_dim > (1u << 29) ||
        uint64_t(c->sequences) * c->table_pages > 0x7FFFFFFFu || c->layers > 16384u)
        return fail(HSPMM_ERR_UNSUPPORTED, "a cache of %u layers, %u pages of %u tokens, %u heads of %u elements, %u sequences of %u pages", c->layers, c->pages,
                    c->page_tokens, c->heads, c->head_dim, c->sequences, c->table_pages);
    const int64_t elements = int64_t(page * c->head_dim);
    if (c->page_stride < 0 || (c->page_stride && c->page_stride < elements)) return fail(HSPMM_ERR_INVALID, "pages of %lld elements, %lld apart", (long long)elements, (long long)c->page_stride);
    if (c->layer_stride < 0) return fail(HSPMM_ERR_INVALID, "layers %lld elements apart", (long long)c->layer_stride);
    if (!c->keys || !c->values || !c->table || !c->lengths || !c->references || !c->scratch) return fail(HSPMM_ERR_INVALID, "a null array of the cache");
    if (reinterpret_cast<uintptr_t>(c->keys) % 16u || reinterpret_cast<uintptr_t>(c->values) % 16u) return fail(HSPMM_ERR_INVALID, "keys and values must be aligned to 16 bytes");
    return HSPMM_OK;
}

int64_t page_stride(const hspmm_cache *c) { return c->page_stride ? c->page_stride : int64_t(c->heads) * c->page_tokens * c->head_dim; }
int64_t layer_stride(const hspmm_cache *c) { return c->layer_stride ? c->layer_stride : page_stride(c) * c->pages; }

PagesArgs pages_of(const hspmm_cache *c, uint32_t layer)
{
    PagesArgs pg{};
    const int64_t at = layer_stride(c) * layer * element_bytes(c->dtype);
    pg.keys = static_cast<char *>(c->keys) + at;
    pg.values = static_cast<char *>(c->values) + at;
    pg.table = c->table; pg.lengths = c->lengths;
    pg.pages = c->pages; pg.sequences = c->sequences; pg.table_pages = c->table_pages; pg.heads = c->heads; pg.head_dim = c->head_dim;
    pg.page_tokens = Divisor::of(c->page_tokens);
    pg.page_stride = page_stride(c);
    pg.head_stride = c->order == HSPMM_HEADS_FIRST ? int64_t(c->page_tokens) * c->head_dim : c->head_dim;
    pg.token_stride = c->order == HSPMM_HEADS_FIRST ? c->head_dim : int64_t(c->heads) * c->head_dim;
    return pg;
}

PoolArgs pool_of(const hspmm_cache *c)
{
    PoolArgs pa{};
    const uint32_t e = element_bytes(c->dtype);
    pa.keys = static_cast<char *>(c->keys); pa.values = static_cast<char *>(c->values);
    pa.table = c->table; pa.lengths = c->lengths; pa.references = c->references; pa.scratch = c->scratch;
    pa.layers = c->layers; pa.pages = c->pages; pa.heads = c->heads; pa.sequences = c->sequences; pa.table_pages = c->table_pages;
    pa.page_tokens = Divisor::of(c->page_tokens);
    pa.token_bytes = c->head_dim * e;
    pa.heads_first = c->order == HSPMM_HEADS_FIRST;
    pa.page_bytes = page_stride(c) * e;
    pa.layer_bytes = layer_stride(c) * e;
    const uint64_t all = uint64_t(pa.token_bytes) | uint64_t(pa.page_bytes) | uint64_t(pa.layer_bytes);
    pa.unit = all % 16u == 0u ? 16u : all % 4u == 0u ? 4u : 2u;
    return pa;
}

int check_batch(const hspmm_cache *c, const hspmm_batch *b)
{
    if (!b) return fail(HSPMM_ERR_INVALID, "null batch");
    if (b->tokens && (!b->sequences || !b->starts)) return fail(HSPMM_ERR_INVALID, "a batch of %u tokens without sequences or their starts", b->tokens);
    if (b->tokens > 0x7FFFFFFEu || b->sequences > 0x7FFFFFFEu) return fail(HSPMM_ERR_UNSUPPORTED, "a batch of %u tokens, %u sequences", b->tokens, b->sequences);
    if (!b->rows && b->sequences > c->sequences) return fail(HSPMM_ERR_INVALID, "a batch of %u sequences for a cache of %u", b->sequences, c->sequences);
    return HSPMM_OK;
}

// `threads` of an entry, in a launch that has fewer than 2^32
int check_launch(uint32_t n, uint32_t threads)
{
    if ((uint64_t(n) + 1u) * threads < (uint64_t(1) << 32)) return HSPMM_OK;
    return fail(HSPMM_ERR_UNSUPPORTED, "a list of %u: in several calls", n);
}

int check_list(const hspmm_cache *c, uint32_t n, const void *list, const char *name)
{
    if (n > c->sequences) return fail(HSPMM_ERR_INVALID, "a list of %u for a cache of %u sequences", n, c->sequences);
    if (n && !list) return fail(HSPMM_ERR_INVALID, "null %s", name);
    return HSPMM_OK;
}

BatchArgs batch_of(const hspmm_batch *b) { return BatchArgs{b->starts, b->rows, b->sequences, b->tokens}; }
HeadsArgs heads_of(const hspmm_heads *x)
{
    return x ? HeadsArgs{static_cast<char *>(x->data), x->token_stride, x->head_stride, x->dim_stride} : HeadsArgs{nullptr, 0, 0, 1};
}

// Elements that the piece kernel moves at a time, 0: it cannot (elements apart, or pairs between two pieces).
uint32_t rotary_piece(int dtype, const RotaryArgs &ra, const hspmm_cache *c)
{
    const uint32_t e = element_bytes(dtype);
    uint64_t all = ra.head_dim | (16u / e);
    if (ra.table) all |= ra.interleaved ? ra.dims : ra.dims / 2u;
    const HeadsArgs *tensors[4] = {ra.q_heads ? &ra.q : nullptr, ra.q_heads ? &ra.q_out : nullptr, ra.k_heads ? &ra.k : nullptr, ra.k_heads ? &ra.v : nullptr};
    for (const HeadsArgs *x : tensors) {
        if (!x) continue;
        if (x->dim_stride != 1) return 0u;
        all |= uint64_t(x->token_stride) | uint64_t(x->head_stride) | (reinterpret_cast<uintptr_t>(x->data) / e);
    }
    if (c) all |= uint64_t(page_stride(c)) | uint64_t(layer_stride(c));
    const uint32_t vec = uint32_t(all & ~(all - 1u));
    if (vec == 1u && ra.table && ra.interleaved) return 0u;
    return vec;
}

// (a launch has fewer than 2^32 threads along x, and 65535 workgroups along z)
int run_rotary(int dtype, const RotaryArgs &ra, const hspmm_cache *c, void *stream)
{
    const uint32_t vec = rotary_piece(dtype, ra, c), heads = ra.q_heads + 2u * ra.k_heads;
    if (!vec) {
        const uint64_t groups = (uint64_t(ra.tokens) + 63u) / 64u * ((ra.head_dim + 63u) / 64u) * heads;
        if (groups >= (1u << 24) || ra.tokens >= (1u << 29) || heads > 65535u)
            return fail(HSPMM_ERR_UNSUPPORTED, "%u tokens of %u heads at these strides: in several calls", ra.tokens, heads);
    } else if (ra.tokens > 4u * ((1u << 24) - 1u)) {
        return fail(HSPMM_ERR_UNSUPPORTED, "%u tokens: in several calls", ra.tokens);
    }
    if (int rc = check_device()) return rc;
    HSPMM_HIP(launch_rotary(dtype, ra, vec, static_cast<hipStream_t>(stream)));
    return HSPMM_OK;
}

}  // namespace

extern "C" {

int hspmm_rotary_table(int kind, uint32_t dims, double base, double factor, double original_length, double fast_turns, double slow_turns,
                       uint32_t positions, float *table)
{
    if (kind < HSPMM_ROTARY_PLAIN || kind > HSPMM_ROTARY_YARN) return fail(HSPMM_ERR_INVALID, "rotary positions of kind %d", kind);
    if (dims == 0 || dims % 2u || dims > 65536u) return fail(HSPMM_ERR_INVALID, "%u elements turn: an even number above 0", dims);
    if (!(base > 1.0) || !std::isfinite(base)) return fail(HSPMM_ERR_INVALID, "base %g", base);
    if (kind != HSPMM_ROTARY_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return fail(HSPMM_ERR_INVALID, "factor %g", factor);
    if (kind == HSPMM_ROTARY_BASE && dims == 2u) return fail(HSPMM_ERR_INVALID, "a scaled base wants more than one pair");
    if (kind == HSPMM_ROTARY_YARN && (!(original_length > 0.0) || !(slow_turns > 0.0) || !(fast_turns > slow_turns) || !std::isfinite(original_length) || !std::isfinite(fast_turns)))
        return fail(HSPMM_ERR_INVALID, "original length %g, turns %g and %g", original_length, fast_turns, slow_turns);
    if (positions && !table) return fail(HSPMM_ERR_INVALID, "null table");
    const uint32_t pairs = dims / 2u;
    try {
        constexpr double kTurn = 6.283185307179586476925286766559;
        const double b = kind == HSPMM_ROTARY_BASE ? base * std::pow(factor, double(dims) / double(dims - 2u)) : base;
        const double scale = kind == HSPMM_ROTARY_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
        // the pair whose wavelength turns that often within the original length
        auto pair_of = [&](double turns) { return double(dims) * std::log(original_length / (turns * kTurn)) / (2.0 * std::log(base)); };
        double low = 0.0, high = 0.0;
        if (kind == HSPMM_ROTARY_YARN) {
            // (whole pairs, dims - 1 and 0.001 are the steps of the authors' published program, to which trained models hold; the paper has none of them)
            low = std::max(std::floor(pair_of(fast_turns)), 0.0);
            high = std::min(std::ceil(pair_of(slow_turns)), double(dims - 1u));
            if (high <= low) high = low + 0.001;
        }
        std::vector<double> f(pairs);
        for (uint32_t i = 0; i < pairs; ++i) {
            f[i] = std::pow(b, -2.0 * i / dims);
            if (kind == HSPMM_ROTARY_LINEAR) f[i] /= factor;
            if (kind == HSPMM_ROTARY_YARN) {
                const double ramp = std::min(std::max((i - low) / (high - low), 0.0), 1.0);
                f[i] = f[i] / factor * ramp + f[i] * (1.0 - ramp);
            }
        }
        parallel_blocks(positions, 256, [&](size_t pb, size_t pe) {
            for (size_t p = pb; p < pe; ++p)
                for (uint32_t i = 0; i < pairs; ++i) {
                    const double angle = double(p) * f[i];
                    table[(p * pairs + i) * 2u] = float(std::cos(angle) * scale);
                    table[(p * pairs + i) * 2u + 1u] = float(std::sin(angle) * scale);
                }
        });
    } catch (const std::bad_alloc &) { return fail(HSPMM_ERR_ALLOC, "out of host memory"); }
    return HSPMM_OK;
}

int hspmm_rotate(const hspmm_rotary *rotary, int dtype, uint32_t tokens, uint32_t heads, uint32_t head_dim, const hspmm_heads *x,
                 const int32_t *positions, const hspmm_heads *y, int backward, void *stream)
{
    if (!rotary) return fail(HSPMM_ERR_INVALID, "null rotary positions");
    if (int rc = check_dtype(dtype)) return rc;
    if (!head_dim || head_dim > 32768u || heads > 32768u || tokens > 0x7FFFFFFEu) return fail(HSPMM_ERR_INVALID, "%u tokens, %u heads of %u elements", tokens, heads, head_dim);
    if (int rc = check_rotary(rotary, head_dim)) return rc;
    if (tokens == 0 || heads == 0) return HSPMM_OK;
    if (int rc = check_heads("x", x, dtype)) return rc;
    if (int rc = check_heads("y", y, dtype)) return rc;
    if (!positions && rotary->dims) return fail(HSPMM_ERR_INVALID, "null positions");
    RotaryArgs ra{};
    ra.q = heads_of(x); ra.q_out = heads_of(y);
    ra.q_heads = heads; ra.head_dim = head_dim; ra.dims = rotary->dims; ra.interleaved = rotary->interleaved != 0; ra.positions = rotary->positions;
    ra.sign = backward ? -1.f : 1.f;
    ra.table = rotary->dims ? rotary->table : nullptr;
    ra.at = positions;
    ra.tokens = tokens;
    return run_rotary(dtype, ra, nullptr, stream);
}

uint64_t hspmm_cache_scratch_words(uint32_t pages, uint32_t sequences, uint32_t table_pages)
{
    const uint64_t lists = uint64_t(sequences) * (4u + uint64_t(table_pages));
    return std::max<uint64_t>(lists, 3u * uint64_t(pages) + sequences) + 16u;
}

int hspmm_cache_append(const hspmm_cache *cache, uint32_t layer, const hspmm_batch *batch, const hspmm_heads *k, const hspmm_heads *v,
                       const hspmm_rotary *rotary, uint32_t q_heads, const hspmm_heads *q, const hspmm_heads *q_out, void *stream)
{
    if (int rc = check_cache(cache)) return rc;
    if (layer >= cache->layers) return fail(HSPMM_ERR_INVALID, "layer %u of %u", layer, cache->layers);
    if (int rc = check_batch(cache, batch)) return rc;
    if (rotary)
        if (int rc = check_rotary(rotary, cache->head_dim)) return rc;
    if (q && q_heads > 32768u) return fail(HSPMM_ERR_INVALID, "%u heads of queries", q_heads);
    if (batch->tokens == 0) return HSPMM_OK;
    if (int rc = check_heads("k", k, cache->dtype)) return rc;
    if (int rc = check_heads("v", v, cache->dtype)) return rc;
    if (q && q_heads) {
        if (int rc = check_heads("q", q, cache->dtype)) return rc;
        if (int rc = check_heads("q_out", q_out, cache->dtype)) return rc;
    }
    RotaryArgs ra{};
    ra.k = heads_of(k); ra.v = heads_of(v); ra.q = heads_of(q); ra.q_out = heads_of(q ? q_out : nullptr);
    ra.q_heads = q ? q_heads : 0u; ra.k_heads = cache->heads;
    ra.head_dim = cache->head_dim;
    if (rotary && rotary->dims) {
        ra.dims = rotary->dims; ra.interleaved = rotary->interleaved != 0; ra.positions = rotary->positions;
        ra.table = rotary->table;
    }
    ra.sign = 1.f;
    ra.tokens = batch->tokens;
    ra.pages = pages_of(cache, layer);
    ra.batch = batch_of(batch);
    return run_rotary(cache->dtype, ra, cache, stream);
}

static int check_attention(const hspmm_cache *c, const hspmm_batch *b, const hspmm_attention *a)
{
    if (int rc = check_cache(c)) return rc;
    if (int rc = check_batch(c, b)) return rc;
    if (!a) return fail(HSPMM_ERR_INVALID, "null attention");
    if (!a->q_heads || a->q_heads % c->heads || a->q_heads > 32768u) return fail(HSPMM_ERR_INVALID, "%u heads of queries for %u of keys", a->q_heads, c->heads);
    if (!std::isfinite(a->scale)) return fail(HSPMM_ERR_INVALID, "scale %g", double(a->scale));
    if (uint64_t(b->tokens) * (a->q_heads / c->heads) + b->sequences > 0x7FFFFFFFu)
        return fail(HSPMM_ERR_UNSUPPORTED, "%u tokens with %u heads that share their keys: in several calls", b->tokens, a->q_heads / c->heads);
    if (a->window && !a->causal) return fail(HSPMM_ERR_INVALID, "a window of %u keys without causal", a->window);
    const uint32_t piece = 16u / element_bytes(c->dtype);
    if (c->head_dim % piece || c->head_dim > 256u) return fail(HSPMM_ERR_UNSUPPORTED, "heads of %u elements: a multiple of %u up to 256", c->head_dim, piece);
    if (c->page_stride % piece || c->layer_stride % piece) return fail(HSPMM_ERR_UNSUPPORTED, "pages or layers that begin between two pieces of 16 bytes");
    return HSPMM_OK;
}

// How an attention is launched, by sizes alone: the same for the call and for its workspace.
struct AttendShape {
    uint32_t rows_log;                   // of a tile: kAttendRowsLog the rows kernel, 7 and 8 the chunk kernel
    uint32_t tiles, splits, part_keys;
    bool past;                           // the rows kernel reads past the L2
    uint64_t bytes;
};

static AttendShape attend_shape(const hspmm_cache *c, const hspmm_batch *b, const hspmm_attention *a)
{
    const uint32_t shared = a->q_heads / c->heads;
    const uint64_t rows = uint64_t(std::min(a->longest_chunk, b->tokens)) * shared;
    AttendShape sh{};
    // keys that a sequence's tokens see at most, and those of a tile of so many rows
    uint64_t keys = uint64_t(c->table_pages) * c->page_tokens;
    if (a->longest && a->longest < keys) keys = a->longest;
    auto seen = [&](uint32_t tile_rows) { return a->window && uint64_t(a->window) + tile_rows < keys ? uint64_t(a->window) + tile_rows : keys; };
    // The rows kernel for up to 16 rows, and where there is little to do: a tile of it is sixteen rows, and its waves share out the keys.  us of it / of the
    // chunk kernel by tiles of 16 rows x heads x keys, bf16, heads of 128: 8 K (60 tokens from the beginning, 32 heads) 6.6 / 9.7; 96 K (8 tokens for each of
    // 3 sequences of up to 2000, 32 heads on 8) 15.3 / 22.7; 180 K (300 tokens from the beginning) 15.0 / 16.7; 256 K (32 sequences of up to 500) 19.7 / 28.3;
    // 384 K (3 of 8000) 30.6 / 38.6; 384 K (3 tokens for each of 64 of 1500, 16 heads on 2) 34.0 / 32.6; 480 K (5 tokens over 30000) 55.9 / 70.8; 512 K (16 over
    // 16000) 48.3 / 44.4; 640 K (64 over 20000, 8 heads on 4) 67.5 / 54.4; 1024 K (32 of 2000) 82 / 70; 1600 K (16 ragged chunks) 65 / 33.  Up to 400 K it lost
    // at 4 of 24 such shapes, by 10 % at most (400 tokens from the beginning 19.9 / 18.1), above 500 K at 11 of 18, by up to a half; of 256 elements it won at
    // 304 K (59.5 / 74) and lost at 480 K (80 / 77).
    const uint64_t rows_work = uint64_t(b->sequences) * ((rows + 15u) / 16u) * c->heads * seen(16u);
    // 256 rows for heads of 97 to 128 elements only - with 128 rows two workgroups share a compute unit, but there only two images fit for each -, where chunks
    // are of one length, tiles for a quarter of the compute units and keys for parts on all of them: few, short and half-filled tiles are the longer ones' loss.  us
    // with 128 / 256 rows, by heads x tiles of 256 (`wide`), 32 heads on 8: 4096 tokens over 16384 keys (520) 1025 / 942; 8192 over 8192 (1032) 597 / 571; 2048 over
    // 8192 (264) 281 / 266; 1024 over 4096 (136) 96 / 82; 512 over 8512 (72) 105 / 99; 16 x 512 over 2000 (1088) 232 / 237; 2048 over 2048 (264) 67 / 71; 500 over
    // 500, 32 heads of keys (64) 22 / 27; few tiles: 256 over 8192 (40) 58 / 60, 700 over 20000, 8 heads on 4 (24) 85 / 103; ragged: 17 chunks of up to 700 over up
    // to 5700 (592) 216 / 279, 16 of up to 300 over 600 (664) 44 / 50, 8 of up to 300 over 2000 (328) 73 / 68.  Heads of 64, 2048 tokens over 8048, 177 / 184.
    const uint64_t wide = uint64_t(c->heads) * ((uint64_t(b->tokens) * shared >> 8) + (b->sequences + 1u) / 2u);
    const bool even = uint64_t(b->tokens) * 8u >= uint64_t(b->sequences) * std::min(a->longest_chunk, b->tokens) * 7u;
    if (c->dtype == HSPMM_TF32 || rows <= 16u || rows_work <= 400000u) sh.rows_log = kAttendRowsLog;
    else sh.rows_log = c->head_dim > 96u && c->head_dim <= 128u && rows > 128u && even && wide >= 64u && wide * seen(256u) >= 200000u ? 8u : 7u;
    keys = seen(1u << sh.rows_log);
    const uint64_t numbered = attend_tiles(b->tokens, b->sequences, shared, sh.rows_log);
    // tiles that have rows, at most: numbers are left out
    const uint64_t tiles = std::min<uint64_t>(numbered, uint64_t(b->sequences) * ((rows + (1u << sh.rows_log) - 1u) >> sh.rows_log));
    // Keys of a part.  Rows kernel: as few as give every compute unit two workgroups, 128 at least (every wave a tile or two) and 512 at most, more only
    // where that is over 4096 workgroups: sequences are of many lengths, and the last ones should not be long.  us by parts of 128 / 256 / 512 keys: one token
    // over 1000 keys, 8 heads 8.1 / 9.2 / 11.9; over 30000 58 / 39 / 30; 8 sequences of up to 8000 56 / 44 / 42.
    // Chunk kernel: as many as run at a time (two a compute unit with 128 rows and heads of up to 128 elements); a part's sums are as much as 130 keys.
    // Of two, twice as many where there are tiles for half of them anyway, which are of different lengths.  us by 512 / 1024 workgroups: 100 tokens for
    // each of 4 sequences of 4000 52 / 64; 512 tokens over 8512 keys, head_dim 64 38 / 48; 17 chunks of up to 700 tokens over up to 5700, 12 heads on 4, 204 / 175.  (One a compute unit, head_dim
    // 256, 1024 tokens over 2048 older keys, by 256 / 512 264 / 338.)
    const uint64_t work = tiles * c->heads * keys;
    const bool two = sh.rows_log == 7u && c->head_dim <= 128u;
    auto whole = [](uint64_t k) { return (k + 127u) & ~uint64_t(127u); };
    const uint64_t part = sh.rows_log == kAttendRowsLog ? std::max(whole(work / 4096u), std::min<uint64_t>(whole(work / 512u), 512u)) :
                                                          whole(work / (!two ? 256u : tiles * c->heads < 256u ? 512u : 1024u));
    sh.part_keys = uint32_t(std::min<uint64_t>(std::max<uint64_t>(part, sh.rows_log == kAttendRowsLog ? 128u : 512u), 1u << 30));
    const uint64_t parts = (keys + 31u + sh.part_keys - 1u) / sh.part_keys;
    sh.splits = numbered * c->heads > kAttendCounters ? 1u : uint32_t(std::min<uint64_t>(std::max<uint64_t>(parts, 1u), 256u));
    sh.tiles = uint32_t(numbered);
    // Keys and values of more than 256 MB by tiles, which no cache holds until they are read again, are read past the L2.  us past it / through it: one token for
    // each of 48 sequences of up to 16000 keys 281 / 310, up to 8000 160 / 163; 32 of up to 2000, 8 heads of 64 24.2 / 22.1; 8 tokens for each of 4 of up to
    // 4000, 16 heads on 2 22.1 / 19.7.
    sh.past = tiles * c->heads * keys * c->head_dim * 2u * element_bytes(c->dtype) > (uint64_t(1) << 28);
    if (sh.splits > 1u) sh.bytes = kAttendCounters * 4u + numbered * c->heads * sh.splits * attend_slot(sh.rows_log, c->head_dim) * 4u;
    return sh;
}

// (a launch has fewer than 2^32 threads, 512 a workgroup at most)
static int check_tiles(const hspmm_cache *c, const hspmm_batch *b, const AttendShape &sh)
{
    if (uint64_t(sh.tiles) * c->heads < (1u << 23)) return HSPMM_OK;
    return fail(HSPMM_ERR_UNSUPPORTED, "%u tokens of %u sequences with %u heads of keys: in several calls", b->tokens, b->sequences, c->heads);
}

int hspmm_cache_attend_workspace(const hspmm_cache *cache, const hspmm_batch *batch, const hspmm_attention *attention, uint64_t *bytes)
{
    if (!bytes) return fail(HSPMM_ERR_INVALID, "null bytes");
    if (int rc = check_attention(cache, batch, attention)) return rc;
    if (batch->tokens == 0) { *bytes = 0; return HSPMM_OK; }
    const AttendShape sh = attend_shape(cache, batch, attention);
    *bytes = sh.bytes;
    return check_tiles(cache, batch, sh);
}

int hspmm_cache_attend(const hspmm_cache *cache, uint32_t layer, const hspmm_batch *batch, const hspmm_attention *attention, const hspmm_heads *q,
                       const hspmm_heads *out, float *lse, void *workspace, uint64_t workspace_bytes, void *stream)
{
    if (int rc = check_attention(cache, batch, attention)) return rc;
    if (layer >= cache->layers) return fail(HSPMM_ERR_INVALID, "layer %u of %u", layer, cache->layers);
    if (batch->tokens == 0) return HSPMM_OK;
    const uint32_t e = element_bytes(cache->dtype), piece = 16u / e;
    if (int rc = check_heads("q", q, cache->dtype)) return rc;
    if (int rc = check_heads("out", out, cache->dtype)) return rc;
    if (q->dim_stride != 1 || q->token_stride % piece || q->head_stride % piece || reinterpret_cast<uintptr_t>(q->data) % 16u)
        return fail(HSPMM_ERR_UNSUPPORTED, "q: a head's elements side by side, tokens and heads at multiples of 16 bytes");
    if (reinterpret_cast<uintptr_t>(lse) % 4u) return fail(HSPMM_ERR_INVALID, "lse is not aligned to its elements");
    const AttendShape sh = attend_shape(cache, batch, attention);
    if (int rc = check_tiles(cache, batch, sh)) return rc;
    if (sh.bytes && (!workspace || workspace_bytes < sh.bytes || reinterpret_cast<uintptr_t>(workspace) % 16u))
        return fail(HSPMM_ERR_INVALID, "a workspace of %llu bytes, aligned to 16, is wanted", (unsigned long long)sh.bytes);
    if (int rc = check_device()) return rc;
    AttendArgs aa{};
    aa.pages = pages_of(cache, layer);
    aa.batch = batch_of(batch);
    aa.q = heads_of(q); aa.out = heads_of(out); aa.lse = lse;
    aa.q_heads = attention->q_heads; aa.shared = Divisor::of(attention->q_heads / cache->heads);
    aa.scale = attention->scale; aa.causal = attention->causal != 0; aa.window = attention->window;
    aa.heads = Divisor::of(cache->heads); aa.tiles = sh.tiles; aa.splits = sh.splits; aa.part_keys = sh.part_keys;
    aa.arrive = static_cast<uint32_t *>(workspace);
    aa.sums = reinterpret_cast<float *>(static_cast<char *>(workspace) + kAttendCounters * 4u);
    if (sh.rows_log == kAttendRowsLog) HSPMM_HIP(launch_attend_rows(cache->dtype, aa, sh.past, static_cast<hipStream_t>(stream)));
    else HSPMM_HIP(launch_attend_chunk(cache->dtype, aa, sh.rows_log, static_cast<hipStream_t>(stream)));
    return HSPMM_OK;
}

int hspmm_cache_extend(const hspmm_cache *cache, uint32_t n, const int32_t *rows, const int32_t *add, int32_t *status, void *stream)
{
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_list(cache, n, add, "add")) return rc;
    if (int rc = check_device()) return rc;
    HSPMM_HIP(launch_pages_extend(pool_of(cache), n, rows, add, status, static_cast<hipStream_t>(stream)));
    return HSPMM_OK;
}

int hspmm_cache_fork(const hspmm_cache *cache, uint32_t n, const int32_t *parents, const int32_t *children, int32_t *status, void *stream)
{
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_list(cache, n, parents, "parents")) return rc;
    if (int rc = check_list(cache, n, children, "children")) return rc;
    if (n == 0 && !status) return HSPMM_OK;
    if (int rc = check_launch(n, 1024u)) return rc;
    if (int rc = check_device()) return rc;
    HSPMM_HIP(launch_pages_fork(pool_of(cache), n, parents, children, status, static_cast<hipStream_t>(stream)));
    return HSPMM_OK;
}

int hspmm_cache_free(const hspmm_cache *cache, uint32_t n, const int32_t *rows, void *stream)
{
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_list(cache, n, rows, "rows")) return rc;
    if (n == 0) return HSPMM_OK;
    if (int rc = check_launch(n, 256u)) return rc;
    if (int rc = check_device()) return rc;
    HSPMM_HIP(launch_pages_free(pool_of(cache), n, rows, static_cast<hipStream_t>(stream)));
    return HSPMM_OK;
}

int hspmm_cache_compact(const hspmm_cache *cache, int32_t *table_out, int32_t *references_out, int32_t *live, void *stream)
{
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_device()) return rc;
    HSPMM_HIP(launch_pages_compact(pool_of(cache), table_out ? table_out : cache->table, references_out ? references_out : cache->references, live,
                                   static_cast<hipStream_t>(stream)));
    return HSPMM_OK;
}

int hspmm_cache_copy(const hspmm_cache *cache, uint32_t n, const int32_t *from, const int32_t *to, void *stream)
{
    if (int rc = check_cache(cache)) return rc;
    if (n > cache->pages) return fail(HSPMM_ERR_INVALID, "%u pages to copy of %u", n, cache->pages);
    if (n && (!from || !to)) return fail(HSPMM_ERR_INVALID, "null list of pages");
    if (n == 0) return HSPMM_OK;
    if (int rc = check_launch(n, 256u)) return rc;
    if (int rc = check_device()) return rc;
    HSPMM_HIP(launch_pages_copy(pool_of(cache), n, from, to, static_cast<hipStream_t>(stream)));
    return HSPMM_OK;
}

}  // extern "C"
