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

static int check_queries(const hspmm_cache *c, const hspmm_heads *q)
{
    const uint32_t piece = 16u / element_bytes(c->dtype);
    if (q->dim_stride != 1 || q->token_stride % piece || q->head_stride % piece || reinterpret_cast<uintptr_t>(q->data) % 16u)
        return fail(HSPMM_ERR_UNSUPPORTED, "q: a head's elements side by side, tokens and heads at multiples of 16 bytes");
    return HSPMM_OK;
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

// sequences: of a batch, or groups of them; chunk: the most tokens that one has; keys: the most that one sees.
static AttendShape attend_shape(const hspmm_cache *c, uint32_t sequences, uint32_t tokens, uint32_t chunk, uint64_t keys, const hspmm_attention *a)
{
    const uint32_t shared = a->q_heads / c->heads;
    const uint64_t rows = uint64_t(std::min(chunk, tokens)) * shared;
    AttendShape sh{};
    // those that a tile of so many rows sees
    auto seen = [&](uint32_t tile_rows) { return a->window && uint64_t(a->window) + tile_rows < keys ? uint64_t(a->window) + tile_rows : keys; };
    // The rows kernel for up to 16 rows, and where there is little to do: a tile of it is sixteen rows, and its waves share out the keys.  us of it / of the
    // chunk kernel by tiles of 16 rows x heads x keys, bf16, heads of 128: 8 K (60 tokens from the beginning, 32 heads) 6.6 / 9.7; 96 K (8 tokens for each of
    // 3 sequences of up to 2000, 32 heads on 8) 15.3 / 22.7; 180 K (300 tokens from the beginning) 15.0 / 16.7; 256 K (32 sequences of up to 500) 19.7 / 28.3;
    // 384 K (3 of 8000) 30.6 / 38.6; 384 K (3 tokens for each of 64 of 1500, 16 heads on 2) 34.0 / 32.6; 480 K (5 tokens over 30000) 55.9 / 70.8; 512 K (16 over
    // 16000) 48.3 / 44.4; 640 K (64 over 20000, 8 heads on 4) 67.5 / 54.4; 1024 K (32 of 2000) 82 / 70; 1600 K (16 ragged chunks) 65 / 33.  Up to 400 K it lost
    // at 4 of 24 such shapes, by 10 % at most (400 tokens from the beginning 19.9 / 18.1), above 500 K at 11 of 18, by up to a half; of 256 elements it won at
    // 304 K (59.5 / 74) and lost at 480 K (80 / 77).
    const uint64_t rows_work = uint64_t(sequences) * ((rows + 15u) / 16u) * c->heads * seen(16u);
    // 256 rows for heads of 97 to 128 elements only - with 128 rows two workgroups share a compute unit, but there only two images fit for each -, where chunks
    // are of one length, tiles for a quarter of the compute units and keys for parts on all of them: few, short and half-filled tiles are the longer ones' loss.  us
    // with 128 / 256 rows, by heads x tiles of 256 (`wide`), 32 heads on 8: 4096 tokens over 16384 keys (520) 1025 / 942; 8192 over 8192 (1032) 597 / 571; 2048 over
    // 8192 (264) 281 / 266; 1024 over 4096 (136) 96 / 82; 512 over 8512 (72) 105 / 99; 16 x 512 over 2000 (1088) 232 / 237; 2048 over 2048 (264) 67 / 71; 500 over
    // 500, 32 heads of keys (64) 22 / 27; few tiles: 256 over 8192 (40) 58 / 60, 700 over 20000, 8 heads on 4 (24) 85 / 103; ragged: 17 chunks of up to 700 over up
    // to 5700 (592) 216 / 279, 16 of up to 300 over 600 (664) 44 / 50, 8 of up to 300 over 2000 (328) 73 / 68.  Heads of 64, 2048 tokens over 8048, 177 / 184.
    const uint64_t wide = uint64_t(c->heads) * ((uint64_t(tokens) * shared >> 8) + (sequences + 1u) / 2u);
    const bool even = uint64_t(tokens) * 8u >= uint64_t(sequences) * std::min(chunk, tokens) * 7u;
    if (c->dtype == HSPMM_TF32 || rows <= 16u || rows_work <= 400000u) sh.rows_log = kAttendRowsLog;
    else sh.rows_log = c->head_dim > 96u && c->head_dim <= 128u && rows > 128u && even && wide >= 64u && wide * seen(256u) >= 200000u ? 8u : 7u;
    keys = seen(1u << sh.rows_log);
    const uint64_t numbered = attend_tiles(tokens, sequences, shared, sh.rows_log);
    // tiles that have rows, at most: numbers are left out
    const uint64_t tiles = std::min<uint64_t>(numbered, uint64_t(sequences) * ((rows + (1u << sh.rows_log) - 1u) >> sh.rows_log));
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

// Keys that a sequence may have, as far as the call says.
static uint64_t most_keys(const hspmm_cache *c, uint32_t longest)
{
    const uint64_t places = uint64_t(c->table_pages) * c->page_tokens;
    return longest && longest < places ? longest : places;
}

static AttendShape attend_shape(const hspmm_cache *c, const hspmm_batch *b, const hspmm_attention *a)
{
    return attend_shape(c, b->sequences, b->tokens, a->longest_chunk, most_keys(c, a->longest), a);
}

// An attention over shared prefixes, by sizes alone: tiles of the prefixes, with a group for a sequence, and of what is behind them.
struct SharedShape {
    bool both;                           // by tiles of the sequences' own rows, all keys: `rest` is an attention's
    AttendShape prefix, rest;
    uint64_t bytes;                      // of the workspace: sums of the parts of either
};

static SharedShape shared_shape(const hspmm_cache *c, const hspmm_batch *b, const hspmm_prefix *p, const hspmm_attention *a)
{
    SharedShape sh{};
    const uint64_t all = most_keys(c, a->longest), common = std::min<uint64_t>(p->longest ? p->longest : all, all);
    // Where sequences' own rows fill some tiles of the chunk kernel each, on average, there is little to win by others' beside them, and sums need not go through memory.  (A chunk of some thousand
    // tokens among 63 single ones does not make these full.)  us so / by tiles of the prefixes' rows and of what is behind them, by rows a sequence, 32 heads on 8 of 128, bf16: 160 (40 tokens for each of 64 behind 8000)
    // 728 / 476, (63 tokens and a chunk of 2500) 800 / 495; 256 755 / 665; 400 (100 tokens behind 8000) 732 / 589, (1500) 128 / 109; 590 (16 chunks of 50 to 250 tokens behind 3000 and 6000, features x
    // tokens) 273 to 283 / 275 to 302; 1000 506 / 416, (1500) 209 / 221; 2000 838 / 843, (1500) 366 / 457.  fp32, whose tiles are of 16 rows either way: 2000 1681 / 1554, but there sums are twice
    // what the call reads and writes else.
    sh.rest = attend_shape(c, b, a);
    const uint64_t all_rows = uint64_t(b->tokens) * (a->q_heads / c->heads), filled = all_rows / b->sequences;
    const bool full = c->dtype == HSPMM_TF32 ? filled >= 4096u : sh.rest.rows_log != kAttendRowsLog && filled >= 512u;
    // The same where all of it is little: a launch less.  us so / by tiles of prefixes and of what is behind them, a token each, 32 heads on 8, fp16, by MB of keys and values that the sequences'
    // own tiles read: 39 13.8 / 16.1, 72 16.7 / 19.7, 79 16.7 / 18.5, 92 20.4 / 18.0, 138 24.9 / 21.0; 12 heads on 4 of 64, fp32: 46 14.7 / 15.2, 69 19.8 / 21.8, 79 19.5 / 18.8, 144 27.9 / 22.6.
    // (no fewer tiles than rows fill, and as many as are numbered where the longest chunk is not told)
    const uint64_t rows = uint64_t(std::min(a->longest_chunk, b->tokens)) * (a->q_heads / c->heads);
    const uint64_t told = a->longest_chunk ? uint64_t(b->sequences) * ((rows + (1u << sh.rest.rows_log) - 1u) >> sh.rest.rows_log) : sh.rest.tiles;
    const uint64_t tiles = std::max<uint64_t>(std::min<uint64_t>(told, sh.rest.tiles), all_rows >> sh.rest.rows_log);
    const bool little = tiles * c->heads * all * c->head_dim * 2u * element_bytes(c->dtype) <= (uint64_t(80) << 20);
    sh.both = little || full;
    if (sh.both) {
        sh.bytes = sh.rest.bytes;
        return sh;
    }
    hspmm_attention whole = *a;
    whole.window = 0u;
    sh.prefix = attend_shape(c, p->groups, b->tokens, p->most_tokens ? p->most_tokens : b->tokens, common, &whole);
    // (keys behind the prefix: the longest sequence is taken to have the longest one)
    const uint64_t behind = std::max<uint64_t>(all - common, std::min<uint64_t>(std::max(a->longest_chunk, 1u), all));
    sh.rest = attend_shape(c, b->sequences, b->tokens, a->longest_chunk, behind, a);
    const uint32_t shared = a->q_heads / c->heads;
    auto tiles_of = [&](AttendShape &x, uint32_t sequences, uint32_t log) { x.rows_log = log; x.tiles = uint32_t(attend_tiles(b->tokens, sequences, shared, log)); };
    auto parts_of = [](AttendShape &x, uint64_t keys, uint64_t part) {
        x.part_keys = uint32_t(std::min<uint64_t>(std::max<uint64_t>((part + 127u) & ~uint64_t(127u), 128u), 1u << 30));
        x.splits = uint32_t(std::min<uint64_t>(std::max<uint64_t>((keys + 31u + x.part_keys - 1u) / x.part_keys, 1u), 256u));
    };
    tiles_of(sh.prefix, p->groups, std::min(sh.prefix.rows_log, 7u));
    if (sh.prefix.rows_log == kAttendRowsLog) sh.rest.rows_log = kAttendRowsLog;
    tiles_of(sh.rest, b->sequences, std::min(sh.rest.rows_log, 7u));
    // Parts cost a row's sums each, written and read, but nobody waits for them.  us by keys of a prefix's part / of what is behind one's: 8 beams over 1000 keys by 128 / 256 / 512 / 1024 17.8 /
    // 15.6 / 16.1 / 19.9; 64 sequences of up to 1500 behind 8000 by 256 / 512 / 768 / 1024 / 1536 102 / 79 / 72 / 67 / 75, and with 1024 there by 256 / 512 / 1024 / 1536 75 / 69 / 67 / 70; fp32 drafts over
    // up to 6000 81 / 67 / - / 60 / 70 and 60 / 60 / 64 / -.
    // Longer ones where tiles alone are workgroups for the chip - as many of the chunk kernel's as run at a time, four times as many of the rows kernel's -, as sums are what parts cost
    // then.  us (MB of workspace) by 1024 keys / 1024 / 768 / 512 workgroups of the chunk kernel, 32 heads on 8 of 128, bf16: 64 x 16 tokens behind 8000 243 (156) / 204 (87) / 193 (69) / 189 (52);
    // 256 x 8 538 (311) / 411 (104) / 414 (104) / 397 (69); 32 x 100 715 (487) / 545 (162) / 594 (108) / 593 (108); 63 tokens and a chunk of 1000 289 (180) / 250 (108) / 225 (72) / 253 (54); 128 x 16 behind
    // 32000 1696 (1142) / 1202 (138) / 1198 (104) / 1200 (104); 256 x 1 behind 128000 902 (549) / 668 (74) / 672 (56) / 670 (43).  By 1024 keys / 2048 workgroups of the rows kernel, fp32: 16 x 60 behind
    // 4000 782 / 739, 16 x 64, 12 heads on 4 of 64, 185 / 181.  (By 768 / 512, 18 such shapes were 2 % above the best on average with either, and 512 wants a third less.)
    auto spread = [&](const AttendShape &x, uint32_t sequences, uint64_t keys) {
        const uint64_t most = uint64_t(sequences) * ((uint64_t(std::min(&x == &sh.prefix ? (p->most_tokens ? p->most_tokens : b->tokens) : a->longest_chunk, b->tokens)) * shared + (1u << x.rows_log) - 1u) >> x.rows_log);
        // (whatever the call says, there are no fewer tiles than its rows fill)
        const uint64_t tiles = std::max<uint64_t>(std::min<uint64_t>(most, x.tiles), uint64_t(b->tokens) * shared >> x.rows_log);
        const uint64_t cells = std::max<uint64_t>(tiles, 1u) * c->heads, at_a_time = x.rows_log == kAttendRowsLog ? 2048u : 512u;
        return std::max<uint64_t>(std::min<uint64_t>(std::max<uint64_t>(cells * keys / 128u, 256u), 1024u), cells * keys / at_a_time);
    };
    parts_of(sh.prefix, common, spread(sh.prefix, p->groups, common));
    parts_of(sh.rest, behind, spread(sh.rest, b->sequences, behind));
    // (behind an attention's counters, so that one workspace serves both)
    sh.bytes = kAttendCounters * 4u + uint64_t(sh.prefix.splits + sh.rest.splits) * b->tokens * a->q_heads * (c->head_dim + kPrefixExtra) * 4u;
    return sh;
}

static int check_prefix(const hspmm_batch *b, const hspmm_prefix *p)
{
    if (!p) return fail(HSPMM_ERR_INVALID, "null prefix");
    if (p->groups > b->sequences) return fail(HSPMM_ERR_INVALID, "%u groups of %u sequences", p->groups, b->sequences);
    if (p->groups && (!p->firsts || !p->tokens)) return fail(HSPMM_ERR_INVALID, "%u groups without their sequences or tokens", p->groups);
    return HSPMM_OK;
}

// (a launch has fewer than 2^32 threads, 512 a workgroup at most)
static int check_tiles(const hspmm_cache *c, const hspmm_batch *b, const AttendShape &sh)
{
    if (uint64_t(sh.tiles) * c->heads < (1u << 23)) return HSPMM_OK;
    return fail(HSPMM_ERR_UNSUPPORTED, "%u tokens of %u sequences with %u heads of keys: in several calls", b->tokens, b->sequences, c->heads);
}

}  // extern "C"

// (launches have fewer than 2^32 threads, 256 a workgroup)
static int check_shared(const hspmm_cache *c, const hspmm_batch *b, const hspmm_attention *a, const SharedShape &sh)
{
    if (sh.both) return check_tiles(c, b, sh.rest);
    const uint64_t groups = uint64_t(c->heads) * (uint64_t(sh.prefix.tiles) * sh.prefix.splits + uint64_t(sh.rest.tiles) * sh.rest.splits), merged = (uint64_t(b->tokens) + 15u) / 16u * a->q_heads;
    if (groups < (1u << 23) && merged < (1u << 24)) return HSPMM_OK;
    return fail(HSPMM_ERR_UNSUPPORTED, "%u tokens of %u sequences with %u heads of keys: in several calls", b->tokens, b->sequences, c->heads);
}

extern "C" {

int hspmm_cache_attend_workspace(const hspmm_cache *cache, const hspmm_batch *batch, const hspmm_attention *attention, uint64_t *bytes)
{
    if (!bytes) return fail(HSPMM_ERR_INVALID, "null bytes");
    if (int rc = check_attention(cache, batch, attention)) return rc;
    if (batch->tokens == 0) { *bytes = 0; return HSPMM_OK; }
    const AttendShape sh = attend_shape(cache, batch, attention);
    *bytes = sh.bytes;
    return check_tiles(cache, batch, sh);
}

}  // extern "C"

// What an attention's calls check alike.
static int check_attend_tensors(const hspmm_cache *cache, uint32_t layer, const hspmm_heads *q, const hspmm_heads *out, const float *lse)
{
    if (layer >= cache->layers) return fail(HSPMM_ERR_INVALID, "layer %u of %u", layer, cache->layers);
    if (int rc = check_heads("q", q, cache->dtype)) return rc;
    if (int rc = check_heads("out", out, cache->dtype)) return rc;
    if (int rc = check_queries(cache, q)) return rc;
    if (reinterpret_cast<uintptr_t>(lse) % 4u) return fail(HSPMM_ERR_INVALID, "lse is not aligned to its elements");
    return HSPMM_OK;
}

static AttendArgs attend_args(const hspmm_cache *cache, uint32_t layer, const hspmm_batch *batch, const hspmm_attention *attention, const hspmm_heads *q,
                              const hspmm_heads *out, float *lse, const AttendShape &sh, void *workspace)
{
    AttendArgs aa{};
    aa.pages = pages_of(cache, layer);
    aa.batch = batch_of(batch);
    aa.q = heads_of(q); aa.out = heads_of(out); aa.lse = lse;
    aa.q_heads = attention->q_heads; aa.shared = Divisor::of(attention->q_heads / cache->heads);
    aa.scale = attention->scale; aa.causal = attention->causal != 0; aa.window = attention->window;
    aa.heads = Divisor::of(cache->heads); aa.tiles = sh.tiles; aa.splits = sh.splits; aa.part_keys = sh.part_keys;
    aa.arrive = static_cast<uint32_t *>(workspace);
    aa.sums = reinterpret_cast<float *>(static_cast<char *>(workspace) + kAttendCounters * 4u);
    return aa;
}

static int check_workspace(const void *workspace, uint64_t bytes, uint64_t wanted)
{
    if (wanted && (!workspace || bytes < wanted || reinterpret_cast<uintptr_t>(workspace) % 16u))
        return fail(HSPMM_ERR_INVALID, "a workspace of %llu bytes, aligned to 16, is wanted", (unsigned long long)wanted);
    return HSPMM_OK;
}

extern "C" {

int hspmm_cache_attend(const hspmm_cache *cache, uint32_t layer, const hspmm_batch *batch, const hspmm_attention *attention, const hspmm_heads *q,
                       const hspmm_heads *out, float *lse, void *workspace, uint64_t workspace_bytes, void *stream)
{
    if (int rc = check_attention(cache, batch, attention)) return rc;
    if (layer >= cache->layers) return fail(HSPMM_ERR_INVALID, "layer %u of %u", layer, cache->layers);
    if (batch->tokens == 0) return HSPMM_OK;
    if (int rc = check_attend_tensors(cache, layer, q, out, lse)) return rc;
    const AttendShape sh = attend_shape(cache, batch, attention);
    if (int rc = check_tiles(cache, batch, sh)) return rc;
    if (int rc = check_workspace(workspace, workspace_bytes, sh.bytes)) return rc;
    if (int rc = check_device()) return rc;
    const AttendArgs aa = attend_args(cache, layer, batch, attention, q, out, lse, sh, workspace);
    if (sh.rows_log == kAttendRowsLog) HSPMM_HIP(launch_attend_rows(cache->dtype, aa, sh.past, false, static_cast<hipStream_t>(stream)));
    else HSPMM_HIP(launch_attend_chunk(cache->dtype, aa, false, sh.rows_log, static_cast<hipStream_t>(stream)));
    return HSPMM_OK;
}

int hspmm_cache_attend_shared_workspace(const hspmm_cache *cache, const hspmm_batch *batch, const hspmm_prefix *prefix, const hspmm_attention *attention, uint64_t *bytes)
{
    if (!bytes) return fail(HSPMM_ERR_INVALID, "null bytes");
    if (int rc = check_attention(cache, batch, attention)) return rc;
    if (int rc = check_prefix(batch, prefix)) return rc;
    if (prefix->groups == 0) return hspmm_cache_attend_workspace(cache, batch, attention, bytes);
    if (batch->tokens == 0) { *bytes = 0; return HSPMM_OK; }
    const SharedShape sh = shared_shape(cache, batch, prefix, attention);
    *bytes = sh.bytes;
    return check_shared(cache, batch, attention, sh);
}

int hspmm_cache_attend_shared(const hspmm_cache *cache, uint32_t layer, const hspmm_batch *batch, const hspmm_prefix *prefix, const hspmm_attention *attention,
                              const hspmm_heads *q, const hspmm_heads *out, float *lse, void *workspace, uint64_t workspace_bytes, void *stream)
{
    if (int rc = check_attention(cache, batch, attention)) return rc;
    if (int rc = check_prefix(batch, prefix)) return rc;
    if (prefix->groups == 0) return hspmm_cache_attend(cache, layer, batch, attention, q, out, lse, workspace, workspace_bytes, stream);
    if (layer >= cache->layers) return fail(HSPMM_ERR_INVALID, "layer %u of %u", layer, cache->layers);
    if (batch->tokens == 0) return HSPMM_OK;
    if (int rc = check_attend_tensors(cache, layer, q, out, lse)) return rc;
    const SharedShape sh = shared_shape(cache, batch, prefix, attention);
    if (int rc = check_shared(cache, batch, attention, sh)) return rc;
    if (int rc = check_workspace(workspace, workspace_bytes, sh.bytes)) return rc;
    if (int rc = check_device()) return rc;
    AttendArgs of_prefix = attend_args(cache, layer, batch, attention, q, out, lse, sh.prefix, workspace), of_rest = attend_args(cache, layer, batch, attention, q, out, lse, sh.rest, workspace);
    of_prefix.prefix = of_rest.prefix = PrefixArgs{prefix->firsts, prefix->tokens, prefix->groups, sh.prefix.splits, sh.prefix.part_keys, of_rest.sums,
                                                   int64_t(batch->tokens) * attention->q_heads * (cache->head_dim + kPrefixExtra)};
    if (sh.both) {
        if (sh.rest.rows_log == kAttendRowsLog) HSPMM_HIP(launch_attend_rows(cache->dtype, of_rest, false, true, static_cast<hipStream_t>(stream)));
        else HSPMM_HIP(launch_attend_chunk(cache->dtype, of_rest, true, sh.rest.rows_log, static_cast<hipStream_t>(stream)));
        return HSPMM_OK;
    }
    HSPMM_HIP(launch_attend_shared(cache->dtype, of_prefix, of_rest, sh.prefix.rows_log != kAttendRowsLog, sh.rest.rows_log != kAttendRowsLog, static_cast<hipStream_t>(stream)));
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

}  // extern "C"

// tokens, sequences: that a head's row has at least, and that have rows which are written at a time (rows side by side are written by different workgroups): from the smallest stride to the
// largest each passes all rows of those below it.
static int check_weights(const hspmm_cache *c, const hspmm_weights *w, uint64_t tokens, uint32_t sequences, uint32_t layers)
{
    if (!w || !w->data) return fail(HSPMM_ERR_INVALID, "null weights");
    if (reinterpret_cast<uintptr_t>(w->data) % 4u) return fail(HSPMM_ERR_INVALID, "weights are not aligned to their elements");
    if (w->layer_stride < 0 || w->sequence_stride < 0 || w->head_stride < 0) return fail(HSPMM_ERR_INVALID, "weights: strides below 0");
    std::pair<uint64_t, uint32_t> rows[3] = {{uint64_t(w->head_stride), c->heads}, {uint64_t(w->sequence_stride), sequences}, {uint64_t(w->layer_stride), layers}};
    std::sort(rows, rows + 3);
    unsigned __int128 reach = tokens;
    for (const auto &r : rows) {
        if (r.second <= 1u) continue;
        if (r.first < reach) return fail(HSPMM_ERR_INVALID, "weights: rows of %llu tokens that overlap", (unsigned long long)tokens);
        reach += static_cast<unsigned __int128>(r.first) * (r.second - 1u);
    }
    return HSPMM_OK;
}

// How a call of hspmm_cache_weigh is launched, by sizes alone: the same for the call and for its workspace.
struct WeighShape {
    bool chunk, few;                     // by the chunk kernel; by the rows kernel, sixteen rows at a time
    uint32_t parts, blocks, part_rows;
    uint64_t cells, bytes;
};

static WeighShape weigh_shape(const hspmm_cache *c, const hspmm_batch *b, const hspmm_attention *a, uint32_t last)
{
    WeighShape sh{};
    const uint64_t keys = most_keys(c, a->longest), heads = uint64_t(b->sequences) * c->heads;
    const uint64_t tokens = std::min(a->longest_chunk, b->tokens), rows = std::max<uint64_t>((last && last < tokens ? last : tokens) * (a->q_heads / c->heads), 1u);
    auto up = [](uint64_t n, uint64_t to) { return (n + to - 1u) / to; };
    // (rows in registers / in LDS, us: a token for each of 48 sequences of up to 16000 178 / 234, of 3 of up to 300 6.8 / 7.0)
    sh.few = rows <= 16u;
    // (up to the rows that the rows kernel has in LDS; us there / by the chunk kernel: 96 rows over 17 of up to 5700 keys 18 / 30, 16384 over 8192 840 / 260)
    sh.chunk = c->dtype != HSPMM_TF32 && rows > 128u;
    if (!sh.chunk) {
        // a wave has a tile of 32 keys or some.  us by 1024 / 2048 / 4096 / 8192 / 16384 workgroups: a token for each of 48 sequences of up to 16000 214 / 195 / 184 / 177 / 182;
        // where a workgroup has rows to load first, the last 32 tokens of 17 of up to 5700 19.6 / 20.2 / 21.0 / 22.0
        const uint64_t groups = (sh.few ? 8192u : 1024u) / std::max<uint64_t>(heads, 1u);
        sh.parts = uint32_t(std::min<uint64_t>(std::max<uint64_t>(std::min<uint64_t>(up(keys, 128u), groups), 1u), 32768u));
        return sh;
    }
    sh.blocks = uint32_t(std::min<uint64_t>(up(keys, kWeighKeys), std::max<uint64_t>((uint64_t(1) << 22) / std::max<uint64_t>(heads, 1u), 1u)));
    sh.cells = heads * sh.blocks;
    // parts of the rows: as many as make some thousand workgroups, 256 rows at least
    sh.part_rows = uint32_t(std::max<uint64_t>(up(up(rows * sh.cells, 1536u), 64u) * 64u, 256u));
    sh.parts = uint32_t(std::min<uint64_t>(up(rows, sh.part_rows), 256u));
    if (sh.cells > kAttendCounters) sh.parts = 1u;
    if (sh.parts > 1u) sh.bytes = kAttendCounters * 4u + sh.cells * sh.parts * kWeighKeys * 4u;
    return sh;
}

static int check_weigh(const hspmm_cache *c, const hspmm_batch *b, const hspmm_attention *a)
{
    if (int rc = check_attention(c, b, a)) return rc;
    // (a launch has fewer than 2^32 threads)
    if (uint64_t(b->sequences) * c->heads >= (1u << 23)) return fail(HSPMM_ERR_UNSUPPORTED, "%u sequences with %u heads of keys: in several calls", b->sequences, c->heads);
    return HSPMM_OK;
}

extern "C" {

int hspmm_cache_weigh_workspace(const hspmm_cache *cache, const hspmm_batch *batch, const hspmm_attention *attention, uint32_t last, uint64_t *bytes)
{
    if (!bytes) return fail(HSPMM_ERR_INVALID, "null bytes");
    if (int rc = check_weigh(cache, batch, attention)) return rc;
    *bytes = batch->tokens ? weigh_shape(cache, batch, attention, last).bytes : 0u;
    return HSPMM_OK;
}

int hspmm_cache_weigh(const hspmm_cache *cache, uint32_t layer, const hspmm_batch *batch, const hspmm_attention *attention, const hspmm_heads *q, const float *lse,
                      const hspmm_weights *weights, float decay, uint32_t last, void *workspace, uint64_t workspace_bytes, void *stream)
{
    if (int rc = check_weigh(cache, batch, attention)) return rc;
    if (layer >= cache->layers) return fail(HSPMM_ERR_INVALID, "layer %u of %u", layer, cache->layers);
    if (!std::isfinite(decay)) return fail(HSPMM_ERR_INVALID, "decay %g", double(decay));
    if (int rc = check_weights(cache, weights, 1u, batch->sequences, 1u)) return rc;
    if (batch->tokens == 0) return HSPMM_OK;
    if (int rc = check_heads("q", q, cache->dtype)) return rc;
    if (int rc = check_queries(cache, q)) return rc;
    if (!lse || reinterpret_cast<uintptr_t>(lse) % 4u) return fail(HSPMM_ERR_INVALID, "lse is null or not aligned to its elements");
    const WeighShape sh = weigh_shape(cache, batch, attention, last);
    if (int rc = check_workspace(workspace, workspace_bytes, sh.bytes)) return rc;
    if (int rc = check_device()) return rc;
    WeighArgs wa{};
    wa.pages = pages_of(cache, layer);
    wa.batch = batch_of(batch);
    wa.q = heads_of(q); wa.lse = lse;
    wa.q_heads = attention->q_heads; wa.shared = Divisor::of(attention->q_heads / cache->heads); wa.heads = Divisor::of(cache->heads);
    wa.scale = attention->scale; wa.decay = decay; wa.causal = attention->causal != 0; wa.window = attention->window; wa.last = last;
    wa.weights = weights->data + weights->layer_stride * layer;
    wa.sequence_stride = weights->sequence_stride; wa.head_stride = weights->head_stride;
    wa.parts = sh.parts;
    if (!sh.chunk) {
        HSPMM_HIP(launch_weigh_rows(cache->dtype, wa, sh.few, static_cast<hipStream_t>(stream)));
        return HSPMM_OK;
    }
    wa.blocks = Divisor::of(sh.blocks); wa.part_rows = sh.part_rows;
    wa.arrive = static_cast<uint32_t *>(workspace);
    wa.sums = reinterpret_cast<float *>(static_cast<char *>(workspace) + kAttendCounters * 4u);
    HSPMM_HIP(launch_weigh_chunk(cache->dtype, wa, static_cast<hipStream_t>(stream)));
    return HSPMM_OK;
}

}  // extern "C"

// Words of an eviction's workspace, one behind another.
struct EvictShape { uint64_t arrive, entries, rows, to, free, kept, weights, words; uint32_t keep_pages; };

static EvictShape evict_shape(const hspmm_cache *c, uint32_t n, uint32_t keep)
{
    EvictShape sh{};
    sh.keep_pages = uint32_t((uint64_t(keep) + c->page_tokens - 1u) / c->page_tokens);
    const uint64_t lists = uint64_t(c->layers) * n * c->heads * keep, pages = uint64_t(n) * sh.keep_pages;
    sh.entries = sh.arrive + kAttendCounters;                    // (an attention's, so that one workspace serves both)
    sh.rows = sh.entries + uint64_t(n) * kEvictEntry;
    sh.to = sh.rows + uint64_t(n) * c->table_pages;
    sh.free = sh.to + pages;
    sh.kept = sh.free + std::min<uint64_t>(pages, c->pages);
    sh.weights = sh.kept + lists;
    sh.words = sh.weights + lists;
    return sh;
}

static int check_eviction(const hspmm_cache *c, uint32_t n, uint32_t keep)
{
    if (int rc = check_cache(c)) return rc;
    if (n > c->sequences) return fail(HSPMM_ERR_INVALID, "a list of %u for a cache of %u sequences", n, c->sequences);
    if (!keep || keep > 0x7FFFFFFFu || keep > uint64_t(c->table_pages) * c->page_tokens) return fail(HSPMM_ERR_INVALID, "%u tokens to keep, of at most %llu", keep, (unsigned long long)c->table_pages * c->page_tokens);
    // (a launch has fewer than 2^32 threads, 1024 a workgroup, or 256 and up to 2 x 16384 + 1 workgroups a head)
    const uint64_t cells = uint64_t(n) * c->layers * c->heads;
    PoolArgs pa{};
    pa.token_bytes = c->head_dim * element_bytes(c->dtype);
    if (n + cells >= (1u << 22) || n + cells * (2u * evict_shares(pa, cells) + 1u) >= (1u << 24)) return fail(HSPMM_ERR_UNSUPPORTED, "a list of %u: in several calls", n);
    return HSPMM_OK;
}

extern "C" {

int hspmm_cache_evict_workspace(const hspmm_cache *cache, uint32_t n, uint32_t keep, uint64_t *bytes)
{
    if (!bytes) return fail(HSPMM_ERR_INVALID, "null bytes");
    if (int rc = check_eviction(cache, n, keep)) return rc;
    *bytes = n ? evict_shape(cache, n, keep).words * 4u : 0u;
    return HSPMM_OK;
}

int hspmm_cache_evict(const hspmm_cache *cache, uint32_t n, const int32_t *parents, const int32_t *children, const hspmm_weights *weights, uint32_t keep, uint32_t first,
                      uint32_t last, int32_t *kept, int32_t *status, void *workspace, uint64_t workspace_bytes, void *stream)
{
    if (int rc = check_eviction(cache, n, keep)) return rc;
    if (int rc = check_list(cache, n, parents, "parents")) return rc;
    if (int rc = check_weights(cache, weights, uint64_t(cache->table_pages) * cache->page_tokens, cache->sequences, cache->layers)) return rc;
    if (uint64_t(first) + last > keep) return fail(HSPMM_ERR_INVALID, "the first %u and the last %u tokens, of %u to keep", first, last, keep);
    if (n == 0 && !status) return HSPMM_OK;
    const EvictShape sh = evict_shape(cache, n, keep);
    if (n)
        if (int rc = check_workspace(workspace, workspace_bytes, sh.words * 4u)) return rc;
    if (int rc = check_device()) return rc;
    // (of nothing there is the status alone)
    if (n == 0) {
        HSPMM_HIP(launch_pages_extend(pool_of(cache), 0u, nullptr, nullptr, status, static_cast<hipStream_t>(stream)));
        return HSPMM_OK;
    }
    int32_t *const words = static_cast<int32_t *>(workspace);
    EvictArgs ea{};
    ea.n = n; ea.parents = parents; ea.children = children; ea.keep = keep; ea.first = first; ea.last = last;
    ea.weights = weights->data; ea.weights_layer = weights->layer_stride; ea.weights_sequence = weights->sequence_stride; ea.weights_head = weights->head_stride;
    ea.kept = kept ? kept : words + sh.kept; ea.status = status;
    ea.arrive = reinterpret_cast<uint32_t *>(words + sh.arrive);
    ea.entries = words + sh.entries; ea.rows = words + sh.rows; ea.to = words + sh.to; ea.free = words + sh.free;
    ea.kept_weights = reinterpret_cast<float *>(words + sh.weights);
    ea.keep_pages = sh.keep_pages;
    HSPMM_HIP(launch_evict(pool_of(cache), ea, static_cast<hipStream_t>(stream)));
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
