// Eviction of cached tokens by the attention weight that they have received.
//
// Per layer, list entry and head of keys: of the tokens that the parent has stored, those that are kept anyway (the first and the last ones) and, of the others, those of the
// greatest weights, ties to the lowest number.  The smallest weight that is taken is found digit by digit (2048, 2048 and 1024 values of a
// digit) from counts in LDS.  Up to 16384 tokens each weight is read once, into a register; of more once a digit, and once more for the list.  Then slot k of the child receives the k-th token kept.
//
// In place - a sequence that is its own child, its pages named by nobody else - no token moves to a higher slot, so a workgroup that has all tokens of a column and
// loads a set of them before it stores the set in front loses none.  Everything else goes to new pages, by as many workgroups as like.
// Columns are shares of 64 bytes and more, and sets wait for each other, so moving all is slower than into other pages, but what keeps its place is not moved: us into others / in place (keys, values and
// weights last used long ago), 12 sequences, 8 layers of 8 heads of 128, bf16: 1024 of up to 8000 tokens 246 / 285, 1024 of 1025 227 / 123; 32 sequences, 32 layers, 1024 of up to 1040 1953 / 1100;
// 4 of 8192 of up to 60000 749 / 891.
// Two launches, as which pages are free has to be known before one is written (page_kernels.hip).
// Moving is memory's: 1024 of up to 8000 tokens of 12 prompts, 8 layers of 8 heads of 128, bf16, 179 us for 0.8 GB, 4.5 TB/s in rows of 256 bytes that lie apart (a copy: 4.8); four rows a thread on their way
// (two or eight: slower), stores past the L2.  Choosing is a chain of sums over the workgroup and of counts, 10 us for 700 tokens and 35 there, so each weight stays in a register (16 a thread) for all digits, and tokens follow each other in
// a thread so that one sum puts them in order.
#include "pages_common.hpp"
#include <algorithm>

namespace hspmm {

namespace {

// An entry of the list, as the first launch leaves it for the second.
struct EvictEntry {
    int32_t tokens;                      // that are kept, below 0: nothing happens to the child
    int32_t need, at;                    // new pages, and the first of them among the free ones
    int32_t in_place;
    int32_t spare[4];
};
static_assert(sizeof(EvictEntry) == kEvictEntry * 4u, "");

__device__ __forceinline__ EvictEntry *entry_of(const EvictArgs &ea, uint32_t i) { return reinterpret_cast<EvictEntry *>(ea.entries) + i; }
__device__ __forceinline__ uint32_t parent_of(const PoolArgs &pa, const EvictArgs &ea, uint32_t i) { return row_of(pa, ea.parents, i); }
__device__ __forceinline__ uint32_t child_of(const PoolArgs &pa, const EvictArgs &ea, uint32_t i) { return ea.children ? row_of(pa, ea.children, i) : parent_of(pa, ea, i); }

// Tokens of place p of a sequence of so many, if it has a page.
__device__ __forceinline__ uint32_t tokens_of_place(const PoolArgs &pa, uint32_t p, int32_t length)
{
    const uint32_t before = p * pa.page_tokens.d, left = uint32_t(length) - before;
    return left < pa.page_tokens.d ? left : pa.page_tokens.d;
}

// Whole numbers that keep the weights' order; NaN, which is less than anything, is 0.
__device__ __forceinline__ uint32_t ordered(float w)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, w);
    if (w != w) return 0u;
    if (u == 0x80000000u) return 0x80000000u;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Entry i of the list: its parent's row of the table, how many tokens it keeps and where they go.  The workgroup that is done last gives out pages.
__device__ void evict_plan(const PoolArgs &pa, const EvictArgs &ea, uint32_t i)
{
    __shared__ uint32_t waves[2u * kScanWaves], last_one;
    uint32_t turn = 0u;
    const uint32_t tid = threadIdx.x, parent = parent_of(pa, ea, i), child = child_of(pa, ea, i);
    // (asked for before it is known which workgroup looks at them)
    const Eight ahead = load_references(pa.references, pa.pages, tid * kEach);
    EvictEntry e{-1, 0, 0, 0, {0, 0, 0, 0}};
    if (parent != kIdxMax && child != kIdxMax) {
        const int32_t length = held(pa, parent);
        const uint32_t used = places_for(pa, length);
        const int32_t *row = pa.table + size_t(parent) * pa.table_pages;
        const bool own = parent == child;
        int32_t *const to = ea.to + size_t(i) * ea.keep_pages;
        // the k-th page that the parent has takes the k-th page of tokens where that can be in place, else a new one does
        uint32_t pages_there = 0u, stored = 0u, total;
        for (uint32_t p0 = 0; p0 < used; p0 += kScanThreads) {
            const uint32_t p = p0 + tid;
            const int32_t id = p < used ? row[p] : -1;
            const bool there = uint32_t(id) < pa.pages;
            if (p < used) ea.rows[size_t(i) * pa.table_pages + p] = there ? id : -1;
            // (a bit more where the last place, which may be filled in part, has a page)
            const uint32_t k = pages_there + (scan(uint32_t(there) + (there && p + 1u == used ? 1u << 16 : 0u), waves, turn, &total) & 0xFFFFu);
            turn ^= 1u;
            pages_there += total & 0xFFFFu;
            stored += (total & 0xFFFFu) * pa.page_tokens.d - (total >> 16 ? pa.page_tokens.d - tokens_of_place(pa, used - 1u, length) : 0u);
            if (there && k < ea.keep_pages) to[k] = own ? id : -1 - int32_t(k);
        }
        if (!own || uint32_t(length) > ea.keep) {
            e.tokens = int32_t(stored < ea.keep ? stored : ea.keep);
            const uint32_t pages = pages_for(pa, e.tokens);
            e.need = int32_t(pages);
            if (own) {
                uint32_t named = 0u;
                for (uint32_t k = tid; k < ea.n; k += kScanThreads) named += parent_of(pa, ea, k) == parent;
                scan(named, waves, turn, &total);
                turn ^= 1u;
                e.in_place = total == 1u;
                // (the pages that follow in `to` are this workgroup's own writes, of other threads: behind the barrier of the sum above)
                uint32_t before = 0u;
                for (uint32_t k0 = 0; k0 < pages; k0 += kScanThreads) {
                    const uint32_t k = k0 + tid;
                    const int32_t id = k < pages ? to[k] : 0;
                    const bool fresh = k < pages && !(e.in_place && pa.references[id] == 1);
                    const uint32_t rank = before + scan(fresh, waves, turn, &total);
                    turn ^= 1u;
                    before += total;
                    if (fresh) to[k] = -1 - int32_t(rank);
                }
                e.need = int32_t(before);
            }
        }
    }
    if (tid == 0u) {
        EvictEntry *const to = entry_of(ea, i);
        to->in_place = e.in_place;
        __hip_atomic_store(&to->tokens, e.tokens, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&to->need, e.need, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_one = __hip_atomic_fetch_add(ea.arrive, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) + 1u == ea.n;
    }
    __syncthreads();
    if (!last_one) return;
    if (tid == 0u) __hip_atomic_store(ea.arrive, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    uint64_t need = 0u;
    for (uint32_t i0 = 0; i0 < ea.n; i0 += kScanThreads) {
        const uint32_t k = i0 + tid;
        const uint32_t mine = k < ea.n ? uint32_t(__hip_atomic_load(&entry_of(ea, k)->need, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) : 0u;
        uint32_t total;
        const uint32_t before = scan(mine, waves, turn, &total);
        turn ^= 1u;
        const uint64_t at = need + before;
        // (an entry that the pool has no pages for stays as it was; those behind it find none either)
        if (k < ea.n) entry_of(ea, k)->at = at + mine <= pa.pages ? int32_t(at) : -1;
        need += total;
    }
    const uint32_t found = find_free(pa.references, pa.pages, need < pa.pages ? uint32_t(need) : pa.pages, ea.free, waves, turn, ahead);
    __syncthreads();
    for (uint32_t k = tid; k < ea.n; k += kScanThreads) {
        EvictEntry *const to = entry_of(ea, k);
        const int32_t mine = __hip_atomic_load(&to->need, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (mine && (to->at < 0 || uint32_t(to->at) + uint32_t(mine) > found)) __hip_atomic_store(&to->tokens, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (ea.status && tid == 0u) {
        const uint64_t missing = need - found;
        *ea.status = missing > 0x7FFFFFFFu ? 0x7FFFFFFF : int32_t(missing);
    }
}

constexpr uint32_t kDigits = 3u, kBins = 2048u;
__device__ __forceinline__ uint32_t digit_of(uint32_t u, uint32_t digit) { return digit == 0u ? u >> 21 : digit == 1u ? u >> 10 & 2047u : u & 1023u; }

// Which tokens of a layer, an entry and a head are kept.  kHeld: tokens a thread has in registers, so that of up to 1024 times as many each weight is read once; of more, the threads look at
// 1024 side by side at a time, and again for every digit.
template <uint32_t kHeld>
__device__ void evict_choose(const PoolArgs &pa, const EvictArgs &ea, uint32_t cell)
{
    __shared__ uint32_t waves[2u * kScanWaves], bins[kBins], found[2];
    uint32_t turn = 0u;
    const uint32_t tid = threadIdx.x, row = cell / pa.heads, head = cell - row * pa.heads, layer = row / ea.n, i = row - layer * ea.n;
    const uint32_t parent = parent_of(pa, ea, i);
    const size_t out = (size_t(row) * pa.heads + head) * ea.keep;
    const int32_t length = parent == kIdxMax ? 0 : held(pa, parent);
    const uint32_t used = places_for(pa, length);
    const int32_t *table = pa.table + size_t(parent == kIdxMax ? 0u : parent) * pa.table_pages;
    const float *weights = ea.weights + int64_t(layer) * ea.weights_layer + int64_t(parent == kIdxMax ? 0u : parent) * ea.weights_sequence + int64_t(head) * ea.weights_head;
    const uint32_t tokens = uint32_t(length) < used * pa.page_tokens.d ? uint32_t(length) : used * pa.page_tokens.d;      // that there are places for
    const int32_t last = length - int32_t(ea.last);            // (below 0 where all are among the last ones)
    auto is_kept_anyway = [&](uint32_t j) __attribute__((always_inline)) { return j < ea.first || int32_t(j) >= last; };
    const bool held_here = tokens <= kHeld * kScanThreads;
    // (a thread's tokens follow each other: one sum over the threads is enough to put them in order)
    const uint32_t each = (tokens + kScanThreads - 1u) / kScanThreads, mine = held_here ? tid * each : 0u;
    float w[kHeld];
    if (held_here) {
#pragma unroll
        for (uint32_t e = 0; e < kHeld; ++e) w[e] = weights[e < each && mine + e < tokens ? mine + e : 0u];
    }
    // whether every place has a page, else they are looked up token by token
    uint32_t missing = 0u, total;
    for (uint32_t p = tid; p < used; p += kScanThreads) missing += uint32_t(table[p]) >= pa.pages;
    scan(missing, waves, turn, &total);
    turn ^= 1u;
    const bool whole = total == 0u;
    auto is_stored = [&](uint32_t j) __attribute__((always_inline)) { return whole || uint32_t(table[pa.page_tokens.quotient(j)]) < pa.pages; };
    // how many are stored, and how many of those are kept anyway
    uint32_t stored = tokens, anyway = min(ea.first, tokens) + (last < int32_t(tokens) ? tokens - uint32_t(max(last, int32_t(min(ea.first, tokens)))) : 0u);
    if (!whole) {
        stored = anyway = 0u;
        for (uint32_t j = tid; j < tokens; j += kScanThreads)
            if (is_stored(j)) {
                ++stored;
                anyway += is_kept_anyway(j);
            }
        scan(stored, waves, turn, &total);
        turn ^= 1u;
        stored = total;
        scan(anyway, waves, turn, &total);
        turn ^= 1u;
        anyway = total;
    }
    const uint32_t stays = stored < ea.keep ? stored : ea.keep;
    // of a thread's tokens: stored ones that are kept anyway, and the others, a bit each
    uint32_t sure_bits = 0u, open_bits = 0u;
    if (held_here) {
#pragma unroll
        for (uint32_t e = 0; e < kHeld; ++e)
            if (e < each && mine + e < tokens && is_stored(mine + e)) (is_kept_anyway(mine + e) ? sure_bits : open_bits) |= 1u << e;
    }
    // the smallest weight that is taken, and how many tokens of it; all of them where no choice is to be made
    uint32_t least = 0u, ties = ~0u;
    if (stays < stored) {
        uint32_t take = stays - anyway;
        least = ~0u;
        ties = 0u;
        if (take) {
            uint32_t prefix = 0u;
            for (uint32_t digit = 0; digit < kDigits; ++digit) {
                const uint32_t shift = digit == 0u ? 32u : digit == 1u ? 21u : 10u;
                for (uint32_t k = tid; k < kBins; k += kScanThreads) bins[k] = 0u;
                __syncthreads();
                auto count = [&](float weight) __attribute__((always_inline)) {
                    const uint32_t u = ordered(weight);
                    if (digit == 0u || u >> shift == prefix) atomicAdd(&bins[digit_of(u, digit)], 1u);
                };
                if (held_here) {
#pragma unroll
                    for (uint32_t e = 0; e < kHeld; ++e)
                        if (open_bits >> e & 1u) count(w[e]);
                } else {
                    for (uint32_t j = tid; j < tokens; j += kScanThreads)
                        if (is_stored(j) && !is_kept_anyway(j)) count(weights[j]);
                }
                __syncthreads();
                // counts from the greatest digit down: a thread has two
                const uint32_t high = kBins - 1u - 2u * tid, n0 = bins[high], n1 = bins[high - 1u];
                const uint32_t above = scan(n0 + n1, waves, turn, &total);
                turn ^= 1u;
                if (above < take && take <= above + n0) { found[0] = high; found[1] = above; }
                else if (above + n0 < take && take <= above + n0 + n1) { found[0] = high - 1u; found[1] = above + n0; }
                __syncthreads();
                prefix = digit == 0u ? found[0] : digit == 1u ? prefix << 11 | found[0] : prefix << 10 | found[0];
                take -= found[1];
                __syncthreads();
            }
            least = prefix;
            ties = take;
        }
    }
    // in the tokens' order
    auto keep = [&](uint32_t at, uint32_t j, float weight) __attribute__((always_inline)) {
        ea.kept[out + at] = int32_t(j);
        ea.kept_weights[out + at] = weight;
    };
    if (held_here) {
        uint32_t tie_bits = 0u;
#pragma unroll
        for (uint32_t e = 0; e < kHeld; ++e)
            if (open_bits >> e & 1u) {
                const uint32_t u = ordered(w[e]);
                if (u > least) sure_bits |= 1u << e;
                else if (u == least) tie_bits |= 1u << e;
            }
        // (both counts in a word: there are 16384 at most)
        const uint32_t both = scan(uint32_t(__popc(sure_bits)) | uint32_t(__popc(tie_bits)) << 16, waves, turn, &total);
        uint32_t sure = both & 0xFFFFu, tie = both >> 16;
#pragma unroll
        for (uint32_t e = 0; e < kHeld; ++e) {
            const bool is_sure = sure_bits >> e & 1u, is_tie = tie_bits >> e & 1u;
            if (is_sure || (is_tie && tie < ties)) keep(sure + min(tie, ties), mine + e, w[e]);
            sure += is_sure;
            tie += is_tie;
        }
    } else {
        uint32_t before = 0u, equal = 0u;
        for (uint32_t j0 = 0; j0 < tokens; j0 += kScanThreads) {
            const uint32_t j = j0 + tid;
            bool sure = false, tie = false;
            float weight = 0.f;
            if (j < tokens && is_stored(j)) {
                weight = weights[j];
                const uint32_t u = ordered(weight);
                sure = is_kept_anyway(j) || u > least;
                tie = !sure && u == least;
            }
            // (both counts in a word: a workgroup has 1024 tokens)
            const uint32_t both = scan(uint32_t(sure) | uint32_t(tie) << 16, waves, turn, &total);
            turn ^= 1u;
            const uint32_t ties_before = equal + (both >> 16);
            if (sure || (tie && ties_before < ties)) keep(before + (both & 0xFFFFu) + min(ties_before, ties), j, weight);
            before += total & 0xFFFFu;
            equal += total >> 16;
        }
    }
    for (uint32_t k = stays + tid; k < ea.keep; k += kScanThreads) ea.kept[out + k] = -1;
}

template <uint32_t kHeld>
__global__ __launch_bounds__(kScanThreads, kHeld <= 8u ? 8 : 4) void evict_choose_kernel(const PoolArgs pa, const EvictArgs ea)
{
    if (blockIdx.x < ea.n) evict_plan(pa, ea, blockIdx.x);
    else evict_choose<kHeld>(pa, ea, blockIdx.x - ea.n);
}

constexpr uint32_t kMoveThreads = 256u, kMoveAtOnce = 4u;

// Keys or values of a layer, an entry and a head, a share of them: columns (in place) or tokens, as only what a workgroup has all tokens of can be rewritten in place.
template <class U>
__device__ void evict_move(const PoolArgs &pa, const EvictArgs &ea, uint32_t row, uint32_t head, uint32_t values, uint32_t share, uint32_t shares)
{
    const uint32_t layer = row / ea.n, i = row - layer * ea.n, tid = threadIdx.x;
    const EvictEntry e = *entry_of(ea, i);
    const uint32_t units = pa.token_bytes / uint32_t(sizeof(U)), tokens = uint32_t(e.tokens);
    uint32_t column0 = 0u, column1 = units, token0 = 0u, token1 = tokens;
    if (e.in_place) {
        column0 = uint32_t(uint64_t(units) * share / shares);
        column1 = uint32_t(uint64_t(units) * (share + 1u) / shares);
    } else {
        token0 = uint32_t(uint64_t(tokens) * share / shares);
        token1 = uint32_t(uint64_t(tokens) * (share + 1u) / shares);
    }
    const int32_t *const kept = ea.kept + (size_t(row) * pa.heads + head) * ea.keep, *const from_row = ea.rows + size_t(i) * pa.table_pages, *const to_row = ea.to + size_t(i) * ea.keep_pages;
    char *const base = (values ? pa.values : pa.keys) + int64_t(layer) * pa.layer_bytes;
    auto slot = [&](uint32_t page, uint32_t in_page) __attribute__((always_inline)) {
        const uint64_t n = pa.heads_first ? uint64_t(head) * pa.page_tokens.d + in_page : uint64_t(in_page) * pa.heads + head;
        return base + int64_t(page) * pa.page_bytes + int64_t(n * pa.token_bytes);
    };
    for (uint32_t column = column0; column < column1; column += kMoveThreads) {
        const uint32_t width = column1 - column < kMoveThreads ? column1 - column : kMoveThreads, each = kMoveThreads / width;      // tokens side by side
        const uint32_t mine = tid / width, c = column + tid - mine * width;
        const bool works = mine < each;
        for (uint32_t k0 = token0; k0 < token1; k0 += kMoveAtOnce * each) {
            U v[kMoveAtOnce];
            char *to[kMoveAtOnce];
#pragma unroll
            for (uint32_t k = 0; k < kMoveAtOnce; ++k) {
                const uint32_t n = k0 + k * each + mine;
                to[k] = nullptr;
                if (!works || n >= token1) continue;
                const uint32_t j = uint32_t(kept[n]), place = pa.page_tokens.quotient(j), to_place = pa.page_tokens.quotient(n);
                const char *const source = slot(uint32_t(from_row[place]), j - place * pa.page_tokens.d);
                int32_t page = to_row[to_place];
                if (page < 0) page = ea.free[e.at + (-1 - page)];
                char *const target = slot(uint32_t(page), n - to_place * pa.page_tokens.d);
                if (target == source) continue;
                to[k] = target + size_t(c) * sizeof(U);
                v[k] = *reinterpret_cast<const U *>(source + size_t(c) * sizeof(U));
            }
            if (e.in_place) {
                // (every thread's loads have come before any thread stores)
                __builtin_amdgcn_s_waitcnt(0);
                __syncthreads();
            }
#pragma unroll
            for (uint32_t k = 0; k < kMoveAtOnce; ++k)
                if (to[k]) __builtin_nontemporal_store(v[k], reinterpret_cast<U *>(to[k]));
        }
    }
}

// Workgroups n and on move: of every layer, entry and head, `shares` keys, `shares` values and one the weights.  Workgroup i < n: entry i's row of the table and references.
template <class U>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(const PoolArgs pa, const EvictArgs ea, const uint32_t shares)
{
    if (blockIdx.x < ea.n) {
        const uint32_t i = blockIdx.x, child = child_of(pa, ea, i), parent = parent_of(pa, ea, i);
        const EvictEntry e = *entry_of(ea, i);
        if (parent == kIdxMax || child == kIdxMax || e.tokens < 0) return;
        const uint32_t pages = pages_for(pa, e.tokens);
        for (uint32_t p = threadIdx.x; p < pa.table_pages; p += kMoveThreads) {
            int32_t &at = pa.table[size_t(child) * pa.table_pages + p];
            const uint32_t old = uint32_t(at);
            int32_t now = -1;
            if (p < pages) {
                now = ea.to[size_t(i) * ea.keep_pages + p];
                if (now < 0) now = ea.free[e.at + (-1 - now)];
            }
            if (old < pa.pages) atomicAdd(pa.references + old, -1);
            if (now >= 0) atomicAdd(pa.references + now, 1);
            at = now;
        }
        if (threadIdx.x == 0u) pa.lengths[child] = e.tokens;
        return;
    }
    const uint32_t number = blockIdx.x - ea.n, parts = 2u * shares + 1u, cell = number / parts, part = number - cell * parts;
    const uint32_t row = cell / pa.heads, head = cell - row * pa.heads, layer = row / ea.n, i = row - layer * ea.n;
    const uint32_t child = child_of(pa, ea, i), parent = parent_of(pa, ea, i);
    const int32_t tokens = entry_of(ea, i)->tokens;
    if (parent == kIdxMax || child == kIdxMax || tokens < 0) return;
    if (part < 2u * shares) {
        evict_move<U>(pa, ea, row, head, part / shares, part % shares, shares);
        return;
    }
    float *const to = ea.weights + int64_t(layer) * ea.weights_layer + int64_t(child) * ea.weights_sequence + int64_t(head) * ea.weights_head;
    const float *const from = ea.kept_weights + (size_t(row) * pa.heads + head) * ea.keep;
    const uint64_t places = uint64_t(pa.table_pages) * pa.page_tokens.d;
    for (uint64_t k = threadIdx.x; k < places; k += kMoveThreads) to[k] = k < uint64_t(tokens) ? from[k] : 0.f;
}

}  // namespace

hipError_t launch_evict(const PoolArgs &pa, const EvictArgs &ea, hipStream_t s)
{
    const uint64_t cells = uint64_t(ea.n) * pa.layers * pa.heads;
    // (two workgroups a compute unit where eight tokens a thread are enough; us, eight / sixteen: 12 prompts of up to 8000 213 / 224, 700 tokens 14.5 / 17.4)
    if (uint64_t(pa.table_pages) * pa.page_tokens.d <= 8u * kScanThreads) evict_choose_kernel<8u><<<dim3(uint32_t(ea.n + cells)), dim3(kScanThreads), 0, s>>>(pa, ea);
    else evict_choose_kernel<16u><<<dim3(uint32_t(ea.n + cells)), dim3(kScanThreads), 0, s>>>(pa, ea);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    const uint32_t shares = evict_shares(pa, cells);
    by_unit(pa, [&](auto u) { evict_move_kernel<decltype(u)><<<dim3(uint32_t(ea.n + cells * (2u * shares + 1u))), dim3(kMoveThreads), 0, s>>>(pa, ea, shares); });
    return hipGetLastError();
}

}  // namespace hspmm
