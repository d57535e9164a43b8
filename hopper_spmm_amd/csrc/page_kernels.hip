// Work on the pages of a cache: giving out, sharing, releasing, moving and copying them.  What decides is integers - the
// table, lengths and references -, what takes time is the pages' bytes, each read and written once, all layers in one launch.  us: 476 pages of 2 MB
// moved 382, 5.2 TB/s (a large copy: 4.8); 192 beams of partly filled pages, all of 32 layers, 57 for 284 MB, 5.0 TB/s; a token more for 64 sequences 4.4, freeing
// them 4.8; small forks and compactions 10, which is two launches, as which pages are free has to be known before one is written: what is decided cannot be decided again by every workgroup that copies
// while others change the table and the references.
#include "pages_common.hpp"
#include <algorithm>

namespace hspmm {

namespace {

// Copies `bytes` (a multiple of the unit) by `threads` threads, four units of each on their way at a time.  Nothing that is written is read again in the
// launch, and of whole pages nothing is read twice either: past the L2 (a pool of 2048 pages of 2 MB, 476 of them moved, 402 -> 389 us, 5.1 TB/s).  A partly
// filled page may be several children's (shared): its loads stay (48 x 4 beams, all layers, 72 -> 68 us).
template <class U, bool Shared>
__device__ __forceinline__ void copy_run(char *to, const char *from, uint32_t bytes, uint32_t thread, uint32_t threads)
{
    constexpr uint32_t kAtOnce = 4u;
    const uint32_t n = bytes / sizeof(U);
    for (uint32_t i = thread; i < n; i += kAtOnce * threads) {
        U v[kAtOnce];
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k)
            if (i + k * threads < n) {
                const U *at = reinterpret_cast<const U *>(from) + i + k * threads;
                v[k] = Shared ? *at : __builtin_nontemporal_load(at);
            }
#pragma unroll
        for (uint32_t k = 0; k < kAtOnce; ++k)
            if (i + k * threads < n) __builtin_nontemporal_store(v[k], reinterpret_cast<U *>(to) + i + k * threads);
    }
}

// The first `tokens` tokens of a page of one layer's keys or values.
template <class U>
__device__ __forceinline__ void copy_tokens(const PoolArgs &pa, uint32_t part, uint32_t to, uint32_t from, uint32_t tokens, uint32_t head0, uint32_t head1)
{
    const int64_t layer = int64_t(part >> 1) * pa.layer_bytes;
    char *base = (part & 1u ? pa.values : pa.keys) + layer;
    char *d = base + int64_t(to) * pa.page_bytes;
    const char *s = base + int64_t(from) * pa.page_bytes;
    if (tokens == pa.page_tokens.d && head0 == 0u && head1 == pa.heads) {
        copy_run<U, false>(d, s, tokens * pa.heads * pa.token_bytes, threadIdx.x, blockDim.x);
    } else if (!pa.heads_first) {
        if (head0 == 0u) copy_run<U, true>(d, s, tokens * pa.heads * pa.token_bytes, threadIdx.x, blockDim.x);
    } else {
        // a head's tokens lie side by side: a wave has a head at a time
        const uint32_t pitch = pa.page_tokens.d * pa.token_bytes, waves = blockDim.x / 64u;
        for (uint32_t h = head0 + threadIdx.x / 64u; h < head1; h += waves)
            copy_run<U, true>(d + size_t(h) * pitch, s + size_t(h) * pitch, tokens * pa.token_bytes, threadIdx.x & 63u, 64u);
    }
}

// One workgroup: pages for more tokens.  scratch: the first request of every list entry, then the free pages.
__global__ __launch_bounds__(kScanThreads) void pages_extend_kernel(const PoolArgs pa, const uint32_t n, const int32_t *rows, const int32_t *add, int32_t *status)
{
    __shared__ uint32_t waves[2u * kScanWaves];
    __shared__ unsigned long long past;                        // pages that no row has a place for
    const Eight ahead = load_references(pa.references, pa.pages, threadIdx.x * kEach);
    int32_t *const first = pa.scratch, *const list = pa.scratch + pa.sequences;
    uint32_t need = 0u, turn = 0u;
    if (threadIdx.x == 0u) past = 0u;
    __syncthreads();
    for (uint32_t i0 = 0; i0 < n; i0 += kScanThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const uint32_t row = i < n ? row_of(pa, rows, i) : kIdxMax;
        uint32_t mine = 0u;
        if (row != kIdxMax) {
            const int32_t have = held(pa, row), now = extended(have, add[i]);
            mine = places_for(pa, now) - places_for(pa, have);
            const uint32_t all = pages_for(pa, now) - pages_for(pa, have);
            if (all > mine) atomicAdd(&past, static_cast<unsigned long long>(all - mine));
        }
        uint32_t total;
        const uint32_t at = need + scan(mine, waves, turn, &total);
        turn ^= 1u;
        if (i < n) first[i] = int32_t(at);
        need += total;
    }
    const uint32_t found = find_free(pa.references, pa.pages, need < pa.pages ? need : pa.pages, list, waves, turn, ahead);
    __syncthreads();
    for (uint32_t i = threadIdx.x / 64u; i < n; i += kScanWaves) {
        const uint32_t row = row_of(pa, rows, i);
        if (row == kIdxMax) continue;
        const int32_t have = held(pa, row), now = extended(have, add[i]);
        const uint32_t p0 = places_for(pa, have), p1 = places_for(pa, now), at = uint32_t(first[i]);
        for (uint32_t p = p0 + (threadIdx.x & 63u); p < p1; p += 64u) {
            const uint32_t k = at + p - p0;
            const int32_t id = k < found ? list[k] : -1;
            pa.table[size_t(row) * pa.table_pages + p] = id;
            if (id >= 0) pa.references[id] = 1;
        }
        if ((threadIdx.x & 63u) == 0u) pa.lengths[row] = now;
    }
    if (status && threadIdx.x == 0u) {
        const unsigned long long missing = past + (need - found);
        *status = missing > 0x7FFFFFFFu ? 0x7FFFFFFF : int32_t(missing);
    }
}

// Fork, first launch: what the second needs to know of the state before the call.  Workgroup 0 finds the new pages; workgroup 1 + i keeps
// the parent's row of entry i.  scratch: per entry the new page, the parent's last page, the parent's tokens; free pages; rows.
struct ForkScratch { int32_t *page, *from, *tokens, *list, *rows; };
__device__ __forceinline__ ForkScratch fork_scratch(const PoolArgs &pa)
{
    int32_t *s = pa.scratch;
    return ForkScratch{s, s + pa.sequences, s + 2u * pa.sequences, s + 3u * pa.sequences, s + 4u * size_t(pa.sequences)};
}
constexpr uint32_t kForkRows = 32768u;          // entries along y of the second launch
__device__ __forceinline__ bool fork_takes_page(const PoolArgs &pa, uint32_t parent, uint32_t child, int32_t tokens)
{
    const uint32_t full = pa.page_tokens.quotient(uint32_t(tokens));
    return parent != kIdxMax && child != kIdxMax && parent != child && full < pa.table_pages && uint32_t(tokens) != full * pa.page_tokens.d;
}

__global__ __launch_bounds__(kScanThreads) void pages_fork_kernel(const PoolArgs pa, const uint32_t n, const int32_t *parents, const int32_t *children, int32_t *status)
{
    const ForkScratch fs = fork_scratch(pa);
    if (blockIdx.x > 0u) {
        const uint32_t i = blockIdx.x - 1u, parent = row_of(pa, parents, i);
        if (parent == kIdxMax) return;
        const uint32_t used = places_for(pa, held(pa, parent));
        for (uint32_t p = threadIdx.x; p < used; p += kScanThreads) fs.rows[size_t(i) * pa.table_pages + p] = pa.table[size_t(parent) * pa.table_pages + p];
        return;
    }
    __shared__ uint32_t waves[2u * kScanWaves];
    const Eight ahead = load_references(pa.references, pa.pages, threadIdx.x * kEach);
    uint32_t need = 0u, turn = 0u;
    for (uint32_t i0 = 0; i0 < n; i0 += kScanThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const uint32_t parent = i < n ? row_of(pa, parents, i) : kIdxMax, child = i < n ? row_of(pa, children, i) : kIdxMax;
        const int32_t tokens = parent != kIdxMax ? held(pa, parent) : 0;
        // (a last page that the parent lacks the child lacks, too: a page of its own would show what its last owner left there)
        const int32_t last = fork_takes_page(pa, parent, child, tokens) ? pa.table[size_t(parent) * pa.table_pages + pages_for(pa, tokens) - 1u] : -1;
        const bool takes = uint32_t(last) < pa.pages;
        uint32_t total;
        const uint32_t at = need + scan(takes, waves, turn, &total);
        turn ^= 1u;
        if (i < n) {
            fs.page[i] = takes ? int32_t(at) : -1;
            fs.tokens[i] = tokens;
            fs.from[i] = last;
        }
        need += total;
    }
    const uint32_t found = find_free(pa.references, pa.pages, need, fs.list, waves, turn, ahead);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kScanThreads) {
        const int32_t k = fs.page[i];
        if (k >= 0) fs.page[i] = uint32_t(k) < found ? fs.list[k] : -1;
    }
    if (status && threadIdx.x == 0u) *status = int32_t(need - found);
}

// Second launch: workgroup (part, i): part 0 entry i's row and references, the others copy its last page's tokens.  (An entry's parts follow each other:
// workgroups go to the eight L2 domains in turn, and where every fourth entry is its own parent, entries in turn would leave two of them with nothing.)
template <class U>
__global__ __launch_bounds__(256) void pages_fork_copy_kernel(const PoolArgs pa, const uint32_t n, const int32_t *parents, const int32_t *children, const uint32_t heads_each, const uint32_t head_parts)
{
    const ForkScratch fs = fork_scratch(pa);
    const uint32_t i = blockIdx.z * kForkRows + blockIdx.y;
    if (i >= n) return;
    const uint32_t parent = row_of(pa, parents, i), child = row_of(pa, children, i);
    if (parent == kIdxMax || child == kIdxMax || parent == child) return;
    const int32_t tokens = fs.tokens[i], page = fs.page[i];
    const uint32_t full = pa.page_tokens.quotient(uint32_t(tokens)), rest = uint32_t(tokens) - full * pa.page_tokens.d;
    if (blockIdx.x == 0u) {
        for (uint32_t p = threadIdx.x; p < pa.table_pages; p += blockDim.x) {
            int32_t &at = pa.table[size_t(child) * pa.table_pages + p];
            const uint32_t old = uint32_t(at);
            const int32_t now = p < full ? fs.rows[size_t(i) * pa.table_pages + p] : p == full && rest ? page : -1;
            if (old < pa.pages) atomicAdd(pa.references + old, -1);
            if (uint32_t(now) < pa.pages) atomicAdd(pa.references + now, 1);
            at = now;
        }
        if (threadIdx.x == 0u) pa.lengths[child] = tokens;
        return;
    }
    const uint32_t from = uint32_t(fs.from[i]), part = (blockIdx.x - 1u) / head_parts, h0 = (blockIdx.x - 1u) % head_parts * heads_each;
    if (!rest || uint32_t(page) >= pa.pages || from >= pa.pages) return;
    copy_tokens<U>(pa, part, uint32_t(page), from, rest, h0, h0 + heads_each < pa.heads ? h0 + heads_each : pa.heads);
}

__global__ __launch_bounds__(256) void pages_free_kernel(const PoolArgs pa, const int32_t *rows)
{
    const uint32_t row = row_of(pa, rows, blockIdx.x);
    if (row == kIdxMax) return;
    for (uint32_t p = threadIdx.x; p < pa.table_pages; p += blockDim.x) {
        int32_t &at = pa.table[size_t(row) * pa.table_pages + p];
        if (uint32_t(at) < pa.pages) atomicAdd(pa.references + at, -1);
        at = -1;
    }
    if (threadIdx.x == 0u) pa.lengths[row] = 0;
}

// Compact, first launch, one workgroup: the live pages' number, and which goes where.  scratch: number, pages that move; per
// page from that number on which of those that move it is, -1: a free one; from; to.
struct CompactScratch { int32_t *count, *map, *from, *to; };
__device__ __forceinline__ CompactScratch compact_scratch(const PoolArgs &pa)
{
    int32_t *s = pa.scratch;
    return CompactScratch{s, s + 2, s + 2 + pa.pages, s + 2 + 2u * size_t(pa.pages)};
}

__global__ __launch_bounds__(kScanThreads) void pages_compact_kernel(const PoolArgs pa, int32_t *live_out)
{
    __shared__ uint32_t waves[2u * kScanWaves], below_live;
    const CompactScratch cs = compact_scratch(pa);
    uint32_t live = 0u, turn = 0u, at = 0u;
    Eight v;
    auto look = [&](uint32_t p0) {
        const uint32_t p = p0 + threadIdx.x * kEach;
        v = load_references(pa.references, pa.pages, p);
        uint32_t count = 0u, total;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) count += p + e < pa.pages && v.r[e] > 0;
        at = scan(count, waves, turn, &total);
        turn ^= 1u;
        return total;
    };
    for (uint32_t p0 = 0; p0 < pa.pages; p0 += kScanThreads * kEach) live += look(p0);
    // Of a page below their number that is free, and of a live one at or above it, the number is the live pages' in front of it, up to a constant.
    // (The references of a pool of one round are in registers.)
    const bool once = pa.pages <= kScanThreads * kEach;
    uint32_t before = 0u;
    for (uint32_t p0 = 0; p0 < pa.pages; p0 += kScanThreads * kEach) {
        const uint32_t total = once ? live : look(p0), p = p0 + threadIdx.x * kEach;
        at += before;
        before += total;
        if (p <= live && live < p + kEach) {
            uint32_t below = at;
#pragma unroll
            for (uint32_t e = 0; e < kEach; ++e) below += p + e < live && v.r[e] > 0;
            below_live = below;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) {
            if (p + e >= pa.pages) continue;
            if (p + e >= live) {
                if (v.r[e] > 0) cs.from[at - below_live] = int32_t(p + e);
                cs.map[p + e] = v.r[e] > 0 ? int32_t(at - below_live) : -1;
            } else if (v.r[e] <= 0) {
                cs.to[p + e - at] = int32_t(p + e);
            }
            at += v.r[e] > 0;
        }
    }
    const uint32_t from = live < pa.pages ? live - below_live : 0u;
    if (threadIdx.x == 0u) {
        cs.count[0] = int32_t(live);
        cs.count[1] = int32_t(from);
        if (live_out) *live_out = int32_t(live);
    }
}

// Second launch: pages, the table, references.
template <class U>
__global__ __launch_bounds__(256) void pages_compact_copy_kernel(const PoolArgs pa, int32_t *table_out, int32_t *references_out)
{
    const CompactScratch cs = compact_scratch(pa);
    const uint32_t live = uint32_t(cs.count[0]), moved = uint32_t(cs.count[1]), parts = pa.layers * 2u;
    const uint64_t tasks = uint64_t(moved) * parts;
    for (uint64_t k = blockIdx.x; k < tasks; k += gridDim.x) {
        const uint32_t m = uint32_t(k / parts), part = uint32_t(k - uint64_t(m) * parts);
        copy_tokens<U>(pa, part, uint32_t(cs.to[m]), uint32_t(cs.from[m]), pa.page_tokens.d, 0u, pa.heads);
    }
    const uint64_t thread = uint64_t(blockIdx.x) * 256u + threadIdx.x, threads = uint64_t(gridDim.x) * 256u, places = uint64_t(pa.sequences) * pa.table_pages;
    for (uint64_t i = thread; i < places; i += threads) {
        const int32_t id = pa.table[i];
        const int32_t m = uint32_t(id) < pa.pages && uint32_t(id) >= live ? cs.map[id] : -1;
        table_out[i] = m >= 0 ? cs.to[m] : id;
    }
    for (uint64_t i = thread; i < pa.pages; i += threads) {
        // (in place, a page that stays keeps its count; the counts of those that move are read by their own thread alone)
        if (references_out != pa.references) {
            const int32_t count = pa.references[i];
            if (i < live ? count > 0 : count <= 0) references_out[i] = i < live ? count : 0;
        }
        if (i < moved) {
            const int32_t from = cs.from[i], count = pa.references[from];
            references_out[cs.to[i]] = count;
            references_out[from] = 0;
        }
    }
}

template <class U>
__global__ __launch_bounds__(256) void pages_copy_kernel(const PoolArgs pa, const int32_t *from, const int32_t *to)
{
    const uint32_t f = uint32_t(from[blockIdx.x]), t = uint32_t(to[blockIdx.x]);
    if (f >= pa.pages || t >= pa.pages || f == t) return;
    copy_tokens<U>(pa, blockIdx.y, t, f, pa.page_tokens.d, 0u, pa.heads);
}

}  // namespace

hipError_t launch_pages_extend(const PoolArgs &pa, uint32_t n, const int32_t *rows, const int32_t *add, int32_t *status, hipStream_t s)
{
    pages_extend_kernel<<<dim3(1), dim3(kScanThreads), 0, s>>>(pa, n, rows, add, status);
    return hipGetLastError();
}

hipError_t launch_pages_fork(const PoolArgs &pa, uint32_t n, const int32_t *parents, const int32_t *children, int32_t *status, hipStream_t s)
{
    pages_fork_kernel<<<dim3(n + 1u), dim3(kScanThreads), 0, s>>>(pa, n, parents, children, status);
    // (nothing is copied by what a launch that failed has not written; for a list of nothing there is the status alone)
    if (const hipError_t e = hipGetLastError(); e != hipSuccess || n == 0u) return e;
    // heads of a page are shared out while that leaves fewer than some thousand workgroups
    const uint64_t groups = uint64_t(n) * pa.layers * 2u;
    uint32_t parts = pa.heads_first && groups < 2048u ? uint32_t(2048u / groups) : 1u;
    if (parts > pa.heads) parts = pa.heads;
    const uint32_t each = (pa.heads + parts - 1u) / parts;
    parts = (pa.heads + each - 1u) / each;
    by_unit(pa, [&](auto u) {
        pages_fork_copy_kernel<decltype(u)><<<dim3(1u + pa.layers * 2u * parts, std::min(n, kForkRows), (n + kForkRows - 1u) / kForkRows), dim3(256), 0, s>>>(pa, n, parents, children, each, parts);
    });
    return hipGetLastError();
}

hipError_t launch_pages_free(const PoolArgs &pa, uint32_t n, const int32_t *rows, hipStream_t s)
{
    pages_free_kernel<<<dim3(n), dim3(256), 0, s>>>(pa, rows);
    return hipGetLastError();
}

hipError_t launch_pages_compact(const PoolArgs &pa, int32_t *table_out, int32_t *references_out, int32_t *live, hipStream_t s)
{
    pages_compact_kernel<<<dim3(1), dim3(kScanThreads), 0, s>>>(pa, live);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    const uint64_t most = uint64_t(pa.pages) * pa.layers;          // (at most half of the pages move)
    by_unit(pa, [&](auto u) {
        pages_compact_copy_kernel<decltype(u)><<<dim3(uint32_t(most < 4096u ? most : 4096u)), dim3(256), 0, s>>>(pa, table_out, references_out);
    });
    return hipGetLastError();
}

hipError_t launch_pages_copy(const PoolArgs &pa, uint32_t n, const int32_t *from, const int32_t *to, hipStream_t s)
{
    by_unit(pa, [&](auto u) { pages_copy_kernel<decltype(u)><<<dim3(n, pa.layers * 2u), dim3(256), 0, s>>>(pa, from, to); });
    return hipGetLastError();
}

}  // namespace hspmm
