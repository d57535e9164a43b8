// The rows kernel's part of attention: a few rows of queries - single new tokens, and the heads that share their keys - over the pages of a cache.
#pragma once
#include "attend_common.hpp"

namespace hspmm {

namespace {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// A tile's keys and values in a wave's registers, and the two products.  kKeys keys at a time; a lane (g, i) = (lane / 16, lane % 16).
//   scores: S^T = K Q^T by matrix instructions of 16 keys x 16 rows; register r of part t: key 16 t + 4 g + r, row i
//   sums:   O^T = V^T P^T, 16 elements x 16 rows at a time: the scores' registers are the second operand as they are, once keys are taken in
//           the order the lanes hold them; the first operand wants a lane's keys side by side per element
// 16-bit types: a lane loads pieces of eight elements (head_dim up to 64: four) of eight keys, 4 g .. + 3 of either part: an 8 x 8 block which 32
// byte permutations transpose.  Elements of an operand's 16 rows are kPiece apart: kPiece i + dt.  Nothing goes through LDS.
template <bool BF, int DP, bool Past>
struct Rows16 {
    typedef typename HalfOps<BF>::elem_t T;
    static constexpr int kKeys = 32, kParts = 2, kElem = 2, kPiece = DP >= 128 ? 8 : 4, kSteps = DP / 32, kBlocks = DP / (16 * kPiece), kTiles = DP / 16;
    u32x4 k[kParts][kSteps];
    uint32_t v[8][kBlocks][kPiece / 2];
    struct Query { u32x4 q[kSteps]; };

    __device__ static __forceinline__ void load_query(Query &Q, const char *row, bool there, uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = 32u * s + 8u * (lane >> 4);
            Q.q[s] = there && d < D ? *reinterpret_cast<const u32x4 *>(row + d * 2u) : u32x4{0u, 0u, 0u, 0u};
        }
    }
    // Past: not kept in the L2.
    template <class P> __device__ static __forceinline__ P fetch(const char *p)
    {
        if constexpr (Past) return __builtin_nontemporal_load(reinterpret_cast<const P *>(p));
        else return *reinterpret_cast<const P *>(p);
    }
    // Key 16 t + i, by its offset.
    __device__ __forceinline__ void load_keys(int t, const char *keys, int64_t at, uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = 32u * s + 8u * (lane >> 4);
            k[t][s] = fetch<u32x4>(keys + (at + (d < D ? d : 0u)) * 2);
        }
    }
    __device__ __forceinline__ void load_values(int t, int r, const char *values, int64_t at, uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const uint32_t d = uint32_t(16 * kPiece * b) + uint32_t(kPiece) * (lane & 15u);
            const char *p = values + (at + (d < D ? d : 0u)) * 2;
            uint32_t *to = v[4 * t + r][b];
            if constexpr (kPiece == 8) {
                const u32x4 x = fetch<u32x4>(p);
                to[0] = x[0]; to[1] = x[1]; to[2] = x[2]; to[3] = x[3];
            } else {
                const t_u32x2 x = fetch<t_u32x2>(p);
                to[0] = x[0]; to[1] = x[1];
            }
        }
    }
    // elements behind the last one
    __device__ __forceinline__ void clear_keys(uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int t = 0; t < kParts; ++t)
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                if (32u * s + 8u * (lane >> 4) >= D) k[t][s] = u32x4{0u, 0u, 0u, 0u};
    }
    // keys that are not stored
    __device__ __forceinline__ void clear_values(uint32_t stored)
    {
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int n = 0; n < kPiece / 2; ++n) v[r][b][n] = stored >> (16 * (r / 4) + r % 4) & 1u ? v[r][b][n] : 0u;
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
    __device__ __forceinline__ void add(const f32x4 (&p)[kParts], f32x4 (&o)[kTiles]) const
    {
        u32x4 w;
#pragma unroll
        for (int t = 0; t < kParts; ++t) {
            w[2 * t] = pack_two<BF>(p[t][0], p[t][1]);
            w[2 * t + 1] = pack_two<BF>(p[t][2], p[t][3]);
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                u32x4 a;
#pragma unroll
                for (int n = 0; n < 4; ++n) a[n] = __builtin_amdgcn_perm(v[2 * n + 1][b][e / 2], v[2 * n][b][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
                o[b * kPiece + e] = HalfOps<BF>::mfma(a, w, o[b * kPiece + e]);
            }
    }
    __device__ __forceinline__ bool not_finite() const
    {
        bool f = false;
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int n = 0; n < kPiece / 2; ++n) f |= word_not_finite<BF>(v[r][b][n]);
        return f;
    }
    // this tile with the values of key `a` alone
    __device__ __forceinline__ Rows16 only(uint32_t a, uint32_t g) const
    {
        Rows16 x = *this;
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int n = 0; n < kPiece / 2; ++n) x.v[r][b][n] = a == uint32_t(16 * (r / 4) + r % 4) + 4u * g ? v[r][b][n] : 0u;
        return x;
    }
};

// fp32: 16 keys at a time, products in fp32 (four keys or elements a matrix instruction).  Scores: element 16 s + 4 g + e is step (s, e)'s.  Sums: step r takes
// keys 4 g + r, which register r of the scores holds; a lane's pieces of four elements are the first operands of four instructions.
template <int DP>
struct Rows32 {
    typedef float T;
    static constexpr int kKeys = 16, kParts = 1, kElem = 4, kPiece = 4, kSteps = DP / 16, kBlocks = DP / 64, kTiles = DP / 16;
    f32x4 k[kSteps];
    f32x4 v[4][kBlocks];
    struct Query { f32x4 q[kSteps]; };
    __device__ static __forceinline__ void load_query(Query &Q, const char *row, bool there, uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = 16u * s + 4u * (lane >> 4);
            Q.q[s] = there && d < D ? *reinterpret_cast<const f32x4 *>(row + d * 4u) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ void load_keys(int, const char *keys, int64_t at, uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = 16u * s + 4u * (lane >> 4);
            k[s] = *reinterpret_cast<const f32x4 *>(keys + (at + (d < D ? d : 0u)) * 4);
        }
    }
    __device__ __forceinline__ void load_values(int, int r, const char *values, int64_t at, uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const uint32_t d = 64u * b + 4u * (lane & 15u);
            v[r][b] = *reinterpret_cast<const f32x4 *>(values + (at + (d < D ? d : 0u)) * 4);
        }
    }
    __device__ __forceinline__ void clear_keys(uint32_t lane, uint32_t D)
    {
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
            if (16u * s + 4u * (lane >> 4) >= D) k[s] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void clear_values(uint32_t stored)
    {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[r][b][e] = stored >> r & 1u ? v[r][b][e] : 0.f;
    }
    __device__ __forceinline__ void scores(const Query &Q, f32x4 (&s)[1]) const
    {
        s[0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kSteps; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[c][e], Q.q[c][e], s[0], 0, 0, 0);
    }
    __device__ __forceinline__ void add(const f32x4 (&p)[1], f32x4 (&o)[kTiles]) const
    {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[b * 4 + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][b][e], p[0][r], o[b * 4 + e], 0, 0, 0);
    }
    __device__ __forceinline__ bool not_finite() const
    {
        bool f = false;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = v[r][b][e];                 // (a bit cast of a vector's element as such takes its first one)
                    f |= (~__builtin_bit_cast(uint32_t, x) & 0x7F800000u) == 0u;
                }
        return f;
    }
    __device__ __forceinline__ Rows32 only(uint32_t a, uint32_t g) const
    {
        Rows32 x = *this;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) x.v[r][b][e] = a == uint32_t(r) + 4u * g ? v[r][b][e] : 0.f;
        return x;
    }
};

constexpr int kRowWaves = 4;

// A workgroup has 16 rows and a part of their keys; its waves take tiles of keys in turn.  The waves' sums are added at the end in LDS, the parts'
// through memory.  Memory bounds it, as keys and values are read once for all heads that share them: one token for each of 48 sequences of up to 16000
// keys, 32 heads on 8 of 128 elements, bf16, 281 us for 1.62 GB, 5.8 TB/s (a large copy: 4.8, read and written).  Short sequences: three of up to 300 keys, fp32, 7.8 us,
// launch and a few dependent loads (starts, table, keys); 30000 keys of one sequence 31 us, 2^18 194, 5.5 TB/s.
// Registers for two workgroups a compute unit (three up to 64 elements): a wave has one tile on its way, 16 KB of keys and values.
// Whole: pages hold a multiple of 16 tokens, so 16 keys of a tile lie in one page, and a wave asks for its next tiles' page numbers 64 at a time;
// else every lane finds a key's row and hands it to the lanes that load it.
// lds: rows_lds(DP) bytes; number, part: of the workgroup.
constexpr uint32_t rows_lds(int DP) { return kRowWaves * 16u * (uint32_t(DP) + 4u + 2u) * 4u + 16u; }
template <class K, bool Whole, int DP, AttendSpan Span>
__device__ __forceinline__ void attend_rows(const AttendArgs &aa, char *lds, uint32_t number, uint32_t part)
{
    constexpr uint32_t kRows = 16u, kPitch = DP + 4u;
    float *const sums = reinterpret_cast<float *>(lds);
    float (*const refs)[kRows] = reinterpret_cast<float (*)[kRows]>(sums + kRowWaves * kRows * kPitch), (*const totals)[kRows] = refs + kRowWaves;
    uint32_t &arrived = *reinterpret_cast<uint32_t *>(totals + kRowWaves);
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, i = lane & 15u;
    const uint32_t D = aa.pages.head_dim;
    const Cell cell = cell_of(aa, number, part);
    const uint32_t head = cell.head;
    RowTile t = find_tile<4, Span>(aa, cell.tile);
    if (!t.there) return;
    constexpr int32_t kKeys = K::kKeys;
    // this part's keys
    const KeyPart keys_here = key_part(aa, t, part);
    constexpr bool kJoins = Span == kSpanAll || Span == kSpanBoth;
    const int32_t parts = kJoins ? keys_here.parts : 1, end = keys_here.end;
    int32_t begin = keys_here.begin;
    if (int32_t(part) >= keys_here.parts) return;

    const RowOf row = row_of_tile<Span>(aa, t, head, i);
    if constexpr (Span == kSpanPrefix) {
        // (rows of several sequences: from the first key that any of them sees)
        int32_t low = i < t.rows ? row.lo : 0x7FFFFFFF;
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) low = min(low, __shfl_xor(low, d));
        begin = max(begin, min(__builtin_amdgcn_readfirstlane(low) & ~31, end));
    }
    typename K::Query Q;
    K::load_query(Q, aa.q.data + (int64_t(row.token) * aa.q.token_stride + int64_t(row.head) * aa.q.head_stride) * K::kElem, i < t.rows, lane, D);
    const float scale = aa.scale * kLog2e;
    const int32_t *table = aa.pages.table + size_t(t.sequence) * aa.pages.table_pages, *const lead = aa.pages.table + size_t(Span == kSpanBoth ? t.leader : t.sequence) * aa.pages.table_pages;
    // (key by key, as a prefix may end within a group of 16)
    static_assert(Span != kSpanBoth || !Whole, "");
    const int64_t head_offset = int64_t(head) * aa.pages.head_stride;
    const char *keys = aa.pages.keys, *values = aa.pages.values;
    // keys that every row of the tile sees
    int32_t all_lo = row.lo, all_hi = i < t.rows ? row.hi : 0x7FFFFFFF;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        all_lo = max(all_lo, __shfl_xor(all_lo, d));
        all_hi = min(all_hi, __shfl_xor(all_hi, d));
    }
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);

    f32x4 o[K::kTiles];
#pragma unroll
    for (int c = 0; c < K::kTiles; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ref = -INFINITY, total = 0.f;

    const int32_t first = begin + int32_t(wave) * kKeys, step = kRowWaves * kKeys;
    const int32_t n_tiles = end > first ? (end - first + step - 1) / step : 0;

    // page numbers of this wave's next 64 / kParts tiles, a lane each (Whole), or offsets of a tile's keys (else)
    int32_t pages_ahead = -1;
    auto look_up_pages = [&](int32_t n) __attribute__((always_inline)) {
        const int32_t tile = n + int32_t(lane) / K::kParts, key = first + tile * step + int32_t(lane) % K::kParts * 16;
        pages_ahead = -1;
        if (tile < n_tiles && key < end) {
            const uint32_t place = aa.pages.page_tokens.quotient(uint32_t(key));
            if (place < aa.pages.table_pages) pages_ahead = table[place];
        }
        asm volatile("" : "+v"(pages_ahead));                  // (waited for here, not wherever it is used, with all that is on its way then)
    };
    K kv;
    // Every request is made, of what is not there for the pool's first row, and what came is cleared before it is used: the number of loads on their way is
    // the same on every path, so that a wait can leave the later ones alone.
    // Keys and values of a tile are asked for as soon as the registers are free: the keys after the scores of the tile in front, the values
    // after its sums.
    struct Place { int64_t at[K::kParts]; uint32_t stored; } now{}, next{};     // of 16 keys (Whole) or of this lane's key; keys that are stored, a bit each
    auto locate = [&](Place &pl, int32_t n) __attribute__((always_inline)) {
        const int32_t j0 = first + n * step;
        const uint32_t in = end - j0 >= kKeys ? ~0u >> (32 - kKeys) : end > j0 ? (1u << (end - j0)) - 1u : 0u;
        pl.stored = 0u;
        if constexpr (Whole) {
#pragma unroll
            for (int p = 0; p < K::kParts; ++p) {
                const uint32_t id = uint32_t(__builtin_amdgcn_readlane(pages_ahead, n % (64 / K::kParts) * K::kParts + p));
                const uint32_t key = uint32_t(j0 + 16 * p), slot = key - aa.pages.page_tokens.quotient(key) * aa.pages.page_tokens.d;
                const bool ok = id < aa.pages.pages;
                if (ok) pl.stored |= 0xFFFFu << (16 * p);
                pl.at[p] = ok ? int64_t(id) * aa.pages.page_stride + head_offset + int64_t(slot) * aa.pages.token_stride : -1;
            }
            pl.stored &= in;
        } else {
            const int32_t key = j0 + int32_t(lane) % kKeys;
            pl.at[0] = key < end ? key_offset(aa.pages, Span == kSpanBoth && key < t.prefix ? lead : table, head_offset, key) : -1;
            pl.stored = uint32_t(__ballot(pl.at[0] >= 0)) & (~0u >> (32 - kKeys));
        }
    };
    // offset of key `a` of the tile, which differs by lane
    auto offset = [&](const Place &pl, int p, uint32_t a) __attribute__((always_inline)) {
        if constexpr (Whole) {
            return pl.at[p] < 0 ? int64_t(-1) : pl.at[p] + int64_t(a - 16u * p) * aa.pages.token_stride;
        } else {
            const int low = int(uint32_t(pl.at[0])), high = int(uint32_t(uint64_t(pl.at[0]) >> 32));
            return int64_t(uint64_t(uint32_t(__shfl(low, int(a)))) | uint64_t(uint32_t(__shfl(high, int(a)))) << 32);
        }
    };
    auto request_keys = [&](const Place &pl) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < K::kParts; ++p) {
            const int64_t at = offset(pl, p, 16u * p + i);
            kv.load_keys(p, keys, at < 0 ? 0 : at, lane, D);
        }
    };
    auto request_values = [&](const Place &pl) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < K::kParts; ++p)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t a = 16u * p + 4u * g + r;
                const int64_t at = offset(pl, p, a);
                kv.load_values(p, r, values, at < 0 ? 0 : at, lane, D);
            }
    };
    constexpr int32_t kAhead = 64 / K::kParts;
    if (n_tiles > 0) {
        if (Whole) look_up_pages(0);
        locate(now, 0);
        request_keys(now);
        request_values(now);
        // (Waits count loads in the order they were asked for, and the compiler takes the worst of all ways that lead to a wait: queries and page numbers are
        // waited for here and where they are asked for, or every tile's keys would be waited for with its values: 807 -> 711 us for fp32 chunks, 2 x 1500 tokens
        // over 2000 keys; 286 -> 281 for one token of 48 sequences of up to 16000.)
#pragma unroll
        for (int x = 0; x < K::kSteps; ++x) asm volatile("" : "+v"(Q.q[x]));
        int32_t n = 0;
#pragma unroll 1
        do {
            const int32_t j0 = first + n * step;
            if (Whole && (n + 1) % kAhead == 0) look_up_pages(n + 1);
            locate(next, n + 1);
            f32x4 s[K::kParts];
            if (D < uint32_t(DP)) {
                asm volatile("");
                kv.clear_keys(lane, D);
            }
            kv.scores(Q, s);
            request_keys(next);
            const bool masked = j0 < all_lo || j0 + kKeys > all_hi || now.stored != (~0u >> (32 - kKeys));
            // (a row's keys, and this lane's of the tile, from the lane's first key on)
            const int32_t low = row.lo - j0 - int32_t(4u * g), high = row.hi - j0 - int32_t(4u * g);
            const uint32_t stored = now.stored >> (4u * g);
            float most = -INFINITY, x[K::kParts][4];
#pragma unroll
            for (int p = 0; p < K::kParts; ++p)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[p][r] = s[p][r] * scale;
                    if (masked) {
                        const int a = 16 * p + r;
                        x[p][r] = select(bool(int(a < low) | int(a >= high) | int(!(stored >> a & 1u))), -INFINITY, x[p][r]);
                    }
                    most = fmaxf(most, x[p][r]);
                }
            most = max_quarters(most);
            constexpr float kLead = kReferenceLead<typename K::T>;
            const bool moves = most > ref + (kReferenceSlack + kLead) || (ref == -INFINITY && most > -INFINITY);
            if (__ballot(moves)) {
                asm volatile("");                                  // (a branch, not multiplications by one every time)
                const float to = most - kLead, by = moves ? __builtin_amdgcn_exp2f(ref - to) : 1.f;
                if (moves) ref = to;
                total *= by;
#pragma unroll
                for (int c = 0; c < K::kTiles; ++c) o[c] *= by;
            }
            const float base = ref == -INFINITY ? 0.f : ref;
#pragma unroll
            for (int p = 0; p < K::kParts; ++p)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[p][r] = __builtin_amdgcn_exp2f(x[p][r] - base);
                    total += x[p][r];
                    s[p][r] = x[p][r];
                }
            if (now.stored != (~0u >> (32 - kKeys))) {
                // (what is not stored may be anything, and no weight of zero undoes a NaN)
                asm volatile("");
                kv.clear_values(stored);
            }
            if (masked && __ballot(kv.not_finite())) {
                // an infinity or a NaN that some rows do not see, which a matrix instruction would multiply by their zeros: a key at a time,
                // taken by the rows that see it
#pragma unroll 1
                for (uint32_t a = 0; a < uint32_t(kKeys); ++a) {
                    const K alone = kv.only(a, g);
                    f32x4 w[K::kParts], sum[K::kTiles];
#pragma unroll
                    for (int p = 0; p < K::kParts; ++p)
#pragma unroll
                        for (int r = 0; r < 4; ++r) w[p][r] = a == 16u * p + 4u * g + r ? x[p][r] : 0.f;
#pragma unroll
                    for (int c = 0; c < K::kTiles; ++c) sum[c] = o[c];
                    alone.add(w, sum);
                    const int32_t j = j0 + int32_t(a);
                    const bool sees = int(j >= row.lo) & int(j < row.hi);
#pragma unroll
                    for (int c = 0; c < K::kTiles; ++c)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[c][r] = select(sees, sum[c][r], o[c][r]);
                }
            } else {
                kv.add(s, o);
            }
            request_values(next);
            now = next;
        } while (++n < n_tiles);
    }
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);

    // the waves' sums, in LDS
#pragma unroll
    for (int c = 0; c < K::kTiles; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            sums[(wave * kRows + i) * kPitch + uint32_t(c / K::kPiece * 16 * K::kPiece) + K::kPiece * (4u * g + r) + uint32_t(c % K::kPiece)] = o[c][r];
    if (g == 0u) { refs[wave][i] = ref; totals[wave][i] = total; }
    __syncthreads();
    // a thread has kEach elements of a row
    constexpr uint32_t kEach = DP / 16u;
    const uint32_t m = tid / 16u, d0 = (tid % 16u) * kEach;
    float most = -INFINITY, sum = 0.f, acc[kEach];
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) most = fmaxf(most, refs[w][m]);
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) acc[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) {
        const float by = refs[w][m] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(refs[w][m] - most);
        // (a wave that has seen nothing has added nothing: its sums are zeros)
        sum += totals[w][m] * by;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) acc[e] += sums[(w * kRows + m) * kPitch + d0 + e] * by;
    }
    if (parts > 1) {
        constexpr uint32_t kSlot = kRows * (DP + 4u);              // floats of a part: per row its sums, its reference and its total
        const uint32_t pair = cell.tile * aa.heads.d + head;
        const __amdgpu_buffer_rsrc_t mem = device_scope_buffer(aa.sums + size_t(pair) * aa.splits * kSlot);
        if (m < t.rows) {
            const uint32_t at = (part * kSlot + m * (DP + 4u)) * 4u;
#pragma unroll
            for (uint32_t e = 0; e < kEach; e += 4) store_device_scope(mem, at + (d0 + e) * 4u, f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]});
            if (tid % 16u == 0u) store_device_scope(mem, at + DP * 4u, f32x4{most, sum, 0.f, 0.f});
        }
        wait_stores_acknowledged();
        __syncthreads();
        if (tid == 0u) arrived = __hip_atomic_fetch_add(aa.arrive + pair, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (arrived + 1u != uint32_t(parts)) return;
        if (tid == 0u) __hip_atomic_store(aa.arrive + pair, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // The parts' sums, in turn by as many sets of threads as the rows leave, kAtOnce parts on their way at a time; then the sets' own, in LDS.
        constexpr uint32_t kAtOnce = 4u;
        uint32_t rows_log = 0u;
        while ((1u << rows_log) < t.rows || (uint32_t(parts) <= kAtOnce && rows_log < 4u)) ++rows_log;
        const uint32_t sets = 16u >> rows_log, set = m >> rows_log, row_here = m & ((1u << rows_log) - 1u);
        float top = -INFINITY;
        sum = 0.f;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) acc[e] = 0.f;
        if (row_here < t.rows)
            for (uint32_t p0 = set; p0 < uint32_t(parts); p0 += kAtOnce * sets) {
                f32x4 s[kAtOnce], x[kAtOnce][kEach / 4u];
#pragma unroll
                for (uint32_t k = 0; k < kAtOnce; ++k) {
                    const uint32_t p = p0 + k * sets, at = ((p < uint32_t(parts) ? p : p0) * kSlot + row_here * (DP + 4u)) * 4u;
                    s[k] = load_device_scope(mem, at + DP * 4u);
#pragma unroll
                    for (uint32_t e = 0; e < kEach / 4u; ++e) x[k][e] = load_device_scope(mem, at + (d0 + 4u * e) * 4u);
                }
#pragma unroll
                for (uint32_t k = 0; k < kAtOnce; ++k) {
                    if (p0 + k * sets >= uint32_t(parts)) break;
                    const float now = fmaxf(top, s[k][0]);
                    const float keep = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now), by = s[k][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s[k][0] - now);
                    sum = sum * keep + s[k][1] * by;
#pragma unroll
                    for (uint32_t e = 0; e < kEach; ++e) acc[e] = acc[e] * keep + x[k][e / 4u][e % 4u] * by;
                    top = now;
                }
            }
        most = top;
        if (sets > 1u) {
            // (the waves' references, totals and sums are used up: their place, a set's at [set][row])
            float *const ref_of = &refs[0][0], *const total_of = &totals[0][0];
            if (tid % 16u == 0u) { ref_of[m] = top; total_of[m] = sum; }
#pragma unroll
            for (uint32_t e = 0; e < kEach; ++e) sums[m * kPitch + d0 + e] = acc[e];
            __syncthreads();
            if (m < t.rows) {
                most = -INFINITY;
                for (uint32_t k = 0; k < sets; ++k) most = fmaxf(most, ref_of[(k << rows_log) + m]);
                sum = 0.f;
#pragma unroll
                for (uint32_t e = 0; e < kEach; ++e) acc[e] = 0.f;
                for (uint32_t k = 0; k < sets; ++k) {
                    const uint32_t at = (k << rows_log) + m;
                    const float by = ref_of[at] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref_of[at] - most);
                    sum += total_of[at] * by;
#pragma unroll
                    for (uint32_t e = 0; e < kEach; ++e) acc[e] += sums[at * kPitch + d0 + e] * by;
                }
            }
        }
    }
    if (m < t.rows) {
        const RowOf r = row_of_tile<Span>(aa, t, head, m);
        if constexpr (!kJoins) {
            float *const to = span_sums<Span>(aa, r, part);
#pragma unroll
            for (uint32_t e = 0; e < kEach; e += 4)
                if (d0 + e < D) *reinterpret_cast<f32x4 *>(to + d0 + e) = f32x4{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]};
            if (tid % 16u == 0u) *reinterpret_cast<f32x4 *>(to + D) = span_header<Span>(aa, t, most, sum, keys_here.parts);
            return;
        }
        const bool any = !(sum == 0.f);
        const float by = any ? 1.f / sum : 0.f;
        typename K::T *og = reinterpret_cast<typename K::T *>(aa.out.data) + int64_t(r.token) * aa.out.token_stride + int64_t(r.head) * aa.out.head_stride;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e)
            if (d0 + e < D) og[int64_t(d0 + e) * aa.out.dim_stride] = typename K::T(acc[e] * by);
        if (aa.lse && tid % 16u == 0u) aa.lse[size_t(r.token) * aa.q_heads + r.head] = any ? (most + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY;
    }
}

}  // namespace

}  // namespace hspmm
