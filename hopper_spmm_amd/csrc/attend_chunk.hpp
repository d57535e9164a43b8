// The chunk kernel's part of attention: many rows of queries - chunks of a prompt - over the pages of a cache, 16-bit types.
#pragma once
#include "attend_common.hpp"

namespace hspmm {

namespace {

// A workgroup's LDS writes are done and every wave is here (loads from memory may be on their way).
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A wave has 32 rows, a lane (h, j) = (lane / 32, lane % 32) row j; keys come in images of 64, two halves of 32.
//   scores: S^T = K Q^T, 32 keys x 32 rows by instructions of 16 elements; register r: key 8 (r / 4) + 4 h + r % 4
//   sums:   O^T = V^T P^T, 32 elements x 32 rows by instructions of 16 keys: scores 8 s .. 8 s + 7 of a lane are its part of the second operand,
//           keys in that order; the first one comes transposed from LDS (ds_read_b64_tr_b16), four keys of an element a read
// Per key and row 4 D operations, an exponential and some ten other instructions.  Matrix instructions bound it where keys are many: 4096 tokens over
// 16384 keys, 32 heads on 8, head_dim 128, bf16, 935 to 1020 us, 940 to 1030 TFLOP/s, by machine (a library's product of 8192^3: 1170); 2048 tokens over 8048 keys, heads of 96 / 64:
// 217 / 180 us, 800 / 650 TFLOP/s, as exponentials weigh more.  What is left there is the exponentials' share of a wave's issue that no matrix
// instruction of the other wave covers.  Short spans: an image's arrival and the last workgroups; 17 chunks of up to 700 tokens, window 1000, 70 us, 360
// TFLOP/s.  A wave has 32 rows, two waves a SIMD: one multiplies while the other one takes exponentials.
// The scores of a half are made among the exponentials of the half in front.  Images go through LDS, kRing of them in turn: while image n is
// multiplied, n + 1 is there and n + 2 on its way, first to registers, then to the place of n - 1; one barrier an image (with two places: two).
// Lds<N>: chunk_lds(DP, W) bytes or more; number: of the workgroup among so many `numbers`; part: of its keys.
// What one kind of call has alone stands behind `if constexpr`, and LDS is named, not pointed to: registers are short with heads of 256 elements.  1024 tokens over 2048 older keys, 16 heads on 4
// of 256, bf16, pages of 24 tokens, 158 us with conditions that are never true and a pointer, 142 so; pages of 16 149 and 151 (without prefixes in the body at all 137 and 155).
constexpr uint32_t chunk_image(int DP) { return 64u * (uint32_t(DP) * 2u + 16u + uint32_t(DP) * 2u + (DP % 128 == 0 || DP == 64 ? 64u : 0u)); }
constexpr uint32_t chunk_ring(int DP, int W) { return 3u * chunk_image(DP) <= (DP <= 128 && W == 4 ? 80u : 160u) * 1024u - 256u ? 3u : 2u; }
constexpr uint32_t chunk_lds(int DP, int W) { return chunk_ring(DP, W) * chunk_image(DP) + (uint32_t(W) * 12u + 15u) / 16u * 16u; }
template <bool BF, int DP, int W, bool Whole, AttendSpan Span, uint32_t N>
__device__ __forceinline__ void attend_chunk(const AttendArgs &aa, uint32_t number, uint32_t numbers, uint32_t part)
{
    typedef typename HalfOps<BF>::elem_t T;
    constexpr uint32_t kThreads = 64u * W, kRows = 32u * W, kKeys = 64u;
    constexpr int kRowsLog = W == 8 ? 8 : 7;
    // (rows whose operands are read together begin in different banks: 16 of keys 16 bytes apart, four of values 64)
    constexpr uint32_t kKeyPitch = DP * 2u + 16u, kValuePitch = DP * 2u + (DP % 128 == 0 || DP == 64 ? 64u : 0u), kImage = kKeys * (kKeyPitch + kValuePitch);
    static_assert(kKeyPitch / 16u % 2u == 1u && kValuePitch / 64u % 2u == 1u && kValuePitch % 64u == 0u, "");
    constexpr uint32_t kRing = chunk_ring(DP, W);
    static_assert(kImage == chunk_image(DP) && N >= chunk_lds(DP, W), "");
    constexpr uint32_t kRowPieces = DP / 8u, kImagePieces = kKeys * kRowPieces;
    constexpr int kSteps = DP / 16, kTiles = DP / 32, kPieces = int((kImagePieces + kThreads - 1u) / kThreads);
    __shared__ uint32_t odd, arrived;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, j = lane & 31u;
    // (the last tiles first: where a token sees what is in front of it they are the longest)
    const uint32_t D = aa.pages.head_dim;
    const Cell cell = cell_of(aa, numbers - 1u - number, 0u);
    const uint32_t head = cell.head, tile_number = cell.tile;
    const RowTile t = find_tile<kRowsLog, Span>(aa, tile_number);
    if (!t.there) return;
    const KeyPart keys_here = key_part(aa, t, part);
    constexpr bool kJoins = Span == kSpanAll || Span == kSpanBoth;
    // (where pages are no multiples of 16 tokens what is alike in all lanes is kept in scalar registers: 1024 tokens over 2048 older keys, heads of 256, 147 -> 142 us; else 151 -> 160)
    auto uniform = [](int32_t x) __attribute__((always_inline)) { return Whole ? x : __builtin_amdgcn_readfirstlane(x); };
    const int32_t parts = kJoins ? keys_here.parts : 1, end = uniform(keys_here.end);
    if (int32_t(part) >= keys_here.parts) return;
    if (tid == 0u) odd = 0u;

    const uint32_t m = wave * 32u + j;
    const bool is_row = m < t.rows;
    const RowOf row = row_of_tile<Span>(aa, t, head, m);
    const float scale = aa.scale == 0.f ? 1.f : fabsf(aa.scale) * kLog2e;
    const uint32_t flip = aa.scale < 0.f ? 0x80008000u : 0u;
    u32x4 q[kSteps];
    {
        const char *from = aa.q.data + (int64_t(row.token) * aa.q.token_stride + int64_t(row.head) * aa.q.head_stride) * 2;
        // (loads without conditions: one wait for all of them)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint32_t d = 16u * s + 8u * h;
            q[s] = *reinterpret_cast<const u32x4 *>(from + (d < D ? d : 0u) * 2u);
        }
        const uint32_t keep = is_row && aa.scale != 0.f ? ~0u : 0u;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) q[s] = (q[s] ^ flip) & keep;
        if (D < uint32_t(DP)) {
            asm volatile("");
#pragma unroll
            for (int s = 0; s < kSteps; ++s) q[s] &= 16u * s + 8u * h < D ? ~0u : 0u;
        }
    }
    // keys that all of the wave's rows see
    int32_t all_lo = is_row ? row.lo : 0, all_hi = is_row ? row.hi : 0x7FFFFFFF, any_lo = is_row ? row.lo : 0x7FFFFFFF;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        all_lo = max(all_lo, __shfl_xor(all_lo, d));
        all_hi = min(all_hi, __shfl_xor(all_hi, d));
        if (Span == kSpanPrefix) any_lo = min(any_lo, __shfl_xor(any_lo, d));
    }
    all_lo = __builtin_amdgcn_readfirstlane(all_lo); all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    // the same of the workgroup's rows
    int32_t group_lo, group_hi;
    if constexpr (Span == kSpanPrefix) {
        // (rows of several sequences)
        int32_t (*const ranges)[3] = reinterpret_cast<int32_t (*)[3]>(Lds<N>::bytes + kRing * kImage);
        if (lane == 0u) { ranges[wave][0] = all_lo; ranges[wave][1] = all_hi; ranges[wave][2] = any_lo; }
        __syncthreads();
        group_lo = all_lo; group_hi = all_hi;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            group_lo = max(group_lo, ranges[w][0]);
            group_hi = min(group_hi, ranges[w][1]);
            any_lo = min(any_lo, ranges[w][2]);
        }
        group_lo = __builtin_amdgcn_readfirstlane(group_lo); group_hi = __builtin_amdgcn_readfirstlane(group_hi);
        any_lo = __builtin_amdgcn_readfirstlane(any_lo);
    } else {
        const int32_t p0 = t.position + int32_t(aa.shared.quotient(t.first_row)), p1 = t.position + int32_t(aa.shared.quotient(t.first_row + t.rows - 1u));
        group_hi = __builtin_amdgcn_readfirstlane(aa.causal ? p0 + 1 : t.length);
        group_lo = __builtin_amdgcn_readfirstlane(aa.window && int64_t(p1) + 1 > int64_t(aa.window) ? p1 + 1 - int32_t(aa.window) : 0);
        if constexpr (Span == kSpanRest) group_lo = max(group_lo, t.prefix);
    }
    // (rows of several sequences: from the first key that any of them sees)
    const int32_t begin = uniform(Span == kSpanPrefix ? max(keys_here.begin, min(any_lo & ~31, end)) : keys_here.begin);
    // Images of 64 keys: of the prefix (kSpanBoth), by its first sequence's pages, then of what is behind it, from where a group of 16 begins.
    int32_t first_images = 0, behind = begin, n_images = end > begin ? (end - begin + 63) / 64 : 0;
    if constexpr (Span == kSpanBoth) {
        if (begin < t.prefix) {
            first_images = (min(end, t.prefix) - begin + 63) / 64;
            behind = t.prefix & ~15;
            n_images = first_images + (end > t.prefix ? (end - behind + 63) / 64 : 0);
        }
    }
    const int32_t *table = aa.pages.table + size_t(t.sequence) * aa.pages.table_pages, *const lead = aa.pages.table + size_t(Span == kSpanBoth ? t.leader : t.sequence) * aa.pages.table_pages;
    // The first key of image n, what its keys end in front of, whose row of the table has them, and those of its 64 places that are its.
    auto key_of = [&](int32_t n) __attribute__((always_inline)) {
        if constexpr (Span == kSpanBoth) return n < first_images ? begin + n * 64 : behind + (n - first_images) * 64;
        else return begin + n * 64;
    };
    auto end_of = [&](int32_t n) __attribute__((always_inline)) {
        if constexpr (Span == kSpanBoth) return n < first_images ? min(end, t.prefix) : end;
        else return end;
    };
    auto table_of = [&](int32_t n) __attribute__((always_inline)) {
        if constexpr (Span == kSpanBoth) return n < first_images ? lead : table;
        else return table;
    };
    auto places_of = [&](int32_t n) __attribute__((always_inline)) {
        const int32_t left = end_of(n) - key_of(n);
        const uint64_t in = left >= 64 ? ~uint64_t(0) : left > 0 ? (uint64_t(1) << left) - 1u : 0u;
        if constexpr (Span == kSpanBoth) return n == first_images && behind < t.prefix ? in & ~uint64_t(0) << (t.prefix - behind) : in;
        else return in;
    };
    const int64_t head_offset = int64_t(head) * aa.pages.head_stride;
    // Where keys lie, in bytes from keys and values: of groups of 16 keys, four an image, of 16 images at a time, a lane each (Whole), or of
    // the keys of an image; and which of them are stored, a bit each.
    uint32_t ahead_low = 0u, ahead_high = 0u;
    uint64_t ahead_there = 0u;
    auto look_up = [&](int32_t n, int32_t in_image) __attribute__((always_inline)) {
        const int32_t key = key_of(n) + in_image;
        const int64_t at = key < end_of(n) ? key_offset(aa.pages, table_of(n), head_offset, key) : -1;
        ahead_there = __ballot(at >= 0);
        const uint64_t bytes = at >= 0 ? uint64_t(at) * 2u : 0u;
        ahead_low = uint32_t(bytes);
        ahead_high = uint32_t(bytes >> 32);
    };
    // a thread's pieces of an image: 16 bytes of a row of keys and of values
    u32x4 k_piece[kPieces], v_piece[kPieces];
    uint32_t groups_there = 0u;                                // of the image in the registers (Whole)
    uint64_t keys_there = 0u;
    // Piece i of a thread: eight elements from `column` on of a row.  Of lanes behind the last element, and of keys that are not stored,
    // something is read and not used.
    auto piece_row = [&](int i) __attribute__((always_inline)) {
        const uint32_t p = tid + kThreads * i;
        return (kImagePieces % kThreads == 0u || p < kImagePieces ? p : kImagePieces - 1u) / kRowPieces;
    };
    auto piece_column = [&](int i) __attribute__((always_inline)) { return (tid + kThreads * i) % kRowPieces * 8u; };
    auto is_piece = [&](int i) __attribute__((always_inline)) { return kImagePieces % kThreads == 0u || tid + kThreads * i < kImagePieces; };
    // A piece's bytes from where its group of 16 begins (Whole), or its key: the latter is made anew, and is one for all of a thread's pieces where its columns are.
    uint32_t in_group_of[Whole ? kPieces : 1];
#pragma unroll
    for (int i = 0; i < (Whole ? kPieces : 1); ++i) {
        const uint32_t c = piece_column(i);
        in_group_of[i] = (Whole ? uint32_t(int64_t(piece_row(i) % 16u) * aa.pages.token_stride) * 2u : 0u) + (c < D ? c : 0u) * 2u;
    }
    auto in_group = [&](int i) __attribute__((always_inline)) {
        if constexpr (Whole || kThreads % kRowPieces == 0u) return in_group_of[Whole ? i : 0];
        else {
            const uint32_t c = piece_column(i);
            return (c < D ? c : 0u) * 2u;
        }
    };
    auto request = [&](int32_t n) __attribute__((always_inline)) {
        if constexpr (Whole) {
            if (n % 16 == 0) look_up(n + int32_t(lane / 4u), int32_t(lane % 4u) * 16);
            const int32_t first = n % 16 * 4;
            groups_there = uint32_t(ahead_there >> first) & 15u;
        } else {
            look_up(n, int32_t(lane));
            keys_there = ahead_there;
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            uint64_t from;
            if constexpr (Whole) {
                // (the rows of a wave's pieces lie in one group of 16: 2 DP / 64 waves have a group's pieces)
                static_assert(16u * kRowPieces % 64u == 0u, "");
                constexpr uint32_t kGroupWaves = 16u * kRowPieces / 64u;
                const uint32_t g = (wave + uint32_t(W) * i) / kGroupWaves;
                const int32_t at = n % 16 * 4 + int32_t(g < 4u ? g : 3u);
                from = uint64_t(uint32_t(__builtin_amdgcn_readlane(int(ahead_low), at))) | uint64_t(uint32_t(__builtin_amdgcn_readlane(int(ahead_high), at))) << 32;
            } else {
                const int at = int(piece_row(i));
                from = uint64_t(uint32_t(__shfl(int(ahead_low), at))) | uint64_t(uint32_t(__shfl(int(ahead_high), at))) << 32;
            }
            k_piece[i] = *reinterpret_cast<const u32x4 *>(aa.pages.keys + from + in_group(i));
            v_piece[i] = *reinterpret_cast<const u32x4 *>(aa.pages.values + from + in_group(i));
        }
    };
    // the stored keys of image n, which is in the registers
    auto stored_keys = [&](int32_t n) __attribute__((always_inline)) {
        const uint64_t in = places_of(n);
        if constexpr (!Whole) return keys_there & in;
        if (groups_there == 15u) return in;
        uint64_t there = 0u;
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (groups_there >> g & 1u) there |= uint64_t(0xFFFFu) << (16 * g);
        return there & in;
    };
    auto write_image = [&](int32_t n, uint32_t to) __attribute__((always_inline)) {
        char *const image = Lds<N>::bytes + to * kImage;
        const uint64_t stored_there = stored_keys(n);
        if (~stored_there || D < uint32_t(DP)) {
            // (what is not stored may be anything, and no weight of zero undoes a NaN)
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                if (piece_column(i) >= D || !(stored_there >> piece_row(i) & 1u)) k_piece[i] = v_piece[i] = u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (!is_piece(i)) continue;
            *reinterpret_cast<u32x4 *>(image + piece_row(i) * kKeyPitch + piece_column(i) * 2u) = k_piece[i];
            *reinterpret_cast<u32x4 *>(image + kKeys * kKeyPitch + piece_row(i) * kValuePitch + piece_column(i) * 2u) = v_piece[i];
        }
        const int32_t key0 = key_of(n);
        if (n < n_images && (key0 < group_lo || key0 + 64 > group_hi || ~stored_there)) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
#pragma unroll
                for (int w = 0; w < 4; ++w) any |= word_not_finite<BF>(v_piece[i][w]);
            if (any) odd = 1u;
        }
        return stored_there;
    };

    f32x16 o[kTiles];
    float ref, total;
    auto begin_sums = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][r] = 0.f;
        ref = -INFINITY;
        total = 0.f;
    };
    const uint32_t key_lane = j * kKeyPitch + h * 16u;
    const uint32_t value_lane = kKeys * kKeyPitch + (4u * h + (lane & 15u) / 4u) * kValuePitch + ((lane >> 4 & 1u) * 16u + (lane & 3u) * 4u) * 2u;
    // The first operands of half of the scores' instructions, asked for well ahead of them.
    struct KeyOperands { u32x4 a[kSteps / 2]; };
    auto ask_keys = [&](KeyOperands &f, auto second, uint32_t image, uint32_t half) __attribute__((always_inline)) {
        const char *const from = Lds<N>::bytes + image * kImage + half * 32u * kKeyPitch + key_lane + decltype(second)::value * (kSteps / 2) * 32;
#pragma unroll
        for (int c = 0; c < kSteps / 2; ++c) f.a[c] = *reinterpret_cast<const u32x4 *>(from + c * 32);
    };
    auto scores = [&](auto second, f32x16 &s, const KeyOperands &f) __attribute__((always_inline)) {
        constexpr int c0 = decltype(second)::value * (kSteps / 2);
        if constexpr (c0 == 0) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < kSteps / 2; ++c) s = Wide<BF>::mfma(f.a[c], q[c0 + c], s);
    };
    auto mask = [&](f32x16 &s, int32_t key0, uint32_t stored) __attribute__((always_inline)) {
        if (key0 >= all_lo && key0 + 32 <= all_hi && stored == ~0u) return;
        const uint32_t mine = stored >> (4u * h);
        const int32_t low = row.lo - key0 - int32_t(4u * h), high = row.hi - key0 - int32_t(4u * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            constexpr int kOf[16] = {0, 1, 2, 3, 8, 9, 10, 11, 16, 17, 18, 19, 24, 25, 26, 27};
            s[r] = select(bool(int(kOf[r] < low) | int(kOf[r] >= high) | int(!(mine >> kOf[r] & 1u))), -INFINITY, s[r]);
        }
    };
    // the largest score of every row; where one is far above its row's reference the sums move to a new one
    auto move_references = [&](const f32x16 &s) __attribute__((always_inline)) {
        float most = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) most = fmaxf(most, s[r]);
        most = max_halves(most) * scale;
        constexpr float kLead = kReferenceLead<T>;
        const bool moves = most > ref + (kReferenceSlack + kLead) || (ref == -INFINITY && most > -INFINITY);
        if (__builtin_expect(__ballot(moves) != 0u, 0)) {
            asm volatile("");                                  // (a branch, not DP / 2 multiplications by one every time)
            const float to = most - kLead, by = moves ? __builtin_amdgcn_exp2f(ref - to) : 1.f;
            if (moves) ref = to;
            total *= by;
#pragma unroll
            for (int c = 0; c < kTiles; ++c) o[c] *= by;
        }
    };
    auto exponentials = [&](f32x16 &s) __attribute__((always_inline)) {
        const float base = ref == -INFINITY ? 0.f : ref;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale, -base));
            total += s[r];
        }
    };
    // The same of the sums' instructions for 16 keys.
    struct ValueOperands { u32x4 a[kTiles]; };
    auto ask_values = [&](ValueOperands &f, auto second, uint32_t image, uint32_t half) __attribute__((always_inline)) {
        constexpr int c = decltype(second)::value;
        const __attribute__((address_space(3))) char *const from = (const __attribute__((address_space(3))) char *)(Lds<N>::bytes + image * kImage + half * 32u * kValuePitch + value_lane);
#pragma unroll
        for (int e = 0; e < kTiles; ++e) {
            const t_u32x2 a0 = __builtin_bit_cast(t_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tile_tr_ptr)(from + (16 * c) * kValuePitch + e * 64)));
            const t_u32x2 a1 = __builtin_bit_cast(t_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tile_tr_ptr)(from + (16 * c + 8) * kValuePitch + e * 64)));
            f.a[e] = u32x4{a0[0], a0[1], a1[0], a1[1]};
        }
    };
    auto add = [&](auto second, const f32x16 &s, const ValueOperands &f) __attribute__((always_inline)) {
        constexpr int c = decltype(second)::value;
        u32x4 p;
#pragma unroll
        for (int w = 0; w < 4; ++w) p[w] = pack_two<BF>(s[8 * c + 2 * w], s[8 * c + 2 * w + 1]);
#pragma unroll
        for (int e = 0; e < kTiles; ++e) o[e] = Wide<BF>::mfma(f.a[e], p, o[e]);
    };
    using first = std::integral_constant<int, 0>;
    using second = std::integral_constant<int, 1>;
    KeyOperands keys_1, keys_2;
    // A half: scores `s` become weights and are added, the scores of the half behind it are made meanwhile (its first operands are asked for
    // already); at the end those of the one behind that are asked for.
    auto half_step = [&](f32x16 &s, f32x16 &s_other, int32_t key0, uint32_t stored, uint32_t image, uint32_t half, uint32_t other_image, uint32_t other_half,
                         uint32_t third_image, uint32_t third_half) __attribute__((always_inline)) {
        mask(s, key0, stored);
        ask_keys(keys_2, second{}, other_image, other_half);
        __builtin_amdgcn_sched_barrier(0);
        scores(first{}, s_other, keys_1);
        move_references(s);
        ValueOperands values_1, values_2;
        ask_values(values_1, first{}, image, half);
        __builtin_amdgcn_sched_barrier(0);
        scores(second{}, s_other, keys_2);
        exponentials(s);
        // (nothing between: the values are asked for among the exponentials, 960 -> 937 us for 4096 tokens over 16384 keys)
        ask_values(values_2, second{}, image, half);
        add(first{}, s, values_1);
        ask_keys(keys_1, first{}, third_image, third_half);
        add(second{}, s, values_2);
    };

    begin_sums();
    if (n_images) {
        f32x16 s_a, s_b;
        request(0);
        lds_barrier();                                         // (`odd` is zero before any wave can set it)
        uint64_t stored_now = write_image(0, 0u);
        request(1);
        uint64_t stored_next = write_image(1, 1u);
        lds_barrier();
        ask_keys(keys_1, first{}, 0u, 0u);
        ask_keys(keys_2, second{}, 0u, 0u);
        scores(first{}, s_a, keys_1);
        scores(second{}, s_a, keys_2);
        ask_keys(keys_1, first{}, 0u, 1u);
        uint32_t now = 0u, next = 1u, free = kRing - 1u;
#pragma unroll 1
        for (int32_t n = 0; n < n_images; ++n) {
            const int32_t key0 = key_of(n);
            request(n + 2);
            half_step(s_a, s_b, key0, uint32_t(stored_now), now, 0u, now, 1u, next, 0u);
            half_step(s_b, s_a, key0 + 32, uint32_t(stored_now >> 32), now, 1u, next, 0u, next, 1u);
            if constexpr (kRing == 2u) { lds_barrier(); free = now; }
            stored_now = stored_next;
            stored_next = write_image(n + 2, free);
            const uint32_t old = now;
            now = next;
            next = free;
            free = old;
            lds_barrier();
        }
        __syncthreads();
        if (odd) {
            // An infinity or a NaN that some rows do not see, which a matrix instruction would multiply by their zeros: once more, the values key by
            // key and by the rows that see it.  Slow, and off the path of finite data.
            begin_sums();
            float *const weights = reinterpret_cast<float *>(Lds<N>::bytes + kImage) + wave * 32u * 32u;
            static_assert(W * 32u * 32u * 4u <= (kRing - 1u) * kImage, "weights in the place of the other images");
#pragma unroll 1
            for (int32_t n = 0; n < n_images; ++n) {
                __syncthreads();
                if (Whole && n % 16) look_up((n & ~15) + int32_t(lane / 4u), int32_t(lane % 4u) * 16);
                request(n);
                const uint64_t stored = write_image(n, 0u);
                __syncthreads();
#pragma unroll 1
                for (uint32_t half = 0; half < 2u; ++half) {
                    const int32_t key0 = key_of(n) + int32_t(half) * 32;
                    ask_keys(keys_1, first{}, 0u, half);
                    ask_keys(keys_2, second{}, 0u, half);
                    scores(first{}, s_a, keys_1);
                    scores(second{}, s_a, keys_2);
                    mask(s_a, key0, uint32_t(stored >> (32u * half)));
                    move_references(s_a);
                    exponentials(s_a);
                    __syncthreads();
#pragma unroll
                    for (int r = 0; r < 16; ++r) weights[(8u * (r / 4) + 4u * h + r % 4) * 32u + j] = s_a[r];
                    __syncthreads();
#pragma unroll 1
                    for (uint32_t a = 0; a < 32u; ++a) {
                        const int32_t key = key0 + int32_t(a);
                        const float w = weights[a * 32u + j];
                        const T *from = reinterpret_cast<const T *>(Lds<N>::bytes + kKeys * kKeyPitch + (32u * half + a) * kValuePitch) + 4u * h;
                        const bool hidden = int(key < row.lo) | int(key >= row.hi);
#pragma unroll
                        for (int c = 0; c < kTiles; ++c)
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[c][r] += select(hidden, 0.f, w * float(from[32 * c + 8 * (r / 4) + r % 4]));
                    }
                }
            }
        }
    }

    // what a row's two lanes have
    total += __shfl_xor(total, 32);
    if (parts > 1) {
        // A part's sums as the lanes hold them: 16 bytes a lane side by side, then the rows' references and totals.
        constexpr uint32_t kWaveSlot = 32u * (DP + 4u), kSlot = kRows * (DP + 4u);
        const uint32_t pair = tile_number * aa.heads.d + head;
        const __amdgpu_buffer_rsrc_t mem = device_scope_buffer(aa.sums + size_t(pair) * aa.splits * kSlot);
        const bool wave_there = wave * 32u < t.rows;
        auto sums_at = [&](uint32_t p, int c, int r) __attribute__((always_inline)) { return (p * kSlot + wave * kWaveSlot + (c * 4u + r / 4u) * 256u + lane * 4u) * 4u; };
        auto scalars_at = [&](uint32_t p) __attribute__((always_inline)) { return (p * kSlot + wave * kWaveSlot + 32u * DP + j * 4u) * 4u; };
        if (wave_there) {
#pragma unroll
            for (int c = 0; c < kTiles; ++c)
#pragma unroll
                for (int r = 0; r < 16; r += 4) store_device_scope(mem, sums_at(part, c, r), f32x4{o[c][r], o[c][r + 1], o[c][r + 2], o[c][r + 3]});
            if (h == 0u) store_device_scope(mem, scalars_at(part), f32x4{ref, total, 0.f, 0.f});
        }
        wait_stores_acknowledged();
        __syncthreads();
        if (tid == 0u) arrived = __hip_atomic_fetch_add(aa.arrive + pair, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (arrived + 1u != uint32_t(parts)) return;
        if (tid == 0u) __hip_atomic_store(aa.arrive + pair, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (!wave_there) return;
        begin_sums();
#pragma unroll 1
        for (int32_t p = 0; p < parts; ++p) {
            const f32x4 s = load_device_scope(mem, scalars_at(uint32_t(p)));
            f32x4 x[kTiles][4];
#pragma unroll
            for (int c = 0; c < kTiles; ++c)
#pragma unroll
                for (int r = 0; r < 16; r += 4) x[c][r / 4] = load_device_scope(mem, sums_at(uint32_t(p), c, r));
            const float top = fmaxf(ref, s[0]);
            const float keep = ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - top), by = s[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s[0] - top);
            total = total * keep + s[1] * by;
#pragma unroll
            for (int c = 0; c < kTiles; ++c)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[c][r] = o[c][r] * keep + x[c][r / 4][r % 4] * by;
            ref = top;
        }
    }
    if (!is_row) return;
    if constexpr (!kJoins) {
        float *const to = span_sums<Span>(aa, row, part);
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const uint32_t d = 32u * c + 2u * r + 4u * h;
                if (d < D) *reinterpret_cast<f32x4 *>(to + d) = f32x4{o[c][r], o[c][r + 1], o[c][r + 2], o[c][r + 3]};
            }
        if (h == 0u) *reinterpret_cast<f32x4 *>(to + D) = span_header<Span>(aa, t, ref, total, keys_here.parts);
        return;
    }
    const bool any = !(total == 0.f);
    const float by = any ? 1.f / total : 0.f;
    T *og = reinterpret_cast<T *>(aa.out.data) + int64_t(row.token) * aa.out.token_stride + int64_t(row.head) * aa.out.head_stride;
    const bool side_by_side = aa.out.dim_stride == 1 && (reinterpret_cast<uintptr_t>(og) & 7u) == 0u;
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const uint32_t d = 32u * c + 2u * r + 4u * h;
            if (d >= D) continue;
            if (side_by_side) {
                *reinterpret_cast<t_u32x2 *>(og + d) = t_u32x2{pack_two<BF>(o[c][r] * by, o[c][r + 1] * by), pack_two<BF>(o[c][r + 2] * by, o[c][r + 3] * by)};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) og[int64_t(d + e) * aa.out.dim_stride] = T(o[c][r + e] * by);
            }
        }
    if (aa.lse && h == 0u) aa.lse[size_t(row.token) * aa.q_heads + row.head] = any ? (ref + __builtin_amdgcn_logf(total)) * kLn2 : -INFINITY;
}

}  // namespace

}  // namespace hspmm
