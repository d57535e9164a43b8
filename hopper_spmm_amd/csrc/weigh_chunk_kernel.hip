// Accumulated attention weights of cached keys by many rows of queries - chunks of a prompt, or their last tokens -, 16-bit types.
#include "weigh_common.hpp"

namespace hspmm {

namespace {

constexpr uint32_t kThreads = 256u, kWaves = kThreads / 64u;

// A workgroup has 128 keys, in LDS for good; its waves take 32 rows in turn, from memory to registers, and meet at the end only.  A lane (h, j) = (lane / 32, lane % 32).
//   scores: S^T = K Q^T, 32 keys x 32 rows by instructions of 16 elements; register r: key 8 (r / 4) + 4 h + r % 4, row j
// so that a row's lse and range of keys are a lane's own, and a key's weights add up in its register, over lanes and waves once at the end.
// Per key and row 2 D operations and an exponential: matrix instructions (32 cycles for 32 x 32 x 16) and exponentials (8 for 64) bound it.  4096 tokens over 8192 keys, 32 heads on 8 of 128, bf16: 253 to 266 us, 775 to 810
// TFLOP/s of products (a library's product of 8192^3: 1170), 840 by the rows kernel; the last 32 tokens of 17 prompts, 96 rows, are 30 us here and 18 there.  What is left: 8 us of a
// workgroup's time before its first product and behind its last, and the exponentials' share of a wave's issue that no product of the other wave covers.  Keys stay and rows move, not the other way round, as a key's
// sum is then a register from the first row to the last; 128 keys and two workgroups a compute unit are what 160 KB hold with rows of 128 elements.
// Rows that see a workgroup's keys are cut into parts; a part leaves its keys' sums, and the workgroup that leaves the last one adds them up in the parts' order.
template <bool BF, int DP>
__global__ __launch_bounds__(kThreads, DP <= 128 ? 2 : 1) void weigh_chunk_kernel(const WeighArgs wa)
{
    constexpr int kSteps = DP / 16, kTiles = kWeighKeys / 32;
    constexpr uint32_t kKeys = kWeighKeys, kPitch = DP * 2u + 16u, kRowPieces = DP / 8u, kPieces = kKeys * kRowPieces / kThreads;
    static_assert(kKeys * kRowPieces % kThreads == 0u && kKeys <= kThreads, "");
    __shared__ __attribute__((aligned(16))) char keys[kKeys * kPitch], rows_of[kWaves][32u * kPitch];
    __shared__ int64_t rows_at[kWaves][32];
    __shared__ __attribute__((aligned(16))) float sums_of[kWaves][kKeys];
    __shared__ uint32_t keys_stored[kTiles], arrived;
    const uint32_t D = wa.pages.head_dim;
    const uint32_t column = wa.heads.quotient(blockIdx.x), head = blockIdx.x - column * wa.heads.d, b = wa.blocks.quotient(column), block0 = column - b * wa.blocks.d;
    const WeighRows w = weigh_rows(wa, b);
    if (!w.there) return;
    const int32_t n_blocks = (w.keys + int32_t(kKeys) - 1) / int32_t(kKeys);
    // (a sequence longer than the call said: nothing is cut, the first workgroups have several blocks)
    const bool cut = n_blocks <= int32_t(wa.blocks.d);
    if (!cut && blockIdx.y) return;
    const float scale = wa.scale * kLog2e;
    const int32_t *table = wa.pages.table + size_t(w.sequence) * wa.pages.table_pages;
    const int64_t head_offset = int64_t(head) * wa.pages.head_stride;
    float *const weights = wa.weights + int64_t(w.sequence) * wa.sequence_stride + int64_t(head) * wa.head_stride;
    const uint32_t step_heads = kWaves * 32u % wa.shared.d, step_tokens = kWaves * 32u / wa.shared.d;
    const int64_t q_step = (int64_t(step_tokens) * wa.q.token_stride + int64_t(step_heads) * wa.q.head_stride) * 2, q_wrap = (wa.q.token_stride - int64_t(wa.shared.d) * wa.q.head_stride) * 2;
    const int64_t lse_step = int64_t(step_tokens) * wa.q_heads + step_heads, lse_wrap = int64_t(wa.q_heads) - wa.shared.d;
    for (int32_t block = int32_t(block0); block < n_blocks; block += int32_t(wa.blocks.d)) {
        // (made anew in every turn, of which there is one: what follows from it is not wanted in registers from here to the end)
        uint32_t tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const uint32_t lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, j = lane & 31u;
        const int32_t key0 = block * int32_t(kKeys);
        const RowRange range = rows_that_see(wa, w, key0, int32_t(kKeys));
        // this part's rows
        const uint32_t all_rows = range.end > range.first ? range.end - range.first : 0u;
        uint32_t parts = 1u, first_row = range.first, end_row = range.end;
        if (cut) {
            // (of one length, and as many as there are workgroups for)
            parts = min((all_rows + wa.part_rows - 1u) / wa.part_rows, gridDim.y);
            const uint32_t each = parts > 1u ? ((all_rows + parts - 1u) / parts + 127u) & ~127u : all_rows;
            parts = all_rows ? (all_rows + each - 1u) / each : 1u;
            if (blockIdx.y >= parts) return;
            first_row = range.first + blockIdx.y * each;
            end_row = blockIdx.y + 1u < parts ? first_row + each : range.end;
        }
        // Rows, 32 a wave, 128 on in the next turn: where those lie follows without a division or a product (`step_heads` heads on, and some tokens), a lane finds out for row j.
        // They are loaded with a row's pieces side by side, of eight elements each, and go through the wave's own LDS to be a product's operand: loaded as that, sixteen bytes of a row
        // a lane, a turn's loads were two thirds of what a compute unit's cache can look up, 277 us of which 70 went for them (4096 tokens over 8192 keys).
        // Of rows behind the last one the first of the tensor is read, and not used; behind a row's last element there are zeros, as those of the keys do not undo an infinity.
        uint32_t at_row = first_row + wave * 32u + j, at_head;
        int64_t at_q, at_lse, lse_at;
        {
            const uint32_t i = wa.shared.quotient(at_row);
            at_head = at_row - i * wa.shared.d;
            at_q = (int64_t(w.first_token + i) * wa.q.token_stride + int64_t(head * wa.shared.d + at_head) * wa.q.head_stride) * 2;
            at_lse = int64_t(w.first_token + i) * wa.q_heads + head * wa.shared.d + at_head;
        }
        constexpr uint32_t kRowsPieces = 32u * kRowPieces / 64u;
        u32x4 rows_piece[kRowsPieces];
        float lse_ahead;
        auto piece_of = [&](uint32_t i) __attribute__((always_inline)) { return (lane + 64u * i) / kRowPieces; };
        auto column_of = [&](uint32_t i) __attribute__((always_inline)) { return (lane + 64u * i) % kRowPieces * 8u; };
        // (what is read for an element behind the last one goes where nobody looks, past the row: in its own place are the zeros that are put there now)
        auto put_column = [&](uint32_t i) __attribute__((always_inline)) { return column_of(i) < D ? column_of(i) : uint32_t(DP); };
        if (D < uint32_t(DP)) {
#pragma unroll 1
            for (uint32_t i = 0; i < kRowsPieces; ++i)
                if (column_of(i) >= D) *reinterpret_cast<u32x4 *>(rows_of[wave] + piece_of(i) * kPitch + column_of(i) * 2u) = u32x4{0u, 0u, 0u, 0u};
        }
        auto find = [&]() __attribute__((always_inline)) {
            const bool there = at_row < w.rows;
            rows_at[wave][j] = there ? at_q : 0;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
            lse_at = there ? at_lse : 0;
            at_row += kWaves * 32u;
            at_head += step_heads;
            const bool wraps = at_head >= wa.shared.d;
            at_head -= wraps ? wa.shared.d : 0u;
            at_q += wraps ? q_step + q_wrap : q_step;
            at_lse += wraps ? lse_step + lse_wrap : lse_step;
        };
        auto request = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t i = 0; i < kRowsPieces; ++i) {
                const uint32_t c = column_of(i);
                rows_piece[i] = *reinterpret_cast<const u32x4 *>(wa.q.data + rows_at[wave][piece_of(i)] + (c < D ? c : 0u) * 2u);
            }
            lse_ahead = wa.lse[lse_at];
        };
        auto put = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (uint32_t i = 0; i < kRowsPieces; ++i) *reinterpret_cast<u32x4 *>(rows_of[wave] + piece_of(i) * kPitch + put_column(i) * 2u) = rows_piece[i];
            // (a wave's LDS accesses are done in the order they are issued in)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
        };
        const uint32_t n_rows = end_row > first_row ? end_row - first_row : 0u, n_tiles = (n_rows + 31u) / 32u;
        find();
        request();
        // keys: what is not stored is not used
        {
            uint32_t at_low = 0u, at_high = 0u, there = 0u;
            if (tid < kKeys) {
                const int32_t key = key0 + int32_t(tid);
                const int64_t at = key < w.keys ? key_offset(wa.pages, table, head_offset, key) : -1;
                there = at >= 0;
                at_low = there ? uint32_t(uint64_t(at)) : 0u;
                at_high = there ? uint32_t(uint64_t(at) >> 32) : 0u;
                const uint64_t stored = __ballot(there);
                if (lane == 0u) { keys_stored[wave * 2u] = uint32_t(stored); keys_stored[wave * 2u + 1u] = uint32_t(stored >> 32); }
                reinterpret_cast<uint2 *>(sums_of)[tid] = uint2{at_low, at_high};
            }
            __syncthreads();
            u32x4 piece[kPieces];
#pragma unroll
            for (uint32_t i = 0; i < kPieces; ++i) {
                const uint32_t p = tid + kThreads * i, c = p % kRowPieces * 8u;
                const uint2 at = reinterpret_cast<const uint2 *>(sums_of)[p / kRowPieces];
                piece[i] = *reinterpret_cast<const u32x4 *>(wa.pages.keys + ((uint64_t(at.x) | uint64_t(at.y) << 32) + (c < D ? c : 0u)) * 2u);
            }
#pragma unroll
            for (uint32_t i = 0; i < kPieces; ++i) {
                const uint32_t p = tid + kThreads * i, c = p % kRowPieces * 8u;
                const uint32_t keep = c < D ? ~0u : 0u;
                *reinterpret_cast<u32x4 *>(keys + p / kRowPieces * kPitch + c * 2u) = piece[i] & keep;
            }
            __syncthreads();
        }
        uint32_t stored[kTiles], all_stored = ~0u;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            stored[t] = keys_stored[t];
            all_stored &= stored[t];
        }
        f32x16 sums[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) sums[t][r] = 0.f;
        if (wave < n_tiles) {
            // A unit is 32 rows and 32 keys.  The scores of the unit behind are made among the exponentials of the one in front: a matrix instruction takes as long as one and a half
            // registers' exponentials.  k: the keys of the unit behind; what their last product leaves free receives those of the unit behind that.
            // q: the rows of the products that are made; after the last ones' first product of a unit, those behind them.
            f32x16 p[2];
            u32x4 k[kSteps], q[kSteps];
            const char *const key_lane = keys + j * kPitch + h * 16u, *const row_lane = rows_of[wave] + j * kPitch + h * 16u;
            auto read_k = [&](int s, int t) __attribute__((always_inline)) { k[s] = *reinterpret_cast<const u32x4 *>(key_lane + t * 32 * kPitch + s * 32); };
            auto read_q = [&](int s) __attribute__((always_inline)) { q[s] = *reinterpret_cast<const u32x4 *>(row_lane + s * 32); };
            auto unit = [&](auto masked, auto tile, uint32_t seen, float base) __attribute__((always_inline)) {
                constexpr int t = decltype(tile)::value, f = t & 1;
                constexpr int kOf[16] = {0, 1, 2, 3, 8, 9, 10, 11, 16, 17, 18, 19, 24, 25, 26, 27};
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    p[f ^ 1] = Wide<BF>::mfma(k[s], q[s], s == 0 ? f32x16{} : p[f ^ 1]);
                    __builtin_amdgcn_sched_barrier(0);
                    read_k(s, (t + 2) % kTiles);
                    if constexpr (t == kTiles - 2) read_q(s);
#pragma unroll
                    for (int r = 16 * s / kSteps; r < 16 * (s + 1) / kSteps; ++r) {
                        float x = __builtin_amdgcn_exp2f(__builtin_fmaf(p[f][r], scale, base));
                        if constexpr (decltype(masked)::value) x = select(seen >> kOf[r] & 1u, x, 0.f);
                        float sum = sums[t][r] + x;
                        asm volatile("" : "+v"(sum));          // (here, not behind the loads that follow)
                        sums[t][r] = sum;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            auto seen_of = [&](const RowOf &row, int t) __attribute__((always_inline)) {
                const int32_t low = row.lo - key0 - 32 * t, high = row.hi - key0 - 32 * t;
                const uint32_t from = low <= 0 ? ~0u : low >= 32 ? 0u : ~0u << low, to = high >= 32 ? ~0u : high <= 0 ? 0u : ~0u >> (32 - high);
                return (stored[t] & from & to) >> (4u * h);
            };
            // sets n, n + 4, .. of 32 rows; the first one's scores of the first keys are in p[0], and the rows behind are asked for
            float base;
            auto turns = [&](auto masked, uint32_t n, uint32_t end) __attribute__((always_inline)) {
#pragma unroll 1
                for (; n < end; n += kWaves) {
                    uint32_t seen[kTiles] = {0u, 0u, 0u, 0u};
                    if constexpr (decltype(masked)::value) {
                        const uint32_t m = first_row + n * 32u + j;
                        const RowOf row = weigh_row(wa, w, head, m < end_row ? m : w.rows);
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) seen[t] = seen_of(row, t);
                    }
                    request();
                    unit(masked, std::integral_constant<int, 0>{}, seen[0], base);
                    unit(masked, std::integral_constant<int, 1>{}, seen[1], base);
                    put();
                    unit(masked, std::integral_constant<int, 2>{}, seen[2], base);
                    find();
                    unit(masked, std::integral_constant<int, 3>{}, seen[3], base);
                    base = moved_by(lse_ahead);
                }
                return n;
            };
            static_assert(kTiles == 4, "");
            put();
            find();
            base = moved_by(lse_ahead);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) read_q(s);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) read_k(s, 0);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) p[0] = Wide<BF>::mfma(k[s], q[s], s == 0 ? f32x16{} : p[0]);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) read_k(s, 1);
            // sets of 32 rows that all see all of the workgroup's keys: behind those that begin in front of one, in front of those whose windows do not reach them any more
            uint32_t clear = n_tiles, clear_end = n_tiles;
            if (all_stored == ~0u) {
                const uint32_t full = n_rows / 32u;
                const int64_t first_clear = wa.causal ? (int64_t(key0) + kKeys - 1 - w.position) * wa.shared.d - first_row : 0;
                const int64_t end_clear = wa.window ? (int64_t(key0) + wa.window - w.position) * wa.shared.d - first_row : int64_t(n_rows);
                clear = first_clear <= 0 ? 0u : uint32_t(min((first_clear + 31) / 32, int64_t(full)));
                clear_end = end_clear <= 0 ? 0u : uint32_t(min(end_clear / 32, int64_t(full)));
            }
            uint32_t n = turns(std::true_type{}, wave, clear);
            n = turns(std::false_type{}, n, clear_end);
            turns(std::true_type{}, n, n_tiles);
        }
        // over the lanes' rows: lane j of sixteen has register j's key
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            float mine_of = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float s = sum_row(sums[t][r]);
                mine_of = (j & 15u) == uint32_t(r) ? s : mine_of;
            }
            mine_of += __shfl_xor(mine_of, 16);
            if (j < 16u) sums_of[wave][32u * t + 8u * (j / 4u) + 4u * h + j % 4u] = mine_of;
        }
        __syncthreads();
        const uint32_t cell = (b * wa.blocks.d + block0) * wa.heads.d + head;
        f32x4 mine = f32x4{0.f, 0.f, 0.f, 0.f};
        if (tid < kKeys / 4u)
#pragma unroll
            for (uint32_t v = 0; v < kWaves; ++v) mine += *reinterpret_cast<const f32x4 *>(sums_of[v] + tid * 4u);
        if (parts > 1u) {
            const __amdgpu_buffer_rsrc_t mem = device_scope_buffer(wa.sums + size_t(cell) * gridDim.y * kKeys);
            if (tid < kKeys / 4u) store_device_scope(mem, (blockIdx.y * kKeys + tid * 4u) * 4u, mine);
            wait_stores_acknowledged();
            __syncthreads();
            if (tid == 0u) arrived = __hip_atomic_fetch_add(wa.arrive + cell, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (arrived + 1u != parts) return;
            if (tid == 0u) __hip_atomic_store(wa.arrive + cell, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            mine = f32x4{0.f, 0.f, 0.f, 0.f};
            if (tid < kKeys / 4u)
                for (uint32_t p = 0; p < parts; ++p) mine += load_device_scope(mem, (p * kKeys + tid * 4u) * 4u);
        }
        if (tid < kKeys / 4u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int32_t key = key0 + int32_t(4u * tid) + e;
                if (key < w.keys) weights[key] = key < w.old ? weights[key] * wa.decay + mine[e] : mine[e];
            }
        }
        __syncthreads();
    }
}

template <bool BF, int DP>
void launch(const WeighArgs &wa, hipStream_t s)
{
    weigh_chunk_kernel<BF, DP><<<dim3(wa.batch.sequences * wa.blocks.d * wa.heads.d, wa.parts), dim3(kThreads), 0, s>>>(wa);
}

template <bool BF>
void launch_type(const WeighArgs &wa, hipStream_t s)
{
    const uint32_t D = wa.pages.head_dim;
    if (D <= 64u) launch<BF, 64>(wa, s);
    else if (D <= 96u) launch<BF, 96>(wa, s);
    else if (D <= 128u) launch<BF, 128>(wa, s);
    else if (D <= 160u) launch<BF, 160>(wa, s);
    else launch<BF, 256>(wa, s);
}

}  // namespace

hipError_t launch_weigh_chunk(int dtype, const WeighArgs &wa, hipStream_t s)
{
    if (dtype == kDtypeF16) launch_type<false>(wa, s);
    else launch_type<true>(wa, s);
    return hipGetLastError();
}

}  // namespace hspmm
