// The product of two e4m3 code matrices under block scales (new with this library; the reference's products are int8):
//   c[i][j] = T(sum over blocks g of 128 channels: a_scale[i][g] * w_scale[j/128][g] * sum of a[i][k] * w[j][k] in g)
// The scales are arbitrary f32 values, so a block's sum has to leave the tensor cores before the next may be added: a
// tcgen05.mma of one block (K = 128, four instructions) goes to one of two accumulators in tensor memory, and eight warps
// read it, scale it and add it to the output they hold in registers, while the other accumulator fills.
//
// Two kernels:
//   wide    a pair of CTAs owns 256 rows of a and 256 of w (as the int8 pair kernel does); an epilogue thread owns one row
//           and 128 outputs, whose scale of a block is one number
//   narrow  few rows of a: 128 rows of w are the M side and up to 192 rows of a the N side of a CTA, the blocks of 128
//           channels are split over a cluster of up to eight CTAs, whose partial outputs are added over distributed shared
//           memory in the order of their rank: no workspace, no atomics, the same bits every time
#include <atomic>

#include "tensor_core.cuh"

namespace krea2 {
namespace {

__device__ int g_product_status = 0;  // folded into krea2_device_status by take_product_status
std::atomic<bool> g_product_launched{false};  // whether the word is worth a copy: a chain's status reads are not to wait for it
constexpr int kProductTimedOut = KREA2_STATUS_GEMM_FP8;

constexpr int kBlock = 128;  // channels under one scale = bytes of K per stage = one 128-byte swizzle row
constexpr int kStep = 32;    // K of one kind::f8f6f4 instruction

struct ProductArgs {
    const float *w_scale, *a_scale;
    uint16_t *c;
    uint32_t m, n, blocks;
    size_t c_stride;
    uint32_t bf16;    // output type
    uint32_t aligned; // rows of c start on 16-byte boundaries
    uint32_t panels;  // wide kernel: column tiles walked together (0: a column of tiles top to bottom)
};

// kind::f8f6f4: f32 accumulate (1 at bit 4), e4m3 A and B (0 at bits 7 and 10), both K-major, N/8 at bit 17, M/16 at bit 24.
__host__ __device__ constexpr uint32_t product_descriptor(int m, int n) {
    return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
template <int kCtas>
__device__ __forceinline__ void issue_product(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kCtas == 2)
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem), "l"(a), "l"(b),
                     "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem), "l"(a), "l"(b),
                     "r"(idesc), "r"(accumulate)
                     : "memory");
}

// ---------------------------------------------------------------- scales
// The rows' scales lie [row][block]: a warp that loads one block's for 32 rows touches 32 lines, and eight epilogue warps
// doing so take the L1's whole time.  So two warps of a CTA load four blocks at a time (16 bytes a row) and lay them out
// [block][row] in a ring in shared memory for all.
template <int kRows, bool kMultiply>
struct ScaleRing {
    static constexpr int kSlots = 3, kRun = 4;                // runs of four blocks
    static constexpr int kWarps = 2, kPerLane = (kRows + 63) / 64;
    static constexpr int kSlotFloats = kRun * kRows + 8;      // and each block's scale of w (of either half), if not multiplied in
    static constexpr int kBytes = kSlots * kSlotFloats * 4;
    float *values;
    uint64_t *full, *empty;

    __device__ __forceinline__ float *slot(uint32_t run) const { return values + (run % kSlots) * kSlotFloats; }
    __device__ __forceinline__ static uint32_t parity(uint32_t run) { return (run / kSlots) & 1u; }

    // Blocks first .. last - 1 of the rows from row0 on, by warp `which` of the two.  `w0`, `w1`: the scales of w (w1 of the
    // second half, not multiplied in).  False when a wait ran out.
    __device__ __forceinline__ bool fill(const float *a_scale, const float *w0, const float *w1, uint32_t row0, uint32_t m, uint32_t blocks, uint32_t first,
                                         uint32_t last, int which, int lane, uint32_t &run, const Abort &abort) const {
        const bool vector = ((blocks | first) & 3u) == 0u && (reinterpret_cast<uintptr_t>(a_scale) & 15u) == 0u;
        const float *from[kPerLane];
#pragma unroll
        for (int i = 0; i < kPerLane; i++)
            from[i] = a_scale + static_cast<size_t>(min(row0 + (2 * i + which) * 32 + lane, m - 1)) * blocks;
        float4 ahead[kPerLane];
        auto request = [&](uint32_t b) {
#pragma unroll
            for (int i = 0; i < kPerLane; i++) {
                if (vector) {
                    ahead[i] = __ldg(reinterpret_cast<const float4 *>(from[i] + b));
                } else {
                    ahead[i].x = __ldg(from[i] + b), ahead[i].y = __ldg(from[i] + min(b + 1, last - 1));
                    ahead[i].z = __ldg(from[i] + min(b + 2, last - 1)), ahead[i].w = __ldg(from[i] + min(b + 3, last - 1));
                }
            }
        };
        request(first);
        for (uint32_t b = first; b < last; b += kRun, run++) {
            if (!barrier_wait_warp(empty + run % kSlots, parity(run) ^ 1u, abort)) return false;
            float *to = slot(run);
            float w[kRun];
            if constexpr (kMultiply) {
#pragma unroll
                for (int k = 0; k < kRun; k++) w[k] = __ldg(w0 + min(b + k, last - 1));
            } else if (which == 0 && lane < 8) {
                to[kRun * kRows + lane] = __ldg((lane < 4 ? w0 : w1) + min(b + (lane & 3), last - 1));
            }
#pragma unroll
            for (int i = 0; i < kPerLane; i++) {
                const int row = (2 * i + which) * 32 + lane;
                const float v[kRun] = {ahead[i].x, ahead[i].y, ahead[i].z, ahead[i].w};
                if (row < kRows)
#pragma unroll
                    for (int k = 0; k < kRun; k++) to[k * kRows + row] = kMultiply ? v[k] * w[k] : v[k];
            }
            __syncwarp();
            if (lane == 0) barrier_arrive(full + run % kSlots);
            if (b + kRun < last) request(b + kRun);
        }
        return true;
    }
};

// ---------------------------------------------------------------- wide
// Bound by what the block scales cost and by the ends of a tile.  A block's four products take 512 clocks of the pair's tensor
// cores, but its 256 x 256 sums also leave tensor memory and pass through the FMA pipes each time: 782 clocks a block.  A tile's
// output holds back the next one's sums, of which two blocks at most are computed ahead: 5200 clocks a tile.  (Both from the
// time times the sampled SM clock of 4608 x 15360 at 1024 to 10240 channels, 15 rounds of tiles.)  4608 x 15360 x 6144 takes
// 380-445 us (2.0-2.3 PFLOP/s, 0.6-0.7 of the e4m3 rate; 441 us at 1432 MHz, back to back at the power cap).  With an eighth
// of the sums read it took 341 us, with a quarter of the products 346, with both 228, each at the clock that the cap left it.
// Sixteen epilogue warps, loads of 32 columns, one product of 256 columns instead of two of 128: no faster.
struct Wide {
    static constexpr int kRows = 128;     // of a, and of w, per CTA
    static constexpr int kColumns = 256;  // of a tile
    static constexpr int kStages = 6;
    static constexpr int kWarps = 8;      // epilogue: two per 32-lane quarter, each with half of the columns
    using Scales = ScaleRing<kRows, false>;
    static constexpr int kWarpColumns = kColumns / (kWarps / 4);
    static constexpr int kThreads = (kWarps + 4) * 32;  // a warpgroup beside them: one loads, one issues, two lay out scales
    // The launch gives each thread 168 registers; the epilogue's two warpgroups, with 128 outputs a thread, take some of
    // the third's.
    static constexpr int kEpilogueRegisters = 208, kOtherRegisters = 64;
    static_assert((kWarps / 4) * kEpilogueRegisters + kOtherRegisters <= (kWarps / 4 + 1) * 168, "registers of the launch");
    static constexpr int kOperandBytes = kRows * kBlock;
    static constexpr int kStageBytes = 2 * kOperandBytes;
    static constexpr int kStagingBytes = 32 * 64;  // per warp: 32 rows of 32 outputs on their way out
    static constexpr int kSharedBytes = kStages * kStageBytes + 1024 + 256 + kWarps * kStagingBytes + Scales::kBytes;
    static_assert(kSharedBytes <= 227 * 1024, "shared memory");
};

// Writes 32 outputs of each of the warp's 32 rows through its staging area, so that rows leave in 64-byte pieces; the
// 16-byte pieces of a row change places from one pair of rows to the next, which spreads a column of them over the banks.
template <bool kBf16>
__device__ __forceinline__ void store_wide(const ProductArgs &g, const float2 *values, uint32_t row0, uint32_t column0, uint8_t *staging, int lane) {
    auto piece = [&](uint32_t row, uint32_t i) { return staging + row * 64 + ((i ^ ((row >> 1) & 3u)) * 16); };
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
        *reinterpret_cast<uint4 *>(piece(lane, i)) =
            make_uint4(pack_pair<kBf16>(values[4 * i].x, values[4 * i].y), pack_pair<kBf16>(values[4 * i + 1].x, values[4 * i + 1].y),
                       pack_pair<kBf16>(values[4 * i + 2].x, values[4 * i + 2].y), pack_pair<kBf16>(values[4 * i + 3].x, values[4 * i + 3].y));
    __syncwarp();
    if (g.aligned) {
        const uint32_t column = column0 + (lane & 3) * 8, row = row0 + (lane >> 2);
        uint4 v[4];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = *reinterpret_cast<const uint4 *>(piece(8 * r + (lane >> 2), lane & 3));
        uint16_t *to = g.c + row * g.c_stride + column;
        if (row0 + 32 <= g.m && column0 + 32 <= g.n) {
#pragma unroll
            for (int r = 0; r < 4; r++) *reinterpret_cast<uint4 *>(to + 8 * r * g.c_stride) = v[r];
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                if (row + 8 * r >= g.m) continue;
                if (column + 8 <= g.n) {
                    *reinterpret_cast<uint4 *>(to + 8 * r * g.c_stride) = v[r];
                } else {
                    const uint32_t words[4] = {v[r].x, v[r].y, v[r].z, v[r].w};
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (column + i < g.n) to[8 * r * g.c_stride + i] = static_cast<uint16_t>(words[i >> 1] >> (16 * (i & 1)));
                }
            }
        }
    } else if (column0 + lane < g.n) {
        for (uint32_t local = 0; local < 32 && row0 + local < g.m; local++)
            g.c[(row0 + local) * g.c_stride + column0 + lane] = reinterpret_cast<const uint16_t *>(piece(local, lane >> 3))[lane & 7];
    }
    __syncwarp();
}

template <bool kBf16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Wide::kThreads, 1)
wide_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const ProductArgs g) {
    using T = Wide;
    extern __shared__ uint8_t shared_raw[];
    uint8_t *shared = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(shared + T::kStages * T::kStageBytes);
    uint64_t *empty = full + T::kStages, *sum_full = empty + T::kStages, *sum_empty = sum_full + 4;  // [half][parity]
    uint64_t *scale_full = sum_empty + 4, *scale_empty = scale_full + T::Scales::kSlots;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(scale_empty + T::Scales::kSlots);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    // [0], [1] the stages each CTA's producer filled (in the leader), [2], [3] each CTA's abort flag (in both)
    volatile uint32_t *exchange = reinterpret_cast<volatile uint32_t *>(tmem_slot + 2);
    uint8_t *staging = shared + T::kStages * T::kStageBytes + 256;
    const T::Scales scales = {reinterpret_cast<float *>(staging + T::kWarps * T::kStagingBytes), scale_full, scale_empty};
    const Abort abort = {abort_flag, &g_product_status, kProductTimedOut};

    const int warp = static_cast<int>(uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const uint32_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t m_tiles = (g.m + 2 * T::kRows - 1) / (2 * T::kRows), n_tiles = (g.n + T::kColumns - 1) / T::kColumns;
    const uint32_t tiles = m_tiles * n_tiles;
    uint32_t issued = 0;
    auto origin = [&](uint32_t tile, uint32_t &row, uint32_t &column) {
        uint32_t tile_m = tile % m_tiles, tile_n = tile / m_tiles;
        if (g.panels != 0) {
            const uint32_t per = m_tiles * g.panels, first = tile / per * g.panels, t = tile % per;
            const uint32_t width = n_tiles - first < g.panels ? n_tiles - first : g.panels;
            tile_m = t / width;
            tile_n = first + t % width;
        }
        row = tile_m * 2 * T::kRows + rank * T::kRows;
        column = tile_n * T::kColumns;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < T::kStages; s++) {
            barrier_init(full + s, 1);
            barrier_init(empty + s, 1);
        }
        for (int s = 0; s < 4; s++) {
            barrier_init(sum_full + s, 1);
            barrier_init(sum_empty + s, T::kWarps);  // the half's warps of both CTAs
        }
        for (int s = 0; s < T::Scales::kSlots; s++) {
            barrier_init(scale_full + s, T::Scales::kWarps);
            barrier_init(scale_empty + s, T::kWarps);
        }
        *abort_flag = 0;
        barrier_init_done();
    }
    if (warp == T::kWarps + 1) {
        __syncwarp();
        tensor_alloc<2>(tmem_slot, 2 * T::kColumns);
    }
    tensor_fence_before();
    cluster_barrier();
    tensor_fence_after();
    const uint32_t tmem = uniform(*tmem_slot);
    if (warp >= T::kWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::kOtherRegisters));
        if (warp == T::kWarps && lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool alive = true;
            for (uint32_t tile = pair; alive && tile < tiles; tile += pairs) {
                uint32_t row, column;
                origin(tile, row, column);
                for (uint32_t b = 0; b < g.blocks; b++) {
                    if (!(alive = barrier_wait(empty + stage, phase ^ 1u, abort))) break;
                    uint8_t *dst = shared + stage * T::kStageBytes;
                    const uint32_t leader_full = cluster_address(full + stage, 0);
                    if (leader) barrier_expect(full + stage, 2 * T::kStageBytes);
                    load_tile_pair(dst, &map_a, leader_full, static_cast<int>(b * kBlock), static_cast<int>(row));
                    // this CTA's 64 rows of either half
                    load_tile_pair(dst + T::kOperandBytes, &map_w, leader_full, static_cast<int>(b * kBlock), static_cast<int>(column + rank * 64));
                    load_tile_pair(dst + T::kOperandBytes + T::kOperandBytes / 2, &map_w, leader_full, static_cast<int>(b * kBlock),
                                   static_cast<int>(column + kBlock + rank * 64));
                    issued++;
                    if (++stage == T::kStages) stage = 0, phase ^= 1u;
                }
            }
        }
        if (warp == T::kWarps + 1 && leader) {
            const bool elected = elect_lane();
            constexpr uint32_t idesc = product_descriptor(2 * T::kRows, T::kColumns / 2);
            uint32_t stage = 0, phase = 0, count = 0;
            bool alive = true;
            bool loaded = false, free0 = false, free1 = false;  // what the next block's barriers said while this one's products ran
            for (uint32_t tile = pair; alive && tile < tiles; tile += pairs) {
                for (uint32_t b = 0; b < g.blocks; b++, count++) {
                    const uint32_t s = count & 1u, parity = ((count >> 1) & 1u) ^ 1u;
                    const uint32_t at = smem_address(shared + stage * T::kStageBytes);
                    const uint64_t a = operand_descriptor(at);
                    if (!(alive = barrier_wait_warp(full + stage, phase, abort, loaded))) break;
#pragma unroll
                    for (uint32_t half = 0; half < 2; half++) {
                        if (!(alive = barrier_wait_warp(sum_empty + 2 * half + s, parity, abort, half == 0 ? free0 : free1))) break;
                        tensor_fence_after();
                        // each CTA holds 128 of the tile's rows of w: its 64 of this half lie at 64 * half
                        const uint64_t w = operand_descriptor(at + T::kOperandBytes + half * (T::kOperandBytes / 2));
                        if (elected) {
#pragma unroll
                            for (int k = 0; k < kBlock / kStep; k++)
                                issue_product<2>(tmem + s * T::kColumns + half * kBlock, a + 2 * k, w + 2 * k, idesc, k != 0);
                            tensor_commit_pair(sum_full + 2 * half + s);
                            if (half == 1) tensor_commit_pair(empty + stage);
                        }
                        __syncwarp();
                    }
                    if (!alive) break;
                    if (++stage == T::kStages) stage = 0, phase ^= 1u;
                    const uint32_t next = (count + 1) & 1u, next_parity = (((count + 1) >> 1) & 1u) ^ 1u;
                    loaded = barrier_peek(full + stage, phase);
                    free0 = barrier_peek(sum_empty + next, next_parity);
                    free1 = barrier_peek(sum_empty + 2 + next, next_parity);
                }
            }
        }
        if (warp >= T::kWarps + 2) {
            uint32_t run = 0;
            const uint32_t scale_rows = (g.n + kBlock - 1) / kBlock;
            for (uint32_t tile = pair; tile < tiles; tile += pairs) {
                uint32_t row, column;
                origin(tile, row, column);
                const float *w0 = g.w_scale + static_cast<size_t>(column / kBlock) * g.blocks;
                const float *w1 = column / kBlock + 1 < scale_rows ? w0 + g.blocks : w0;
                if (!scales.fill(g.a_scale, w0, w1, row, g.m, g.blocks, 0, g.blocks, warp - T::kWarps - 2, lane, run, abort)) break;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::kEpilogueRegisters));
        const int quarter = warp & 3, half = warp >> 2;
        uint32_t count = 0, run = 0;
        bool alive = true;
        const uint32_t release[2] = {cluster_address(sum_empty + 2 * half, 0), cluster_address(sum_empty + 2 * half + 1, 0)};
        for (uint32_t tile = pair; alive && tile < tiles; tile += pairs) {
            uint32_t row0, column0;
            origin(tile, row0, column0);
            row0 += quarter * 32;
            column0 += half * T::kWarpColumns;
            float2 out[T::kWarpColumns / 2];
#pragma unroll
            for (int i = 0; i < T::kWarpColumns / 2; i++) out[i] = make_float2(0.0f, 0.0f);
            bool ready = false;
            for (uint32_t b = 0; b < g.blocks; b++, count++) {
                const uint32_t s = count & 1u;
                if ((b & 3u) == 0u && !(alive = barrier_wait_warp(scale_full + run % T::Scales::kSlots, T::Scales::parity(run), abort))) break;
                const float *run_scales = scales.slot(run);
                const float one = run_scales[(b & 3u) * T::kRows + quarter * 32 + lane] * run_scales[4 * T::kRows + half * 4 + (b & 3u)];
                const float2 scale = make_float2(one, one);
                if ((b & 3u) == 3u || b + 1 == g.blocks) {
                    __syncwarp();
                    if (lane == 0) barrier_arrive(scale_empty + run % T::Scales::kSlots);
                    run++;
                }
                if (!(alive = barrier_wait_warp(sum_full + 2 * half + s, (count >> 1) & 1u, abort, ready))) break;
                tensor_fence_after();
                const uint32_t from = tmem + s * T::kColumns + half * T::kWarpColumns + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
                for (int c = 0; c < T::kWarpColumns / 16; c++) {
                    float sums[16];
                    tensor_load_16(from + c * 16, sums);
                    tensor_loads_done_16(sums);
                    if (c == T::kWarpColumns / 16 - 1) {  // everything has been read: the accumulator may be overwritten
                        tensor_fence_before();
                        __syncwarp();
                        if (lane == 0) barrier_arrive_at(release[s]);
                        ready = barrier_peek(sum_full + 2 * half + (s ^ 1u), ((count + 1) >> 1) & 1u);
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) out[c * 8 + i] = fma_pair(make_float2(sums[2 * i], sums[2 * i + 1]), scale, out[c * 8 + i]);
                }
            }
            if (!alive) break;
#pragma unroll
            for (int c = 0; c < T::kWarpColumns / 32; c++)
                store_wide<kBf16>(g, out + c * 16, row0, column0 + c * 32, staging + warp * T::kStagingBytes, lane);
        }
    }

    tensor_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t mine = *abort_flag ? 1u : 0u;
        cluster_store(cluster_address(const_cast<uint32_t *>(exchange) + 2 + rank, 0), mine);
        cluster_store(cluster_address(const_cast<uint32_t *>(exchange) + 2 + rank, 1), mine);
    }
    if (warp == T::kWarps && lane == 0) cluster_store(cluster_address(const_cast<uint32_t *>(exchange) + rank, 0), issued);
    __syncwarp();
    cluster_barrier();  // neither CTA frees tensor memory or exits while the other may still use it
    tensor_fence_after();
    if (exchange[2] | exchange[3]) {
        // A wait ran out.  All loads of the pair complete on the leader's barriers: its producer waits for the last load
        // into every stage, after putting the byte count right where only one CTA issued its half.
        if (leader && warp == T::kWarps && lane == 0) {
            const uint32_t by_leader = exchange[0], by_peer = exchange[1], high = max(by_leader, by_peer);
            const uint64_t start = clock_ns();
            for (uint32_t i = high > T::kStages ? high - T::kStages : 0u; i < high; i++) {
                const uint32_t s = i % T::kStages;
                if (i >= by_peer)
                    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_address(full + s)), "r"(T::kStageBytes) : "memory");
                if (i >= by_leader) barrier_expect(full + s, T::kStageBytes);
                barrier_drain(full + s, (i / T::kStages) & 1u, start);
            }
        }
        __syncwarp();
        cluster_barrier();  // the other CTA stays until its loads have been seen to land
    }
    if (warp == T::kWarps + 1) {
        __syncwarp();
        tensor_free<2>(tmem, 2 * T::kColumns);
    }
}

// ---------------------------------------------------------------- narrow
// One row: bound by HBM once the weights are large (15360 x 16384: 46 us, 5.5 TB/s), by the start, the ramp of the loads and
// the addition of the shares below (6144 x 6144: 11.2 us against 5.9 for the bytes).  A few hundred rows: by what the tiles
// take out of L2, 13-15 TB/s (275 x 6144 x 16384: 43 us).
constexpr int power_of_two(int n) { return n <= 32 ? 32 : 2 * power_of_two((n + 1) / 2); }

template <int kTokens>
struct Narrow {
    static constexpr int kRows = 128;                        // of w
    static constexpr int kWarps = kTokens <= 32 ? 4 : 8;  // epilogue
    static constexpr int kThreads = (kWarps + 4) * 32;       // and one warp that loads, one that issues, two that lay out scales
    using Scales = ScaleRing<kTokens, true>;
    static constexpr int kColumns = kTokens / (kWarps / 4);  // tokens of one epilogue thread
    static constexpr int kStageBytes = (kRows + kTokens) * kBlock;
    // Up to 64 tokens two CTAs share an SM, so that one streams while the other starts or adds up.  Above, a thread's
    // outputs want the registers of one; and where two sets of accumulators exceed tensor memory (512 columns, 2 * kTokens
    // each) the shared memory has to keep the second out, since a CTA that waits for tensor memory holds up its cluster.
    static constexpr int kPerSm = kTokens <= 64 ? 2 : 1;
    // Blocks between the products and the epilogue: each is short, and the way to the epilogue's warps and back long.
    static constexpr int kSums = kTokens <= 32 ? 8 : kTokens <= 128 ? 4 : kTokens <= 160 ? 3 : 2;
    static constexpr int kTensorColumns = power_of_two(kSums * kTokens);
    static_assert(kPerSm * kTensorColumns <= 512, "tensor memory");
    static constexpr int kStages = ((kPerSm == 2 ? 108 : 216) * 1024 - 2048 - Scales::kBytes) / kStageBytes;
    static constexpr int kSharedBytes = kStages * kStageBytes + 1024 + 512 + Scales::kBytes;
    static constexpr int kPitch = kRows + 4;  // of the partial outputs, in floats: a fragment's four tokens fall into different banks
    static_assert(kStages >= 2 && kStages * kStageBytes >= kPitch * kTokens * 4, "the partial outputs take the stages' place");
    static_assert(kPerSm * kSharedBytes <= 227 * 1024 && (kPerSm + 1) * (kSharedBytes + 1024) > 228 * 1024, "CTAs per SM");
};

template <int kTokens>
__global__ void __launch_bounds__(Narrow<kTokens>::kThreads, Narrow<kTokens>::kPerSm)
narrow_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const ProductArgs g) {
    using T = Narrow<kTokens>;
    extern __shared__ uint8_t shared_raw[];
    uint8_t *shared = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(shared + T::kStages * T::kStageBytes);
    uint64_t *empty = full + T::kStages, *sum_full = empty + T::kStages, *sum_empty = sum_full + T::kSums;
    uint64_t *scale_full = sum_empty + T::kSums, *scale_empty = scale_full + T::Scales::kSlots;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(scale_empty + T::Scales::kSlots);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const typename T::Scales scales = {reinterpret_cast<float *>(shared + T::kStages * T::kStageBytes + 512), scale_full, scale_empty};
    float *partial = reinterpret_cast<float *>(shared);                                     // [kTokens][kPitch], once the stages are done with
    const Abort abort = {abort_flag, &g_product_status, kProductTimedOut};

    const int warp = static_cast<int>(uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x, shares = gridDim.x;  // a cluster spans x: the split of the blocks
    const uint32_t n0 = blockIdx.y * T::kRows, m0 = blockIdx.z * kTokens;
    const uint32_t first = static_cast<uint32_t>(static_cast<uint64_t>(g.blocks) * rank / shares);
    const uint32_t last = static_cast<uint32_t>(static_cast<uint64_t>(g.blocks) * (rank + 1) / shares);
    uint32_t issued = 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < T::kStages; s++) {
            barrier_init(full + s, 1);
            barrier_init(empty + s, 1);
        }
        for (int s = 0; s < T::kSums; s++) {
            barrier_init(sum_full + s, 1);
            barrier_init(sum_empty + s, T::kWarps);
        }
        for (int s = 0; s < T::Scales::kSlots; s++) {
            barrier_init(scale_full + s, T::Scales::kWarps);
            barrier_init(scale_empty + s, T::kWarps);
        }
        *abort_flag = 0;
        barrier_init_done();
    }
    if (warp == T::kWarps + 1) {
        __syncwarp();
        tensor_alloc<1>(tmem_slot, T::kTensorColumns);
    }
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t tmem = uniform(*tmem_slot);

    if (warp == T::kWarps) {
        if (lane == 0) {
            for (uint32_t b = first; b < last; b++, issued++) {
                const uint32_t stage = issued % T::kStages, phase = (issued / T::kStages) & 1u;
                if (!barrier_wait(empty + stage, phase ^ 1u, abort)) break;
                uint8_t *dst = shared + stage * T::kStageBytes;
                barrier_expect(full + stage, T::kStageBytes);
                load_tile(dst, &map_w, full + stage, static_cast<int>(b * kBlock), static_cast<int>(n0));
                load_tile(dst + T::kRows * kBlock, &map_a, full + stage, static_cast<int>(b * kBlock), static_cast<int>(m0));
            }
        }
    } else if (warp == T::kWarps + 1) {
        {
            const bool elected = elect_lane();
            constexpr uint32_t idesc = product_descriptor(T::kRows, kTokens);
            bool loaded = false, free = false;  // what the next block's barriers said while this one's products ran
            uint32_t s = 0, stage = 0, sum_phase = 1, load_phase = 0;
            for (uint32_t b = first; b < last; b++) {
                if (!barrier_wait_warp(full + stage, load_phase, abort, loaded) || !barrier_wait_warp(sum_empty + s, sum_phase, abort, free)) break;
                tensor_fence_after();
                const uint32_t at = smem_address(shared + stage * T::kStageBytes);
                const uint64_t w = operand_descriptor(at), a = operand_descriptor(at + T::kRows * kBlock);
                if (elected) {
#pragma unroll
                    for (int k = 0; k < kBlock / kStep; k++) issue_product<1>(tmem + s * kTokens, w + 2 * k, a + 2 * k, idesc, k != 0);
                    tensor_commit(empty + stage);
                    tensor_commit(sum_full + s);
                }
                __syncwarp();
                if (++stage == T::kStages) stage = 0, load_phase ^= 1u;
                if (++s == T::kSums) s = 0, sum_phase ^= 1u;
                loaded = barrier_peek(full + stage, load_phase);
                free = barrier_peek(sum_empty + s, sum_phase);
            }
        }
    } else if (warp >= T::kWarps + 2) {
        uint32_t run = 0;
        const float *w_scale = g.w_scale + static_cast<size_t>(blockIdx.y) * g.blocks;
        scales.fill(g.a_scale, w_scale, w_scale, m0, g.m, g.blocks, first, last, warp - T::kWarps - 2, lane, run, abort);
    } else {
        // A warp owns 32 rows of w and kColumns tokens, a thread four of the rows (lane / 4 + 0, 8, 16, 24) and every
        // fourth pair of tokens, so that a scale it reads from shared memory serves four outputs.  (With a row and all
        // tokens per thread, each scale is handed to 32 lanes for one output each: four clocks of shared memory a token
        // and block, twice what the product takes.)
        const int quarter = warp & 3, group = warp >> 2;
        float2 out[T::kColumns / 8][4];
#pragma unroll
        for (int i = 0; i < T::kColumns / 8; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) out[i][r] = make_float2(0.0f, 0.0f);
        uint32_t run = 0, s = 0, sum_phase = 0;
        bool ready = false;
        for (uint32_t b = first, count = 0; b < last; b++, count++) {
            const uint32_t k = count & 3u;
            if (k == 0u && !barrier_wait_warp(scale_full + run % T::Scales::kSlots, T::Scales::parity(run), abort)) break;
            if (!barrier_wait_warp(sum_full + s, sum_phase, abort, ready)) break;
            tensor_fence_after();
            const uint32_t from = tmem + s * kTokens + group * T::kColumns + (static_cast<uint32_t>(quarter * 32) << 16);
            const float *mine = scales.slot(run) + k * kTokens + group * T::kColumns + 2 * (lane & 3);
#pragma unroll
            for (int c = 0; c < T::kColumns; c += 16) {
                float sums[16];  // rows lane / 4 + 0 and 8, then + 16 and 24
                tensor_load_fragment(from + c, sums);
                tensor_load_fragment(from + c + (16u << 16), sums + 8);
                float2 scale[2];
#pragma unroll
                for (int j = 0; j < 2; j++) scale[j] = *reinterpret_cast<const float2 *>(mine + c + 8 * j);
                tensor_loads_done_16(sums);
                if (c + 16 == T::kColumns) {
                    tensor_fence_before();
                    __syncwarp();
                    if (lane == 0) barrier_arrive(sum_empty + s);
                    if (++s == T::kSums) s = 0, sum_phase ^= 1u;
                    ready = barrier_peek(sum_full + s, sum_phase);
                }
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float *sum = sums + 8 * (r >> 1) + 4 * j + 2 * (r & 1);
                        out[c / 8 + j][r] = fma_pair(make_float2(sum[0], sum[1]), scale[j], out[c / 8 + j][r]);
                    }
            }
            if (k == 3u || b + 1 == last) {
                __syncwarp();
                if (lane == 0) barrier_arrive(scale_empty + run % T::Scales::kSlots);
                run++;
            }
        }
        // The last sum has been read, so every product has read its stage and every load has landed.
        asm volatile("bar.sync 1, %0;" ::"n"(T::kWarps * 32) : "memory");
        if (!*abort_flag) {
            float *to = partial + (group * T::kColumns + 2 * (lane & 3)) * T::kPitch + quarter * 32 + lane / 4;
#pragma unroll
            for (int i = 0; i < T::kColumns / 8; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    to[8 * i * T::kPitch + 8 * r] = out[i][r].x;
                    to[(8 * i + 1) * T::kPitch + 8 * r] = out[i][r].y;
                }
        }
    }

    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    if (*abort_flag && warp == T::kWarps && lane == 0) {
        const uint64_t start = clock_ns();
        for (uint32_t i = issued > T::kStages ? issued - T::kStages : 0u; i < issued; i++)
            barrier_drain(full + i % T::kStages, (i / T::kStages) & 1u, start);
    }
    if (warp == T::kWarps + 1) {
        __syncwarp();
        tensor_free<1>(tmem, T::kTensorColumns);
    }
    cluster_barrier();  // every share of this tile is in shared memory
    // This CTA adds the shares of its part of the tokens, in the order of their rank, four outputs per thread at a time.
    const uint32_t token_first = kTokens * rank / shares, token_last = kTokens * (rank + 1) / shares;
    for (uint32_t item = token_first * 32 + threadIdx.x; item < token_last * 32; item += T::kThreads) {
        const uint32_t token = item / 32, column = n0 + (item % 32) * 4;
        if (m0 + token >= g.m || column >= g.n) continue;
        float4 total = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float4 share[8];  // requested together: a load from another CTA takes as long as one from L2
#pragma unroll
        for (uint32_t r = 0; r < 8; r++)
            if (r < shares) share[r] = cluster_load(cluster_address(partial + token * T::kPitch + (item % 32) * 4, r));
#pragma unroll
        for (uint32_t r = 0; r < 8; r++)
            if (r < shares) total.x += share[r].x, total.y += share[r].y, total.z += share[r].z, total.w += share[r].w;
        const uint2 packed = g.bf16 ? make_uint2(pack_pair<true>(total.x, total.y), pack_pair<true>(total.z, total.w))
                                    : make_uint2(pack_pair<false>(total.x, total.y), pack_pair<false>(total.z, total.w));
        uint16_t *to = g.c + (m0 + token) * g.c_stride + column;
        if (g.aligned && column + 4 <= g.n) {
            *reinterpret_cast<uint2 *>(to) = packed;
        } else {
            const uint32_t words[2] = {packed.x, packed.y};
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (column + i < g.n) to[i] = static_cast<uint16_t>(words[i >> 1] >> (16 * (i & 1)));
        }
    }
    cluster_barrier();  // the others have read this CTA's share
}

// ---------------------------------------------------------------- host side
int operand_map(CUtensorMap *map, const void *base, size_t rows, size_t k, size_t stride, uint32_t box_rows) {
    const cuuint64_t dims[2] = {k, rows}, strides[1] = {stride};
    const cuuint32_t box[2] = {kBlock, box_rows};
    return make_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box);
}

template <int kTokens>
cudaLaunchConfig_t narrow_config(const ProductArgs &g, uint32_t shares, cudaLaunchAttribute &attribute) {
    using T = Narrow<kTokens>;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(shares, (g.n + T::kRows - 1) / T::kRows, (g.m + kTokens - 1) / kTokens);
    config.blockDim = dim3(T::kThreads);
    config.dynamicSmemBytes = T::kSharedBytes;
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = shares;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return config;
}

// A launch of the narrow kernel and what it is expected to take.
struct NarrowPlan {
    uint32_t shares = 1;
    float microseconds = 0.0f;
};

// The split of the blocks that keeps all clusters resident (more CTAs than that run in a second round, which costs more
// than the shorter first one saves: 1 x 6144 x 6144 takes 11 us in four shares, 15.8 in six), and its time from
// measured parts: a CTA's start and end 5 us, a block 0.18 us + 1.65 ns a token (a third more where two CTAs share an SM
// that is full), and no less than its tiles take out of L2 at 13 TB/s.
template <int kTokens>
int plan_narrow(const ProductArgs &g, NarrowPlan *plan) {
    using T = Narrow<kTokens>;
    static Prepared prepared;
    static std::atomic<int> known[64][9];  // clusters of so many CTAs that a device holds at once
    if (int status = prepare_kernel(prepared, narrow_kernel<kTokens>, T::kSharedBytes)) return status;
    int device = 0;
    KREA2_CUDA(cudaGetDevice(&device));
    const uint32_t tiles = ((g.n + T::kRows - 1) / T::kRows) * ((g.m + kTokens - 1) / kTokens);
    uint32_t resident = 1;
    for (uint32_t shares = 1; shares <= 8 && shares <= g.blocks; shares++) {
        int clusters = known[device][shares].load(std::memory_order_relaxed);
        if (clusters == 0) {
            cudaLaunchAttribute attribute = {};
            const cudaLaunchConfig_t config = narrow_config<kTokens>(g, shares, attribute);
            KREA2_CUDA(cudaOccupancyMaxActiveClusters(&clusters, narrow_kernel<kTokens>, &config));
            if (clusters < 1) clusters = 1;
            known[device][shares].store(clusters, std::memory_order_relaxed);
        }
        if (shares > 1 && tiles > static_cast<uint32_t>(clusters)) break;
        plan->shares = shares;
        resident = static_cast<uint32_t>(clusters);
    }
    const uint32_t rounds = (tiles + resident - 1) / resident, steps = (g.blocks + plan->shares - 1) / plan->shares;
    const bool full = T::kPerSm == 2 && tiles * plan->shares > static_cast<uint32_t>(multiprocessors());
    const float block = (0.18f + 0.00165f * kTokens) * (full ? 1.33f : 1.0f);
    const float bytes = static_cast<float>(tiles) * g.blocks * T::kStageBytes;
    const float busy = rounds * (steps * block + 5.0f) + 4.0f, fed = bytes / 13e6f + 9.0f;
    plan->microseconds = busy > fed ? busy : fed;
    return KREA2_OK;
}

template <int kTokens>
int launch_narrow(cudaStream_t stream, const void *a, const void *w, size_t k, size_t a_stride, size_t w_stride, uint32_t shares, const ProductArgs &g) {
    CUtensorMap map_a, map_w;
    if (int status = operand_map(&map_a, a, g.m, k, a_stride, kTokens)) return status;
    if (int status = operand_map(&map_w, w, g.n, k, w_stride, Narrow<kTokens>::kRows)) return status;
    cudaLaunchAttribute attribute = {};
    cudaLaunchConfig_t config = narrow_config<kTokens>(g, shares, attribute);
    config.stream = stream;
    const cudaError_t status = cudaLaunchKernelEx(&config, narrow_kernel<kTokens>, map_a, map_w, g);
    if (status != cudaSuccess) return fail(KREA2_RUNTIME, "gemm_fp8_128 launch failed: %s", cudaGetErrorString(status));
    return KREA2_OK;
}

template <bool kBf16>
int launch_wide(cudaStream_t stream, const void *a, const void *w, size_t k, size_t a_stride, size_t w_stride, ProductArgs g) {
    using T = Wide;
    static Prepared prepared;
    if (int status = prepare_kernel(prepared, wide_kernel<kBf16>, T::kSharedBytes)) return status;
    CUtensorMap map_a, map_w;
    if (int status = operand_map(&map_a, a, g.m, k, a_stride, T::kRows)) return status;
    if (int status = operand_map(&map_w, w, g.n, k, w_stride, T::kRows / 2)) return status;
    // As in the int8 product: while a stays in L2 a column of tiles is walked top to bottom, once it is larger than that
    // groups of w panels of up to 48 MB are walked row by row.
    if (static_cast<size_t>(g.m) * k > (size_t(48) << 20)) {
        const size_t panel = static_cast<size_t>(T::kColumns) * k;
        g.panels = static_cast<uint32_t>((size_t(48) << 20) / panel);
        if (g.panels == 0) g.panels = 1;
    }
    const uint32_t tiles = ((g.m + 2 * T::kRows - 1) / (2 * T::kRows)) * ((g.n + T::kColumns - 1) / T::kColumns);
    const uint32_t pairs = static_cast<uint32_t>(multiprocessors()) / 2;
    wide_kernel<kBf16><<<2 * (tiles < pairs ? tiles : pairs), T::kThreads, T::kSharedBytes, stream>>>(map_a, map_w, g);
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return fail(KREA2_RUNTIME, "gemm_fp8_128 launch failed: %s", cudaGetErrorString(status));
    return KREA2_OK;
}

// The kernel and tile that are expected to take least.  The wide kernel takes 7.5 us and, for each round of tiles over the
// pairs of SMs, 1 us and 0.4 us a block.  It has the rows that fill its tiles: of 6144 columns and channels it takes 26 us for
// 128 to 512 rows and 29 for 768, the narrow one (its best tile) 16 for 64, 17 for 128, 20 for 192, 26 for 384, 32 for 512
// and 47 for 768.  Beyond 1024 rows the wide kernel is taken without an estimate.  That is right where its tiles fill the pairs
// (1043 x 6144 x 6144 48.6 us, narrow 59.6; 2048 x 1536 x 6144 25.3 and 30.4; 4608 x 1536 x 6144 47.3 and 59.8).  It costs
// few columns, which leave most pairs idle and whose channels it does not split: 1043 x 1536 x 6144 24.4 us, narrow 19.0;
// 1043 x 1536 x 16384 55.1 and 36.1; 4608 x 256 x 6144 25.0 and 16.4; 2048 x 256 x 16384 55.2 and 20.5; 1025 x 128 x 16384
// 54.1 and 11.4.
int launch_product(cudaStream_t stream, const void *a, const void *w, size_t k, size_t a_stride, size_t w_stride, const ProductArgs &g) {
    NarrowPlan plan;
#define KREA2_NARROW(tokens)                                                                       \
    do {                                                                                           \
        if (int status = plan_narrow<tokens>(g, &plan)) return status;                             \
        return launch_narrow<tokens>(stream, a, w, k, a_stride, w_stride, plan.shares, g);         \
    } while (0)
    if (g.m <= 16) KREA2_NARROW(16);
    if (g.m <= 32) KREA2_NARROW(32);
#undef KREA2_NARROW
    if (g.m <= 1024) {
        const uint32_t tiles = ((g.m + 2 * Wide::kRows - 1) / (2 * Wide::kRows)) * ((g.n + Wide::kColumns - 1) / Wide::kColumns);
        const uint32_t pairs = static_cast<uint32_t>(multiprocessors()) / 2;
        float least = ((tiles + pairs - 1) / pairs) * (0.40f * g.blocks + 1.0f) + 7.5f;
        int tokens = 0;
        uint32_t shares = 1;
#define KREA2_NARROW(candidate)                                                                    \
    do {                                                                                           \
        plan = NarrowPlan();                                                                       \
        if (int status = plan_narrow<candidate>(g, &plan)) return status;                          \
        if (plan.microseconds < least) least = plan.microseconds, tokens = candidate, shares = plan.shares; \
    } while (0)
        KREA2_NARROW(64);
        if (g.m > 64) KREA2_NARROW(96);
        if (g.m > 96) KREA2_NARROW(128);
        if (g.m > 128) KREA2_NARROW(160);
        if (g.m > 160) KREA2_NARROW(192);
#undef KREA2_NARROW
        switch (tokens) {
            case 64: return launch_narrow<64>(stream, a, w, k, a_stride, w_stride, shares, g);
            case 96: return launch_narrow<96>(stream, a, w, k, a_stride, w_stride, shares, g);
            case 128: return launch_narrow<128>(stream, a, w, k, a_stride, w_stride, shares, g);
            case 160: return launch_narrow<160>(stream, a, w, k, a_stride, w_stride, shares, g);
            case 192: return launch_narrow<192>(stream, a, w, k, a_stride, w_stride, shares, g);
            default: break;
        }
    }
    return g.bf16 ? launch_wide<true>(stream, a, w, k, a_stride, w_stride, g) : launch_wide<false>(stream, a, w, k, a_stride, w_stride, g);
}

}  // namespace

int take_product_status(int mask, int *value) {
    *value = 0;
    return g_product_launched.load(std::memory_order_relaxed) ? take_status_bits(g_product_status, mask, value) : KREA2_OK;
}

}  // namespace krea2

using namespace krea2;

extern "C" int krea2_gemm_fp8_128(krea2_stream stream, size_t m, const void *a, const void *w, const float *scale, const float *a_scale,
                                  void *c, size_t k_size, size_t a_stride, size_t w_stride, size_t n_size, size_t c_stride, int kind) {
    clear_error();
    const char *name = "gemm_fp8_128";
    KREA2_REQUIRE(m >= 1 && m <= 16777216, "%s: m %zu outside 1..16777216", name, m);
    KREA2_REQUIRE(k_size >= 1 && k_size <= 65536, "%s: k_size %zu outside 1..65536", name, k_size);
    KREA2_REQUIRE(n_size >= 1 && n_size <= 262144, "%s: n_size %zu outside 1..262144", name, n_size);
    KREA2_REQUIRE(a_stride >= k_size && a_stride % 16 == 0, "%s: a_stride %zu must be a multiple of 16, at least k_size %zu", name, a_stride, k_size);
    KREA2_REQUIRE(w_stride >= k_size && w_stride % 16 == 0, "%s: w_stride %zu must be a multiple of 16, at least k_size %zu", name, w_stride, k_size);
    KREA2_REQUIRE(c_stride >= n_size, "%s: c_stride %zu is below n_size %zu", name, c_stride, n_size);
    KREA2_REQUIRE(kind == KREA2_F16 || kind == KREA2_BF16, "%s: kind %d is neither KREA2_F16 nor KREA2_BF16", name, kind);
    KREA2_REQUIRE(a && w && scale && a_scale && c, "%s: null buffer", name);
    KREA2_REQUIRE(aligned16(a) && aligned16(w), "%s: the codes must be 16-byte aligned", name);
    KREA2_REQUIRE(reinterpret_cast<uintptr_t>(c) % 2 == 0 && reinterpret_cast<uintptr_t>(scale) % 4 == 0 &&
                      reinterpret_cast<uintptr_t>(a_scale) % 4 == 0,
                  "%s: buffers must be aligned to their element size", name);
    const ProductArgs g = {scale, a_scale, static_cast<uint16_t *>(c), static_cast<uint32_t>(m), static_cast<uint32_t>(n_size),
                           static_cast<uint32_t>((k_size + kBlock - 1) / kBlock), c_stride, kind == KREA2_BF16 ? 1u : 0u,
                           aligned16(c) && c_stride % 8 == 0 ? 1u : 0u, 0u};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    g_product_launched.store(true, std::memory_order_relaxed);
    return launch_product(s, a, w, k_size, a_stride, w_stride, g);
}
