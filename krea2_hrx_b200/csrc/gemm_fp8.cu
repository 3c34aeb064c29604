// The product of two e4m3 code matrices under block scales (new with this library; the reference's products are int8):
//   c[i][j] = T(sum over blocks g of 128 channels: a_scale[i][g] * w_scale[j/128][g] * sum of a[i][k] * w[j][k] in g)
// The scales are arbitrary f32 values, so a block's sum has to leave the tensor cores before the next may be added: a
// tcgen05.mma of one block (K = 128, four instructions) goes to one of two accumulators in tensor memory, and eight warps
// read it, scale it and add it to the output they hold in registers, while the other accumulator fills.
//
// Two kernels:
//   wide    a pair of CTAs owns 256 rows of a and 256 of w (as the int8 pair kernel does); an epilogue thread owns one row
//           and 128 outputs, whose scale of a block is one number
//   narrow  few rows of a: 128 rows of w are the M side and up to 256 rows of a the N side of a CTA, the blocks of 128
//           channels are split over a cluster of up to eight CTAs, whose partial outputs are added over distributed shared
//           memory in the order of their rank: no workspace, no atomics, the same bits every time
#include "tensor_core.cuh"

namespace krea2 {
namespace {

__device__ int g_product_status = 0;  // folded into krea2_device_status by take_product_status
constexpr int kProductTimedOut = 64;

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

__device__ __forceinline__ uint32_t pack_outputs(float lo, float hi, uint32_t bf16) {
    if (bf16) return bits_of<true>(lo) | (static_cast<uint32_t>(bits_of<true>(hi)) << 16);
    return bits_of<false>(lo) | (static_cast<uint32_t>(bits_of<false>(hi)) << 16);
}

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

// ---------------------------------------------------------------- wide
struct Wide {
    static constexpr int kStages = 6;
    static constexpr int kRows = 128;     // of a, and of w, per CTA
    static constexpr int kColumns = 256;  // of a tile
    static constexpr int kWarps = 8;      // epilogue: two per 32-lane quarter, each with half of the columns
    static constexpr int kThreads = (kWarps + 2) * 32;
    static constexpr int kOperandBytes = kRows * kBlock;
    static constexpr int kStageBytes = 2 * kOperandBytes;
    static constexpr int kStagingRow = 80;             // 32 outputs, and 16 bytes that spread the rows over the banks
    static constexpr int kStagingBytes = 32 * kStagingRow;  // per warp
    static constexpr int kSharedBytes = kStages * kStageBytes + 1024 + 256 + kWarps * kStagingBytes;
};

// Writes 32 outputs of each of the warp's 32 rows through its staging area, so that rows leave in 64-byte pieces.
__device__ __forceinline__ void store_wide(const ProductArgs &g, const float2 *values, uint32_t row0, uint32_t column0, uint8_t *staging, int lane) {
    uint4 *mine = reinterpret_cast<uint4 *>(staging + lane * Wide::kStagingRow);
#pragma unroll
    for (int i = 0; i < 4; i++)
        mine[i] = make_uint4(pack_outputs(values[4 * i].x, values[4 * i].y, g.bf16), pack_outputs(values[4 * i + 1].x, values[4 * i + 1].y, g.bf16),
                             pack_outputs(values[4 * i + 2].x, values[4 * i + 2].y, g.bf16), pack_outputs(values[4 * i + 3].x, values[4 * i + 3].y, g.bf16));
    __syncwarp();
    if (g.aligned) {
        const uint32_t column = column0 + (lane & 3) * 8;
#pragma unroll
        for (int r = 0; r < 32; r += 8) {
            const uint32_t local = r + (lane >> 2), row = row0 + local;
            if (row >= g.m || column >= g.n) continue;
            const uint8_t *from = staging + local * Wide::kStagingRow + (lane & 3) * 16;
            uint16_t *to = g.c + row * g.c_stride + column;
            if (column + 8 <= g.n) {
                *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(from);
            } else {
                for (uint32_t i = 0; column + i < g.n; i++) to[i] = reinterpret_cast<const uint16_t *>(from)[i];
            }
        }
    } else if (column0 + lane < g.n) {
        for (uint32_t local = 0; local < 32 && row0 + local < g.m; local++)
            g.c[(row0 + local) * g.c_stride + column0 + lane] = reinterpret_cast<const uint16_t *>(staging + local * Wide::kStagingRow)[lane];
    }
    __syncwarp();
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Wide::kThreads, 1)
wide_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const ProductArgs g) {
    using T = Wide;
    extern __shared__ uint8_t shared_raw[];
    uint8_t *shared = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(shared + T::kStages * T::kStageBytes);
    uint64_t *empty = full + T::kStages, *sum_full = empty + T::kStages, *sum_empty = sum_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sum_empty + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    // [0], [1] the stages each CTA's producer filled (in the leader), [2], [3] each CTA's abort flag (in both)
    volatile uint32_t *exchange = reinterpret_cast<volatile uint32_t *>(tmem_slot + 2);
    uint8_t *staging = shared + T::kStages * T::kStageBytes + 256;
    const Abort abort = {abort_flag, &g_product_status, kProductTimedOut};

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
        for (int s = 0; s < 2; s++) {
            barrier_init(sum_full + s, 1);
            barrier_init(sum_empty + s, 2 * T::kWarps);
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
    const uint32_t tmem = *tmem_slot;

    if (warp == T::kWarps) {
        if (lane == 0) {
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
                    load_tile_pair(dst + T::kOperandBytes, &map_w, leader_full, static_cast<int>(b * kBlock), static_cast<int>(column + rank * T::kRows));
                    issued++;
                    if (++stage == T::kStages) stage = 0, phase ^= 1u;
                }
            }
        }
    } else if (warp == T::kWarps + 1) {
        if (leader && lane == 0) {
            constexpr uint32_t idesc = product_descriptor(2 * T::kRows, T::kColumns);
            uint32_t stage = 0, phase = 0, count = 0;
            bool alive = true;
            for (uint32_t tile = pair; alive && tile < tiles; tile += pairs) {
                for (uint32_t b = 0; b < g.blocks; b++, count++) {
                    const uint32_t s = count & 1u;
                    if (!(alive = barrier_wait(sum_empty + s, ((count >> 1) & 1u) ^ 1u, abort) && barrier_wait(full + stage, phase, abort))) break;
                    tensor_fence_after();
                    const uint32_t at = smem_address(shared + stage * T::kStageBytes);
                    const uint64_t a = operand_descriptor(at), w = operand_descriptor(at + T::kOperandBytes);
#pragma unroll
                    for (int k = 0; k < kBlock / kStep; k++) issue_product<2>(tmem + s * T::kColumns, a + 2 * k, w + 2 * k, idesc, k != 0);
                    tensor_commit_pair(empty + stage);
                    tensor_commit_pair(sum_full + s);
                    if (++stage == T::kStages) stage = 0, phase ^= 1u;
                }
            }
        }
    } else {
        const int quarter = warp & 3, half = warp >> 2;
        uint32_t count = 0;
        bool alive = true;
        const uint32_t scale_rows = (g.n + kBlock - 1) / kBlock;
        for (uint32_t tile = pair; alive && tile < tiles; tile += pairs) {
            uint32_t row0, column0;
            origin(tile, row0, column0);
            row0 += quarter * 32;
            column0 += half * kBlock;
            const uint32_t row = min(row0 + lane, g.m - 1), scale_row = min(column0 / kBlock, scale_rows - 1);
            const float *a_scale = g.a_scale + static_cast<size_t>(row) * g.blocks, *w_scale = g.w_scale + static_cast<size_t>(scale_row) * g.blocks;
            float2 out[64];
#pragma unroll
            for (int i = 0; i < 64; i++) out[i] = make_float2(0.0f, 0.0f);
            float next = __ldg(a_scale) * __ldg(w_scale);
            for (uint32_t b = 0; b < g.blocks; b++, count++) {
                const uint32_t s = count & 1u;
                const float2 scale = make_float2(next, next);
                if (b + 1 < g.blocks) next = __ldg(a_scale + b + 1) * __ldg(w_scale + b + 1);
                alive = __all_sync(0xffffffffu, barrier_wait(sum_full + s, (count >> 1) & 1u, abort));
                if (!alive) break;
                tensor_fence_after();
                const uint32_t from = tmem + s * T::kColumns + half * kBlock + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    float part[16];
                    tensor_load_16(from + c * 16, part);
                    tensor_loads_done();
                    if (c == 7) {  // everything has been read: the accumulator may be overwritten
                        tensor_fence_before();
                        __syncwarp();
                        if (lane == 0) barrier_arrive_at(cluster_address(sum_empty + s, 0));
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) out[c * 8 + i] = fma_pair(make_float2(part[2 * i], part[2 * i + 1]), scale, out[c * 8 + i]);
                }
            }
            if (!alive) break;
#pragma unroll
            for (int c = 0; c < 4; c++)
                store_wide(g, out + c * 16, row0, column0 + c * 32, staging + warp * T::kStagingBytes, lane);
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
constexpr int power_of_two(int n) { return n <= 32 ? 32 : 2 * power_of_two((n + 1) / 2); }

template <int kTokens>
struct Narrow {
    static constexpr int kRows = 128;                        // of w
    static constexpr int kWarps = kTokens <= 64 ? 4 : 8;     // epilogue
    static constexpr int kThreads = (kWarps + 2) * 32;
    static constexpr int kColumns = kTokens / (kWarps / 4);  // tokens of one epilogue thread
    static constexpr int kStageBytes = (kRows + kTokens) * kBlock;
    // Two CTAs share an SM where both sets of accumulators fit its tensor memory (512 columns, 2 * kTokens each): their
    // shared memory has to keep a second one out otherwise, since a CTA that waits for tensor memory holds up its cluster.
    static constexpr int kTensorColumns = power_of_two(2 * kTokens);
    static constexpr int kPerSm = kTensorColumns <= 256 ? 2 : 1;
    static constexpr int kStages = ((kPerSm == 2 ? 108 : 216) * 1024 - 2048 - 2 * kTokens * 4) / kStageBytes;
    static constexpr int kSharedBytes = kStages * kStageBytes + 1024 + 256 + 2 * kTokens * 4;
    static_assert(kStages >= 2 && kStages * kStageBytes >= kRows * kTokens * 4, "the partial outputs take the stages' place");
    static_assert(kPerSm * kSharedBytes <= 227 * 1024 && (kPerSm + 1) * (kSharedBytes + 1024) > 228 * 1024, "CTAs per SM");
};

template <int kTokens>
__global__ void __launch_bounds__(Narrow<kTokens>::kThreads, Narrow<kTokens>::kPerSm)
narrow_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const ProductArgs g) {
    using T = Narrow<kTokens>;
    extern __shared__ uint8_t shared_raw[];
    uint8_t *shared = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(shared + T::kStages * T::kStageBytes);
    uint64_t *empty = full + T::kStages, *sum_full = empty + T::kStages, *sum_empty = sum_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sum_empty + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    float *scales = reinterpret_cast<float *>(shared + T::kStages * T::kStageBytes + 256);  // two blocks' token scales
    float *partial = reinterpret_cast<float *>(shared);                                     // [kTokens][128], once the stages are done with
    const Abort abort = {abort_flag, &g_product_status, kProductTimedOut};

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
        for (int s = 0; s < 2; s++) {
            barrier_init(sum_full + s, 1);
            barrier_init(sum_empty + s, T::kWarps);
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
    const uint32_t tmem = *tmem_slot;

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
        if (lane == 0) {
            constexpr uint32_t idesc = product_descriptor(T::kRows, kTokens);
            for (uint32_t b = first, count = 0; b < last; b++, count++) {
                const uint32_t s = count & 1u, stage = count % T::kStages;
                if (!barrier_wait(sum_empty + s, ((count >> 1) & 1u) ^ 1u, abort) || !barrier_wait(full + stage, (count / T::kStages) & 1u, abort)) break;
                tensor_fence_after();
                const uint32_t at = smem_address(shared + stage * T::kStageBytes);
                const uint64_t w = operand_descriptor(at), a = operand_descriptor(at + T::kRows * kBlock);
#pragma unroll
                for (int k = 0; k < kBlock / kStep; k++) issue_product<1>(tmem + s * kTokens, w + 2 * k, a + 2 * k, idesc, k != 0);
                tensor_commit(empty + stage);
                tensor_commit(sum_full + s);
            }
        }
    } else {
        // A thread owns one row of w and kColumns tokens.  The tokens' scales of a block (times the weights', which the
        // whole CTA shares) lie in shared memory, two blocks of them in turn.
        const int quarter = warp & 3, group = warp >> 2;
        const float *w_scale = g.w_scale + static_cast<size_t>(blockIdx.y) * g.blocks;
        const uint32_t token = threadIdx.x;
        const float *a_scale = g.a_scale + static_cast<size_t>(min(m0 + token, g.m - 1)) * g.blocks;
        const bool loads = token < kTokens;
        float2 out[T::kColumns / 2];
#pragma unroll
        for (int i = 0; i < T::kColumns / 2; i++) out[i] = make_float2(0.0f, 0.0f);
        float next = loads ? __ldg(a_scale + first) * __ldg(w_scale + first) : 0.0f;
        for (uint32_t b = first, count = 0; b < last; b++, count++) {
            const uint32_t s = count & 1u;
            if (loads) {
                scales[s * kTokens + token] = next;
                if (b + 1 < last) next = __ldg(a_scale + b + 1) * __ldg(w_scale + b + 1);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(T::kWarps * 32) : "memory");
            if (!__all_sync(0xffffffffu, barrier_wait(sum_full + s, (count >> 1) & 1u, abort))) *abort_flag = 1;  // all leave the loop below
            tensor_fence_after();
            const uint32_t from = tmem + s * kTokens + group * T::kColumns + (static_cast<uint32_t>(quarter * 32) << 16);
            const float *mine = scales + s * kTokens + group * T::kColumns;
#pragma unroll
            for (int c = 0; c < T::kColumns; c += 16) {
                float part[16];
                tensor_load_16(from + c, part);
                tensor_loads_done();
                if (c + 16 == T::kColumns) {
                    tensor_fence_before();
                    __syncwarp();
                    if (lane == 0) barrier_arrive(sum_empty + s);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4 scale = *reinterpret_cast<const float4 *>(mine + c + 4 * i);
                    float2 &lo = out[(c + 4 * i) / 2], &hi = out[(c + 4 * i) / 2 + 1];
                    lo = fma_pair(make_float2(part[4 * i], part[4 * i + 1]), make_float2(scale.x, scale.y), lo);
                    hi = fma_pair(make_float2(part[4 * i + 2], part[4 * i + 3]), make_float2(scale.z, scale.w), hi);
                }
            }
        }
        // The last sum has been read, so every product has read its stage and every load has landed.
        asm volatile("bar.sync 1, %0;" ::"n"(T::kWarps * 32) : "memory");
        if (!*abort_flag) {
            const uint32_t row = quarter * 32 + lane;
#pragma unroll
            for (int i = 0; i < T::kColumns / 2; i++) {
                partial[(group * T::kColumns + 2 * i) * T::kRows + row] = out[i].x;
                partial[(group * T::kColumns + 2 * i + 1) * T::kRows + row] = out[i].y;
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
        for (uint32_t r = 0; r < shares; r++) {
            const float4 share = cluster_load(cluster_address(partial + item * 4, r));
            total.x += share.x, total.y += share.y, total.z += share.z, total.w += share.w;
        }
        const uint2 packed = make_uint2(pack_outputs(total.x, total.y, g.bf16), pack_outputs(total.z, total.w, g.bf16));
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
int launch_narrow(cudaStream_t stream, const void *a, const void *w, size_t k, size_t a_stride, size_t w_stride, uint32_t shares, const ProductArgs &g) {
    using T = Narrow<kTokens>;
    static Prepared prepared;
    if (int status = prepare_kernel(prepared, narrow_kernel<kTokens>, T::kSharedBytes)) return status;
    CUtensorMap map_a, map_w;
    if (int status = operand_map(&map_a, a, g.m, k, a_stride, kTokens)) return status;
    if (int status = operand_map(&map_w, w, g.n, k, w_stride, T::kRows)) return status;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(shares, (g.n + T::kRows - 1) / T::kRows, (g.m + kTokens - 1) / kTokens);
    config.blockDim = dim3(T::kThreads);
    config.dynamicSmemBytes = T::kSharedBytes;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = shares;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    const cudaError_t status = cudaLaunchKernelEx(&config, narrow_kernel<kTokens>, map_a, map_w, g);
    if (status != cudaSuccess) return fail(KREA2_RUNTIME, "gemm_fp8_128 launch failed: %s", cudaGetErrorString(status));
    return KREA2_OK;
}

int launch_wide(cudaStream_t stream, const void *a, const void *w, size_t k, size_t a_stride, size_t w_stride, ProductArgs g) {
    using T = Wide;
    static Prepared prepared;
    if (int status = prepare_kernel(prepared, wide_kernel, T::kSharedBytes)) return status;
    CUtensorMap map_a, map_w;
    if (int status = operand_map(&map_a, a, g.m, k, a_stride, T::kRows)) return status;
    if (int status = operand_map(&map_w, w, g.n, k, w_stride, T::kRows)) return status;
    // As in the int8 product: while a stays in L2 a column of tiles is walked top to bottom, once it is larger than that
    // groups of w panels of up to 48 MB are walked row by row.
    if (static_cast<size_t>(g.m) * k > (size_t(48) << 20)) {
        const size_t panel = static_cast<size_t>(T::kColumns) * k;
        g.panels = static_cast<uint32_t>((size_t(48) << 20) / panel);
        if (g.panels == 0) g.panels = 1;
    }
    const uint32_t tiles = ((g.m + 2 * T::kRows - 1) / (2 * T::kRows)) * ((g.n + T::kColumns - 1) / T::kColumns);
    const uint32_t pairs = static_cast<uint32_t>(multiprocessors()) / 2;
    wide_kernel<<<2 * (tiles < pairs ? tiles : pairs), T::kThreads, T::kSharedBytes, stream>>>(map_a, map_w, g);
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return fail(KREA2_RUNTIME, "gemm_fp8_128 launch failed: %s", cudaGetErrorString(status));
    return KREA2_OK;
}

}  // namespace

int take_product_status(int *value) {
    KREA2_CUDA(cudaMemcpyFromSymbol(value, g_product_status, sizeof(int)));
    if (*value != 0) {
        const int zero = 0;
        KREA2_CUDA(cudaMemcpyToSymbol(g_product_status, &zero, sizeof(int)));
    }
    return KREA2_OK;
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
    if (m > 256) return launch_wide(s, a, w, k_size, a_stride, w_stride, g);
    // Narrow: as many shares as give each SM two CTAs of work, a block of channels each at least.
    const uint32_t columns = (g.n + 127) / 128;
    uint32_t shares = 1;
    while (shares < 8 && 2 * shares <= g.blocks && columns * shares < 2u * static_cast<uint32_t>(multiprocessors())) shares *= 2;
    if (m <= 16) return launch_narrow<16>(s, a, w, k_size, a_stride, w_stride, shares, g);
    if (m <= 32) return launch_narrow<32>(s, a, w, k_size, a_stride, w_stride, shares, g);
    if (m <= 64) return launch_narrow<64>(s, a, w, k_size, a_stride, w_stride, shares, g);
    if (m <= 96) return launch_narrow<96>(s, a, w, k_size, a_stride, w_stride, shares, g);
    return launch_narrow<128>(s, a, w, k_size, a_stride, w_stride, shares, g);
}
