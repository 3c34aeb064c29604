// Attention of queries to an encoder's states of another length (new with this library: the reference's attention is
// over one sequence, whose values it transposes first): batches whose items count different numbers of keys, a key
// mask, bf16 and f16, heads of 8 to 128 channels, rows at any 16-byte pitch.
//   out[b][i][h] = sum_j p_j v[b][j][h'] / sum_j p_j,  p_j = exp(scale q[b][i][h] . k[b][j][h'])
// over the keys j < kv_lengths[b] whose mask byte is not zero, h' = h / (q_heads / kv_heads); zero where there is none.
//
// One pass over the keys with a running maximum and sum.  A CTA owns up to 128 rows of one key head: the query heads that
// share it are packed (row r is query r / shares, head r % shares of the key head's), so a single query fills as many rows as
// heads share its keys, and one tile load or store moves the rows of 128 / shares queries.  S = Q K^T and O += P V are
// tcgen05.mma kind::f16 with f32 accumulators in tensor memory; K and V tiles of 128 keys arrive by TMA as they lie (V is
// the second product's B operand with its channels innermost, so nothing is transposed), a thread owns one row's softmax
// and writes P over S in tensor memory.  Two CTAs share an SM: one's softmax, its start and its output run under the
// other's products.
//
// Bound by the chain of a row tile, scores -> softmax -> second product, of which an SM has two under way: 16384 queries of
// 48/12 heads of 128 to 512 keys take 240-265 us (0.78-0.86 PFLOP/s: four key tiles a CTA, so its start and end weigh), 4608
// to 4608 480 us (1.09 PFLOP/s, tensor pipe 0.5 active).  Heads of 64 do half the products for the same exponentials and are
// bound by those; a mask's selects cost 22-30 % more softmax.  One row tile per head of a single query: 7.3-10 us for 512 keys.
// Where the rows do not fill the device, a cluster of up to eight CTAs splits the keys of a row tile and adds its partial
// outputs over distributed shared memory in the order of their rank: no workspace, the same bits every time.
#include <atomic>
#include <cmath>

#include "tensor_core.cuh"

namespace krea2 {
namespace {

__device__ int g_cross_status = 0;  // folded into krea2_device_status by take_cross_status
std::atomic<bool> g_cross_launched{false};  // whether the word is worth a copy: a chain's status reads are not to wait for it
constexpr int kCrossTimedOut = KREA2_STATUS_CROSS_ATTENTION;

constexpr int kRows = 128;  // query rows of a CTA, keys of a tile

// Weights are rounded to the tensors' type for the second product (half a step each; their sum is taken before), as the tensor
// cores need them: the error of an output against 64 bits is 1.2-1.4 times that of weights in f32 (bf16 0.0021-0.0023 against
// 0.0017 of it, f16 0.00026-0.00029 against 0.00021).  A weight
// far below its row's largest would be lost in f16, whose numbers end at 2^-25, and many such may count, so f16 weights
// carry a factor of 2^7, which drops out with the sum: the largest is 2^15 (the reference lags by 2^8 at most), and what is
// 2^-32 of the reference still counts.
template <bool kBf16>
constexpr float kLift = kBf16 ? 0.0f : 7.0f;

struct CrossArgs {
    const int32_t *kv_lengths;
    const uint8_t *key_mask;
    uint16_t *out;
    uint32_t q_len, kv_len, shares, queries, head_dim;  // shares: query heads of a key head; queries of a row tile: 128 / shares
    size_t out_batch_stride, out_stride, mask_stride;
    uint32_t q_batches, k_batches, v_batches;  // 1 where every item of the batch shares its queries (keys, values), 0 otherwise
    float scale_log2;                          // softmax scale times log2(e)
};

// kD: channels of a head as the tiles hold them, 64 or 128; those past head_dim are zero.
template <int kD>
struct Cross {
    static constexpr int kSoftmaxWarps = 4, kLoadWarp = 4, kProductWarp = 5, kValueWarp = 6, kMaskWarp = 7;
    static constexpr int kThreads = 8 * 32;  // a warpgroup of softmax, one of the others
    // A row's 128 scores stay in registers: the softmax takes what the other warpgroup does without of the launch's 128.
    static constexpr int kSoftmaxRegisters = 192, kOtherRegisters = 64;
    static_assert(kSoftmaxRegisters + kOtherRegisters <= 2 * 128, "registers of the launch");
    static constexpr int kSubtileBytes = kRows * 128;  // 128 rows of 64 channels: one 128-byte swizzled column block
    static constexpr int kTileBytes = kD / 64 * kSubtileBytes;
    static constexpr int kStages = kD == 64 ? 2 : 1;
    static constexpr int kTensorColumns = 256;  // S (then P) at 0, O at 128
    static constexpr int kBarrierBytes = 256, kStatsBytes = kRows * 8;
    static constexpr int kSharedBytes = (1 + 2 * kStages) * kTileBytes + 1024 + kBarrierBytes + kStatsBytes;
    static_assert(2 * kStages * kTileBytes >= kRows * kD * 4, "the partial outputs take the place of keys and values");
    static_assert(2 * (kSharedBytes + 1024) <= 228 * 1024 && 3 * kSharedBytes > 228 * 1024, "two CTAs share an SM and its tensor memory");
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The largest of three; a NaN among them stays one, so that a row that meets a NaN becomes NaN through its maximum.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// kind::f16: f32 accumulate (1 at bit 4), A and B f16 (0) or bf16 (1) at bits 7 and 10, B with its N side innermost at bit
// 16, N/8 at bit 17, M/16 at bit 24.
template <bool kBf16>
__device__ constexpr uint32_t attention_descriptor(int n, bool n_inner) {
    return (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | (n_inner ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
           (static_cast<uint32_t>(kRows >> 4) << 24);
}
// A tile whose N side is innermost: rows of 64 channels (128 bytes, swizzled), eight rows of K to the next 1024 bytes, the
// next 64 channels one subtile on.
__device__ __forceinline__ uint64_t value_descriptor(uint32_t address, uint32_t subtile_bytes) {
    return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | (static_cast<uint64_t>(subtile_bytes >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void issue_f16(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem), "l"(a), "l"(b), "r"(idesc),
                 "r"(accumulate)
                 : "memory");
}
// A from tensor memory: 128 lanes of 16-bit pairs, eight columns per K = 16.
__device__ __forceinline__ void issue_f16_tensor_a(uint32_t tmem, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(tmem), "r"(a), "l"(b),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}

// Which keys of a tile count where the first `left` of them do.
__device__ __forceinline__ void tail_words(uint32_t left, uint32_t (&word)[4]) {
#pragma unroll
    for (uint32_t w = 0; w < 4; w++) word[w] = left >= 32 * w + 32 ? 0xffffffffu : left <= 32 * w ? 0u : (1u << (left - 32 * w)) - 1u;
}

template <int kD, bool kBf16>
__global__ void __launch_bounds__(Cross<kD>::kThreads, 2)
cross_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ CUtensorMap map_out, const CrossArgs g) {
    using T = Cross<kD>;
    extern __shared__ uint8_t shared_raw[];
    uint8_t *q_tile = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *k_tiles = q_tile + T::kTileBytes, *v_tiles = k_tiles + T::kStages * T::kTileBytes;
    uint64_t *q_full = reinterpret_cast<uint64_t *>(v_tiles + T::kStages * T::kTileBytes);
    uint64_t *k_full = q_full + 1, *k_empty = k_full + T::kStages, *v_full = k_empty + T::kStages, *v_empty = v_full + T::kStages;
    uint64_t *v_ready = v_empty + T::kStages, *s_full = v_ready + T::kStages, *p_full = s_full + 1, *o_full = p_full + 2, *out_full = o_full + 1, *words_full = out_full + 1;
    uint32_t *words = reinterpret_cast<uint32_t *>(words_full + 4);  // [4][4]: which keys of a tile count, four tiles in turn
    uint32_t *tmem_slot = words + 16;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    float *stats = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(q_full) + T::kBarrierBytes);  // [128][2]: reference and sum of a row
    float *partial = reinterpret_cast<float *>(k_tiles);                                              // [128][kD], once the products are done
    const Abort abort = {abort_flag, &g_cross_status, kCrossTimedOut};

    const int warp = static_cast<int>(uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const uint32_t parts = cluster_size(), rank = cluster_rank();
    const uint32_t query0 = blockIdx.x / parts * g.queries, kv_head = blockIdx.y, batch = blockIdx.z;
    const uint32_t rows = min(g.queries, g.q_len - query0) * g.shares;
    int32_t length = static_cast<int32_t>(g.kv_len);
    if (g.kv_lengths) length = min(max(g.kv_lengths[batch], 0), length);
    const uint32_t keys = static_cast<uint32_t>(length), tiles = (keys + kRows - 1) / kRows;
    const uint32_t first = static_cast<uint32_t>(static_cast<uint64_t>(tiles) * rank / parts);
    const uint32_t last = static_cast<uint32_t>(static_cast<uint64_t>(tiles) * (rank + 1) / parts);
    const uint32_t count = last - first;
    uint32_t issued = 0;  // loader warps: tiles requested

    if (threadIdx.x == 0) {
        barrier_init(q_full, 1);
        for (int s = 0; s < T::kStages; s++) {
            barrier_init(k_full + s, 1);
            barrier_init(k_empty + s, 1);
            barrier_init(v_full + s, 1);
            barrier_init(v_empty + s, 1);
            barrier_init(v_ready + s, 1);
        }
        barrier_init(s_full, 1);
        barrier_init(p_full, T::kSoftmaxWarps);
        barrier_init(p_full + 1, T::kSoftmaxWarps);
        barrier_init(o_full, 1);
        barrier_init(out_full, T::kSoftmaxWarps);
        for (int s = 0; s < 4; s++) barrier_init(words_full + s, 1);
        *abort_flag = 0;
        barrier_init_done();
    }
    if (warp == T::kProductWarp) {
        __syncwarp();
        tensor_alloc<1>(tmem_slot, T::kTensorColumns);
    }
    tensor_fence_before();
    __syncthreads();
    tensor_fence_after();
    const uint32_t tmem = uniform(*tmem_slot);
    float reference = -INFINITY, sum = 0.0f;  // a softmax thread's row, in units of log2
    bool alive = true;

    if (warp >= T::kSoftmaxWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::kOtherRegisters));
        // Keys that do not count have the weight zero, but zero times what lies in their values may be NaN: a warp clears their
        // rows once the tile is there and before the second product reads it.
        auto clear = [&](uint32_t i, const uint32_t (&word)[4]) {
            const uint32_t s = i % T::kStages;
            if (!barrier_wait_warp(v_full + s, (i / T::kStages) & 1u, abort)) return false;
            uint8_t *tile = v_tiles + s * T::kTileBytes;
            constexpr uint32_t kPieces = kD / 8, kAtOnce = 32 / kPieces;  // of 16 bytes in a row, rows
            const uint32_t at = lane % kPieces, base = (at >> 3) * T::kSubtileBytes + (at & 7u) * 16;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                if (word[w] == 0xffffffffu) continue;
#pragma unroll 4
                for (uint32_t bit = lane / kPieces; bit < 32; bit += kAtOnce)
                    if (!((word[w] >> bit) & 1u)) *reinterpret_cast<uint4 *>(tile + base + (w * 32 + bit) * 128) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) barrier_arrive(v_ready + s);
            return true;
        };
        if (warp == T::kLoadWarp) {
            const bool elected = elect_lane();
            if (count && elected) {
                barrier_expect(q_full, kD / 64 * g.queries * g.shares * 128);
#pragma unroll
                for (int sub = 0; sub < kD / 64; sub++)
                    load_tile_4d(q_tile + sub * T::kSubtileBytes, &map_q, q_full, sub * 64, static_cast<int>(kv_head * g.shares), static_cast<int>(query0),
                                 static_cast<int>(g.q_batches ? 0 : batch));
            }
            __syncwarp();
            for (uint32_t i = 0; i < count; i++, issued++) {
                const uint32_t s = i % T::kStages;
                if (!barrier_wait_warp(k_empty + s, ((i / T::kStages) & 1u) ^ 1u, abort)) break;
                if (elected) {
                    barrier_expect(k_full + s, T::kTileBytes);
#pragma unroll
                    for (int sub = 0; sub < kD / 64; sub++)
                        load_tile_4d(k_tiles + s * T::kTileBytes + sub * T::kSubtileBytes, &map_k, k_full + s, sub * 64, static_cast<int>(kv_head),
                                     static_cast<int>((first + i) * kRows), static_cast<int>(g.k_batches ? 0 : batch));
                }
                __syncwarp();
            }
        } else if (warp == T::kValueWarp) {
            const bool elected = elect_lane();
            for (uint32_t i = 0; i < count; i++, issued++) {
                const uint32_t s = i % T::kStages;
                if (!barrier_wait_warp(v_empty + s, ((i / T::kStages) & 1u) ^ 1u, abort)) break;
                if (elected) {
                    barrier_expect(v_full + s, T::kTileBytes);
#pragma unroll
                    for (int sub = 0; sub < kD / 64; sub++)
                        load_tile_4d(v_tiles + s * T::kTileBytes + sub * T::kSubtileBytes, &map_v, v_full + s, sub * 64, static_cast<int>(kv_head),
                                     static_cast<int>((first + i) * kRows), static_cast<int>(g.v_batches ? 0 : batch));
                }
                __syncwarp();
                if (!g.key_mask && (first + i + 1) * kRows > keys) {
                    uint32_t word[4];
                    tail_words(keys - (first + i) * kRows, word);
                    if (!clear(i, word)) break;
                }
            }
        } else if (warp == T::kMaskWarp && g.key_mask) {
            // Which keys of a tile count goes to the softmax two tiles ahead, and their values are cleared as they land.  (Every
            // tile of a masked launch waits for this warp, so that it meets each phase of the barriers.)
            auto words_of = [&](uint32_t i, uint32_t (&word)[4]) {
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const uint32_t key = (first + i) * kRows + w * 32 + lane;
                    word[w] = __ballot_sync(0xffffffffu, i < count && key < keys && g.key_mask[batch * g.mask_stride + key] != 0);
                }
            };
            auto publish = [&](uint32_t i, const uint32_t (&word)[4]) {
                if (i >= count) return;
                if (lane < 4) words[(i & 3u) * 4 + lane] = lane == 0 ? word[0] : lane == 1 ? word[1] : lane == 2 ? word[2] : word[3];
                __syncwarp();
                if (lane == 0) barrier_arrive(words_full + (i & 3u));
            };
            uint32_t word[4], next[4], after[4];
            words_of(0, word);
            words_of(1, next);
            publish(0, word);
            publish(1, next);
            for (uint32_t i = 0; i < count; i++) {
                words_of(i + 2, after);
                if (!clear(i, word)) break;
                // The tile that used these words four tiles ago has been through its second product: this tile's values came
                // in its place or a later one's.
                publish(i + 2, after);
#pragma unroll
                for (int w = 0; w < 4; w++) word[w] = next[w], next[w] = after[w];
            }
        } else if (warp == T::kProductWarp) {
            const bool elected = elect_lane();
            constexpr uint32_t scores_idesc = attention_descriptor<kBf16>(kRows, false), values_idesc = attention_descriptor<kBf16>(kD, true);
            if (count) alive = barrier_wait_warp(q_full, 0, abort);
            // The pipe runs one thread's products in issue order and a commit covers all that was issued before it: the scores of
            // a tile overwrite the weights of the one before only after the second product has read them, and the softmax that
            // sees new scores may rescale O.
            auto scores = [&](uint32_t i) {
                const uint32_t s = i % T::kStages;
                if (!barrier_wait_warp(k_full + s, (i / T::kStages) & 1u, abort)) return false;
                tensor_fence_after();
                if (elected) {
#pragma unroll
                    for (int sub = 0; sub < kD / 64; sub++) {
                        const uint64_t a = operand_descriptor(smem_address(q_tile + sub * T::kSubtileBytes));
                        const uint64_t b = operand_descriptor(smem_address(k_tiles + s * T::kTileBytes + sub * T::kSubtileBytes));
#pragma unroll
                        for (int k = 0; k < 4; k++) issue_f16(tmem, a + 2 * k, b + 2 * k, scores_idesc, sub != 0 || k != 0);
                    }
                    tensor_commit(s_full);
                    tensor_commit(k_empty + s);
                }
                __syncwarp();
                return true;
            };
            if (count && alive) alive = scores(0);
            for (uint32_t i = 0; alive && i < count; i++) {
                const uint32_t s = i % T::kStages;
                const bool cleared = g.key_mask || (first + i + 1) * kRows > keys;
                alive = cleared ? barrier_wait_warp(v_ready + s, g.key_mask ? (i / T::kStages) & 1u : 0u, abort)
                                : barrier_wait_warp(v_full + s, (i / T::kStages) & 1u, abort);
                // The weights arrive in halves: the first half's products run under the softmax of the second.
                const uint64_t v = value_descriptor(smem_address(v_tiles + s * T::kTileBytes), T::kSubtileBytes);
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    alive = alive && barrier_wait_warp(p_full + half, i & 1u, abort);
                    if (!alive) break;
                    tensor_fence_after();
                    if (elected) {
#pragma unroll
                        for (int k = 4 * half; k < 4 * half + 4; k++)
                            issue_f16_tensor_a(tmem + kRows, tmem + 8 * k, v + 128 * k, values_idesc, i != 0 || k != 0);
                        if (half == 1) {
                            tensor_commit(v_empty + s);
                            if (i + 1 == count) tensor_commit(o_full);
                        }
                    }
                    __syncwarp();
                }
                if (!alive) break;
                if (i + 1 < count) alive = scores(i + 1);
            }
        }
    } else {
        // ---- softmax: thread = row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::kSoftmaxRegisters));
        const uint32_t lane_bits = static_cast<uint32_t>(warp * 32) << 16;
        const uint32_t s_at = tmem + lane_bits, o_at = tmem + kRows + lane_bits;
        // Rows past the tile's queries belong to nobody and hold what an earlier CTA left in shared memory: they have no say in
        // whether the warp rescales O (a NaN there would have it do so for every tile).
        const bool owned = static_cast<uint32_t>(warp * 32 + lane) < rows;
        for (uint32_t i = 0; i < count; i++) {
            uint32_t word[4];
            const uint32_t key0 = (first + i) * kRows;
            bool all = true;
            if (g.key_mask) {
                if (!(alive = barrier_wait_warp(words_full + (i & 3u), (i >> 2) & 1u, abort))) break;
#pragma unroll
                for (int w = 0; w < 4; w++) word[w] = words[(i & 3u) * 4 + w];
                all = (word[0] & word[1] & word[2] & word[3]) == 0xffffffffu;
            } else if (key0 + kRows > keys) {
                all = false;
                tail_words(keys - key0, word);
            }
            if (!(alive = barrier_wait_warp(s_full, i & 1u, abort))) break;
            tensor_fence_after();
            float v[kRows];
#pragma unroll
            for (int c = 0; c < 4; c++) tensor_load_32(s_at + c * 32, v + c * 32);
#pragma unroll
            for (int c = 0; c < 4; c++) tensor_loads_done_32(v + c * 32);
            if (!all) {
#pragma unroll
                for (int k = 0; k < kRows; k++)
                    if (!((word[k >> 5] >> (k & 31)) & 1u)) v[k] = -INFINITY;
            }
            float part[8];
#pragma unroll
            for (int t = 0; t < 8; t++) part[t] = max3_nan(v[t], v[8 + t], v[16 + t]);
#pragma unroll
            for (int k = 24; k < kRows - 8; k += 16)
#pragma unroll
                for (int t = 0; t < 8; t++) part[t] = max3_nan(part[t], v[k + t], v[k + 8 + t]);
#pragma unroll
            for (int t = 0; t < 8; t++) part[t] = max_nan(part[t], v[kRows - 8 + t]);
            const float top = max3_nan(max3_nan(part[0], part[1], part[2]), max3_nan(part[3], part[4], part[5]), max_nan(part[6], part[7])) * g.scale_log2;
            // The exponents' reference moves only when the maximum has grown by more than 2^8 (a weight of 256 is exact
            // enough in either type, and neither O nor the sum changes its ratio); NaN and infinity make the row NaN for good.
            float alpha = 1.0f;
            const bool move = owned && !(top <= reference + 8.0f);
            if (move) {
                const float next = top < INFINITY ? top : NAN;
                alpha = exp2_approx(reference - next);
                reference = next;
                sum *= alpha;
            }
            if (i > 0 && __any_sync(0xffffffffu, move)) {
#pragma unroll 1
                for (int c = 0; c < kD; c += 32) {
                    float o[32];
                    tensor_load_32(o_at + c, o);
                    tensor_loads_done_32(o);
#pragma unroll
                    for (int k = 0; k < 32; k++) o[k] *= alpha;
                    tensor_store_32(o_at + c, reinterpret_cast<const uint32_t *>(o));
                }
                tensor_stores_done();
            }
            const float shift = reference == -INFINITY ? 0.0f : kLift<kBf16> - reference;  // nothing counted yet: the weights are zero, not NaN
            float2 total[4];
#pragma unroll
            for (int t = 0; t < 4; t++) total[t] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int half = 0; half < 2; half++) {
                uint32_t packed[32];
#pragma unroll
                for (int k = 0; k < 32; k++) {
                    const float2 x = fma_pair(make_float2(v[64 * half + 2 * k], v[64 * half + 2 * k + 1]), make_float2(g.scale_log2, g.scale_log2),
                                              make_float2(shift, shift));
                    const float2 p = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                    total[k & 3] = add_pair(total[k & 3], p);
                    packed[k] = pack_pair<kBf16>(p.x, p.y);
                }
                tensor_store_32(s_at + half * 32, packed);
                tensor_stores_done();
                tensor_fence_before();
                __syncwarp();
                if (lane == 0) barrier_arrive(p_full + half);
            }
            total[0] = add_pair(add_pair(total[0], total[1]), add_pair(total[2], total[3]));
            sum += total[0].x + total[0].y;
        }
        alive = alive && (count == 0 || barrier_wait_warp(o_full, 0, abort));
        tensor_fence_after();
        if (alive && parts == 1) {
            // Through the Q tile, which no product reads any more: one tile store moves all rows (and leaves out the queries
            // past the last).
            const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
            const uint32_t local = warp * 32 + lane;
#pragma unroll
            for (int c = 0; c < kD; c += 32) {
                float o[32];
                if (count) {
                    tensor_load_32(o_at + c, o);
                    tensor_loads_done_32(o);
                }
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) w[j] = count ? pack_pair<kBf16>(o[k + 2 * j] * inverse, o[k + 2 * j + 1] * inverse) : 0u;
                    const uint32_t at = (c + k) / 8;
                    *reinterpret_cast<uint4 *>(q_tile + (at >> 3) * T::kSubtileBytes + local * 128 + (((at & 7u) ^ (local & 7u)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) barrier_arrive(out_full);
            if (threadIdx.x == 0 && barrier_wait(out_full, 0, abort)) {
#pragma unroll
                for (int sub = 0; sub < kD / 64; sub++)
                    if (sub * 64 < g.head_dim)
                        store_tile_4d(q_tile + sub * T::kSubtileBytes, &map_out, sub * 64, static_cast<int>(kv_head * g.shares), static_cast<int>(query0),
                                      static_cast<int>(batch));
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the tile has to outlive the reading
            }
        } else if (alive && static_cast<uint32_t>(warp * 32) < rows) {
            // A share of the keys: the row's reference, sum and unscaled output for the others to read.
            const uint32_t local = warp * 32 + lane;
            stats[2 * local] = reference;
            stats[2 * local + 1] = sum;
#pragma unroll 1
            for (int c = 0; c < kD; c += 32) {
                float o[32];
                if (count) {
                    tensor_load_32(o_at + c, o);
                    tensor_loads_done_32(o);
                }
#pragma unroll
                for (int k = 0; k < 32; k += 4)
                    *reinterpret_cast<float4 *>(partial + local * kD + (((c + k) / 4) ^ (local & 7u)) * 4) =
                        count ? make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
    }

    tensor_fence_before();
    __syncthreads();  // every role is done: the abort flag is final
    tensor_fence_after();
    if (*abort_flag && (warp == T::kLoadWarp || warp == T::kValueWarp) && lane == 0) {
        uint64_t *full = warp == T::kLoadWarp ? k_full : v_full;
        const uint64_t start = clock_ns();
        if (warp == T::kLoadWarp && count) barrier_drain(q_full, 0, start);
        for (uint32_t i = issued > T::kStages ? issued - T::kStages : 0u; i < issued; i++) barrier_drain(full + i % T::kStages, (i / T::kStages) & 1u, start);
    }
    if (warp == T::kProductWarp) {
        __syncwarp();
        tensor_free<1>(tmem, T::kTensorColumns);
    }
    if (parts == 1) return;
    cluster_barrier();  // every share of this row tile is in shared memory
    const uint32_t pieces = g.head_dim / 4;
    for (uint32_t item = threadIdx.x * parts + rank; item < rows * pieces; item += T::kThreads * parts) {
        const uint32_t local = item / pieces, at = item % pieces;
        float references[8], top = -INFINITY, total = 0.0f;
        float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f), share[8];
        float sums[8];
#pragma unroll
        for (uint32_t r = 0; r < 8; r++) {
            if (r >= parts) continue;
            const float2 stat = cluster_load_pair(cluster_address(stats + 2 * local, r));
            share[r] = cluster_load(cluster_address(partial + local * kD + (at ^ (local & 7u)) * 4, r));
            references[r] = stat.x, sums[r] = stat.y;
        }
#pragma unroll
        for (uint32_t r = 0; r < 8; r++)
            if (r < parts) top = max_nan(top, references[r]);
        const float shift = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (uint32_t r = 0; r < 8; r++) {
            if (r >= parts) continue;
            const float weight = exp2_approx(references[r] - shift);
            total += weight * sums[r];
            value.x += weight * share[r].x, value.y += weight * share[r].y, value.z += weight * share[r].z, value.w += weight * share[r].w;
        }
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
        const uint32_t query = query0 + local / g.shares, head = kv_head * g.shares + local % g.shares;
        *reinterpret_cast<uint2 *>(g.out + batch * g.out_batch_stride + query * g.out_stride + static_cast<size_t>(head) * g.head_dim + at * 4) =
            make_uint2(pack_pair<kBf16>(value.x * inverse, value.y * inverse), pack_pair<kBf16>(value.z * inverse, value.w * inverse));
    }
    cluster_barrier();  // the others have read this CTA's share
}

// ---------------------------------------------------------------- host side
// [batch][rows][heads][head_dim] as boxes of 64 channels of `box_heads` heads and `box_rows` rows.
int states_map(CUtensorMap *map, bool bf16, const void *base, size_t head_dim, size_t heads, size_t rows, size_t batch, size_t stride, size_t batch_stride,
               uint32_t box_heads, uint32_t box_rows) {
    const cuuint64_t dims[4] = {head_dim, heads, rows, batch};
    const cuuint64_t strides[3] = {head_dim * 2, stride * 2, batch > 1 ? batch_stride * 2 : stride * 2};
    const cuuint32_t box[4] = {64, box_heads, box_rows, 1};
    return make_tensor_map(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides, box);
}

struct CrossMaps {
    CUtensorMap q, k, v, out;
};

template <int kD, bool kBf16>
int launch_cross(cudaStream_t stream, const CrossMaps &maps, size_t batch, size_t kv_heads, const CrossArgs &g) {
    using T = Cross<kD>;
    static Prepared prepared;
    static std::atomic<int> known[64][9];  // clusters of so many CTAs that a device holds at once
    if (int status = prepare_kernel(prepared, cross_attention_kernel<kD, kBf16>, T::kSharedBytes)) return status;
    int device = 0;
    KREA2_CUDA(cudaGetDevice(&device));
    cudaLaunchConfig_t config = {};
    config.blockDim = dim3(T::kThreads);
    config.dynamicSmemBytes = T::kSharedBytes;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    const uint32_t row_tiles = (g.q_len + g.queries - 1) / g.queries, key_tiles = (g.kv_len + kRows - 1) / kRows;
    const size_t tiles = row_tiles * batch * kv_heads;
    // The split of the keys that takes least by the measured parts: a tile of keys 2.2 us where two CTAs share an SM and 1.5
    // where one has it alone (in the last round, if it fills half of the device at most), a CTA's start and end 4 us, or 5 us
    // and for the addition of the shares 1.6 us a share, less where a row tile is not full.  (4 row tiles of 100 rows to 1000
    // keys: 17.6 us in one part, 15.3, 13.7, 12.5 in two to four, 13.8 in six or eight; 96 of 128 rows to 4096 keys: 54 in
    // one, 42 in two, 60 in three.)
    const float addition = 1.6f / kRows * static_cast<float>((g.q_len < g.queries ? g.q_len : g.queries) * g.shares);
    uint32_t parts = 1;
    float least = INFINITY;
    for (uint32_t more = 1; more <= 8 && more <= (key_tiles ? key_tiles : 1u); more++) {
        int clusters = known[device][more].load(std::memory_order_relaxed);
        if (clusters == 0) {
            config.gridDim = dim3(more, 1, 1);
            attribute.val.clusterDim.x = more;
            KREA2_CUDA(cudaOccupancyMaxActiveClusters(&clusters, cross_attention_kernel<kD, kBf16>, &config));
            // The query counts the registers that the softmax holds after the exchange for every thread, and so one CTA an SM;
            // two are launched.  (24 row tiles of 600 queries to 4096 keys in two parts, 43 us; in one, as if they did not
            // fit, 52.)
            clusters = clusters < 1 ? 2 : 2 * clusters;
            known[device][more].store(clusters, std::memory_order_relaxed);
        }
        const uint32_t resident = static_cast<uint32_t>(clusters);
        const float walk = static_cast<float>((key_tiles + more - 1) / more), ends = more > 1 ? 5.0f + addition * static_cast<float>(more) : 4.0f;
        const float shared = 2.2f * walk + ends, alone = 1.5f * walk + ends;
        const size_t rest = tiles % resident;
        const float time = static_cast<float>(tiles / resident) * shared + (rest == 0 ? 0.0f : 2 * rest <= resident ? alone : shared);
        if (time < least) least = time, parts = more;
    }
    attribute.val.clusterDim.x = parts;
    config.gridDim = dim3(row_tiles * parts, static_cast<unsigned>(kv_heads), static_cast<unsigned>(batch));
    const cudaError_t status = cudaLaunchKernelEx(&config, cross_attention_kernel<kD, kBf16>, maps.q, maps.k, maps.v, maps.out, g);
    if (status != cudaSuccess) return fail(KREA2_RUNTIME, "cross_attention launch failed: %s", cudaGetErrorString(status));
    return KREA2_OK;
}

}  // namespace

int take_cross_status(int mask, int *value) {
    *value = 0;
    return g_cross_launched.load(std::memory_order_relaxed) ? take_status_bits(g_cross_status, mask, value) : KREA2_OK;
}

}  // namespace krea2

using namespace krea2;

extern "C" int krea2_cross_attention(krea2_stream stream, size_t batch, size_t q_len, size_t kv_len, const void *q, const void *k,
                                     const void *v, const int32_t *kv_lengths, const void *key_mask, void *out, size_t q_heads,
                                     size_t kv_heads, size_t head_dim, size_t q_batch_stride, size_t q_stride, size_t k_batch_stride,
                                     size_t k_stride, size_t v_batch_stride, size_t v_stride, size_t out_batch_stride,
                                     size_t out_stride, size_t mask_stride, float scale, int kind) {
    clear_error();
    const char *name = "cross_attention";
    KREA2_REQUIRE(batch >= 1 && batch <= 65535, "%s: batch %zu outside 1..65535", name, batch);
    KREA2_REQUIRE(q_len >= 1 && q_len <= 16777216, "%s: q_len %zu outside 1..16777216", name, q_len);
    KREA2_REQUIRE(kv_len <= 16777216, "%s: kv_len %zu outside 0..16777216", name, kv_len);
    KREA2_REQUIRE(kv_heads >= 1 && q_heads >= kv_heads && q_heads <= 1024 && q_heads % kv_heads == 0,
                  "%s: %zu query heads must be a multiple of %zu key heads, up to 1024", name, q_heads, kv_heads);
    KREA2_REQUIRE(head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0, "%s: head_dim %zu must be a multiple of 8 up to 128", name, head_dim);
    KREA2_REQUIRE(q_stride >= q_heads * head_dim && out_stride >= q_heads * head_dim, "%s: a query row holds %zu values, the strides are %zu and %zu",
                  name, q_heads * head_dim, q_stride, out_stride);
    KREA2_REQUIRE(kv_len == 0 || (k_stride >= kv_heads * head_dim && v_stride >= kv_heads * head_dim),
                  "%s: a key row holds %zu values, the strides are %zu and %zu", name, kv_heads * head_dim, k_stride, v_stride);
    KREA2_REQUIRE((q_batch_stride | q_stride | k_batch_stride | k_stride | v_batch_stride | v_stride | out_batch_stride | out_stride) % 8 == 0,
                  "%s: strides must be multiples of 8 elements", name);
    KREA2_REQUIRE(batch == 1 || out_batch_stride >= (q_len - 1) * out_stride + q_heads * head_dim ||
                      (out_batch_stride >= q_heads * head_dim && out_stride >= (batch - 1) * out_batch_stride + q_heads * head_dim),
                  "%s: the batch's outputs overlap", name);
    KREA2_REQUIRE(!key_mask || batch == 1 || mask_stride == 0 || mask_stride >= kv_len, "%s: mask_stride %zu is below kv_len %zu", name, mask_stride, kv_len);
    const float scale_log2 = scale * 1.44269504088896340736f;  // infinite for the largest scales, which would make zero scores NaN
    KREA2_REQUIRE(std::isfinite(scale_log2) && scale > 0.0f, "%s: scale must be a positive number below 2^127", name);
    KREA2_REQUIRE(kind == KREA2_F16 || kind == KREA2_BF16, "%s: kind %d is neither KREA2_F16 nor KREA2_BF16", name, kind);
    KREA2_REQUIRE(q && out && (kv_len == 0 || (k && v)), "%s: null buffer", name);
    KREA2_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), "%s: buffers must be 16-byte aligned", name);
    KREA2_REQUIRE(reinterpret_cast<uintptr_t>(kv_lengths) % 4 == 0, "%s: kv_lengths must be 4-byte aligned", name);
    const size_t shares = q_heads / kv_heads;
    KREA2_REQUIRE(shares <= kRows, "%s: %zu query heads share a key head, %d are served", name, shares, kRows);
    const uint32_t queries = static_cast<uint32_t>(kRows / shares), h = static_cast<uint32_t>(shares);
    const bool bf16 = kind == KREA2_BF16, q_shared = batch > 1 && q_batch_stride == 0, k_shared = batch > 1 && k_batch_stride == 0,
               v_shared = batch > 1 && v_batch_stride == 0;
    const CrossArgs g = {kv_lengths, static_cast<const uint8_t *>(key_mask), static_cast<uint16_t *>(out), static_cast<uint32_t>(q_len),
                         static_cast<uint32_t>(kv_len), h, queries, static_cast<uint32_t>(head_dim), out_batch_stride, out_stride, mask_stride,
                         q_shared ? 1u : 0u, k_shared ? 1u : 0u, v_shared ? 1u : 0u, scale_log2};
    CrossMaps maps = {};  // without keys none is loaded
    if (int status = states_map(&maps.q, bf16, q, head_dim, q_heads, q_len, q_shared ? 1 : batch, q_stride, q_batch_stride, h, queries)) return status;
    if (int status = states_map(&maps.out, bf16, out, head_dim, q_heads, q_len, batch, out_stride, out_batch_stride, h, queries)) return status;
    if (kv_len != 0) {
        if (int status = states_map(&maps.k, bf16, k, head_dim, kv_heads, kv_len, k_shared ? 1 : batch, k_stride, k_batch_stride, 1, kRows)) return status;
        if (int status = states_map(&maps.v, bf16, v, head_dim, kv_heads, kv_len, v_shared ? 1 : batch, v_stride, v_batch_stride, 1, kRows)) return status;
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    g_cross_launched.store(true, std::memory_order_relaxed);
    if (head_dim <= 64) return bf16 ? launch_cross<64, true>(s, maps, batch, kv_heads, g) : launch_cross<64, false>(s, maps, batch, kv_heads, g);
    return bf16 ? launch_cross<128, true>(s, maps, batch, kv_heads, g) : launch_cross<128, false>(s, maps, batch, kv_heads, g);
}
