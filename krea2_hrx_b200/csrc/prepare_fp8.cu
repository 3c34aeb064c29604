// Activations as e4m3 codes with one scale per 128 channels (new with this library; the reference's projections are int8):
//   krea2_prepare_norm_fp8   the residual's addition, the RMS norm and the codes of its result in one pass
//   krea2_prepare_plain_fp8  the codes of rows as they are
#include <cuda_fp8.h>

#include <atomic>

#include "tensor_core.cuh"

namespace krea2 {
namespace {

constexpr int kGroup = 128;           // channels under one scale
constexpr float kE4m3Max = 448.0f;
constexpr float kScaleFloor = 1.17549435e-38f;  // 2^-126: a group of zeros keeps a scale that has a reciprocal

struct PrepareArgs {
    const uint16_t *x, *residual;
    const float *weight;
    uint16_t *sum;
    uint8_t *q;
    float *q_scale;
    uint32_t tokens, width, groups;
    size_t x_stride, residual_stride, sum_stride, out_stride;
    float eps, weight_offset;
};

// The channels of a thread's run of eight.  Where rows are aligned they are neighbours, moved by one 16-byte access, and
// sixteen lanes own a scale's group; otherwise they lie 32 apart, so that a warp's single-element accesses are contiguous,
// and all lanes own half of two groups.
template <bool kVector>
__device__ __forceinline__ uint32_t channel_of(uint32_t run, int i) {
    return kVector ? run * 8 + i : (run & ~31u) * 8 + i * 32 + (run & 31u);
}
template <bool kVector>
__device__ __forceinline__ uint4 load8(const uint16_t *row, uint32_t run, uint32_t width) {
    if constexpr (kVector) {
        return run * 8 < width ? *reinterpret_cast<const uint4 *>(row + run * 8) : make_uint4(0, 0, 0, 0);
    } else {
        uint32_t v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t at = channel_of<false>(run, i);
            v[i] = at < width ? row[at] : 0u;
        }
        return make_uint4(v[0] | (v[1] << 16), v[2] | (v[3] << 16), v[4] | (v[5] << 16), v[6] | (v[7] << 16));
    }
}
template <bool kVector>
__device__ __forceinline__ void store8(uint16_t *row, uint32_t run, uint32_t width, uint4 v) {
    if constexpr (kVector) {
        if (run * 8 < width) *reinterpret_cast<uint4 *>(row + run * 8) = v;
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t at = channel_of<false>(run, i);
            if (at < width) row[at] = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
        }
    }
}
template <bool kBf16>
__device__ __forceinline__ void unpack8(uint4 raw, float (&v)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = value_of<kBf16>(static_cast<uint16_t>(w[i]));
        v[2 * i + 1] = value_of<kBf16>(static_cast<uint16_t>(w[i] >> 16));
    }
}

// The sum over the block; `shared` [32] may be used again two calls later.
__device__ __forceinline__ float block_sum(float v, float *shared) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if (blockDim.x == 32) return v;
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < (blockDim.x >> 5) ? shared[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// bf16 rows whose squares leave the range of f32 on either side (those of f16 stay within 2^-48..2^32): where they overflow some
// value is 2^56 at least, and above a mean (and eps) of 2^-100 what the squares lose, 2^-150 each, is below the sum's rounding.
__device__ __forceinline__ bool out_of_range(float mean) { return mean == INFINITY || mean < 0x1p-100f; }

// Takes such rows, among those that the block has walked, again times 2^-80 or 2^80.  Apart from the walk and as a call,
// because they are rare: scaled where they lie in registers they cost every row spills (136-176 bytes with three runs a thread
// and a residual); inlined here they cost 4608 rows of 6150, on single elements, 100 us instead of 79.  (Without them it
// takes 77 us, and 38.0 instead of 38.2 us for 4608 rows of 6144 and their residual.)
template <bool kVector>
__device__ __noinline__ void take_again(const PrepareArgs g, int per, float (*partial)[32]) {
    const uint32_t lane = threadIdx.x & 31;
    __syncthreads();
    for (size_t row = blockIdx.x, count = 0; row < g.tokens; row += gridDim.x, count++) {
        auto value = [&](uint32_t at) {
            if (at >= g.width) return 0.0f;
            if (g.sum != nullptr) return value_of<true>(g.sum[row * g.sum_stride + at]);  // it may have replaced x or the residual
            const float v = value_of<true>(g.x[row * g.x_stride + at]);
            return g.residual != nullptr ? bf_round(v + value_of<true>(g.residual[row * g.residual_stride + at])) : v;
        };
        auto mean_of = [&](float by, float *shared) {  // in the walk's order, so that by = 1 gives its mean to the bit
            float squares = 0.0f;
            for (int j = 0; j < per; j++)
                for (int i = 0; i < 8; i++) {
                    const float v = value(channel_of<kVector>(threadIdx.x + j * blockDim.x, i)) * by;
                    squares = fmaf(v, v, squares);
                }
            return block_sum(squares, shared) / static_cast<float>(g.width) + g.eps * by * by;
        };
        const float mean = mean_of(1.0f, partial[0]);
        if (!out_of_range(mean)) {
            __syncthreads();  // partial[0] is next
            continue;
        }
        const float by = mean < 1.0f ? 0x1p80f : 0x1p-80f, rinv = 1.0f / sqrtf(mean_of(by, partial[1]));
        for (uint32_t group = threadIdx.x >> 5; group < g.groups; group += blockDim.x >> 5) {
            float v[4], top = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t at = group * kGroup + i * 32 + lane;
                v[i] = at < g.width ? value(at) * by * rinv * (g.weight_offset + (g.weight != nullptr ? g.weight[at] : 0.0f)) : 0.0f;
                top = fmaxf(top, fabsf(v[i]));
            }
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const float scale = fmaxf(__fdiv_rn(top, kE4m3Max), kScaleFloor), inverse = __frcp_rn(scale);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t at = group * kGroup + i * 32 + lane;
                if (at < g.width) g.q[row * g.out_stride + at] = __nv_cvt_float_to_fp8(v[i] * inverse, __NV_SATFINITE, __NV_E4M3);
            }
            if (lane == 0) g.q_scale[row * g.groups + group] = scale;
        }
    }
}

// A thread owns kPer runs of eight channels, blockDim.x runs apart; the row stays in registers between the sum of squares and
// the codes.  HBM-bound: a block walks rows gridDim.x apart and requests the next one before it works on the present one
// (not the widest rows, whose values fill the registers).
template <bool kBf16, bool kNorm, bool kResidual, bool kVector, int kPer>
__global__ void __launch_bounds__(kPer <= 2 ? 1024 : kPer == 3 ? 256 : 512, kPer == 3 ? 4 : 1)
prepare_fp8_kernel(const PrepareArgs g) {
    constexpr bool kAhead = kVector && kPer <= 3;  // single elements are packed as they arrive: asking early would wait for them
    __shared__ float partial[2][32];
    const bool wide_weight = kVector && (reinterpret_cast<uintptr_t>(g.weight) & 15u) == 0u;
    uint4 x[kPer], residual[kResidual ? kPer : 1];
    auto run_of = [&](int j) { return threadIdx.x + j * blockDim.x; };
    auto request = [&](size_t row) {
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            x[j] = load8<kVector>(g.x + row * g.x_stride, run_of(j), g.width);
            if constexpr (kResidual) residual[j] = load8<kVector>(g.residual + row * g.residual_stride, run_of(j), g.width);
        }
    };
    if (kAhead) request(blockIdx.x);
    __shared__ int again;  // some row is out of range: not in a register, of which three runs a thread leave none
    if (kNorm && kBf16 && threadIdx.x == 0) again = 0;
    for (size_t row = blockIdx.x, count = 0; row < g.tokens; row += gridDim.x, count++) {
        if (!kAhead) request(row);
        float v[kPer][8];
        float squares = 0.0f;
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            unpack8<kBf16>(x[j], v[j]);
            if constexpr (kResidual) {
                // The next layer reads the sum rounded to the stream's type, so the norm is taken of that.
                float other[8];
                unpack8<kBf16>(residual[j], other);
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = pack_pair<kBf16>(v[j][2 * i] + other[2 * i], v[j][2 * i + 1] + other[2 * i + 1]);
                const uint4 total = make_uint4(w[0], w[1], w[2], w[3]);
                unpack8<kBf16>(total, v[j]);
                if (g.sum != nullptr) store8<kVector>(g.sum + row * g.sum_stride, run_of(j), g.width, total);
            }
            if constexpr (kNorm) {
#pragma unroll
                for (int i = 0; i < 8; i++) squares = fmaf(v[j][i], v[j][i], squares);
            }
        }
        if (kAhead && row + gridDim.x < g.tokens) request(row + gridDim.x);
        if constexpr (kNorm) {
            const float mean = block_sum(squares, partial[count & 1]) / static_cast<float>(g.width) + g.eps;
            if (kBf16 && threadIdx.x == 0 && out_of_range(mean)) again = 1;
            const float rinv = 1.0f / sqrtf(mean);
#pragma unroll
            for (int j = 0; j < kPer; j++) {
                float weight[8] = {};
                if (g.weight != nullptr) {
                    if (wide_weight) {
                        if (run_of(j) * 8 < g.width) {
                            *reinterpret_cast<float4 *>(weight) = __ldg(reinterpret_cast<const float4 *>(g.weight + run_of(j) * 8));
                            *reinterpret_cast<float4 *>(weight + 4) = __ldg(reinterpret_cast<const float4 *>(g.weight + run_of(j) * 8 + 4));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const uint32_t at = channel_of<kVector>(run_of(j), i);
                            if (at < g.width) weight[i] = __ldg(g.weight + at);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; i++) v[j][i] = v[j][i] * rinv * (g.weight_offset + weight[i]);
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const uint32_t run = run_of(j);
            // What lies past the row's end was read as zero; a weight cannot make it more than that (a norm of such a zero
            // may be NaN in a row that is, which no maximum shows).
            float top[2] = {0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 8; i++) top[kVector ? 0 : i >> 2] = fmaxf(top[kVector ? 0 : i >> 2], fabsf(v[j][i]));
#pragma unroll
            for (int off = kVector ? 8 : 16; off >= 1; off >>= 1) {
                top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], off));
                if constexpr (!kVector) top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], off));
            }
            float scale[2], inverse[2];
#pragma unroll
            for (int h = 0; h < (kVector ? 1 : 2); h++) {
                scale[h] = fmaxf(__fdiv_rn(top[h], kE4m3Max), kScaleFloor);
                inverse[h] = __frcp_rn(scale[h]);
            }
            uint32_t w[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float by = inverse[kVector ? 0 : i];
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[j][4 * i] * by, v[j][4 * i + 1] * by), __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[j][4 * i + 2] * by, v[j][4 * i + 3] * by), __NV_SATFINITE, __NV_E4M3);
                w[i] = lo | (hi << 16);
            }
            uint8_t *q = g.q + row * g.out_stride;
            if constexpr (kVector) {
                if (run * 8 >= g.width) continue;
                *reinterpret_cast<uint2 *>(q + run * 8) = make_uint2(w[0], w[1]);
                if ((run & 15u) == 0u) g.q_scale[row * g.groups + run / 16] = scale[0];
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t at = channel_of<false>(run, i);
                    if (at < g.width) q[at] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
                }
                const uint32_t group = run / 32 * 2 + (run & 1u);
                if ((run & 31u) < 2u && group < g.groups) g.q_scale[row * g.groups + group] = scale[run & 1u];
            }
        }
    }
    if constexpr (kNorm && kBf16) {
        __syncthreads();
        if (again) take_again<kVector>(g, kPer, partial);
    }
}

template <bool kBf16, bool kNorm, bool kResidual, bool kVector, int kPer>
int launch_runs(cudaStream_t stream, const PrepareArgs &g, uint32_t runs) {
    static std::atomic<int> known[64][33];  // blocks of so many warps that an SM holds
    const uint32_t threads = ((runs + kPer - 1) / kPer + 31) / 32 * 32;
    int device = 0;
    KREA2_CUDA(cudaGetDevice(&device));
    if (device < 0 || device >= 64) return fail(KREA2_INTERNAL, "device index %d out of range", device);
    int blocks = known[device][threads / 32].load(std::memory_order_relaxed);
    if (blocks == 0) {
        KREA2_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, prepare_fp8_kernel<kBf16, kNorm, kResidual, kVector, kPer>,
                                                                 static_cast<int>(threads), 0));
        if (blocks < 1) blocks = 1;
        known[device][threads / 32].store(blocks, std::memory_order_relaxed);
    }
    const uint32_t resident = static_cast<uint32_t>(blocks) * static_cast<uint32_t>(multiprocessors());
    prepare_fp8_kernel<kBf16, kNorm, kResidual, kVector, kPer><<<g.tokens < resident ? g.tokens : resident, threads, 0, stream>>>(g);
    return KREA2_OK;
}

// Few rows (or narrow ones): one run a thread, for the latency (2.7 us for one row of 6144).  Many: two or three, so that
// four blocks of up to 256 threads share an SM and one's loads run under another's sums: 4608 rows of 6144 and their
// residual take 38 us (82 % of the HBM rate, 91 % for 16896 rows), 70 us with one run a thread and a block per row.  Wider
// rows: two runs in up to 1024 threads, 28 us for 1043 rows of 16384 and their residual, 32 us with four runs in 512.
// Narrow rows have a block of one warp, of which an SM holds 32: 110592 rows of 256 and their residual take 37 us (83 %),
// 221184 rows of 128, where half of the lanes idle, 69 us (45 %).
template <bool kBf16, bool kNorm, bool kResidual, bool kVector>
int launch_prepare(cudaStream_t stream, const PrepareArgs &g) {
    const uint32_t runs = (g.width + 7) / 8;
    if (runs <= 1024 && (!kVector || g.tokens <= static_cast<uint32_t>(multiprocessors()) || runs <= 128))
        return launch_runs<kBf16, kNorm, kResidual, kVector, 1>(stream, g, runs);
    if constexpr (kVector)
        if (runs > 512 && runs <= 768) return launch_runs<kBf16, kNorm, kResidual, kVector, 3>(stream, g, runs);
    if (runs <= 2048) return launch_runs<kBf16, kNorm, kResidual, kVector, 2>(stream, g, runs);
    return launch_runs<kBf16, kNorm, kResidual, kVector, 8>(stream, g, runs);
}

template <bool kBf16, bool kNorm>
int launch_residual(cudaStream_t stream, const PrepareArgs &g, bool vector) {
    if constexpr (kNorm) {
        if (g.residual) return vector ? launch_prepare<kBf16, true, true, true>(stream, g) : launch_prepare<kBf16, true, true, false>(stream, g);
    }
    return vector ? launch_prepare<kBf16, kNorm, false, true>(stream, g) : launch_prepare<kBf16, kNorm, false, false>(stream, g);
}

template <bool kNorm>
int run_prepare(const char *name, cudaStream_t stream, const PrepareArgs &g, int kind) {
    const bool vector = g.width % 8 == 0 && g.x_stride % 8 == 0 && aligned16(g.x) &&
                        (!g.residual || (g.residual_stride % 8 == 0 && aligned16(g.residual))) &&
                        (!g.sum || (g.sum_stride % 8 == 0 && aligned16(g.sum)));
    if (int status = kind == KREA2_BF16 ? launch_residual<true, kNorm>(stream, g, vector) : launch_residual<false, kNorm>(stream, g, vector)) return status;
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return fail(KREA2_RUNTIME, "%s launch failed: %s", name, cudaGetErrorString(status));
    return KREA2_OK;
}

int check_prepare(const char *name, size_t tokens, const void *x, const void *q, const float *q_scale, size_t width, size_t x_stride,
                  size_t out_stride, int kind) {
    KREA2_REQUIRE(tokens >= 1 && tokens <= 16777216, "%s: tokens %zu outside 1..16777216", name, tokens);
    KREA2_REQUIRE(width >= 1 && width <= 32768, "%s: width %zu outside 1..32768", name, width);
    KREA2_REQUIRE(x_stride >= width, "%s: x_stride %zu is below the width %zu", name, x_stride, width);
    KREA2_REQUIRE(out_stride >= width && out_stride % 16 == 0, "%s: out_stride %zu must be a multiple of 16, at least the width %zu", name,
                  out_stride, width);
    KREA2_REQUIRE(kind == KREA2_F16 || kind == KREA2_BF16, "%s: kind %d is neither KREA2_F16 nor KREA2_BF16", name, kind);
    KREA2_REQUIRE(x && q && q_scale, "%s: null buffer", name);
    KREA2_REQUIRE(aligned16(q), "%s: the codes must be 16-byte aligned", name);
    KREA2_REQUIRE(reinterpret_cast<uintptr_t>(x) % 2 == 0 && reinterpret_cast<uintptr_t>(q_scale) % 4 == 0,
                  "%s: buffers must be aligned to their element size", name);
    return KREA2_OK;
}

}  // namespace
}  // namespace krea2

using namespace krea2;

extern "C" int krea2_prepare_norm_fp8(krea2_stream stream, size_t tokens, const void *x, const void *residual, const float *weight,
                                      void *sum, void *q, float *q_scale, size_t width, size_t x_stride, size_t residual_stride,
                                      size_t sum_stride, size_t out_stride, float eps, float weight_offset, int kind) {
    clear_error();
    const char *name = "prepare_norm_fp8";
    if (int status = check_prepare(name, tokens, x, q, q_scale, width, x_stride, out_stride, kind)) return status;
    KREA2_REQUIRE(eps >= 0.0f && eps <= 1.0f, "%s: eps outside 0..1", name);
    KREA2_REQUIRE(weight_offset >= -1e30f && weight_offset <= 1e30f, "%s: weight_offset is not a finite number", name);
    KREA2_REQUIRE(residual || !sum, "%s: a sum is written only where there is a residual", name);
    KREA2_REQUIRE(!residual || residual_stride >= width, "%s: residual_stride %zu is below the width %zu", name, residual_stride, width);
    KREA2_REQUIRE(!sum || sum_stride >= width, "%s: sum_stride %zu is below the width %zu", name, sum_stride, width);
    KREA2_REQUIRE((sum != x || sum_stride == x_stride) && (!sum || sum != residual || sum_stride == residual_stride),
                  "%s: a sum in place needs the stride of the buffer that it replaces", name);
    KREA2_REQUIRE(reinterpret_cast<uintptr_t>(residual) % 2 == 0 && reinterpret_cast<uintptr_t>(sum) % 2 == 0 &&
                      reinterpret_cast<uintptr_t>(weight) % 4 == 0,
                  "%s: buffers must be aligned to their element size", name);
    const PrepareArgs g = {static_cast<const uint16_t *>(x), static_cast<const uint16_t *>(residual), weight, static_cast<uint16_t *>(sum),
                           static_cast<uint8_t *>(q), q_scale, static_cast<uint32_t>(tokens), static_cast<uint32_t>(width),
                           static_cast<uint32_t>((width + kGroup - 1) / kGroup), x_stride, residual_stride, sum_stride, out_stride, eps, weight_offset};
    return run_prepare<true>(name, static_cast<cudaStream_t>(stream), g, kind);
}

extern "C" int krea2_prepare_plain_fp8(krea2_stream stream, size_t tokens, const void *x, void *q, float *q_scale, size_t width,
                                       size_t x_stride, size_t out_stride, int kind) {
    clear_error();
    const char *name = "prepare_plain_fp8";
    if (int status = check_prepare(name, tokens, x, q, q_scale, width, x_stride, out_stride, kind)) return status;
    const PrepareArgs g = {static_cast<const uint16_t *>(x), nullptr, nullptr, nullptr, static_cast<uint8_t *>(q), q_scale,
                           static_cast<uint32_t>(tokens), static_cast<uint32_t>(width), static_cast<uint32_t>((width + kGroup - 1) / kGroup),
                           x_stride, 0, 0, out_stride, 0.0f, 0.0f};
    return run_prepare<false>(name, static_cast<cudaStream_t>(stream), g, kind);
}
