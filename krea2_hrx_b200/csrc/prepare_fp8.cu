// Activations as e4m3 codes with one scale per 128 channels (new with this library; the reference's projections are int8):
//   krea2_prepare_norm_fp8   the residual's addition, the RMS norm and the codes of its result in one pass
//   krea2_prepare_plain_fp8  the codes of rows as they are
#include <cuda_fp8.h>

#include "common.cuh"

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

// Eight consecutive channels from `at` of one row: one 16-byte access where rows are aligned to it, single
// elements (zero past the row's end) otherwise.
template <bool kVector>
__device__ __forceinline__ void load8(const uint16_t *row, uint32_t at, uint32_t width, uint16_t (&v)[8]) {
    if constexpr (kVector) {
        const uint4 raw = *reinterpret_cast<const uint4 *>(row + at);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; i++) v[2 * i] = static_cast<uint16_t>(w[i]), v[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = at + i < width ? row[at + i] : uint16_t(0);
    }
}

__device__ __forceinline__ float block_sum(float v, float *shared) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < (blockDim.x >> 5) ? shared[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// One block per row.  A thread owns kPer runs of eight channels, blockDim.x runs apart, so sixteen neighbouring
// lanes own one scale's group; the row stays in registers between the sum of squares and the codes.
template <bool kBf16, bool kNorm, bool kVector, int kPer>
__global__ void __launch_bounds__(1024)
prepare_fp8_kernel(const PrepareArgs g) {
    __shared__ float partial[32];
    const size_t row = blockIdx.x;
    const uint16_t *x = g.x + row * g.x_stride;
    float v[kPer][8];
    float squares = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const uint32_t at = (threadIdx.x + j * blockDim.x) * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) v[j][i] = 0.0f;
        if (at >= g.width) continue;
        uint16_t raw[8];
        load8<kVector>(x, at, g.width, raw);
#pragma unroll
        for (int i = 0; i < 8; i++) v[j][i] = value_of<kBf16>(raw[i]);
        if constexpr (kNorm) {
            if (g.residual != nullptr) {
                uint16_t other[8];
                load8<kVector>(g.residual + row * g.residual_stride, at, g.width, other);
                // The next layer reads the sum rounded to the stream's type, so the norm is taken of that.
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    raw[i] = bits_of<kBf16>(v[j][i] + value_of<kBf16>(other[i]));
                    v[j][i] = value_of<kBf16>(raw[i]);
                }
                if (g.sum != nullptr) {
                    uint16_t *sum = g.sum + row * g.sum_stride + at;
                    if constexpr (kVector) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) w[i] = raw[2 * i] | (static_cast<uint32_t>(raw[2 * i + 1]) << 16);
                        *reinterpret_cast<uint4 *>(sum) = make_uint4(w[0], w[1], w[2], w[3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if (at + i < g.width) sum[i] = raw[i];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) squares = fmaf(v[j][i], v[j][i], squares);
        }
    }
    float rinv = 1.0f;
    if constexpr (kNorm) rinv = 1.0f / sqrtf(block_sum(squares, partial) / static_cast<float>(g.width) + g.eps);
#pragma unroll
    for (int j = 0; j < kPer; j++) {
        const uint32_t at = (threadIdx.x + j * blockDim.x) * 8;
        if constexpr (kNorm) {
            if (at < g.width) {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (kVector || at + i < g.width) v[j][i] = v[j][i] * rinv * (g.weight_offset + (g.weight ? g.weight[at + i] : 0.0f));
            }
        }
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(v[j][i]));
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float scale = fmaxf(top / kE4m3Max, kScaleFloor);
        const float inverse = 1.0f / scale;
        if (at >= g.width) continue;
        uint8_t *q = g.q + row * g.out_stride + at;
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[j][4 * i] * inverse, v[j][4 * i + 1] * inverse), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[j][4 * i + 2] * inverse, v[j][4 * i + 3] * inverse), __NV_SATFINITE, __NV_E4M3);
            w[i] = lo | (hi << 16);
        }
        if (at + 8 <= g.width) {
            *reinterpret_cast<uint2 *>(q) = make_uint2(w[0], w[1]);
        } else {
            for (uint32_t i = 0; at + i < g.width; i++) q[i] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
        }
        if (((at / 8) & 15) == 0) g.q_scale[row * g.groups + at / kGroup] = scale;
    }
}

template <bool kBf16, bool kNorm, bool kVector>
void launch_prepare(cudaStream_t stream, const PrepareArgs &g) {
    const uint32_t runs = (g.width + 7) / 8;
    auto threads = [&](uint32_t per) { return ((runs + per - 1) / per + 31) / 32 * 32; };
    if (runs <= 1024) prepare_fp8_kernel<kBf16, kNorm, kVector, 1><<<g.tokens, threads(1), 0, stream>>>(g);
    else if (runs <= 2048) prepare_fp8_kernel<kBf16, kNorm, kVector, 2><<<g.tokens, threads(2), 0, stream>>>(g);
    else prepare_fp8_kernel<kBf16, kNorm, kVector, 4><<<g.tokens, threads(4), 0, stream>>>(g);
}

template <bool kNorm>
int run_prepare(const char *name, cudaStream_t stream, const PrepareArgs &g, int kind) {
    const bool vector = g.width % 8 == 0 && g.x_stride % 8 == 0 && aligned16(g.x) &&
                        (!g.residual || (g.residual_stride % 8 == 0 && aligned16(g.residual))) &&
                        (!g.sum || (g.sum_stride % 8 == 0 && aligned16(g.sum)));
    if (kind == KREA2_BF16) vector ? launch_prepare<true, kNorm, true>(stream, g) : launch_prepare<true, kNorm, false>(stream, g);
    else vector ? launch_prepare<false, kNorm, true>(stream, g) : launch_prepare<false, kNorm, false>(stream, g);
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
