// Rotary positions computed from position and frequency (new with this library; krea2_rope_qknorm_f16 takes the
// reference's finished tables): both pair layouts, any even part of a head, frequencies scaled for long contexts,
// forwards and backwards.
//   krea2_rotary_frequencies  radians per position of each pair, in f64, on the host
//   krea2_rotary              queries and keys turned, in place or into other buffers
#include <cmath>

#include "common.cuh"

namespace krea2 {
namespace {

struct RotaryArgs {
    const uint16_t *q, *k;
    const int32_t *positions;
    const double *frequencies;
    uint16_t *q_out, *k_out;
    uint32_t q_heads, kv_heads, head_dim, half;
    size_t q_stride, k_stride, q_out_stride, k_out_stride;
    float magnitude, direction;
};

// cos and sin of position * frequency.  The product and its remainder by whole turns are taken in f64 (at position
// 10^6 an f32 product is off by 0.06 radians), what is left is below half a turn and exact enough in f32.
__device__ __forceinline__ void turn_of(int32_t position, double frequency, float &cosine, float &sine) {
    const double turns = static_cast<double>(position) * frequency * 0.15915494309189533577;  // 1 / (2 pi)
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sine, &cosine);
}

// One block per token: the token's cosines and sines go to shared memory, then its heads are turned pair by pair.
template <bool kBf16, bool kInterleaved>
__global__ void __launch_bounds__(256)
rotary_kernel(const RotaryArgs g) {
    __shared__ float cosines[256], sines[256];
    const size_t token = blockIdx.x;
    const int32_t position = g.positions ? g.positions[token] : static_cast<int32_t>(token);
    for (uint32_t i = threadIdx.x; i < g.half; i += blockDim.x) {
        float c, s;
        turn_of(position, g.frequencies[i], c, s);
        cosines[i] = c * g.magnitude;
        sines[i] = s * g.magnitude * g.direction;
    }
    __syncthreads();
    const uint32_t units = g.head_dim - g.half;  // pairs, then the channels that are not turned
    const uint32_t count = (g.q_heads + g.kv_heads) * units;
    for (uint32_t item = threadIdx.x; item < count; item += blockDim.x) {
        const uint32_t head = item / units, unit = item % units;
        const bool is_q = head < g.q_heads;
        const uint16_t *in = is_q ? g.q + token * g.q_stride + head * g.head_dim : g.k + token * g.k_stride + (head - g.q_heads) * g.head_dim;
        uint16_t *out = is_q ? g.q_out + token * g.q_out_stride + head * g.head_dim : g.k_out + token * g.k_out_stride + (head - g.q_heads) * g.head_dim;
        if (unit < g.half) {
            const uint32_t first = kInterleaved ? 2 * unit : unit, second = kInterleaved ? first + 1 : unit + g.half;
            const float a = value_of<kBf16>(in[first]), b = value_of<kBf16>(in[second]);
            const float c = cosines[unit], s = sines[unit];
            out[first] = bits_of<kBf16>(a * c - b * s);
            out[second] = bits_of<kBf16>(b * c + a * s);
        } else {
            out[unit + g.half] = in[unit + g.half];
        }
    }
}

}  // namespace
}  // namespace krea2

using namespace krea2;

extern "C" int krea2_rotary_frequencies(size_t rotary_dim, double base, int scaling, double factor, double trained, double slow,
                                        double fast, double *host_frequencies, float *host_magnitude) {
    clear_error();
    const char *name = "rotary_frequencies";
    KREA2_REQUIRE(rotary_dim >= 2 && rotary_dim <= 512 && rotary_dim % 2 == 0, "%s: rotary_dim %zu must be even, in 2..512", name, rotary_dim);
    KREA2_REQUIRE(std::isfinite(base) && base > 1.0, "%s: base must be a finite number above 1", name);
    KREA2_REQUIRE(scaling >= KREA2_ROTARY_PLAIN && scaling <= KREA2_ROTARY_PARTS, "%s: scaling %d is none of KREA2_ROTARY_*", name, scaling);
    KREA2_REQUIRE(host_frequencies && host_magnitude, "%s: null output", name);
    if (scaling != KREA2_ROTARY_PLAIN)
        KREA2_REQUIRE(std::isfinite(factor) && factor >= 1.0, "%s: factor must be a finite number of at least 1", name);
    if (scaling == KREA2_ROTARY_PARTS)
        KREA2_REQUIRE(std::isfinite(trained) && trained >= 1.0 && std::isfinite(fast) && std::isfinite(slow) && slow >= 0.0 && fast > slow,
                      "%s: parts need a trained length of at least 1 and 0 <= slow < fast turns", name);
    const double dim = static_cast<double>(rotary_dim);
    // Raising the base leaves the fastest pair as it is and slows the slowest by `factor`.
    if (scaling == KREA2_ROTARY_BASE) base *= std::pow(factor, dim / (rotary_dim > 2 ? dim - 2.0 : 1.0));
    KREA2_REQUIRE(std::isfinite(base), "%s: the raised base is not finite", name);
    for (size_t i = 0; i < rotary_dim / 2; i++) {
        const double plain = std::pow(base, -2.0 * static_cast<double>(i) / dim);
        double frequency = plain;
        if (scaling == KREA2_ROTARY_LINEAR) frequency = plain / factor;
        if (scaling == KREA2_ROTARY_PARTS) {
            // Pairs that turn `fast` times or more within the trained length keep their frequency, those that turn
            // `slow` times or less are slowed by `factor`, the ones between are blended (Peng et al. 2023, eq. 17-20).
            const double turns = trained * plain / 6.28318530717958647693;
            double kept = (turns - slow) / (fast - slow);
            kept = kept < 0.0 ? 0.0 : kept > 1.0 ? 1.0 : kept;
            frequency = plain * kept + plain / factor * (1.0 - kept);
        }
        host_frequencies[i] = frequency;
    }
    *host_magnitude = scaling == KREA2_ROTARY_PARTS ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0f;
    return KREA2_OK;
}

extern "C" int krea2_rotary(krea2_stream stream, size_t tokens, const void *q, const void *k, const int32_t *positions,
                            const double *frequencies, void *q_out, void *k_out, size_t q_heads, size_t kv_heads, size_t head_dim,
                            size_t rotary_dim, size_t q_stride, size_t k_stride, size_t q_out_stride, size_t k_out_stride,
                            float magnitude, int layout, int inverse, int kind) {
    clear_error();
    const char *name = "rotary";
    KREA2_REQUIRE(tokens >= 1 && tokens <= 16777216, "%s: tokens %zu outside 1..16777216", name, tokens);
    KREA2_REQUIRE(q_heads >= 1 && q_heads <= 1024 && kv_heads <= 1024, "%s: %zu query heads and %zu key heads, 1..1024 and 0..1024 are served", name,
                  q_heads, kv_heads);
    KREA2_REQUIRE(head_dim >= 2 && head_dim <= 512, "%s: head_dim %zu outside 2..512", name, head_dim);
    KREA2_REQUIRE(rotary_dim >= 2 && rotary_dim <= head_dim && rotary_dim % 2 == 0, "%s: rotary_dim %zu must be even, in 2..head_dim %zu", name,
                  rotary_dim, head_dim);
    KREA2_REQUIRE(q_stride >= q_heads * head_dim && q_out_stride >= q_heads * head_dim, "%s: a query row holds %zu values, the strides are %zu and %zu",
                  name, q_heads * head_dim, q_stride, q_out_stride);
    KREA2_REQUIRE(kv_heads == 0 || (k_stride >= kv_heads * head_dim && k_out_stride >= kv_heads * head_dim),
                  "%s: a key row holds %zu values, the strides are %zu and %zu", name, kv_heads * head_dim, k_stride, k_out_stride);
    KREA2_REQUIRE(std::isfinite(magnitude), "%s: magnitude is not a finite number", name);
    KREA2_REQUIRE(layout == KREA2_ROTARY_INTERLEAVED || layout == KREA2_ROTARY_HALF, "%s: layout %d is neither interleaved nor half", name, layout);
    KREA2_REQUIRE(inverse == 0 || inverse == 1, "%s: inverse must be 0 or 1", name);
    KREA2_REQUIRE(kind == KREA2_F16 || kind == KREA2_BF16, "%s: kind %d is neither KREA2_F16 nor KREA2_BF16", name, kind);
    KREA2_REQUIRE(q && q_out && frequencies && (kv_heads == 0 || (k && k_out)), "%s: null buffer", name);
    KREA2_REQUIRE(q != q_out || q_stride == q_out_stride, "%s: turning queries in place needs equal strides", name);
    KREA2_REQUIRE(kv_heads == 0 || k != k_out || k_stride == k_out_stride, "%s: turning keys in place needs equal strides", name);
    KREA2_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(q_out) |
                   reinterpret_cast<uintptr_t>(k_out)) % 2 == 0 &&
                      reinterpret_cast<uintptr_t>(positions) % 4 == 0 && reinterpret_cast<uintptr_t>(frequencies) % 8 == 0,
                  "%s: buffers must be aligned to their element size", name);
    const RotaryArgs g = {static_cast<const uint16_t *>(q), static_cast<const uint16_t *>(k), positions, frequencies,
                          static_cast<uint16_t *>(q_out), static_cast<uint16_t *>(k_out), static_cast<uint32_t>(q_heads),
                          static_cast<uint32_t>(kv_heads), static_cast<uint32_t>(head_dim), static_cast<uint32_t>(rotary_dim / 2),
                          q_stride, k_stride, q_out_stride, k_out_stride, magnitude, inverse ? -1.0f : 1.0f};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = static_cast<unsigned>(tokens);
    const bool interleaved = layout == KREA2_ROTARY_INTERLEAVED;
    if (kind == KREA2_BF16) interleaved ? rotary_kernel<true, true><<<grid, 256, 0, s>>>(g) : rotary_kernel<true, false><<<grid, 256, 0, s>>>(g);
    else interleaved ? rotary_kernel<false, true><<<grid, 256, 0, s>>>(g) : rotary_kernel<false, false><<<grid, 256, 0, s>>>(g);
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return fail(KREA2_RUNTIME, "%s launch failed: %s", name, cudaGetErrorString(status));
    return KREA2_OK;
}
