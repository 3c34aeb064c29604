// Rotary positions computed from position and frequency (new with this library; krea2_rope_qknorm_f16 takes the
// reference's finished tables): both pair layouts, any even part of a head, frequencies scaled for long contexts,
// forwards and backwards.
//   krea2_rotary_frequencies  radians per position of each pair, in f64, on the host
//   krea2_rotary              queries and keys turned, in place or into other buffers
#include <cmath>

#include "tensor_core.cuh"

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

__device__ __forceinline__ const uint16_t *head_in(const RotaryArgs &g, size_t token, uint32_t head) {
    return head < g.q_heads ? g.q + token * g.q_stride + static_cast<size_t>(head) * g.head_dim
                            : g.k + token * g.k_stride + static_cast<size_t>(head - g.q_heads) * g.head_dim;
}
__device__ __forceinline__ uint16_t *head_out(const RotaryArgs &g, size_t token, uint32_t head) {
    return head < g.q_heads ? g.q_out + token * g.q_out_stride + static_cast<size_t>(head) * g.head_dim
                            : g.k_out + token * g.k_out_stride + static_cast<size_t>(head - g.q_heads) * g.head_dim;
}

// cos and sin of position * frequency.  The product and its remainder by whole turns are taken in f64 (at position
// 10^6 an f32 product is off by 0.06 radians), what is left is below half a turn and exact enough in f32.
__device__ __forceinline__ void turn_of(int32_t position, double frequency, float &cosine, float &sine) {
    const double turns = static_cast<double>(position) * frequency * 0.15915494309189533577;  // 1 / (2 pi)
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &sine, &cosine);
}

template <bool kBf16>
__device__ __forceinline__ float low_value(uint32_t word) { return value_of<kBf16>(static_cast<uint16_t>(word)); }
template <bool kBf16>
__device__ __forceinline__ float high_value(uint32_t word) { return value_of<kBf16>(static_cast<uint16_t>(word >> 16)); }

// HBM-bound: 4608 tokens of 48 + 12 heads of 128 take 26.4-28.1 us (5.0-5.4 TB/s of reads and writes, 0.78-0.83 of the copy
// rate), 55 us with a lane per pair and element-wise accesses; one token 2.6-3.6 us.  A warp walks heads of one token, four
// heads' loads in flight (the first are under way before the angles are taken); `warps` warps share a token's heads where the
// tokens do not fill the device.  The token's cosines and sines are taken once per warp, a pair per lane, and lie in shared
// memory; a lane keeps those of its piece in registers.
constexpr int kBatch = 4;

__device__ __forceinline__ void take_turns(const RotaryArgs &g, size_t token, uint32_t lane, float2 *turn) {
    const int32_t position = g.positions ? g.positions[token] : static_cast<int32_t>(token);
    for (uint32_t pair = lane; pair < g.half; pair += 32) {
        float c, s;
        turn_of(position, __ldg(g.frequencies + pair), c, s);
        turn[pair] = make_float2(c * g.magnitude, s * g.magnitude * g.direction);
    }
    __syncwarp();
}

// Heads on 16-byte boundaries: a lane owns one piece of eight channels.  A piece of the half layout meets its partners, half
// a rotary part away in the same head, by shuffles, so that every load and store of a warp is contiguous.
template <bool kBf16, bool kInterleaved>
__global__ void __launch_bounds__(256)
rotary_pieces_kernel(const RotaryArgs g, uint32_t tokens, uint32_t warps) {
    __shared__ float2 turns_of_warp[8][256];
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const size_t token = item / warps;
    if (token >= tokens) return;
    const uint32_t share = static_cast<uint32_t>(item % warps), lane = threadIdx.x & 31;
    const uint32_t pieces = g.head_dim / 8, heads = g.q_heads + g.kv_heads;
    bool taken = false;
    for (uint32_t piece0 = 0; piece0 < pieces; piece0 += 32) {
        const uint32_t here = min(32u, pieces - piece0), per_pass = 32 / here;  // heads side by side in a warp
        const uint32_t piece = piece0 + lane % here, offset = lane / here, stride = warps * per_pass;
        const bool idle = offset >= per_pass;
        uint4 x[kBatch];
        auto request = [&](uint32_t head0) {
#pragma unroll
            for (int b = 0; b < kBatch; b++) {
                const uint32_t head = head0 + offset + b * stride;
                x[b] = make_uint4(0, 0, 0, 0);
                if (!idle && head < heads) x[b] = *reinterpret_cast<const uint4 *>(head_in(g, token, head) + piece * 8);
            }
        };
        request(share * per_pass);
        float2 *turn = turns_of_warp[threadIdx.x >> 5];
        if (!taken) take_turns(g, token, lane, turn);
        taken = true;
        constexpr int kPairs = kInterleaved ? 4 : 8;
        const uint32_t away = kInterleaved ? 0u : g.half / 8;  // pieces to a piece's partner
        const bool second = !kInterleaved && piece >= away;
        const uint32_t pair0 = (second ? piece - away : piece) * kPairs;
        const uint32_t inside = kInterleaved ? (g.half > pair0 ? min(4u, g.half - pair0) : 0u) : (piece < 2 * away ? 8u : 0u);  // pairs that turn
        const uint32_t partner = second ? lane - away : lane + away;
        float2 by[kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            by[i] = make_float2(1.0f, 0.0f);
            if (i < inside) by[i] = turn[pair0 + i];
            if (!kInterleaved && !second) by[i].y = -by[i].y;  // own * cos + partner * sin, the first of a pair against -sin
        }
        for (uint32_t head0 = share * per_pass; head0 < heads; head0 += kBatch * stride) {
#pragma unroll
            for (int b = 0; b < kBatch; b++) {
                uint32_t *own = reinterpret_cast<uint32_t *>(&x[b]);
                if constexpr (kInterleaved) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float p = low_value<kBf16>(own[i]), q = high_value<kBf16>(own[i]);
                        if (i < inside) own[i] = pack_pair<kBf16>(p * by[i].x - q * by[i].y, q * by[i].x + p * by[i].y);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t other = __shfl_sync(0xffffffffu, own[i], partner & 31u);
                        const float2 c0 = by[2 * i], c1 = by[2 * i + 1];
                        const uint32_t turned = pack_pair<kBf16>(low_value<kBf16>(own[i]) * c0.x + low_value<kBf16>(other) * c0.y,
                                                               high_value<kBf16>(own[i]) * c1.x + high_value<kBf16>(other) * c1.y);
                        if (inside) own[i] = turned;  // a channel that is not turned is copied, whatever it holds
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < kBatch; b++) {
                const uint32_t head = head0 + offset + b * stride;
                if (!idle && head < heads) *reinterpret_cast<uint4 *>(head_out(g, token, head) + piece * 8) = x[b];
            }
            if (head0 + kBatch * stride < heads) request(head0 + kBatch * stride);
        }
    }
}

// Other heads: a lane owns one pair; the channels from `copied` on, which are not turned and fall on 16-byte boundaries, are
// copied in pieces, those between one by one.
template <bool kBf16, bool kInterleaved>
__global__ void __launch_bounds__(256)
rotary_pairs_kernel(const RotaryArgs g, uint32_t tokens, uint32_t warps, uint32_t copied) {
    __shared__ float2 turns_of_warp[8][256];
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const size_t token = item / warps;
    if (token >= tokens) return;
    const uint32_t share = static_cast<uint32_t>(item % warps), lane = threadIdx.x & 31;
    float2 *turn = turns_of_warp[threadIdx.x >> 5];
    take_turns(g, token, lane, turn);
    const uint32_t heads = g.q_heads + g.kv_heads, units = copied - g.half;
    for (uint32_t unit0 = 0; unit0 < units; unit0 += 32) {
        const uint32_t here = min(32u, units - unit0), per_pass = 32 / here, stride = warps * per_pass;
        const uint32_t unit = unit0 + lane % here, offset = lane / here;
        if (offset >= per_pass) continue;
        const bool turns = unit < g.half;
        const float2 by = turns ? turn[unit] : make_float2(1.0f, 0.0f);
        const uint32_t first = !turns ? unit + g.half : kInterleaved ? 2 * unit : unit;
        const uint32_t second = !turns ? first : kInterleaved ? first + 1 : unit + g.half;
        for (uint32_t head = share * per_pass + offset; head < heads; head += kBatch * stride) {
            uint16_t a[kBatch], b[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; k++) {
                if (head + k * stride >= heads) break;
                const uint16_t *in = head_in(g, token, head + k * stride);
                a[k] = in[first], b[k] = in[second];
            }
#pragma unroll
            for (int k = 0; k < kBatch; k++) {
                if (head + k * stride >= heads) break;
                uint16_t *out = head_out(g, token, head + k * stride);
                if (turns) {
                    const float x = value_of<kBf16>(a[k]), y = value_of<kBf16>(b[k]);
                    out[second] = bits_of<kBf16>(y * by.x + x * by.y);
                    out[first] = bits_of<kBf16>(x * by.x - y * by.y);
                } else {
                    out[first] = a[k];
                }
            }
        }
    }
    const uint32_t pieces = (g.head_dim - copied) / 8;
    for (uint32_t item8 = lane; item8 < heads * pieces; item8 += 32) {
        const uint32_t head = item8 / pieces, at = copied + item8 % pieces * 8;
        if (head % warps == share) *reinterpret_cast<uint4 *>(head_out(g, token, head) + at) = *reinterpret_cast<const uint4 *>(head_in(g, token, head) + at);
    }
}

template <bool kBf16, bool kInterleaved>
void launch_rotary(cudaStream_t stream, uint32_t tokens, const RotaryArgs &g, bool aligned) {
    // Pieces need partners a whole number of pieces away, within the 32 pieces that a warp holds of a head.
    const bool pieces = aligned && (kInterleaved || (g.half % 8 == 0 && g.head_dim <= 256));
    const uint32_t copied = aligned ? (2 * g.half + 7) / 8 * 8 : g.head_dim;
    const uint32_t units = min(32u, pieces ? g.head_dim / 8 : copied - g.half), per_pass = 32 / units;
    // About 32 warps an SM, each with a pass over the heads at least.
    const uint32_t passes = (g.q_heads + g.kv_heads + per_pass - 1) / per_pass, wanted = 32u * static_cast<uint32_t>(multiprocessors()) / tokens;
    const uint32_t warps = max(1u, min(wanted, passes));
    const unsigned blocks = static_cast<unsigned>((static_cast<uint64_t>(tokens) * warps + 7) / 8);
    if (pieces) rotary_pieces_kernel<kBf16, kInterleaved><<<blocks, 256, 0, stream>>>(g, tokens, warps);
    else rotary_pairs_kernel<kBf16, kInterleaved><<<blocks, 256, 0, stream>>>(g, tokens, warps, copied);
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
    const uint32_t n = static_cast<uint32_t>(tokens);
    const bool interleaved = layout == KREA2_ROTARY_INTERLEAVED;
    const bool aligned = head_dim % 8 == 0 && aligned16(q) && aligned16(q_out) && q_stride % 8 == 0 && q_out_stride % 8 == 0 &&
                         (kv_heads == 0 || (aligned16(k) && aligned16(k_out) && k_stride % 8 == 0 && k_out_stride % 8 == 0));
    if (kind == KREA2_BF16) interleaved ? launch_rotary<true, true>(s, n, g, aligned) : launch_rotary<true, false>(s, n, g, aligned);
    else interleaved ? launch_rotary<false, true>(s, n, g, aligned) : launch_rotary<false, false>(s, n, g, aligned);
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return fail(KREA2_RUNTIME, "%s launch failed: %s", name, cudaGetErrorString(status));
    return KREA2_OK;
}
