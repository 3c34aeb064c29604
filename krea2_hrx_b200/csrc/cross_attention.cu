// Attention of queries to an encoder's states of another length (new with this library: the reference's attention is
// over one sequence, whose values it transposes first): batches whose items count different numbers of keys, a key
// mask, bf16 and f16, heads of 8 to 128 channels, rows at any 16-byte pitch.
//   out[b][i][h] = sum_j p_j v[b][j][h'] / sum_j p_j,  p_j = exp(scale q[b][i][h] . k[b][j][h'])
// over the keys j < kv_lengths[b] whose mask byte is not zero, h' = h / (q_heads / kv_heads); zero where there is none.
#include <cmath>

#include "common.cuh"

namespace krea2 {
namespace {

struct CrossArgs {
    const uint16_t *q, *k, *v;
    const int32_t *kv_lengths;
    const uint8_t *key_mask;
    uint16_t *out;
    uint32_t q_len, kv_len, q_heads, shares, head_dim;
    size_t q_batch_stride, q_stride, k_batch_stride, k_stride, v_batch_stride, v_stride, out_batch_stride, out_stride, mask_stride;
    float scale_log2;
};

// A warp per query row and head, four channels per lane, one pass over the keys with the running maximum and sum.
template <bool kBf16>
__global__ void __launch_bounds__(256)
cross_attention_kernel(const CrossArgs g) {
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (item >= static_cast<uint64_t>(g.q_len) * g.q_heads) return;
    const uint32_t batch = blockIdx.y, row = static_cast<uint32_t>(item / g.q_heads), head = static_cast<uint32_t>(item % g.q_heads);
    const uint32_t kv_head = head / g.shares;
    int32_t length = static_cast<int32_t>(g.kv_len);
    if (g.kv_lengths) length = min(max(g.kv_lengths[batch], 0), length);
    const uint16_t *q = g.q + batch * g.q_batch_stride + row * g.q_stride + head * g.head_dim;
    float query[4], out[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) query[i] = lane + 32 * i < g.head_dim ? value_of<kBf16>(q[lane + 32 * i]) * g.scale_log2 : 0.0f;
    float top = -INFINITY, sum = 0.0f;
    for (int32_t j = 0; j < length; j++) {
        if (g.key_mask && g.key_mask[batch * g.mask_stride + j] == 0) continue;
        const uint16_t *k = g.k + batch * g.k_batch_stride + j * g.k_stride + kv_head * g.head_dim;
        const uint16_t *v = g.v + batch * g.v_batch_stride + j * g.v_stride + kv_head * g.head_dim;
        float score = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < g.head_dim) score = fmaf(query[i], value_of<kBf16>(k[lane + 32 * i]), score);
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) score += __shfl_xor_sync(0xffffffffu, score, off);
        const float next = fmaxf(top, score), shift = next == -INFINITY ? 0.0f : next;
        const float keep = exp2f(top - shift), p = exp2f(score - shift);
        top = next;
        sum = sum * keep + p;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane + 32 * i < g.head_dim) out[i] = fmaf(p, value_of<kBf16>(v[lane + 32 * i]), out[i] * keep);
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t *dst = g.out + batch * g.out_batch_stride + row * g.out_stride + head * g.head_dim;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (lane + 32 * i < g.head_dim) dst[lane + 32 * i] = bits_of<kBf16>(out[i] * inverse);
}

}  // namespace
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
    KREA2_REQUIRE(batch == 1 || out_batch_stride >= (q_len - 1) * out_stride + q_heads * head_dim, "%s: the batch's outputs overlap", name);
    KREA2_REQUIRE(!key_mask || mask_stride >= kv_len, "%s: mask_stride %zu is below kv_len %zu", name, mask_stride, kv_len);
    KREA2_REQUIRE(std::isfinite(scale) && scale > 0.0f, "%s: scale must be a positive number", name);
    KREA2_REQUIRE(kind == KREA2_F16 || kind == KREA2_BF16, "%s: kind %d is neither KREA2_F16 nor KREA2_BF16", name, kind);
    KREA2_REQUIRE(q && out && (kv_len == 0 || (k && v)), "%s: null buffer", name);
    KREA2_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out), "%s: buffers must be 16-byte aligned", name);
    KREA2_REQUIRE(reinterpret_cast<uintptr_t>(kv_lengths) % 4 == 0, "%s: kv_lengths must be 4-byte aligned", name);
    const CrossArgs g = {static_cast<const uint16_t *>(q), static_cast<const uint16_t *>(k), static_cast<const uint16_t *>(v), kv_lengths, static_cast<const uint8_t *>(key_mask),
                         static_cast<uint16_t *>(out), static_cast<uint32_t>(q_len), static_cast<uint32_t>(kv_len), static_cast<uint32_t>(q_heads),
                         static_cast<uint32_t>(q_heads / kv_heads), static_cast<uint32_t>(head_dim), q_batch_stride, q_stride, k_batch_stride,
                         k_stride, v_batch_stride, v_stride, out_batch_stride, out_stride, mask_stride, scale * 1.44269504088896340736f};
    const size_t blocks = (q_len * q_heads + 7) / 8;
    KREA2_REQUIRE(blocks <= 0x7fffffff, "%s: %zu query rows of %zu heads exceed the grid", name, q_len, q_heads);
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(batch));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (kind == KREA2_BF16) cross_attention_kernel<true><<<grid, 256, 0, s>>>(g);
    else cross_attention_kernel<false><<<grid, 256, 0, s>>>(g);
    const cudaError_t status = cudaGetLastError();
    if (status != cudaSuccess) return fail(KREA2_RUNTIME, "%s launch failed: %s", name, cudaGetErrorString(status));
    return KREA2_OK;
}
