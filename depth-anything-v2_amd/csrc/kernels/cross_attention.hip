// Attention of queries to keys and values of another length (an encoder's
// tokens): softmax(scale * q k^T) v over the keys that a batch sees.

#include "decoder.h"

using namespace dav2k;

namespace {

// One wave per query row and head, 64 keys at a time: lane l scores key l,
// then takes features l and l + 64 of the values.
template <typename E>
__global__ __launch_bounds__(64) void cross_attention_kernel(dav2_cross_attention_args a) {
    __shared__ float qs[128], w[64];
    const uint32_t h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x, d = a.head_dim;
    const uint32_t kvh = h / (a.heads / a.kv_heads);
    uint32_t keys = a.key_tokens;
    if (a.key_lengths) keys = min(keys, static_cast<uint32_t>(max(a.key_lengths[b], 0)));
    const E* k = static_cast<const E*>(a.keys) + b * a.key_batch_stride + uint64_t(kvh) * d;
    const E* v = static_cast<const E*>(a.values) + b * a.value_batch_stride + uint64_t(kvh) * d;
    const uint8_t* mask = a.key_mask ? a.key_mask + static_cast<uint64_t>(b) * a.key_tokens : nullptr;
    for (uint32_t row = blockIdx.x; row < a.query_tokens; row += gridDim.x) {
        const E* x = static_cast<const E*>(a.query) + b * a.query_batch_stride + row * a.query_stride + uint64_t(h) * d;
        __syncthreads();
        for (uint32_t f = lane; f < d; f += 64u) qs[f] = static_cast<float>(x[f]) * a.scale;
        __syncthreads();
        float most = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
        for (uint32_t j0 = 0; j0 < keys; j0 += 64u) {
            const uint32_t j = j0 + lane;
            const bool seen = j < keys && (!mask || mask[j]);
            const uint64_t visible = __ballot(seen);
            if (!visible) continue;
            float score = -INFINITY;
            if (seen) {
                const E* kr = k + j * a.key_stride;
                score = 0.0f;
                for (uint32_t f = 0; f < d; ++f) score = fmaf(qs[f], static_cast<float>(kr[f]), score);
            }
            const float grown = fmaxf(most, wave_max(score));
            const float keep = most == -INFINITY ? 0.0f : expf(most - grown);
            const float weight = seen ? expf(score - grown) : 0.0f;
            most = grown;
            sum = fmaf(sum, keep, wave_sum_tree(weight));
            o0 *= keep;
            o1 *= keep;
            __syncthreads();
            w[lane] = weight;
            __syncthreads();
            for (uint32_t i = 0; i < 64u; ++i) {
                if (!(visible >> i & 1u)) continue;
                const E* vr = v + (j0 + i) * a.value_stride;
                if (lane < d) o0 = fmaf(w[i], static_cast<float>(vr[lane]), o0);
                if (lane + 64u < d) o1 = fmaf(w[i], static_cast<float>(vr[lane + 64u]), o1);
            }
        }
        E* y = static_cast<E*>(a.output) + b * a.output_batch_stride + row * a.output_stride + uint64_t(h) * d;
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (lane < d) y[lane] = static_cast<E>(o0 * inverse);
        if (lane + 64u < d) y[lane + 64u] = static_cast<E>(o1 * inverse);
    }
}

}  // namespace

extern "C" {

uint64_t dav2_hip_cross_attention_scratch_bytes(const dav2_cross_attention_args*) { return 0; }

int dav2_hip_cross_attention(const dav2_cross_attention_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_cross_attention_args& a = *args;
    if (a.batch == 0 || a.query_tokens == 0) return hipSuccess;
    const uint64_t row = static_cast<uint64_t>(a.heads) * a.head_dim;
    const uint64_t key_row = static_cast<uint64_t>(a.kv_heads) * a.head_dim;
    const uint64_t strides = a.query_stride | a.key_stride | a.value_stride | a.output_stride | a.query_batch_stride |
                             a.key_batch_stride | a.value_batch_stride | a.output_batch_stride;
    if (!a.query || !a.output || (a.key_tokens && (!a.keys || !a.values)) || !aligned16(a.query) ||
        !aligned16(a.output) || !aligned16(a.keys) || !aligned16(a.values) || strides % 8 ||
        a.dtype > DAV2_DTYPE_BF16 || a.batch > 65535u || a.query_tokens > 0x7fffffffu || a.key_tokens > 0x7fffffffu ||
        a.heads == 0 || a.heads > 65535u || a.kv_heads == 0 || a.heads % a.kv_heads || a.head_dim < 16 ||
        a.head_dim > 128 || a.head_dim % 16 ||
        (a.query_tokens > 1 && (a.query_stride < row || a.output_stride < row)) ||
        (a.key_tokens > 1 && (a.key_stride < key_row || a.value_stride < key_row)))
        return hipErrorInvalidValue;
    const uint64_t need = dav2_hip_cross_attention_scratch_bytes(args);
    if (need && (!a.scratch || !aligned16(a.scratch) || a.scratch_bytes < need)) return hipErrorInvalidValue;
    const dim3 grid(a.query_tokens, a.heads, a.batch);
    with_dtype(a.dtype, [&](auto* e) {
        dispatch(cross_attention_kernel<std::remove_pointer_t<decltype(e)>>, grid, dim3(64), 0,
                 static_cast<hipStream_t>(stream), a);
    });
    return hipGetLastError();
}

}  // extern "C"
