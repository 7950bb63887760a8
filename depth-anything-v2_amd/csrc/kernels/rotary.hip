// Rotary positions, alone and behind the norm of each query and key head.
//
// (a, b) -> A (a cos t - b sin t, b cos t + a sin t), t = p f_i. The angle is
// formed in 64 bits and reduced to a fraction of a turn there: in fp32 a
// position of 10^6 would leave 0.06 radians of it uncertain.

#include "decoder.h"

using namespace dav2k;

namespace {

constexpr double kTurnsPerRadian = 0.15915494309189533577;

// One wave per head of a token: lane l has features l, l + 64, ...
template <typename E, bool NORM>
__global__ __launch_bounds__(256) void rotary_kernel(dav2_qk_norm_rotary_args a) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t heads = a.query_heads + a.key_heads;
    const uint64_t item = static_cast<uint64_t>(blockIdx.x) * 4u + (threadIdx.x >> 6);
    if (item >= static_cast<uint64_t>(a.tokens) * heads) return;
    const uint64_t token = item / heads;
    uint32_t head = static_cast<uint32_t>(item - token * heads);
    const bool is_key = head >= a.query_heads;
    if (is_key) head -= a.query_heads;
    const E* x = static_cast<const E*>(is_key ? a.key : a.query) + token * (is_key ? a.key_stride : a.query_stride) +
                 static_cast<uint64_t>(head) * a.head_dim;
    E* y = static_cast<E*>(is_key ? a.key_out : a.query_out) +
           token * (is_key ? a.key_out_stride : a.query_out_stride) + static_cast<uint64_t>(head) * a.head_dim;
    const float* weight = is_key ? a.key_weight : a.query_weight;
    const uint32_t d = a.head_dim;
    float mean = 0.0f, factor = 1.0f;
    if (NORM) {
        if (a.norm == DAV2_QK_NORM_LAYER) {
            float sum = 0.0f;
            for (uint32_t i = lane; i < d; i += 64u) sum += static_cast<float>(x[i]);
            mean = wave_sum_tree(sum) / static_cast<float>(d);
        }
        float squares = 0.0f;
        for (uint32_t i = lane; i < d; i += 64u) {
            const float v = static_cast<float>(x[i]) - mean;
            squares = fmaf(v, v, squares);
        }
        factor = 1.0f / sqrtf(wave_sum_tree(squares) / static_cast<float>(d) + a.epsilon);
    }
    auto at = [&](uint32_t i) {
        float v = static_cast<float>(x[i]);
        if (NORM) {
            v = (v - mean) * factor;
            if (weight) v *= weight[i];
        }
        return v;
    };
    const uint32_t half = a.rotary_dim / 2;
    for (uint32_t i = lane; i < half; i += 64u) {
        const uint32_t i0 = a.layout == DAV2_ROTARY_HALVES ? i : 2 * i;
        const uint32_t i1 = a.layout == DAV2_ROTARY_HALVES ? i + half : 2 * i + 1;
        const double turns = static_cast<double>(a.positions[token]) * (a.frequencies[i] * kTurnsPerRadian);
        float s, c;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
        s *= a.amplitude;
        c *= a.amplitude;
        const float u = at(i0), v = at(i1);
        y[i0] = static_cast<E>(u * c - v * s);
        y[i1] = static_cast<E>(v * c + u * s);
    }
    for (uint32_t i = a.rotary_dim + lane; i < d; i += 64u) y[i] = static_cast<E>(at(i));
}

bool valid(const dav2_qk_norm_rotary_args& a) {
    if (a.dtype > DAV2_DTYPE_BF16 || a.layout > DAV2_ROTARY_PAIRS || a.norm > DAV2_QK_NORM_LAYER) return false;
    if (a.head_dim == 0 || a.head_dim > 1024 || a.rotary_dim > a.head_dim || a.rotary_dim % 2) return false;
    if (a.rotary_dim && (!a.positions || !a.frequencies)) return false;
    if (a.query_heads > 65535 || a.key_heads > 65535 || a.tokens > 0x7fffffffu) return false;
    auto side = [&](const void* in, const void* out, uint32_t heads, uint64_t in_stride, uint64_t out_stride) {
        const uint64_t row = static_cast<uint64_t>(heads) * a.head_dim;
        return heads == 0 || (in && out && (a.tokens == 1 || (in_stride >= row && out_stride >= row)) &&
                              (in != out || a.tokens == 1 || in_stride == out_stride));
    };
    return side(a.query, a.query_out, a.query_heads, a.query_stride, a.query_out_stride) &&
           side(a.key, a.key_out, a.key_heads, a.key_stride, a.key_out_stride);
}

template <bool NORM>
int launch(const dav2_qk_norm_rotary_args& a, void* stream) {
    const uint64_t items = static_cast<uint64_t>(a.tokens) * (a.query_heads + a.key_heads);
    if ((items + 3) / 4 > 0x7fffffffull) return hipErrorInvalidValue;
    with_dtype(a.dtype, [&](auto* e) {
        dispatch(rotary_kernel<std::remove_pointer_t<decltype(e)>, NORM>, dim3(ceil_div(items, 4)), dim3(256), 0,
                 static_cast<hipStream_t>(stream), a);
    });
    return hipGetLastError();
}

}  // namespace

extern "C" {

int dav2_hip_rotary(const dav2_rotary_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    if (args->tokens == 0 || args->heads == 0) return hipSuccess;
    dav2_qk_norm_rotary_args a{};
    a.query = args->input;
    a.query_out = args->output;
    a.query_stride = args->input_stride;
    a.query_out_stride = args->output_stride;
    a.positions = args->positions;
    a.frequencies = args->frequencies;
    a.tokens = args->tokens;
    a.query_heads = args->heads;
    a.head_dim = args->head_dim;
    a.rotary_dim = args->rotary_dim;
    a.layout = args->layout;
    a.dtype = args->dtype;
    a.amplitude = args->amplitude;
    if (args->rotary_dim == 0 || !valid(a)) return hipErrorInvalidValue;
    return launch<false>(a, stream);
}

int dav2_hip_qk_norm_rotary(const dav2_qk_norm_rotary_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    if (args->tokens == 0 || (args->query_heads == 0 && args->key_heads == 0)) return hipSuccess;
    if (!valid(*args) || !(args->epsilon > 0.0f)) return hipErrorInvalidValue;
    return launch<true>(*args, stream);
}

}  // extern "C"
