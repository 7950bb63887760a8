// A residual's addition, the root-mean-square norm and rows in 8 bits.
//
//   h = x + r in the type, f = fp32(1 / sqrt(mean h^2 + epsilon)), y = (h f) w,
//   code = rint(y / s), s = max(absmax y / 127, 1e-8).
//
// The squares are summed in 64 bits, which costs nothing beside the loads: f is
// then the same for any order of the sum, and a code next to a border does not
// go by how many lanes share a row.

#include <algorithm>
#include <type_traits>

#include "decoder.h"

using namespace dav2k;

namespace {

DAV2_DEV double wave_sum(double v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}
DAV2_DEV uint32_t wave_max_bits(uint32_t v) {
    for (int o = 32; o > 0; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o, kWave)));
    return v;
}

// A workgroup for each row, which is read again for its largest value and for its outputs.
template <typename E>
__global__ __launch_bounds__(256) void rms_norm_kernel(dav2_add_rms_norm_args a) {
    typedef Vec<E> V;
    constexpr int N = V::N;
    __shared__ double sums[4];
    __shared__ uint32_t largest[4];
    const uint32_t wave = threadIdx.x >> 6, columns = a.columns;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const E* x = static_cast<const E*>(a.input) + row * a.input_stride;
        const E* r = a.residual ? static_cast<const E*>(a.residual) + row * a.residual_stride : nullptr;
        E* sum = a.sum ? static_cast<E*>(a.sum) + row * a.sum_stride : nullptr;
        auto load = [&](uint32_t c, float (&v)[N]) {
            V::load(x, c, columns, v);
            if (r) {
                float w[N];
                V::load(r, c, columns, w);
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = static_cast<float>(static_cast<E>(keep_fp32(v[i] + w[i])));
            }
        };
        double squares = 0.0;
        for (uint32_t c = threadIdx.x * N; c < columns; c += 256u * N) {
            float v[N];
            load(c, v);
            if (sum) V::store(sum, c, columns, v);
#pragma unroll
            for (int i = 0; i < N; ++i) squares = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), squares);
        }
        if (sum) {  // which may be x or r: what was added is there now
            x = sum;
            r = nullptr;
        }
        squares = wave_sum(squares);
        __syncthreads();
        if ((threadIdx.x & 63u) == 0) sums[wave] = squares;
        __syncthreads();
        squares = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        const float factor = static_cast<float>(1.0 / sqrt(squares / columns + static_cast<double>(a.epsilon)));
        auto norm = [&](uint32_t c, float (&v)[N]) {
            load(c, v);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = v[i] * factor;
            if (!a.weight) return;
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                float w[4];
                Vec<float>::load(a.weight, c + j, columns, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[j + i] *= w[i];
            }
        };
        float scale = 1.0f, inverse = 1.0f;
        if (a.codes) {
            uint32_t most = 0;
            for (uint32_t c = threadIdx.x * N; c < columns; c += 256u * N) {
                float v[N];
                norm(c, v);
#pragma unroll
                for (int i = 0; i < N; ++i) most = max(most, __float_as_uint(fabsf(v[i])));  // NaN above all
            }
            most = wave_max_bits(most);
            if ((threadIdx.x & 63u) == 0) largest[wave] = most;
            __syncthreads();
            most = max(max(largest[0], largest[1]), max(largest[2], largest[3]));
            scale = __uint_as_float(max(__float_as_uint(div_rn(__uint_as_float(most), 127.0f)), __float_as_uint(1.0e-8f)));
            inverse = div_rn(1.0f, scale);
            if (threadIdx.x == 0) a.scales[row] = scale;
        }
        E* y = a.output ? static_cast<E*>(a.output) + row * a.output_stride : nullptr;
        int8_t* q = a.codes ? a.codes + row * a.code_stride : nullptr;
        const uint64_t width = q ? a.code_stride : columns;
        for (uint64_t c = threadIdx.x * N; c < width; c += 256u * N) {
            uint32_t words[N / 4] = {};
            if (c < columns) {
                float v[N];
                norm(static_cast<uint32_t>(c), v);
                if (y) V::store(y, static_cast<uint32_t>(c), columns, v);
                if (q)
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (c + i < columns)
                            words[i / 4] |= (static_cast<uint32_t>(quantize_div(v[i], scale, inverse)) & 0xffu) << (8 * (i % 4));
            }
            if (q)
#pragma unroll
                for (int i = 0; i < N / 4; ++i) reinterpret_cast<uint32_t*>(q + c)[i] = words[i];
        }
    }
}

}  // namespace

extern "C" {

int dav2_hip_add_rms_norm(const dav2_add_rms_norm_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_add_rms_norm_args& a = *args;
    if (a.rows == 0 || a.columns == 0) return hipSuccess;
    auto strided = [&](uint64_t stride) { return a.rows == 1 || stride >= a.columns; };
    auto placed = [&](const void* out, uint64_t stride) {  // as an input, with its stride
        return !out || (strided(stride) && (out != a.input || a.rows == 1 || stride == a.input_stride) &&
                        (out != a.residual || a.rows == 1 || stride == a.residual_stride));
    };
    if (!a.input || (!a.sum && !a.output && !a.codes) || a.dtype > DAV2_DTYPE_BF16 || !(a.epsilon > 0.0f) ||
        a.rows > 0x7fffffffu || a.columns >= (1u << 20) || !strided(a.input_stride) ||
        (a.residual && !strided(a.residual_stride)) || !placed(a.sum, a.sum_stride) ||
        !placed(a.output, a.output_stride) || (a.sum && a.sum == a.output) ||
        (a.codes && (!a.scales || !aligned16(a.codes) || a.code_stride % 64 || a.code_stride < a.columns)))
        return hipErrorInvalidValue;
    return with_dtype(a.dtype, [&](auto* e) -> int {
        typedef std::remove_pointer_t<decltype(e)> E;
        dispatch(rms_norm_kernel<E>, dim3(std::min(a.rows, 1u << 22)), dim3(256), 0, static_cast<hipStream_t>(stream), a);
        return hipGetLastError();
    });
}

}  // extern "C"
