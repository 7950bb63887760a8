// A residual's addition, the root-mean-square norm and rows in 8 bits.
//
//   h = x + r in the type, f = fp32(1 / sqrt(mean h^2 + epsilon)), y = (h f) w,
//   code = rint(y / s), s = max(absmax y / 127, 1e-8).
//
// The squares are summed in 64 bits, which costs nothing beside the loads: orders
// of the sum differ by some 2^-52, so that f is the same for any of them unless
// the root lies that near to a border of fp32, one row in 2^28. A code next to a
// border then hardly ever goes by how many lanes share a row.

#include <algorithm>
#include <type_traits>

#include "decoder.h"

using namespace dav2k;

namespace {

// Over the wave, received by all lanes: sums and maxima run up to lane 63.
template <int CTRL, int ROWS>
DAV2_DEV double moved(double v) {
    return __longlong_as_double(static_cast<long long>(moved64<CTRL, ROWS>(static_cast<uint64_t>(__double_as_longlong(v)))));
}
DAV2_DEV double wave_sum(double v) {
    v += moved<0x111, 0xf>(v);  // row_shr:1
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);  // row_shr:8
    v += moved<0x142, 0xa>(v);  // row_bcast:15
    v += moved<0x143, 0xc>(v);  // row_bcast:31
    const long long bits = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_readlane(static_cast<int>(bits), 63);
    const int hi = __builtin_amdgcn_readlane(static_cast<int>(bits >> 32), 63);
    return __hiloint2double(hi, lo);
}
template <int CTRL, int ROWS>
DAV2_DEV uint32_t larger(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, true)));
}
DAV2_DEV uint32_t wave_max_bits(uint32_t v) {
    v = larger<0x111, 0xf>(v);
    v = larger<0x112, 0xf>(v);
    v = larger<0x114, 0xf>(v);
    v = larger<0x118, 0xf>(v);
    v = larger<0x142, 0xa>(v);
    v = larger<0x143, 0xc>(v);
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

DAV2_DEV float factor_of(double squares, const dav2_add_rms_norm_args& a) {
    return static_cast<float>(1.0 / sqrt(squares / a.columns + static_cast<double>(a.epsilon)));
}
DAV2_DEV float scale_of(uint32_t most) {  // the largest value's bits
    return __uint_as_float(max(__float_as_uint(div_rn(__uint_as_float(most), 127.0f)), __float_as_uint(1.0e-8f)));
}

// N codes of a row from element c on, those past its last zero.
template <int N>
DAV2_DEV void store_codes(int8_t* row, uint32_t c, uint32_t columns, const float (&v)[N], float scale, float inverse) {
    uint32_t words[N / 4] = {};
    // a value past the last is 0, and so is its code unless the scale is no number
#pragma unroll
    for (int i = 0; i < N; ++i)
        words[i / 4] |= (c + i < columns ? static_cast<uint32_t>(quantize_div(v[i], scale, inverse)) & 0xffu : 0u) << (8 * (i % 4));
    if constexpr (N == 8) *reinterpret_cast<uint2*>(row + c) = make_uint2(words[0], words[1]);
    else *reinterpret_cast<uint32_t*>(row + c) = words[0];
}

// LANES lanes share a row and keep it in registers, PIECES vectors each: one
// read of the inputs and one write of each output. Bound by memory: 8191 rows of
// 4096, bf16, sum, norm and codes (302 MB): 55 us, 5.5 TB/s, where a kernel that
// reads the row again from the caches takes 71. The weights stay in registers
// from row to row. Rows that are not multiples of 16 bytes are read as they lie:
// 8191 of 5003 100 us, of 5008 81.
template <typename E, int LANES, int PIECES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void rms_norm_kept_kernel(dav2_add_rms_norm_args a) {
    typedef Vec<E> V;
    constexpr int N = V::N, kThreads = LANES < 256 ? 256 : LANES, kRows = kThreads / LANES, kWaves = LANES / 64;
    __shared__ double sums[2][kThreads / 64];
    __shared__ uint32_t largest[2][kThreads / 64];
    const uint32_t columns = a.columns, lane = threadIdx.x % LANES, wave = threadIdx.x >> 6, wave0 = wave / kWaves * kWaves;
    float weight[PIECES][N];
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            float w[4] = {1.0f, 1.0f, 1.0f, 1.0f};
            if (a.weight) Vec<float>::load(a.weight, (p * LANES + lane) * N + j, columns, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) weight[p][j + i] = w[i];
        }
    uint32_t turn = 0;
    for (uint64_t first = static_cast<uint64_t>(blockIdx.x) * kRows; first < a.rows;
         first += static_cast<uint64_t>(gridDim.x) * kRows, turn ^= 1u) {
        const uint64_t row = min(first + threadIdx.x / LANES, static_cast<uint64_t>(a.rows) - 1u);
        const bool mine = first + threadIdx.x / LANES < a.rows;
        const E* x = static_cast<const E*>(a.input) + row * a.input_stride;
        float v[PIECES][N];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) V::load(x, (p * LANES + lane) * N, columns, v[p]);
        if (a.residual) {
            const E* r = static_cast<const E*>(a.residual) + row * a.residual_stride;
            float w[PIECES][N];
#pragma unroll
            for (int p = 0; p < PIECES; ++p) V::load(r, (p * LANES + lane) * N, columns, w[p]);
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int i = 0; i < N; ++i) v[p][i] = static_cast<float>(static_cast<E>(keep_fp32(v[p][i] + w[p][i])));
        }
        if (a.sum && mine) {
            E* sum = static_cast<E*>(a.sum) + row * a.sum_stride;
#pragma unroll
            for (int p = 0; p < PIECES; ++p) V::store(sum, (p * LANES + lane) * N, columns, v[p]);
        }
        double squares = 0.0;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int i = 0; i < N; ++i) squares = fma(static_cast<double>(v[p][i]), static_cast<double>(v[p][i]), squares);
        squares = wave_sum(squares);
        if constexpr (kWaves > 1) {
            if ((threadIdx.x & 63u) == 0) sums[turn][wave] = squares;
            __syncthreads();
            squares = 0.0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) squares += sums[turn][wave0 + w];
        }
        const float factor = factor_of(squares, a);
        uint32_t most = 0;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[p][i] = (v[p][i] * factor) * weight[p][i];
                most = max(most, __float_as_uint(fabsf(v[p][i])));  // NaN above all
            }
        if (a.output && mine) {
            E* y = static_cast<E*>(a.output) + row * a.output_stride;
#pragma unroll
            for (int p = 0; p < PIECES; ++p) V::store(y, (p * LANES + lane) * N, columns, v[p]);
        }
        if (!a.codes) continue;
        most = wave_max_bits(most);
        if constexpr (kWaves > 1) {
            if ((threadIdx.x & 63u) == 0) largest[turn][wave] = most;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaves; ++w) most = max(most, largest[turn][wave0 + w]);
        }
        if (!mine) continue;
        const float scale = scale_of(most), inverse = div_rn(1.0f, scale);
        if (lane == 0) a.scales[row] = scale;
        int8_t* q = a.codes + row * a.code_stride;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const uint32_t c = (p * LANES + lane) * N;
            if (c < a.code_stride) store_codes(q, c, columns, v[p], scale, inverse);
        }
        for (uint64_t c = static_cast<uint64_t>(PIECES * LANES + lane) * N; c < a.code_stride; c += LANES * N)
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<uint32_t*>(q + c + i) = 0u;
    }
}

// Rows that are too long for that: a workgroup for each, which is read again for
// its largest value and for its outputs.
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
        const float factor = factor_of(squares, a);
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
            scale = scale_of(most);
            inverse = div_rn(1.0f, scale);
            if (threadIdx.x == 0) a.scales[row] = scale;
        }
        E* y = a.output ? static_cast<E*>(a.output) + row * a.output_stride : nullptr;
        int8_t* q = a.codes ? a.codes + row * a.code_stride : nullptr;
        const uint64_t width = q ? a.code_stride : columns;
        for (uint64_t c = threadIdx.x * N; c < width; c += 256u * N) {
            float v[N] = {};
            if (c < columns) {
                norm(static_cast<uint32_t>(c), v);
                if (y) V::store(y, static_cast<uint32_t>(c), columns, v);
            }
            if (q) store_codes(q + (c - static_cast<uint32_t>(c)), static_cast<uint32_t>(c), columns, v, scale, inverse);
        }
    }
}

template <int I>
using Lanes = std::integral_constant<int, I>;
// Workgroups of a kernel for `groups` groups of rows. Wide rows: as many as run at
// once, LANES * PIECES of 1024 and less by four to a CU (against a workgroup for
// each row, us, bf16 with sum, norm and codes: 8191 of 6144 87 / 94, of 8192 115 /
// 126, 4096 of 16384 125 / 135, 2048 of 32768 140 / 172). Others: two groups each,
// and sixteen workgroups a CU before that (30000 of 4096 199 with one or two
// groups each, 208 with sixteen workgroups a CU; 8191 of 4096 55 with two, 58 with
// one; 32768 of 1024 54 with two, 58 with one). Never more than 2^22: threads of a
// launch stay below 2^32.
constexpr uint32_t kMostGroups = 1u << 22;
constexpr uint32_t workgroups_of(uint32_t groups, uint32_t lanes, uint32_t pieces) {
    if (lanes * pieces > 512u) return std::min(groups, lanes * pieces <= 1024u ? 1024u : 1048576u / (lanes * pieces));
    return std::min({groups, std::max(4096u, (groups + 1u) / 2u), kMostGroups});
}
// From this many rows on a wave for each narrow one, instead of a workgroup: us,
// 512 wide 1024 rows 3.9 / 5.1, 32768 rows 26 / 64, 256 rows alike; 1024 wide 256
// rows 4.4 / 4.1, 32768 rows 55 / 85.
constexpr uint32_t kNarrowRows = 512;

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
        const hipStream_t s = static_cast<hipStream_t>(stream);
        constexpr uint32_t N = Vec<E>::N;
        // workgroups that share the rows out
        auto kept = [&](auto lanes, auto pieces) {
            constexpr int LANES = decltype(lanes)::value, kThreads = LANES < 256 ? 256 : LANES, kRows = kThreads / LANES;
            constexpr int PIECES = decltype(pieces)::value;
            static_assert(uint64_t(workgroups_of(0x7fffffffu / kRows + 1u, LANES, PIECES)) * kThreads < 1ull << 32);
            dispatch(rms_norm_kept_kernel<E, LANES, PIECES>,
                     dim3(workgroups_of((a.rows + kRows - 1u) / kRows, LANES, PIECES)), dim3(kThreads), 0, s, a);
        };
        const uint32_t vectors = (a.columns + N - 1u) / N;
        // a lane's vectors: rows of 8192 in bf16, 8191 of them, us: 512 lanes of two 121,
        // 256 of four 137, 1024 of one 144; 4096 of 16384 in 1024 of two 135, 512 of
        // four 179; 2048 of 32768 in registers 172, read again 192
        if (vectors <= 128 && a.rows >= kNarrowRows) {
            if (vectors <= 64) kept(Lanes<64>(), Lanes<1>());
            else kept(Lanes<64>(), Lanes<2>());
        } else if (vectors <= 256) {
            kept(Lanes<256>(), Lanes<1>());
        } else if (vectors <= 512) {
            kept(Lanes<256>(), Lanes<2>());
        } else if (vectors <= 768) {
            kept(Lanes<256>(), Lanes<3>());
        } else if (vectors <= 1024) {
            kept(Lanes<512>(), Lanes<2>());
        } else if (vectors <= 2048) {
            kept(Lanes<1024>(), Lanes<2>());
        } else if (vectors <= 4096) {
            kept(Lanes<1024>(), Lanes<4>());
        } else {
            dispatch(rms_norm_kernel<E>, dim3(std::min(a.rows, kMostGroups)), dim3(256), 0, s, a);
        }
        return hipGetLastError();
    });
}

}  // extern "C"
