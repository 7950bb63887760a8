// Rotary positions, alone and behind the norm of each query and key head.
//
// (a, b) -> A (a cos t - b sin t, b cos t + a sin t), t = p f_i. The angle is
// formed in 64 bits and reduced to a fraction of a turn there: in fp32 a
// position of 10^6 would leave 0.06 radians of it uncertain.

#include <algorithm>

#include "decoder.h"

using namespace dav2k;

namespace {

constexpr double kTurnsPerRadian = 0.15915494309189533577;
constexpr uint64_t kMostTiles = 1u << 22;  // workgroups along x: threads of a launch stay below 2^32

// One wave per head of a token: lane l has features l, l + 64, ...
template <typename E, bool NORM>
DAV2_DEV void rotary_head(const dav2_qk_norm_rotary_args& a, uint64_t item, uint32_t lane) {
    const uint32_t heads = a.query_heads + a.key_heads;
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

template <typename E, bool NORM>
__global__ __launch_bounds__(256) void rotary_kernel(dav2_qk_norm_rotary_args a) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t heads = a.query_heads + a.key_heads;
    const uint64_t items = static_cast<uint64_t>(a.tokens) * heads, step = static_cast<uint64_t>(gridDim.x) * 4u;
    for (uint64_t item = static_cast<uint64_t>(blockIdx.x) * 4u + (threadIdx.x >> 6); item < items; item += step)
        rotary_head<E, NORM>(a, item, lane);
}

// Sum over groups of LANES neighbouring lanes, received by all of them: within
// 16 lanes by DPP moves (quad permutations, then mirrors, whose partners hold
// the same partial sums as the lanes 4 and 8 further), beyond by lane swaps.
template <int LANES>
DAV2_DEV float sum_lanes(float v) {
    auto moved = [](float x, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, true));
    };
    v += moved(v, std::integral_constant<int, 0xB1>{});  // quad_perm [1,0,3,2]
    v += moved(v, std::integral_constant<int, 0x4E>{});  // quad_perm [2,3,0,1]
    if constexpr (LANES >= 8) v += moved(v, std::integral_constant<int, 0x141>{});   // row_half_mirror
    if constexpr (LANES >= 16) v += moved(v, std::integral_constant<int, 0x140>{});  // row_mirror
    if constexpr (LANES >= 32) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
    if constexpr (LANES >= 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    }
    return v;
}

// The same for heads that are whole multiples of U = 2 VEC features, rotated in
// a multiple of U. LANES lanes (a power of two) share a head, each with U
// features in two vectors of VEC: features f .. f + VEC - 1 and their partners
// half a rotated part further (HALVES), or 2 VEC neighbours (PAIRS, and what
// is only copied).
//
// A workgroup takes `tile` tokens: it puts their angles' cosines and sines
// (and the norms' weights) into LDS once for all heads, then walks over the
// tile's heads in memory order, kTogether per thread at a time so that their
// loads overlap; the first loads are under way while the angles are formed.
// Bound by memory: nothing but the heads is read or written. 8191 tokens, 32
// heads of 128 half of which turns, bf16 (134 MB): 26.5 us, 5.1 TB/s, the rate
// of a large copy; 16411 tokens, 32 + 8 normed heads of 128, f16 (336 MB):
// 64.9 us, 5.2 TB/s. The wave per head above takes 80 and 283 us; a thread
// that keeps one token's angles in registers and walks over its heads 34 and
// 84, as each wave then reads 256-byte pieces of eight rows; kTogether 1, 3,
// 4: 28.2, 27.1, 28.0 and 71.3, 70.1, 70.9 (with eight heads a thread).
constexpr int kTogether = 2;
constexpr uint32_t kMostPairs = 2048;  // of a tile: 16 KB of cosines and sines

template <typename E, int VEC, int LANES, bool NORM, bool HALVES>
__global__ __launch_bounds__(256) void rotary_lanes_kernel(dav2_qk_norm_rotary_args a, uint32_t tile) {
    typedef E V __attribute__((ext_vector_type(VEC)));
    constexpr uint32_t U = 2 * VEC, kStep = 256u / LANES;
    extern __shared__ __attribute__((aligned(16))) float table[];  // [tile][cosines, sines][rotary_dim / 2]
    const uint32_t lane = threadIdx.x & (LANES - 1);
    const uint32_t d = a.head_dim, half = a.rotary_dim / 2;
    const bool active = lane * U < d;             // LANES lanes may be more than a head needs
    const bool turned = lane * U < a.rotary_dim;  // else this lane's features are copied
    // this lane's two vectors: features f0 .. and f1 ..
    const uint32_t f0 = !active ? 0u : HALVES && turned ? lane * VEC : lane * U;
    const uint32_t f1 = HALVES && turned ? f0 + half : f0 + VEC;
    const float share = 1.0f / static_cast<float>(d);
    float* const weights = table + static_cast<size_t>(tile) * a.rotary_dim;  // [query, key][head_dim]
    if (NORM)
        for (uint32_t i = threadIdx.x; i < 2 * d; i += 256u) {
            const float* weight = i < d ? a.query_weight : a.key_weight;
            weights[i] = weight ? weight[i < d ? i : i - d] : 1.0f;
        }
    for (uint64_t first = static_cast<uint64_t>(blockIdx.x) * tile; first < a.tokens;
         first += static_cast<uint64_t>(gridDim.x) * tile) {
        const uint32_t tokens = static_cast<uint32_t>(min(static_cast<uint64_t>(tile), a.tokens - first));
        // the query heads (side 0), then the key heads: each with its weight in registers
        for (uint32_t side = 0; side < 2; ++side) {
            const uint32_t heads = side ? a.key_heads : a.query_heads, items = tokens * heads;
            const uint64_t in_stride = side ? a.key_stride : a.query_stride;
            const uint64_t out_stride = side ? a.key_out_stride : a.query_out_stride;
            const E* x = static_cast<const E*>(side ? a.key : a.query) + first * in_stride;
            E* y = static_cast<E*>(side ? a.key_out : a.query_out) + first * out_stride;
            V in0[kTogether], in1[kTogether];
            auto load = [&](uint32_t item0) {
#pragma unroll
                for (int t = 0; t < kTogether; ++t) {
                    const uint32_t item = item0 + t * kStep;
                    if (!active || item >= items) continue;
                    const uint32_t token = item / heads, head = item - token * heads;
                    const E* from = x + token * in_stride + static_cast<uint64_t>(head) * d;
                    in0[t] = *reinterpret_cast<const V*>(from + f0);
                    in1[t] = *reinterpret_cast<const V*>(from + f1);
                }
            };
            const uint32_t item1 = threadIdx.x / LANES;
            load(item1);
            if (side == 0) {
                for (uint32_t i = threadIdx.x; i < tokens * half; i += 256u) {
                    const uint32_t token = i / half, pair = i - token * half;
                    const double turns =
                        static_cast<double>(a.positions[first + token]) * (a.frequencies[pair] * kTurnsPerRadian);
                    float s, c;
                    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
                    table[token * 2 * half + pair] = c * a.amplitude;
                    table[token * 2 * half + half + pair] = s * a.amplitude;
                }
                __syncthreads();
            }
            float w[U];
            if (NORM) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    w[i] = weights[side * d + f0 + i];
                    w[VEC + i] = weights[side * d + f1 + i];
                }
            }
            for (uint32_t item0 = item1; item0 < items; item0 += kTogether * kStep) {
                if (item0 != item1) load(item0);
#pragma unroll
                for (int t = 0; t < kTogether; ++t) {
                    const uint32_t item = item0 + t * kStep;
                    if (item >= items) break;
                    const uint32_t token = item / heads, head = item - token * heads;
                    float v[U];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        v[i] = active ? static_cast<float>(in0[t][i]) : 0.0f;
                        v[VEC + i] = active ? static_cast<float>(in1[t][i]) : 0.0f;
                    }
                    if (NORM) {
                        if (a.norm == DAV2_QK_NORM_LAYER) {
                            float sum = 0.0f;
#pragma unroll
                            for (int i = 0; i < static_cast<int>(U); ++i) sum += v[i];
                            const float mean = sum_lanes<LANES>(sum) * share;
#pragma unroll
                            for (int i = 0; i < static_cast<int>(U); ++i) v[i] -= mean;
                        }
                        float squares = 0.0f;
#pragma unroll
                        for (int i = 0; i < static_cast<int>(U); ++i) squares = fmaf(v[i], v[i], squares);
                        if (!active) squares = 0.0f;
                        const float variance = sum_lanes<LANES>(squares) * share + a.epsilon;
                        // the instruction takes a subnormal number for zero
                        const bool small = variance < 0x1p-100f;
                        const float factor = __builtin_amdgcn_rsqf(small ? variance * 0x1p64f : variance) *
                                             (small ? 0x1p32f : 1.0f);
#pragma unroll
                        for (int i = 0; i < static_cast<int>(U); ++i) v[i] *= factor * w[i];
                    }
                    if (turned) {
                        const float* cosines = table + token * 2 * half + lane * VEC;
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            const float c = cosines[i], s = cosines[half + i];
                            float& p = HALVES ? v[i] : v[2 * i];
                            float& q = HALVES ? v[VEC + i] : v[2 * i + 1];
                            const float u = p;
                            p = u * c - q * s;
                            q = q * c + u * s;
                        }
                    }
                    if (active) {
                        V out0, out1;
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            out0[i] = static_cast<E>(v[i]);
                            out1[i] = static_cast<E>(v[VEC + i]);
                        }
                        E* to = y + token * out_stride + static_cast<uint64_t>(head) * d;
                        *reinterpret_cast<V*>(to + f0) = out0;
                        *reinterpret_cast<V*>(to + f1) = out1;
                    }
                }
            }
        }
        __syncthreads();  // before the next tile's angles
    }
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

// Whether every head is a multiple of 2 vec features, rotated in one, at
// addresses that are multiples of vec elements.
bool divides(const dav2_qk_norm_rotary_args& a, uint32_t vec) {
    const uint32_t size = dtype_bytes(a.dtype), bytes = vec * size;
    if (a.head_dim % (2 * vec) || a.rotary_dim % (2 * vec) || a.head_dim / (2 * vec) > 64) return false;
    auto side = [&](const void* p, uint64_t stride) {
        return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (a.tokens == 1 || stride * size % bytes == 0);
    };
    return (!a.query_heads || (side(a.query, a.query_stride) && side(a.query_out, a.query_out_stride))) &&
           (!a.key_heads || (side(a.key, a.key_stride) && side(a.key_out, a.key_out_stride)));
}

template <typename E, int VEC, int LANES, bool NORM>
int launch_lanes(const dav2_qk_norm_rotary_args& a, hipStream_t stream) {
    // Tokens of a tile: two heads for each thread, four with the norm, whose
    // weights a tile loads (16411 tokens, 40 heads of 128: four 64.9 us, eight
    // 70.3, sixteen 73.5), unless that leaves fewer than kWorkgroups workgroups.
    constexpr uint32_t kWorkgroups = 1024;
    const uint32_t heads = a.query_heads + a.key_heads;
    uint32_t tile = std::max(1u, (NORM ? 4 : 2) * 256u / LANES / heads);
    tile = std::min({tile, std::max(1u, a.tokens / kWorkgroups), std::max(1u, kMostPairs / std::max(1u, a.rotary_dim / 2))});
    const dim3 grid(static_cast<uint32_t>(std::min<uint64_t>(kMostTiles, ceil_div(a.tokens, tile))));
    const size_t lds = (static_cast<size_t>(tile) * a.rotary_dim + (NORM ? 2 * a.head_dim : 0)) * sizeof(float);
    if (a.layout == DAV2_ROTARY_HALVES)
        dispatch(rotary_lanes_kernel<E, VEC, LANES, NORM, true>, grid, dim3(256), lds, stream, a, tile);
    else
        dispatch(rotary_lanes_kernel<E, VEC, LANES, NORM, false>, grid, dim3(256), lds, stream, a, tile);
    return hipGetLastError();
}

template <typename E, int VEC, bool NORM>
int launch_vectors(const dav2_qk_norm_rotary_args& a, hipStream_t stream) {
    const uint32_t lanes = a.head_dim / (2 * VEC);
    if (lanes <= 4) return launch_lanes<E, VEC, 4, NORM>(a, stream);
    if (lanes <= 8) return launch_lanes<E, VEC, 8, NORM>(a, stream);
    if (lanes <= 16) return launch_lanes<E, VEC, 16, NORM>(a, stream);
    if (lanes <= 32) return launch_lanes<E, VEC, 32, NORM>(a, stream);
    return launch_lanes<E, VEC, 64, NORM>(a, stream);
}

template <bool NORM>
int launch(const dav2_qk_norm_rotary_args& a, void* stream) {
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return with_dtype(a.dtype, [&](auto* e) -> int {
        typedef std::remove_pointer_t<decltype(e)> E;
        constexpr int kWide = 16 / sizeof(E);
        if (divides(a, kWide)) return launch_vectors<E, kWide, NORM>(a, s);
        if (divides(a, kWide / 2)) return launch_vectors<E, kWide / 2, NORM>(a, s);
        if constexpr (kWide == 8)
            if (divides(a, 2)) return launch_vectors<E, 2, NORM>(a, s);
        const uint64_t items = static_cast<uint64_t>(a.tokens) * (a.query_heads + a.key_heads);
        dispatch(rotary_kernel<E, NORM>, dim3(static_cast<uint32_t>(std::min<uint64_t>(kMostTiles, (items + 3) / 4))), dim3(256), 0, s,
                 a);
        return hipGetLastError();
    });
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
