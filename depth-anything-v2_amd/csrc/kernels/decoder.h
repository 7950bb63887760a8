// Shared by the decoder operators' kernels (rotary.hip, cache_i8.hip,
// cross_attention.hip): element types and their checks.
#pragma once

#include "common.h"
#include "dav2_hip.h"

namespace dav2k {

// An activation type: E as stored, widened to fp32 on load, rounded to
// nearest even on store.
template <uint32_t DTYPE>
struct Activation;
template <>
struct Activation<DAV2_DTYPE_F32> {
    typedef float E;
};
template <>
struct Activation<DAV2_DTYPE_F16> {
    typedef _Float16 E;
};
template <>
struct Activation<DAV2_DTYPE_BF16> {
    typedef __bf16 E;
};

inline uint32_t dtype_bytes(uint32_t dtype) { return dtype == DAV2_DTYPE_F32 ? 4u : 2u; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Calls f with the element type of a valid dtype as a value of type E*.
template <typename F>
auto with_dtype(uint32_t dtype, F&& f) {
    switch (dtype) {
        case DAV2_DTYPE_F16: return f(static_cast<_Float16*>(nullptr));
        case DAV2_DTYPE_BF16: return f(static_cast<__bf16*>(nullptr));
        default: return f(static_cast<float*>(nullptr));
    }
}

inline bool valid_cache(const dav2_cache_i8& c) {
    return c.keys && c.values && c.key_scales && c.value_scales && aligned16(c.keys) && aligned16(c.values) &&
           c.pages > 0 && c.pages <= 0x7fffffffu && c.kv_heads > 0 && c.kv_heads <= 65535u && c.page_size >= 16 &&
           c.page_size <= 256 && c.page_size % 16 == 0 && c.head_dim >= 16 && c.head_dim <= 128 &&
           c.head_dim % 16 == 0;
}

// What one sequence of a ragged batch has: rows [begin, end) of the new
// tokens and `length` tokens in all, as the arrays give them, with rows
// outside [0, tokens) cut off.
struct Sequence {
    int32_t begin, end, length;
};
DAV2_DEV Sequence sequence_of(const int32_t* starts, const int32_t* lengths, uint32_t s, uint32_t tokens) {
    Sequence q;
    const int32_t most = static_cast<int32_t>(tokens);
    q.begin = min(max(starts[s], 0), most);
    q.end = min(max(starts[s + 1], q.begin), most);
    q.length = max(lengths[s], 0);
    return q;
}

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

// The running maximum of a softmax before its first score. Finite, so that
// exp2(maximum - larger maximum) is 0 and never the difference of infinities.
constexpr float kNoScore = -3.0e38f;

// op over the four lanes l, l ^ 16, l ^ 32, l ^ 48, received by all of them.
template <typename Op>
DAV2_DEV float over_groups(float v, Op op) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// ... over the two lanes l, l ^ 32.
template <typename Op>
DAV2_DEV float over_halves(float v, Op op) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
struct Larger {
    DAV2_DEV float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Plus {
    DAV2_DEV float operator()(float a, float b) const { return a + b; }
};

}  // namespace dav2k
