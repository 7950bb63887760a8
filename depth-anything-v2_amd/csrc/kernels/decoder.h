// Shared by the decoder operators' kernels (rotary.hip, cache_i8.hip,
// cross_attention.hip): element types and head widths, sequences and rows, LDS
// reads beside copies, and the join of what splits of the keys leave.
#pragma once

#include <type_traits>

#include "common.h"
#include "dav2_hip.h"

namespace dav2k {

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

// Calls f with a valid head_dim as a constant: the attention kernels are made
// for each, as a branch around a matrix instruction keeps the compiler from
// overlapping it with anything (4 x 2048 queries of 128 features against 5477
// keys: 873 us with, 575 without).
template <typename F>
auto with_head_dim(uint32_t d, F&& f) {
    switch (d / 16) {
        case 1: return f(std::integral_constant<int, 16>{});
        case 2: return f(std::integral_constant<int, 32>{});
        case 3: return f(std::integral_constant<int, 48>{});
        case 4: return f(std::integral_constant<int, 64>{});
        case 5: return f(std::integral_constant<int, 80>{});
        case 6: return f(std::integral_constant<int, 96>{});
        case 7: return f(std::integral_constant<int, 112>{});
        default: return f(std::integral_constant<int, 128>{});
    }
}

// LDS reads beside copies into LDS that are under way. The compiler would have
// a read wait for every such copy, so these are written out, each block with
// its own wait: nothing of it is in flight behind it. What was copied is
// visible after DAV2_WAIT_VMCNT and lds_turn.
typedef int v4i_t __attribute__((ext_vector_type(4)));
typedef short s4_t __attribute__((ext_vector_type(4)));
DAV2_DEV uint32_t lds_address(const void* p) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr_t)p)); }

// 16 bytes each at a and a + STEP (and b and b + STEP)
template <uint32_t STEP>
DAV2_DEV void lds_read2(uint32_t a, v4i_t (&v)[2]) {
    asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]) : "v"(a), "n"(STEP) : "memory");
}
template <uint32_t STEP>
DAV2_DEV void lds_read4(uint32_t a, uint32_t b, v4i_t (&v)[4]) {
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:%6\n\t"
                 "ds_read_b128 %2, %5\n\tds_read_b128 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]) : "v"(a), "v"(b), "n"(STEP) : "memory");
}
DAV2_DEV void lds_read_pair(uint32_t a, uint32_t b, v4i_t& v, v4i_t& w) {
    asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v), "=&v"(w) : "v"(a), "v"(b) : "memory");
}
// transposing reads: four rows by 16 columns of 16 bits for each 16 lanes, at
// a[i] and a[i] + STEP
template <uint32_t STEP, int N>
DAV2_DEV void lds_read_transposed(const uint32_t (&a)[N], s4_t (&v)[2 * N]) {
    static_assert(N >= 1 && N <= 4);
    if constexpr (N == 1)
        asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(v[0]), "=&v"(v[1]) : "v"(a[0]), "n"(STEP) : "memory");
    else if constexpr (N == 2)
        asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
                     "ds_read_b64_tr_b16 %2, %5\n\tds_read_b64_tr_b16 %3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]) : "v"(a[0]), "v"(a[1]), "n"(STEP) : "memory");
    else if constexpr (N == 3)
        asm volatile("ds_read_b64_tr_b16 %0, %6\n\tds_read_b64_tr_b16 %1, %6 offset:%9\n\t"
                     "ds_read_b64_tr_b16 %2, %7\n\tds_read_b64_tr_b16 %3, %7 offset:%9\n\t"
                     "ds_read_b64_tr_b16 %4, %8\n\tds_read_b64_tr_b16 %5, %8 offset:%9\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5])
                     : "v"(a[0]), "v"(a[1]), "v"(a[2]), "n"(STEP) : "memory");
    else
        asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
                     "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
                     "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
                     "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]),
                       "=&v"(v[7])
                     : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(STEP) : "memory");
}
// one float each at a, a + ROW, a + 2 ROW, a + 3 ROW
template <uint32_t ROW>
DAV2_DEV v4f lds_read_column(uint32_t a) {
    float x, y, z, w;
    asm volatile("ds_read_b32 %0, %4\n\tds_read_b32 %1, %4 offset:%5\n\tds_read_b32 %2, %4 offset:%6\n\t"
                 "ds_read_b32 %3, %4 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x), "=&v"(y), "=&v"(z), "=&v"(w) : "v"(a), "n"(ROW), "n"(2 * ROW), "n"(3 * ROW) : "memory");
    return v4f{x, y, z, w};
}

// A barrier that waits for this wave's LDS accesses and for nothing else.
DAV2_DEV void lds_turn() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Inside a branch: keeps the compiler from doing the branch's work always and
// selecting its results afterwards.
DAV2_DEV void stay_in_branch() { asm volatile(""); }

inline bool valid_cache(const dav2_cache_i8& c) {
    return c.keys && c.values && c.key_scales && c.value_scales && aligned16(c.keys) && aligned16(c.values) &&
           c.pages > 0 && c.pages <= 0x7fffffffu && c.kv_heads > 0 && c.kv_heads <= 32767u && c.page_size >= 16 &&
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
    // in scalar registers: what is formed from them is the same for all lanes
    q.begin = __builtin_amdgcn_readfirstlane(min(max(starts[s], 0), most));
    q.end = __builtin_amdgcn_readfirstlane(min(max(starts[s + 1], q.begin), most));
    q.length = __builtin_amdgcn_readfirstlane(max(lengths[s], 0));
    return q;
}

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

constexpr float kLog2e = 1.44269504f;

// Token and head of N rows from row `first` on: row r is token r / group, head
// r % group. One division for all; behind it (t < group + N) a compare, or for
// groups below N <= 128 a product with 2^16 / group that is exact there.
template <uint32_t N>
struct Rows {
    uint32_t token, head, group, magic, most;
    DAV2_DEV Rows(uint32_t first, uint32_t group_, uint32_t rows)
        : token(first / group_), group(group_), magic(65536u / group_ + 1u), most(min(rows - first, N) - 1u) {
        head = first - token * group;
    }
    // row first + i, i < N; past the last row that one
    DAV2_DEV void find(uint32_t i, uint32_t& t, uint32_t& h) const {
        const uint32_t at = head + min(i, most);
        const uint32_t more = group >= N ? (at >= group ? 1u : 0u) : (at * magic) >> 16;
        t = token + more;
        h = at - more * group;
    }
};

// What splits of the keys leave for the join: for each row and split the
// output's sums and {maximum in units of log2, sum of weights}.
constexpr uint32_t kMostSplits = 64;
struct Parts {
    float* sums;    // [rows * splits][head_dim]
    float2* stats;  // [rows * splits]
};
DAV2_DEV Parts parts_at(void* scratch, uint64_t count) {
    float2* stats = static_cast<float2*>(scratch);
    return {reinterpret_cast<float*>(stats + ((count + 1u) & ~uint64_t(1))), stats};
}
inline uint64_t parts_bytes(uint64_t count, uint32_t head_dim) {
    return ((count + 1u) & ~uint64_t(1)) * sizeof(float2) + count * head_dim * sizeof(float);
}

// Which of the two joins below: lanes, FEW = 4 or 8 splits of a row at a time,
// where there are rows enough to fill the chip (1536 rows of eight splits: 2 us
// less of 22 for the whole call), a workgroup per row (FEW = 0) else (64 to 256
// rows of eight: 1.5 us less of 10 to 31).
inline int join_kind(uint64_t rows, uint32_t splits) { return rows <= 1024 ? 0 : splits <= 4 ? 4 : 8; }

// The lanes that have a row, as a power of two: of 4 features each.
DAV2_DEV uint32_t join_lanes_log2(uint32_t d) { return 32u - __clz(d / 4u - 1u); }
inline uint32_t join_rows(uint32_t d) {  // of a workgroup of 256
    uint32_t lanes = 4;
    while (4 * lanes < d) lanes *= 2;
    return 256 / lanes;
}

// The splits of a row joined by its lanes, the features 4 f4 .. each, FEW at a
// time whose loads are under way together, none under a condition (18464 rows
// of three splits of 64 features: 5 us, 3.9 TB/s). A split that saw nothing has
// a sum of 0 and drops out.
template <int FEW, typename E>
DAV2_DEV void join_few(const Parts& parts, uint64_t slot, uint32_t splits, uint32_t d, uint32_t f4, E* y) {
    typedef E V4 __attribute__((ext_vector_type(4)));
    const uint32_t f = min(4u * f4, d - 4u);
    v4f sum = {0.f, 0.f, 0.f, 0.f};
    float total = 0.0f, top = kNoScore;
    for (uint32_t i0 = 0; i0 < splits; i0 += FEW) {
        float2 stats[FEW];
        v4f sums[FEW];
#pragma unroll
        for (uint32_t i = 0; i < FEW; ++i) {
            const uint64_t at = slot + min(i0 + i, splits - 1u);
            stats[i] = parts.stats[at];
            sums[i] = *reinterpret_cast<const v4f*>(parts.sums + at * d + f);
        }
        float grown = top;
#pragma unroll
        for (uint32_t i = 0; i < FEW; ++i) grown = fmaxf(grown, stats[i].x);
        const float keep = __builtin_amdgcn_exp2f(top - grown);
        top = grown;
        total *= keep;
        sum *= keep;
#pragma unroll
        for (uint32_t i = 0; i < FEW; ++i) {
            if (i0 + i >= splits) break;
            const float weight = __builtin_amdgcn_exp2f(stats[i].x - top);
            total = fmaf(stats[i].y, weight, total);
            sum += sums[i] * weight;
        }
    }
    if (4u * f4 >= d) return;
    const float scale = total == 0.0f ? 0.0f : 1.0f / total;
    V4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = static_cast<E>(sum[i] * scale);
    *reinterpret_cast<V4*>(y + f) = out;
}

// The splits of one row, parts slot .. slot + splits - 1, joined by a workgroup
// of 256: thread (i, f) has the four features 4 f .. of splits i, i + 8, ...,
// so that few loads follow one another (a wave per row that walked over 64
// splits took 60 us).
template <typename E>
DAV2_DEV void join_row(const Parts& parts, uint64_t slot, uint32_t splits, uint32_t d, E* y) {
    __shared__ float share[kMostSplits];
    __shared__ __attribute__((aligned(16))) v4f partial[8][32];
    const uint32_t lane = threadIdx.x & 63u, f4 = threadIdx.x & 31u, from = threadIdx.x >> 5;
    const float2 stat = lane < splits ? parts.stats[slot + lane] : make_float2(kNoScore, 0.0f);
    v4f mine[kMostSplits / 8];
#pragma unroll
    for (uint32_t i = 0; i < kMostSplits / 8; ++i) {
        mine[i] = v4f{0.f, 0.f, 0.f, 0.f};
        if (from + 8 * i < splits && 4 * f4 < d)
            mine[i] = *reinterpret_cast<const v4f*>(parts.sums + (slot + from + 8 * i) * d + 4 * f4);
    }
    const float top = wave_max(stat.x);
    const float weight = __builtin_amdgcn_exp2f(stat.x - top);  // 1 for all, if no split saw anything
    const float total = wave_sum_tree(stat.y * weight);
    __syncthreads();  // the row before has been read
    if (threadIdx.x < kMostSplits) share[lane] = weight;
    __syncthreads();
    v4f sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t i = 0; i < kMostSplits / 8; ++i)
        if (from + 8 * i < splits) sum += mine[i] * share[from + 8 * i];
    partial[from][f4] = sum;
    __syncthreads();
    if (threadIdx.x < 32 && 4 * f4 < d) {
        sum = partial[0][f4];
#pragma unroll
        for (int i = 1; i < 8; ++i) sum += partial[i][f4];
        const float scale = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[4 * f4 + i] = static_cast<E>(sum[i] * scale);
    }
}

}  // namespace dav2k
