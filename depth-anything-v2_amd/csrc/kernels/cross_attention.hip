// Attention of queries to keys and values of another length (an encoder's
// tokens): softmax(scale * q k^T) v over the keys that a batch sees.
//
// Products run on the matrix cores in the tensors' own type (binary16 and
// bfloat16: exact products, fp32 sums; fp32: v_mfma_f32_32x32x2_f32). Weights
// are rounded to that type for the second product (half a step, 2^-11 or 2^-8
// of each); their sum is taken in fp32 from the unrounded ones.
//
// A key mask becomes a list of the keys that a batch sees, made by a kernel
// of its own before the attention: hidden keys are never loaded, so what they
// hold does not matter, and cost nothing.

#include <algorithm>
#include <type_traits>

#include "decoder.h"

using namespace dav2k;

namespace {

// Where the lists are in scratch: behind the parts of the splits.
struct Lists {
    uint32_t* keys;    // [batch][key_tokens]
    uint32_t* counts;  // [batch]
};
uint64_t list_bytes(const dav2_cross_attention_args& a) {
    if (!a.key_mask) return 0;
    return ((static_cast<uint64_t>(a.batch) * a.key_tokens + a.batch) * sizeof(uint32_t) + 15u) & ~uint64_t(15);
}

DAV2_DEV uint32_t length_of(const dav2_cross_attention_args& a, uint32_t b) {
    if (!a.key_lengths) return a.key_tokens;
    return min(a.key_tokens, static_cast<uint32_t>(max(a.key_lengths[b], 0)));
}

// The keys that a batch sees, in order: one workgroup per batch, eight bytes of
// the mask for each thread at a time.
__global__ __launch_bounds__(1024) void list_keys_kernel(dav2_cross_attention_args a, Lists lists) {
    __shared__ uint32_t of_wave[16];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t b = blockIdx.x; b < a.batch; b += gridDim.x) {
        const uint8_t* mask = a.key_mask + static_cast<uint64_t>(b) * a.key_tokens;
        uint32_t* out = lists.keys + static_cast<uint64_t>(b) * a.key_tokens;
        const uint32_t length = length_of(a, b);
        uint32_t base = 0;
        for (uint64_t j0 = 0; j0 < length; j0 += 8192u) {
            const uint64_t j = j0 + threadIdx.x * 8u;
            uint32_t seen = 0;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                if (j + i < length && mask[j + i]) seen |= 1u << i;
            const uint32_t mine = __popc(seen);
            uint32_t upto = mine;  // inclusive sum over the wave
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t v = __shfl_up(upto, o, kWave);
                if (lane >= static_cast<uint32_t>(o)) upto += v;
            }
            __syncthreads();
            if (lane == 63u) of_wave[wave] = upto;
            __syncthreads();
            uint32_t before = 0, all = 0;
#pragma unroll
            for (uint32_t w = 0; w < 16; ++w) {
                before += w < wave ? of_wave[w] : 0u;
                all += of_wave[w];
            }
            uint32_t at = base + before + upto - mine;
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i)
                if (seen >> i & 1u) out[at++] = static_cast<uint32_t>(j + i);
            base += all;
        }
        if (threadIdx.x == 0) lists.counts[b] = base;
    }
}

// Matrix instructions of one 16-byte piece per lane of each operand: lane l
// has row (column) l % 32 and inner indices (l / 32) * n .. of 2 n, n values
// in 16 bytes.
DAV2_DEV v16f multiply(h8 a, h8 b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
DAV2_DEV v16f multiply(b8 a, b8 b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
DAV2_DEV v16f multiply(v4f a, v4f b, v16f c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

// A workgroup has 128 rows (row r: token r / group, query head r % group) of
// one batch and key head, 32 for each of four waves, and goes through the keys
// kTile at a time, copied straight into LDS (two buffers, one barrier for a
// tile, the next tile's copies under way during a tile's products).
//
// S^T = K Q^T and O^T = V^T P^T. Lane l holds, for query l % 32, the scores of
// keys 8 (r / 4) + 4 (l / 32) + r % 4 of a 32-key block in registers r: the
// right operand of the second product as it stands, if the left one takes its
// keys in that order. In 16 bits that is two transposing LDS reads of four
// keys by 16 features each; in fp32 four plain ones.
template <typename E, int D>
__global__ __launch_bounds__(256, 2) void cross_tiles_kernel(dav2_cross_attention_args a, Lists lists, uint32_t splits,
                                                             uint32_t tiles) {
    constexpr bool kFloat = std::is_same_v<E, float>;
    constexpr int kTile = kFloat ? 32 : 64, kBlocks = kTile / 32;
    constexpr int N = 16 / sizeof(E);                  // values of a piece
    constexpr int HEAD = D <= 64 ? 64 : 128;           // features of a row in LDS
    constexpr int KS = D / (2 * N), FB = (D + 31) / 32;  // steps over the features, blocks of 32 features
    constexpr uint32_t d = D;
    constexpr uint32_t kRow = HEAD * sizeof(E);        // bytes of a key in LDS
    constexpr uint32_t kChunks = kRow / 16, kRowsPerCopy = 64 / kChunks;
    constexpr int kCopies = kTile * kRow / 4096;       // of each wave, for the keys and again for the values
    constexpr float kSlack = 6.0f;                     // as in cache_tiles_kernel: weights below 2^6
    typedef E V __attribute__((ext_vector_type(N)));
    __shared__ __attribute__((aligned(16))) int8_t lds[2][2][kTile * kRow];  // [buffer][keys, values]
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col = lane & 31u, hf = lane >> 5;
    const uint32_t group = a.heads / a.kv_heads;
    const uint32_t b = blockIdx.x / a.kv_heads, h = blockIdx.x - b * a.kv_heads;
    const uint32_t split = blockIdx.y % splits;
    const uint32_t rows = a.query_tokens * group;  // batch * query_tokens * heads is below 2^32
    const uint32_t row_tiles = (rows + 127u) / 128u;
    const uint32_t* list = lists.keys ? lists.keys + static_cast<uint64_t>(b) * a.key_tokens : nullptr;
    // in a scalar register: the loop and the branch for its last tile are the same for all lanes
    const uint32_t count = __builtin_amdgcn_readfirstlane(lists.keys ? lists.counts[b] : length_of(a, b));
    const uint32_t blocks = (count + kTile - 1u) / kTile, per = (blocks + splits - 1u) / splits;
    const uint32_t first = split * per, last = min(first + per, blocks);
    const E* keys = static_cast<const E*>(a.keys) + b * a.key_batch_stride + static_cast<uint64_t>(h) * d;
    const E* values = static_cast<const E*>(a.values) + b * a.value_batch_stride + static_cast<uint64_t>(h) * d;
    const Parts parts = parts_at(a.scratch, static_cast<uint64_t>(a.batch) * a.query_tokens * a.heads * splits);

    // Copies: this wave's copy i brings rows kRowsPerCopy (kCopies wave + i) ..;
    // lane l row + l / kChunks, place l % kChunks of it. A row's chunks are
    // permuted so that what one LDS read takes from several rows lies in
    // different banks: for the keys, 16 rows at one chunk; for the values in 16
    // bits, four neighbouring rows at 32 (two times 32) bytes.
    uint32_t place[kCopies];  // key of the copy's row in the next tile to be copied
    auto find = [&](uint32_t block) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const uint32_t r = kRowsPerCopy * (kCopies * wave + i) + lane / kChunks;
            const uint32_t at = min(block * kTile + r, count - 1u);  // past the last key that one
            place[i] = list ? list[at] : at;
        }
    };
    auto copy = [&](uint32_t buffer) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const uint32_t r = kRowsPerCopy * (kCopies * wave + i) + lane / kChunks, c = lane % kChunks;
            uint32_t kc = kRow >= 256u ? c ^ (r & 15u) : c ^ ((r >> 1) & 7u);
            uint32_t vc = kFloat ? c : kRow >= 256u ? c ^ ((r & 3u) << 2) : c ^ (((r >> 1) & 1u) << 2);
            // a head may end inside the row; what is behind it is not used
            if (kc * N >= d) kc = 0;
            if (vc * N >= d) vc = 0;
            const uint32_t to = (kCopies * wave + i) * 1024u;
            copy16_to_lds(keys + place[i] * a.key_stride + kc * N, &lds[buffer][0][to]);
            copy16_to_lds(values + place[i] * a.value_stride + vc * N, &lds[buffer][1][to]);
        }
    };
    auto key_piece = [&](uint32_t buffer, uint32_t r, uint32_t c) {
        const uint32_t at = kRow >= 256u ? c ^ (r & 15u) : c ^ ((r >> 1) & 7u);
        return *reinterpret_cast<const V*>(&lds[buffer][0][r * kRow + at * 16u]);
    };

    for (uint32_t tile = blockIdx.y / splits; tile < row_tiles; tile += tiles) {
        const uint32_t row0 = tile * 128u + wave * 32u;
        const bool any_row = row0 < rows;
        const Rows<32> of(any_row ? row0 : tile * 128u, group, rows);
        uint32_t token, head;
        of.find(col, token, head);
        head += h * group;
        __syncthreads();  // the row tile before has been read
        if (first < last) {
            find(first);
            copy(0);
            if (first + 1u < last) find(first + 1u);
        }
        // the right operand of the scores; a negative scale turns its sign
        V qf[KS];
        {
            const E* x = static_cast<const E*>(a.query) + b * a.query_batch_stride + token * a.query_stride +
                         static_cast<uint64_t>(head) * d + N * hf;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                qf[k] = *reinterpret_cast<const V*>(x + 2 * N * k);
                if (a.scale < 0.0f) qf[k] = -qf[k];
            }
        }
        // not 0, for -infinity times it has to stay what it is
        const float c = a.scale == 0.0f ? 1.0e-37f : fabsf(a.scale) * kLog2e;
        v16f o[FB];
#pragma unroll
        for (int f = 0; f < FB; ++f)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[f][r] = 0.0f;
        float maximum = kNoScore, sum = 0.0f;  // sum: this lane's keys only
        DAV2_WAIT_VMCNT(0);
        __syncthreads();
        for (uint32_t block = first; block < last; ++block) {
            const uint32_t buffer = (block - first) & 1u;
            if (block + 1u < last) {
                copy(buffer ^ 1u);
                if (block + 2u < last) find(block + 2u);
            }
            if (any_row) {
                v16f sc[kBlocks];
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[i][r] = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int i = 0; i < kBlocks; ++i)
                        sc[i] = multiply(key_piece(buffer, 32u * i + col, 2u * k + hf), qf[k], sc[i]);
                // reads kAhead pieces ahead of their products
                constexpr int kAhead = KS * kBlocks < 8 ? KS * kBlocks : 8, kEach = kFloat ? 4 : 1;
                DAV2_ORDER(kLdsReads, kAhead);
#pragma unroll
                for (int i = 0; i < KS * kBlocks; ++i) {
                    DAV2_ORDER(kProducts, kEach);
                    if (i + kAhead < KS * kBlocks) DAV2_ORDER(kLdsReads, 1);
                }
                if ((block + 1u) * kTile > count) {
                    stay_in_branch();
#pragma unroll
                    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const uint32_t key = block * kTile + 32u * i + 8u * (r >> 2) + 4u * hf + (r & 3);
                            if (key >= count) sc[i][r] = -INFINITY;
                        }
                }
                float largest = sc[0][0];
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) largest = fmaxf(largest, sc[i][r]);
                largest = over_halves(fmaxf(kNoScore, largest * c), Larger());
                if (__any(largest > maximum + kSlack)) {
                    stay_in_branch();
                    const float grown = fmaxf(maximum, largest);
                    const float keep = __builtin_amdgcn_exp2f(maximum - grown);
                    maximum = grown;
                    sum *= keep;
#pragma unroll
                    for (int f = 0; f < FB; ++f)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[f][r] *= keep;
                }
                // step t: keys 2 N t ..; its weights are formed among the products of the step before
                constexpr int T = kTile / (2 * N);
                V pf[T];
                float parts_of_sum[T];
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    parts_of_sum[t] = 0.0f;
#pragma unroll
                    for (int r = 0; r < N; ++r) {
                        const int at = N * t + r;
                        const float w = __builtin_amdgcn_exp2f(fmaf(sc[at >> 4][at & 15], c, -maximum));
                        parts_of_sum[t] += w;
                        pf[t][r] = static_cast<E>(w);
                    }
                }
#pragma unroll
                for (int t = 0; t < T; ++t) sum += parts_of_sum[t];
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int f = 0; f < FB; ++f) {
                        V vf;
                        if constexpr (kFloat) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                vf[e] = *reinterpret_cast<const float*>(
                                    &lds[buffer][1][(8u * t + 4u * hf + e) * kRow + (32u * f + col) * 4u]);
                        } else {
                            // lane j of 16 points at row j / 4, features 4 (j % 4) ..; it gets feature j of the four rows
                            const uint32_t j = lane & 15u, half16 = (lane >> 4) & 1u;
                            const uint32_t turn = kRow >= 256u ? j >> 2 : j >> 3;
                            const uint32_t at = (((static_cast<uint32_t>(f) ^ turn) << 2 | half16 << 1 | (j & 3u) >> 1) << 4) +
                                                8u * (j & 1u);
                            typedef short s4 __attribute__((ext_vector_type(4)));
                            typedef __attribute__((address_space(3))) s4* lds_s4;
                            int8_t* row = &lds[buffer][1][(16u * t + 4u * hf + (j >> 2)) * kRow + at];
                            union {
                                s4 part[2];
                                V all;
                            } both;
                            both.part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)row);
                            both.part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(row + 8u * kRow));
                            vf = both.all;
                        }
                        o[f] = multiply(vf, pf[t], o[f]);
                    }
                // a step's values are read, and its weights formed, among the products of the step before
                constexpr int kReads = kFloat ? 4 : 2;
                DAV2_ORDER(kLdsReads, FB * kReads);
                DAV2_ORDER(kVector, 3 * N);
                DAV2_ORDER(kExponentials, N);
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int f = 0; f < FB; ++f) {
                        DAV2_ORDER(kProducts, kEach);
                        if (t + 1 < T) {
                            DAV2_ORDER(kLdsReads, kReads);
                            DAV2_ORDER(kVector, (3 * N + FB - 1) / FB);
                            DAV2_ORDER(kExponentials, (N + FB - 1) / FB);
                        }
                    }
            }
            DAV2_WAIT_VMCNT(0);
            __syncthreads();
        }
        sum = over_halves(sum, Plus());
        // register r of o[f]: feature 32 f + 8 (r / 4) + 4 hf + r % 4 of row col
        if (row0 + col < rows) {
            const uint64_t slot = ((static_cast<uint64_t>(b) * a.query_tokens + token) * a.heads + head) * splits + split;
            const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
            typedef E V4 __attribute__((ext_vector_type(4)));
            E* y = static_cast<E*>(a.output) + b * a.output_batch_stride + token * a.output_stride +
                   static_cast<uint64_t>(head) * d;
#pragma unroll
            for (int f = 0; f < FB; ++f)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t feature = 32u * f + 8u * r + 4u * hf;
                    if (feature >= d) continue;
                    if (splits > 1) {
                        *reinterpret_cast<v4f*>(parts.sums + slot * d + feature) =
                            v4f{o[f][4 * r], o[f][4 * r + 1], o[f][4 * r + 2], o[f][4 * r + 3]};
                    } else {
                        V4 out;
#pragma unroll
                        for (int i = 0; i < 4; ++i) out[i] = static_cast<E>(o[f][4 * r + i] * scale);
                        *reinterpret_cast<V4*>(y + feature) = out;
                    }
                }
            if (splits > 1 && hf == 0) parts.stats[slot] = make_float2(maximum, sum);
        }
    }
}

template <typename E>
__global__ __launch_bounds__(256) void cross_join_kernel(dav2_cross_attention_args a, uint32_t splits,
                                                         bool by_lanes) {
    const uint64_t per_batch = static_cast<uint64_t>(a.query_tokens) * a.heads, rows = a.batch * per_batch;
    const Parts parts = parts_at(a.scratch, rows * splits);
    auto output = [&](uint64_t r) {
        const uint32_t row = static_cast<uint32_t>(r), each = static_cast<uint32_t>(per_batch);  // below 2^32
        const uint32_t b = row / each, in = row - b * each, token = in / a.heads, head = in - token * a.heads;
        return static_cast<E*>(a.output) + b * a.output_batch_stride + token * a.output_stride + head * a.head_dim;
    };
    if (by_lanes) {
        for (uint64_t r = blockIdx.x * 8ull + threadIdx.x / 32u; r < rows; r += gridDim.x * 8ull)
            join_few(parts, r * splits, splits, a.head_dim, output(r));
        return;
    }
    for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) join_row(parts, r * splits, splits, a.head_dim, output(r));
}

struct Plan {
    uint32_t tiles, splits;
};
Plan plan_of(const dav2_cross_attention_args& a) {
    Plan p{1, 1};
    if (a.kv_heads == 0 || a.heads < a.kv_heads || a.batch == 0 || a.query_tokens == 0) return p;
    const uint64_t rows = static_cast<uint64_t>(a.query_tokens) * (a.heads / a.kv_heads);
    p.tiles = static_cast<uint32_t>(std::min<uint64_t>((rows + 127) / 128, 512));
    const uint64_t have = static_cast<uint64_t>(p.tiles) * a.kv_heads * a.batch;
    p.splits = static_cast<uint32_t>(
        std::clamp<uint64_t>(std::min<uint64_t>(512 / have, a.key_tokens / 128), 1, kMostSplits));
    return p;
}
uint64_t split_bytes(const dav2_cross_attention_args& a, const Plan& p) {
    if (p.splits == 1) return 0;
    return (parts_bytes(static_cast<uint64_t>(a.batch) * a.query_tokens * a.heads * p.splits, a.head_dim) + 15u) & ~uint64_t(15);
}

}  // namespace

extern "C" {

uint64_t dav2_hip_cross_attention_scratch_bytes(const dav2_cross_attention_args* args) {
    return args ? split_bytes(*args, plan_of(*args)) + list_bytes(*args) : 0;
}

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
        a.head_dim > 128 || a.head_dim % 16 || static_cast<uint64_t>(a.batch) * a.kv_heads > 0x7fffffull ||
        static_cast<uint64_t>(a.query_tokens) * a.heads > 0xffffff00ull / a.batch ||
        (a.query_tokens > 1 && (a.query_stride < row || a.output_stride < row)) ||
        (a.key_tokens > 1 && (a.key_stride < key_row || a.value_stride < key_row)))
        return hipErrorInvalidValue;
    const uint64_t need = dav2_hip_cross_attention_scratch_bytes(args);
    if (need && (!a.scratch || !aligned16(a.scratch) || a.scratch_bytes < need)) return hipErrorInvalidValue;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const Plan p = plan_of(a);
    Lists lists{nullptr, nullptr};
    if (a.key_mask && a.key_tokens) {
        lists.keys = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.scratch) + split_bytes(a, p));
        lists.counts = lists.keys + static_cast<uint64_t>(a.batch) * a.key_tokens;
        dispatch(list_keys_kernel, dim3(a.batch), dim3(1024), 0, s, a, lists);
    }
    const dim3 grid(a.batch * a.kv_heads, p.tiles * p.splits);
    return with_dtype(a.dtype, [&](auto* e) -> int {
        typedef std::remove_pointer_t<decltype(e)> E;
        with_head_dim(a.head_dim, [&](auto dim) {
            dispatch(cross_tiles_kernel<E, decltype(dim)::value>, grid, dim3(256), 0, s, a, lists, p.splits, p.tiles);
        });
        if (p.splits > 1) {
            const uint64_t rows = static_cast<uint64_t>(a.batch) * a.query_tokens * a.heads;
            const bool by_lanes = join_by_lanes(rows, p.splits);
            const uint64_t all = by_lanes ? (rows + 7) / 8 : rows;
            dispatch(cross_join_kernel<E>, dim3(static_cast<uint32_t>(std::min<uint64_t>(all, 65536))), dim3(256), 0, s, a,
                     p.splits, by_lanes);
        }
        return hipGetLastError();
    });
}

}  // extern "C"
