// Attention of queries to keys and values of another length (an encoder's
// tokens): softmax(scale * q k^T) v over the keys that a batch sees.
//
// Products run on the matrix cores in the tensors' own type (binary16 and
// bfloat16: exact products, fp32 sums; fp32: v_mfma_f32_32x32x2_f32). Weights
// are rounded to that type for the second product (half a step, 2^-11 or 2^-8
// of each); their sum is taken in fp32 from the unrounded ones. Binary16 ends at
// 2^-24: its weights are formed kBias powers of two larger, which cancels in the
// quotient, so that against the largest they keep 2^-11 down to 2^-27 and lose
// at most 2^-38 below.
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
    if (a.key_tokens == 0) return 0;
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

// A workgroup has 32 rows (row r: token r / group, query head r % group) of one
// batch and key head for each of its waves, and goes through the keys kTile at
// a time.
//
// S^T = K Q^T and O^T = V^T P^T. Lane l holds, for query l % 32, the scores of
// keys 8 (r / 4) + 4 (l / 32) + r % 4 of a 32-key block in registers r: the
// right operand of the second product as it stands, if the left one takes its
// keys in that order. In 16 bits that is two transposing LDS reads of four
// keys by 16 features each; in fp32 four plain ones.
template <typename E_, int D_, bool LISTED, int WAVES>
struct Tiles {
    typedef E_ E;
    static constexpr int D = D_;
    static constexpr bool kFloat = std::is_same_v<E, float>;
    static constexpr int kTile = kFloat ? 32 : 64, kBlocks = kTile / 32;
    static constexpr int N = 16 / sizeof(E);                  // values of a piece
    static constexpr int HEAD = D <= 64 ? 64 : 128;           // features of a row in LDS
    static constexpr int KS = D / (2 * N), FB = (D + 31) / 32;  // steps over the features, blocks of 32 features
    static constexpr int T = kTile / (2 * N);                 // steps over the keys; step t: keys 2 N t ..
    static constexpr uint32_t kRow = HEAD * sizeof(E);        // bytes of a key in LDS
    static constexpr uint32_t kChunks = kRow / 16, kRowsPerCopy = 64 / kChunks;
    static constexpr int kCopies = kTile * kRow / (1024 * WAVES);  // of each wave, for the keys and again for the values
    // rescale when a score passes the running maximum by kSlack: most tiles
    // leave the sums alone. Weights stay below 2^(kBias + kSlack).
    static constexpr bool kHalf = std::is_same_v<E, _Float16>;
    static constexpr float kSlack = kHalf ? 2.0f : 6.0f, kBias = kHalf ? 13.0f : 0.0f;
    typedef E V __attribute__((ext_vector_type(N)));

    // of the workgroup
    const dav2_cross_attention_args& a;
    uint32_t b, h, group, rows, count, lane, col, hf, wave;
    const uint32_t* list;
    const E *keys, *values;
    // of the wave's rows
    uint32_t token, head;
    float c;
    V qf[KS];       // the right operand of the scores
    v16f o[FB];     // register r of o[f]: feature 32 f + 8 (r / 4) + 4 hf + r % 4 of row col
    float base, sum;  // the running maximum less kBias; sum: this lane's keys only
    // The wave has met a maximum past kFar, where fp32 has too few bits for a
    // bias and a fused score minus base would keep bits that base has lost,
    // more of them than an exponential bears: base is the maximum itself then.
    bool far;
    static constexpr float kFar = 1048576.0f;
    V pf[T];

    DAV2_DEV Tiles(const dav2_cross_attention_args& args, const Lists& lists, uint32_t plane) : a(args) {
        lane = threadIdx.x & 63u;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        col = lane & 31u;
        hf = lane >> 5;
        group = a.heads / a.kv_heads;
        b = plane / a.kv_heads;
        h = plane - b * a.kv_heads;
        rows = a.query_tokens * group;  // batch * query_tokens * heads is below 2^32
        if (LISTED) list = lists.keys + static_cast<uint64_t>(b) * a.key_tokens;
        // in a scalar register: the loop and the branch for its last tile are the same for all lanes
        count = __builtin_amdgcn_readfirstlane(LISTED ? lists.counts[b] : length_of(a, b));
        keys = static_cast<const E*>(a.keys) + b * a.key_batch_stride + static_cast<uint64_t>(h) * D;
        values = static_cast<const E*>(a.values) + b * a.value_batch_stride + static_cast<uint64_t>(h) * D;
        // not 0, for -infinity times it has to stay what it is: the query is zeros then
        c = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
    }

    // Copies: this wave's copy i brings rows kRowsPerCopy (kCopies wave + i) ..;
    // lane l row + l / kChunks, place l % kChunks of it. A row's chunks are
    // permuted so that what one LDS read takes from several rows lies in
    // different banks: for the keys, 16 rows at one chunk; for the values in 16
    // bits, four neighbouring rows at 32 (two times 32) bytes.
    DAV2_DEV static uint32_t key_chunk(uint32_t r, uint32_t c) { return kRow >= 256u ? c ^ (r & 15u) : c ^ ((r >> 1) & 7u); }
    DAV2_DEV static uint32_t value_chunk(uint32_t r, uint32_t c) {
        return kFloat ? c : kRow >= 256u ? c ^ ((r & 3u) << 2) : c ^ (((r >> 1) & 1u) << 2);
    }
    // The keys of this lane's rows in tile `block`; past the last key that one.
    // Called without a condition: registers that are loaded in one branch only
    // are waited for where the branches meet.
    DAV2_DEV void find(uint32_t block, uint32_t (&place)[kCopies]) const {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const uint32_t r = kRowsPerCopy * (kCopies * wave + i) + lane / kChunks;
            const uint32_t at = min(block * kTile + r, count - 1u);
            place[i] = LISTED ? list[at] : at;
        }
    }
    // where this lane's piece of copy i is, in memory
    DAV2_DEV const E* key_at(int i, uint32_t place) const {
        const uint32_t r = kRowsPerCopy * (kCopies * wave + i) + lane / kChunks;
        const uint32_t chunk = key_chunk(r, lane % kChunks);
        // a head may end inside the row; what is behind it is not used
        return keys + place * a.key_stride + (chunk * N >= D ? 0 : chunk * N);
    }
    DAV2_DEV const E* value_at(int i, uint32_t place) const {
        const uint32_t r = kRowsPerCopy * (kCopies * wave + i) + lane / kChunks;
        const uint32_t chunk = value_chunk(r, lane % kChunks);
        return values + place * a.value_stride + (chunk * N >= D ? 0 : chunk * N);
    }
    // The tile at `place` into LDS; then place is that of tile `next`. Its loads
    // are started before the copies, so that who uses it waits for them without
    // the copies, and straight into its registers, which nobody has to move.
    DAV2_DEV void copy(int8_t* to_keys, int8_t* to_values, uint32_t (&place)[kCopies], uint32_t next) const {
        const E *from_keys[kCopies], *from_values[kCopies];
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            from_keys[i] = key_at(i, place[i]);
            from_values[i] = value_at(i, place[i]);
        }
        find(next, place);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            copy16_to_lds(from_keys[i], to_keys + (kCopies * wave + i) * 1024u);
            copy16_to_lds(from_values[i], to_values + (kCopies * wave + i) * 1024u);
        }
    }

    // Rows row0 .. row0 + 31 (row0 < rows): the query, and nothing seen yet.
    DAV2_DEV void begin(uint32_t row0) {
        const Rows<32> of(row0, group, rows);
        of.find(col, token, head);
        head += h * group;
        const E* x = static_cast<const E*>(a.query) + b * a.query_batch_stride + token * a.query_stride +
                     static_cast<uint64_t>(head) * D + N * hf;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            qf[k] = *reinterpret_cast<const V*>(x + 2 * N * k);
            if (a.scale < 0.0f) qf[k] = -qf[k];
            if (a.scale == 0.0f) qf[k] *= static_cast<E>(0.0f);
        }
#pragma unroll
        for (int f = 0; f < FB; ++f)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[f][r] = 0.0f;
        base = kNoScore;
        sum = 0.0f;
        far = false;
    }

    // A step's pieces are read before the products of the step before, which run
    // while the read waits.
    DAV2_DEV void multiply_keys(const int8_t* from, v16f (&sc)[kBlocks]) const {
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[i][r] = 0.0f;
        // one block of reads for two steps; rows 32 apart have their chunks at the same places
        constexpr int S = (KS + 1) / 2;
        v4i_t in[2][4];
        const uint32_t base = lds_address(from) + col * kRow;
        auto at = [&](int k) { return base + key_chunk(col, 2u * k + hf) * 16u; };
        auto read = [&](int s, v4i_t (&v)[4]) {
            if constexpr (kBlocks == 2) {
                if (2 * s + 1 < KS) {
                    lds_read4<32 * kRow>(at(2 * s), at(2 * s + 1), v);
                } else {
                    v4i_t w[2];
                    lds_read2<32 * kRow>(at(2 * s), w);
                    v[0] = w[0];
                    v[1] = w[1];
                }
            }
        };
        if constexpr (kBlocks == 2) {
            read(0, in[0]);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                if (s + 1 < S) read(s + 1, in[(s + 1) & 1]);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (2 * s + j / 2 < KS)
                        sc[j & 1] = multiply(__builtin_bit_cast(V, in[s & 1][j]), qf[2 * s + j / 2], sc[j & 1]);
            }
        } else {
            // KS is even: fp32 steps are 8 features
            lds_read_pair(at(0), at(1), in[0][0], in[0][1]);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                if (s + 1 < S) lds_read_pair(at(2 * s + 2), at(2 * s + 3), in[(s + 1) & 1][0], in[(s + 1) & 1][1]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    sc[0] = multiply(__builtin_bit_cast(V, in[s & 1][j]), qf[2 * s + j], sc[0]);
            }
        }
    }

    // The scores of tile `block` as weights: the running maximum, the sums so
    // far brought to it, pf and the sum of the weights.
    DAV2_DEV void weigh(uint32_t block, v16f (&sc)[kBlocks]) {
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
        if (__any(largest > base + (far ? 0.0f : kBias + kSlack))) {
            stay_in_branch();
            const float grown = fmaxf(base + (far ? 0.0f : kBias), largest);
            far = far || __any(fabsf(grown) >= kFar && grown != kNoScore);
            const float moved = grown - (far ? 0.0f : kBias);
            const float keep = __builtin_amdgcn_exp2f(base - moved);
            base = moved;
            sum *= keep;
#pragma unroll
            for (int f = 0; f < FB; ++f)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[f][r] *= keep;
        }
        float factor = c;
        if (far) {
            stay_in_branch();
#pragma unroll
            for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) sc[i][r] *= c;
            factor = 1.0f;
        }
        float of_step[T];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            of_step[t] = 0.0f;
#pragma unroll
            for (int r = 0; r < N; ++r) {
                const int at = N * t + r;
                const float w = __builtin_amdgcn_exp2f(fmaf(sc[at >> 4][at & 15], factor, -base));
                of_step[t] += w;
                pf[t][r] = static_cast<E>(w);
            }
        }
#pragma unroll
        for (int t = 0; t < T; ++t) sum += of_step[t];
    }

    // The values of step t, left operands of FB products. In 16 bits by
    // transposing reads: lane j of 16 points at row j / 4, features 4 (j % 4) ..,
    // and gets feature j of the four rows.
    DAV2_DEV void read_values(const int8_t* from, const int t, V (&v)[FB]) const {
        if constexpr (kFloat) {
            const uint32_t base = lds_address(from) + (8u * t + 4u * hf) * kRow + col * 4u;
#pragma unroll
            for (int f = 0; f < FB; ++f) v[f] = lds_read_column<kRow>(base + 128u * f);
        } else {
            const uint32_t j = lane & 15u, half16 = (lane >> 4) & 1u, turn = kRow >= 256u ? j >> 2 : j >> 3;
            const uint32_t base = lds_address(from) + (16u * t + 4u * hf + (j >> 2)) * kRow +
                                  ((half16 << 1 | (j & 3u) >> 1) << 4) + 8u * (j & 1u);
            s4_t p[2 * FB];
            uint32_t at[FB];
#pragma unroll
            for (int f = 0; f < FB; ++f) at[f] = base + ((static_cast<uint32_t>(f) ^ turn) << 6);
            lds_read_transposed<8 * kRow>(at, p);
#pragma unroll
            for (int f = 0; f < FB; ++f) {
                union {
                    s4_t part[2];
                    V all;
                } both;
                both.part[0] = p[2 * f];
                both.part[1] = p[2 * f + 1];
                v[f] = both.all;
            }
        }
    }
    // A step's values are read before the products of the step before, which
    // run while the read waits.
    DAV2_DEV void multiply_values(const int8_t* from) {
        V v[2][FB];
        read_values(from, 0, v[0]);
#pragma unroll
        for (int t = 0; t < T; ++t) {
            if (t + 1 < T) read_values(from, t + 1, v[(t + 1) & 1]);
#pragma unroll
            for (int f = 0; f < FB; ++f) o[f] = multiply(v[t & 1][f], pf[t], o[f]);
        }
    }

    DAV2_DEV void end(uint32_t row0, uint32_t split, uint32_t splits) {
        sum = over_halves(sum, Plus());
        if (row0 + col >= rows) return;
        const uint64_t slot = ((static_cast<uint64_t>(b) * a.query_tokens + token) * a.heads + head) * splits + split;
        const Parts parts = parts_at(a.scratch, static_cast<uint64_t>(a.batch) * a.query_tokens * a.heads * splits);
        const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
        typedef E V4 __attribute__((ext_vector_type(4)));
        E* y = static_cast<E*>(a.output) + b * a.output_batch_stride + token * a.output_stride +
               static_cast<uint64_t>(head) * D;
#pragma unroll
        for (int f = 0; f < FB; ++f)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t feature = 32u * f + 8u * r + 4u * hf;
                if (feature >= D) continue;
                if (splits > 1) {
                    *reinterpret_cast<v4f*>(parts.sums + slot * D + feature) =
                        v4f{o[f][4 * r], o[f][4 * r + 1], o[f][4 * r + 2], o[f][4 * r + 3]};
                } else {
                    V4 out;
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[i] = static_cast<E>(o[f][4 * r + i] * scale);
                    *reinterpret_cast<V4*>(y + feature) = out;
                }
            }
        if (splits > 1 && hf == 0) parts.stats[slot] = make_float2(base, sum);
    }
};

// Four or eight waves, 128 or 256 rows, two buffers and one barrier for a tile,
// whose copies go straight into LDS during the products of the tile before.
//
// Bound by the matrix cores and, as long again in 16 bits, the exponentials of
// the vector units beside them: 8 x 2048 queries of 32 heads of 128 on 4096
// keys of 8, bf16, 1.12 ms, 980 TFLOP/s, where a large library product runs at
// 1190 (four waves 4 % more); f16 1.18 ms, whose weights take a bias; heads of
// 64 in f16 740. fp32: 129 TFLOP/s of 152 at 8 x 1024 queries, 16 heads of 64,
// 4096 keys; 82 at 2 x 577 queries and 1370 keys, where 160 workgroups are
// split in three. Tried and not kept: eight waves in two groups that multiply
// and weigh in turns (barriers between; no difference), a tile's scores one
// tile ahead among the exponentials (spills), a step's exponentials between the
// products of the step before (556 -> 563 us at a masked case of 8 prompts),
// tiles through registers (575 -> 610 us), workgroups of one wave for up to 32
// rows (one query each, 1370 keys, 16 heads of 64: 16 in fp32 57 -> 48 us, but
// 4 in f16 10.3 -> 11.4, 16 20.9 -> 22.7).
template <typename E, int D, bool LISTED, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2)
void cross_tiles_kernel(dav2_cross_attention_args a, Lists lists, uint32_t splits, uint32_t tiles) {
    constexpr uint32_t kTileRows = 32 * WAVES;
    typedef Tiles<E, D, LISTED, WAVES> K;
    __shared__ __attribute__((aligned(16))) int8_t lds[2][2][K::kTile * K::kRow];  // [buffer][keys, values]
    K k(a, lists, blockIdx.x);
    const uint32_t split = blockIdx.y % splits, row_tiles = (k.rows + kTileRows - 1u) / kTileRows;
    const uint32_t blocks = (k.count + K::kTile - 1u) / K::kTile, per = (blocks + splits - 1u) / splits;
    const uint32_t first = split * per, last = min(first + per, blocks);
    for (uint32_t tile = blockIdx.y / splits; tile < row_tiles; tile += tiles) {
        const uint32_t row0 = tile * kTileRows + k.wave * 32u;
        const bool any_row = row0 < k.rows;
        uint32_t place[K::kCopies];  // of the tile that is copied next
        __syncthreads();             // the row tile before has been read
        if (first < last) {
            k.find(first, place);
            k.copy(lds[0][0], lds[0][1], place, first + 1u);
        }
        k.begin(any_row ? row0 : tile * kTileRows);
        DAV2_WAIT_VMCNT(0);
        __syncthreads();
        for (uint32_t block = first; block < last; ++block) {
            const uint32_t buffer = (block - first) & 1u;
            k.copy(lds[buffer ^ 1u][0], lds[buffer ^ 1u][1], place, block + 2u);  // behind the last tile its last key, unread
            if (any_row) {
                v16f sc[K::kBlocks];
                k.multiply_keys(lds[buffer][0], sc);
                k.weigh(block, sc);
                k.multiply_values(lds[buffer][1]);
            }
            DAV2_WAIT_VMCNT(0);
            lds_turn();
        }
        k.end(row0, split, splits);
    }
}

template <typename E, int FEW>
__global__ __launch_bounds__(256) void cross_join_kernel(dav2_cross_attention_args a, uint32_t splits) {
    const uint64_t per_batch = static_cast<uint64_t>(a.query_tokens) * a.heads, rows = a.batch * per_batch;
    const Parts parts = parts_at(a.scratch, rows * splits);
    auto output = [&](uint64_t r) {
        const uint32_t row = static_cast<uint32_t>(r), each = static_cast<uint32_t>(per_batch);  // below 2^32
        const uint32_t b = row / each, in = row - b * each, token = in / a.heads, head = in - token * a.heads;
        return static_cast<E*>(a.output) + b * a.output_batch_stride + token * a.output_stride + head * a.head_dim;
    };
    if constexpr (FEW > 0) {
        const uint32_t lanes = join_lanes_log2(a.head_dim), each = 256u >> lanes, f4 = threadIdx.x & ((1u << lanes) - 1u);
        for (uint64_t r = static_cast<uint64_t>(blockIdx.x) * each + (threadIdx.x >> lanes); r < rows;
             r += static_cast<uint64_t>(gridDim.x) * each)
            join_few<FEW>(parts, r * splits, splits, a.head_dim, f4, output(r));
    } else {
        for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) join_row(parts, r * splits, splits, a.head_dim, output(r));
    }
}

// How a call is dealt out: 128 rows a workgroup, two on a CU, or 256 and one,
// where wide heads of 16 bits leave no room for a third and the larger tiles
// add no rows that do not exist and fill the chip (us, 256 against 128: 8 x 2048
// queries, 4096 keys 1150 / 1200; 16 x 100 queries, 577 keys 29.2 / 30.5; 2 x 1024
// queries and keys 38.6 / 38.9). The keys are split while all workgroups run at
// once, down to two tiles each (fp32: 128 queries, 12 heads of 64, 1024 keys,
// 20.0 us in 16, 21.9 in 8). us: 64 workgroups of one query each and 1370 keys,
// f16, 11.9 in 4, 10.1 in 8, 10.7 in 10; 160 of 577 queries, 25.6 whole, 22.5 in
// 3, fp32 102 whole, 110 in 2, 75 in 3; 80 of 300 queries, 32 heads of 8 of 128,
// 4096 keys, bf16, 40.8 in 3, 39.5 in 6.
struct Plan {
    uint32_t tile;  // rows of a workgroup: 128 or 256
    uint32_t tiles, splits;
};
Plan plan_of(const dav2_cross_attention_args& a) {
    Plan p{128, 1, 1};
    if (a.kv_heads == 0 || a.heads < a.kv_heads || a.batch == 0 || a.query_tokens == 0) return p;
    const uint64_t rows = static_cast<uint64_t>(a.query_tokens) * (a.heads / a.kv_heads);
    // a call's planes are below 2^23; sizes that no call has may not overflow below
    const uint64_t planes = std::min<uint64_t>(static_cast<uint64_t>(a.kv_heads) * a.batch, 1u << 23);
    const uint64_t most = std::clamp<uint64_t>(a.key_tokens / (a.dtype == DAV2_DTYPE_F32 ? 64 : 128), 1, kMostSplits);
    if (a.head_dim > 64 && a.dtype != DAV2_DTYPE_F32 && (rows + 127) / 128 % 2 == 0 &&
        (rows + 255) / 256 * planes * most >= 256)
        p.tile = 256;
    p.tiles = static_cast<uint32_t>(std::min<uint64_t>((rows + p.tile - 1) / p.tile, 512));
    p.splits = static_cast<uint32_t>(std::clamp<uint64_t>((p.tile == 256 ? 256 : 512) / (p.tiles * planes), 1, most));
    return p;
}
uint64_t split_bytes(const dav2_cross_attention_args& a, const Plan& p) {
    if (p.splits == 1) return 0;
    return (parts_bytes(static_cast<uint64_t>(a.batch) * a.query_tokens * a.heads * p.splits, a.head_dim) + 15u) & ~uint64_t(15);
}

}  // namespace

// dav2_hip_cross_attention_scratch_bytes() goes by the sizes alone and always
// has room for a mask's lists; this is whether a call touches it.
namespace dav2k {
bool cross_attention_uses_scratch(const dav2_cross_attention_args& a) {
    return plan_of(a).splits > 1 || (a.key_mask && a.key_tokens);
}
}  // namespace dav2k

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
        (a.batch > 1 && a.output_batch_stride < row) ||
        (a.key_tokens > 1 && (a.key_stride < key_row || a.value_stride < key_row)))
        return hipErrorInvalidValue;
    if (cross_attention_uses_scratch(a) && (!a.scratch || !aligned16(a.scratch) ||
                                            a.scratch_bytes < dav2_hip_cross_attention_scratch_bytes(args)))
        return hipErrorInvalidValue;
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
            constexpr int D = decltype(dim)::value;
            if constexpr (D > 64 && sizeof(E) == 2) {
                if (p.tile == 256)
                    return dispatch(lists.keys ? cross_tiles_kernel<E, D, true, 8> : cross_tiles_kernel<E, D, false, 8>, grid,
                                    dim3(512), 0, s, a, lists, p.splits, p.tiles);
            }
            dispatch(lists.keys ? cross_tiles_kernel<E, D, true, 4> : cross_tiles_kernel<E, D, false, 4>, grid, dim3(256), 0,
                     s, a, lists, p.splits, p.tiles);
        });
        if (p.splits > 1) {
            const uint64_t rows = static_cast<uint64_t>(a.batch) * a.query_tokens * a.heads;
            const int few = join_kind(rows, p.splits);
            const uint64_t each = few ? join_rows(a.head_dim) : 1;
            const dim3 join(static_cast<uint32_t>(std::min<uint64_t>((rows + each - 1) / each, 65536)));
            dispatch(few == 4   ? cross_join_kernel<E, 4>
                     : few == 8 ? cross_join_kernel<E, 8>
                                : cross_join_kernel<E, 0>,
                     join, dim3(256), 0, s, a, p.splits);
        }
        return hipGetLastError();
    });
}

}  // extern "C"
