// The int8 key/value cache: storing new tokens, and attention over it.
//
// One scale per page and head, s = max over the page of |x| / 127, so a page's
// codes are bounded by its largest value and a scale is read once per page.

#include <algorithm>
#include <type_traits>

#include "cache.h"

using namespace dav2k;

namespace {

// max over the workgroup of non-negative floats by their bits: unsigned order
// puts NaN above infinity above every number, so a NaN is kept.
DAV2_DEV uint32_t workgroup_max_bits(uint32_t v, uint32_t* shared) {
    for (int o = 32; o > 0; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o, kWave)));
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
    for (uint32_t w = 1; w < blockDim.x / 64u; ++w) v = max(v, shared[w]);
    return v;
}

// A code at another scale (see dav2_cache_store_i8_args).
DAV2_DEV int requantize(int code, float old, float now, float inverse) {
    return quantize_div(static_cast<float>(code) * old, now, inverse);
}

DAV2_DEV uint32_t byte_of(uint32_t word, uint32_t i, int code) {
    return (word & ~(0xffu << (8u * i))) | ((static_cast<uint32_t>(code) & 0xffu) << (8u * i));
}

// A workgroup per (touched page, head and side, sequence); side 0 keys, 1
// values. The new rows are read once for their largest value and again for
// their codes, which keys keep in registers (up to kKept pieces of 16 features
// a thread) and values take from the caches: their pages are feature-major, so
// a thread needs 16 tokens of one 4-byte piece of features. Codes are written
// 16 at a time; a value chunk that also holds older or later tokens is read,
// changed and written back. 8 prompts of up to 2048 tokens, 8 heads of 128, f16
// (55 MB): 30 us, 1.8 TB/s, a third of a copy's rate: the vector units are busy
// for half of it, the waves wait for loads and stores for two thirds.
template <typename E, bool ALIGNED>
__global__ __launch_bounds__(256, 8) void cache_store_kernel(dav2_cache_store_i8_args a) {
    constexpr int kKept = 1;
    constexpr int kWords = sizeof(E);  // 16-byte words of 16 elements
    __shared__ uint32_t shared[4];
    typedef E V __attribute__((ext_vector_type(16 / sizeof(E))));
    constexpr int N = 16 / sizeof(E);
    const uint32_t h = blockIdx.y >> 1, side = blockIdx.y & 1u, s = blockIdx.z;
    const uint32_t page_size = a.cache.page_size, d = a.cache.head_dim, pieces = d / 16u;
    const Sequence q = sequence_of(a.starts, a.lengths, s, a.tokens);
    // positions [first, last) are new; in 64 bits, as a length may be anything
    const int64_t origin = static_cast<int64_t>(q.length) - (q.end - q.begin);  // row r has position origin + r - begin
    const int64_t first = max(origin, int64_t(0));
    const int64_t last = min(static_cast<int64_t>(q.length), static_cast<int64_t>(a.table_pages) * page_size);
    // nothing new: the page that the next token goes to is left alone, it may be another sequence's by now
    if (first >= last) return;
    const uint64_t stride = side ? a.value_stride : a.key_stride;
    const E* x = static_cast<const E*>(side ? a.values : a.keys) + static_cast<uint64_t>(h) * d;
    for (int64_t p = first / page_size + blockIdx.x; p * page_size < last; p += gridDim.x) {
        const int32_t page = a.page_table[static_cast<uint64_t>(s) * a.table_pages + p];
        if (page < 0 || static_cast<uint32_t>(page) >= a.cache.pages) continue;  // the same for the whole workgroup
        const int64_t base = p * page_size;
        const uint32_t from = static_cast<uint32_t>(max(first - base, int64_t(0)));
        const uint32_t to = static_cast<uint32_t>(min(last - base, static_cast<int64_t>(page_size)));
        const uint64_t plane = static_cast<uint64_t>(page) * a.cache.kv_heads + h;
        int8_t* codes = (side ? a.cache.values : a.cache.keys) + plane * page_size * d;
        float* scale = (side ? a.cache.value_scales : a.cache.key_scales) + plane;
        const E* slot0 = x + (q.begin + (base - origin)) * static_cast<int64_t>(stride);  // of slot 0, new or not
        auto load = [&](uint32_t item, E (&v)[16]) {
            const E* in = slot0 + (from + item / pieces) * stride + 16u * (item % pieces);
            if constexpr (ALIGNED) {
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    const V word = *reinterpret_cast<const V*>(in + N * w);
#pragma unroll
                    for (int i = 0; i < N; ++i) v[N * w + i] = word[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = in[i];
            }
        };
        const float old = from ? *scale : 0.0f;
        const uint32_t items = (to - from) * pieces;
        E kept[kKept][16];
        uint32_t most = 0;
#pragma unroll
        for (int k = 0; k < kKept; ++k) {
            if (threadIdx.x + 256u * k >= items) continue;
            load(threadIdx.x + 256u * k, kept[k]);
#pragma unroll
            for (int i = 0; i < 16; ++i) most = max(most, __float_as_uint(fabsf(static_cast<float>(kept[k][i]))));
        }
        for (uint32_t item = threadIdx.x + 256u * kKept; item < items; item += 256u) {
            E v[16];
            load(item, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) most = max(most, __float_as_uint(fabsf(static_cast<float>(v[i]))));
        }
        most = workgroup_max_bits(most, shared);
        // fmaxf would drop a NaN: compare bits again
        uint32_t bits = max(__float_as_uint(div_rn(__uint_as_float(most), 127.0f)), __float_as_uint(1.0e-8f));
        bits = max(bits, __float_as_uint(old) & 0x7fffffffu);
        const float now = __uint_as_float(bits), inverse = div_rn(1.0f, now);
        __syncthreads();  // every thread has read the old scale
        if (threadIdx.x == 0) *scale = now;
        const bool again = from && now != old;  // the older codes change
        if (side == 0) {
            auto put = [&](uint32_t item, const E (&v)[16]) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = pack4(quantize_div(static_cast<float>(v[4 * i]), now, inverse),
                                 quantize_div(static_cast<float>(v[4 * i + 1]), now, inverse),
                                 quantize_div(static_cast<float>(v[4 * i + 2]), now, inverse),
                                 quantize_div(static_cast<float>(v[4 * i + 3]), now, inverse));
                *reinterpret_cast<uint4*>(codes + from * d + 16u * item) = make_uint4(w[0], w[1], w[2], w[3]);
            };
#pragma unroll
            for (int k = 0; k < kKept; ++k)
                if (threadIdx.x + 256u * k < items) put(threadIdx.x + 256u * k, kept[k]);
            for (uint32_t item = threadIdx.x + 256u * kKept; item < items; item += 256u) {
                E v[16];
                load(item, v);
                put(item, v);
            }
            if (again)
                for (uint32_t i = threadIdx.x; i < from * d / 4u; i += 256u) {
                    uint32_t* word = reinterpret_cast<uint32_t*>(codes) + i;
                    const uint32_t w = *word;
                    *word = pack4(requantize(static_cast<int8_t>(w), old, now, inverse),
                                  requantize(static_cast<int8_t>(w >> 8), old, now, inverse),
                                  requantize(static_cast<int8_t>(w >> 16), old, now, inverse),
                                  requantize(static_cast<int8_t>(w >> 24), old, now, inverse));
                }
            continue;
        }
        constexpr uint32_t F = ALIGNED ? 4 / sizeof(E) : 1;  // features of an item
        typedef E Piece __attribute__((ext_vector_type(F)));
        const uint32_t features = d / F, chunk0 = again ? 0u : from / 16u, chunks = (to + 15u) / 16u - chunk0;
        for (uint32_t item = threadIdx.x; item < features * chunks; item += 256u) {
            const uint32_t chunk = chunk0 + item / features, f = item % features * F, s0 = chunk * 16u;
            uint4* out[F];
            uint32_t w[F][4] = {};
#pragma unroll
            for (uint32_t j = 0; j < F; ++j) out[j] = reinterpret_cast<uint4*>(codes + (f + j) * page_size + s0);
            const bool whole = s0 >= from && s0 + 16u <= to;
            if (!whole) {
#pragma unroll
                for (uint32_t j = 0; j < F; ++j) {
                    const uint4 o = *out[j];
                    w[j][0] = o.x, w[j][1] = o.y, w[j][2] = o.z, w[j][3] = o.w;
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                const uint32_t slot = s0 + i;
                if (slot >= from && slot < to) {
                    const Piece piece = *reinterpret_cast<const Piece*>(slot0 + slot * stride + f);
#pragma unroll
                    for (uint32_t j = 0; j < F; ++j)
                        w[j][i / 4] = byte_of(w[j][i / 4], i % 4, quantize_div(static_cast<float>(piece[j]), now, inverse));
                } else if (again && slot < from) {
#pragma unroll
                    for (uint32_t j = 0; j < F; ++j)
                        w[j][i / 4] = byte_of(w[j][i / 4], i % 4,
                                              requantize(static_cast<int8_t>(w[j][i / 4] >> (8 * (i % 4))), old, now, inverse));
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < F; ++j) *out[j] = make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]);
        }
    }
}

// ---------------------------------------------------------------------------
// Attention over the cache.
//
// Codes are exact in binary16, so both products run on the binary16 MFMA with
// fp32 sums. A query row is multiplied by the power of two that puts its
// largest value into [2^14, 2^15) and rounded to binary16: exact for binary16
// and bfloat16 queries down to 2^-28 of the largest; an fp32 row is kept as
// two such parts (22 bits).
//
// A value's scale sv goes with the weight of its key: with sv = 2^e f,
// 1 <= f < 2, and t = s log2(e) + e for a score s,
//   w = exp2(t - base),  O = sum (w f) c,  L = sum w 2^-e,  o = O / L.
// L is summed in fp32 from the unrounded w. For the product w f is rounded to
// binary16, whose smallest step is 2^-24: base lies kBias below the running
// maximum of t, so that the largest weights are near 2^15 and small ones, of
// which a long context has many, keep their bits. Against a weight of the
// maximum, w f is good to half a step (2^-11) down to 2^(-14 - kBias), and loses
// at most 2^(-25 - kBias) below. The fp32 mode, and every type where rows are
// few, has a second part: the rest times 2^11, whose product takes the codes
// times 2^-11 (exact in binary16), so that it ends 2^11 later: 2^-23 of a weight
// down to 2^(-14 - kBias), at most 2^(-36 - kBias) below.

// Eight codes as binary16: the byte c + 128 below the exponent of 1024 is the
// number 1152 + c.
DAV2_DEV h8 widen(uint32_t lo, uint32_t hi) {
    const uint32_t x = lo ^ 0x80808080u, y = hi ^ 0x80808080u;
    const h2 shift = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - shift;
    const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - shift;
    const h2 c = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, y, 0x04010400u)) - shift;
    const h2 d = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, y, 0x04030402u)) - shift;
    return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

DAV2_DEV Parts parts_of(const dav2_attention_cache_i8_args& a, uint32_t splits) {
    return parts_at(a.scratch, static_cast<uint64_t>(a.tokens) * a.heads * splits);
}

// Few query rows for a cache head (single tokens, drafts): bound by reading
// the cache. A workgroup has 16 rows (token-major: row r is token r / group,
// query head r % group) of one sequence and cache head and a run of 64-key
// blocks, which its four waves take in turn; each wave goes through its blocks
// alone, and their sums are joined through LDS at the end. One token each of 32
// sequences of up to 32768, 32 heads of 8, 128 features, bf16: 230 us for 1.2
// GB, 5.3 TB/s, where a large copy runs at 5.1.
//
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16. The cache's layout
// is such that both left operands are 16-byte pieces of global memory, taken
// straight into registers: lane l has 16 features 64 kc + 16 (l / 16) .. of a
// key, and the 16 keys of chunk l / 16 of one feature. Row i of score tile a
// is key 16 (i / 4) + 4 a + i % 4 of the block; a lane then holds the scores of
// chunk l / 16 in order, which is the right operand of the second product as
// it stands, and the scales it needs are those of one page.
template <typename E, int D>
__global__ __launch_bounds__(256, 2) void cache_rows_kernel(dav2_attention_cache_i8_args a, uint32_t splits,
                                                            uint32_t tiles) {
    constexpr bool kFloat = std::is_same_v<E, float>;
    constexpr int KC = (D + 63) / 64, FT = D / 16, NP = kFloat ? 2 : 1;
    constexpr uint32_t d = D;
    constexpr int kPad = 17;  // row length of the joining waves' sums in LDS
    constexpr float kBias = 14.0f;  // a weight times a fraction stays below 2^15
    __shared__ float joined[4][D * kPad];
    __shared__ float shared_base[4][16], shared_sum[4][16];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col = lane & 15u, g = lane >> 4;
    const uint32_t split = blockIdx.x % splits, h = blockIdx.y, s = blockIdx.z;
    const uint32_t page_size = a.cache.page_size, kv_heads = a.cache.kv_heads;
    const uint32_t group = a.heads / kv_heads;
    const Sequence q = sequence_of(a.starts, a.lengths, s, a.tokens);
    const uint32_t n = static_cast<uint32_t>(q.end - q.begin);
    const uint32_t rows = n * group;  // tokens * heads is below 2^32
    const int64_t span = static_cast<int64_t>(a.table_pages) * page_size;
    const Pages pages = pages_of(a, s);
    const Parts parts = parts_of(a, splits);

    for (uint32_t tile = blockIdx.x / splits; tile < (rows + 15u) / 16u; tile += tiles) {
        const Rows<16> of(tile * 16u, group, rows);
        const uint32_t row = tile * 16u + col;
        uint32_t token, head;
        of.find(col, token, head);
        head += h * group;
        // keys that this lane's row sees, and the most that a row of the tile does
        auto seen = [&](uint32_t i) {
            int64_t t = q.length;
            if (a.causal) t += 1 + static_cast<int64_t>(i) - n;
            return static_cast<uint32_t>(max(min(t, span), int64_t(0)));
        };
        const uint32_t limit = row < rows ? seen(token) : 0u;
        uint32_t last_token, last_head;
        of.find(15u, last_token, last_head);
        const uint32_t most = seen(last_token), least = seen(of.token);
        const uint32_t blocks = (most + 63u) / 64u, per = (blocks + splits - 1u) / splits;
        const uint32_t first = split * per, last = min(first + per, blocks);

        v4f o[FT];
#pragma unroll
        for (int f = 0; f < FT; ++f) o[f] = v4f{0.f, 0.f, 0.f, 0.f};
        float maximum = kNoScore, base = kNoScore, sum = 0.0f;  // sum: this lane's keys only

        // A block's keys are loaded when the scores of the block before are
        // done, its values and scales behind that block's values, its places
        // in the table a block before those.
        uint4 kraw[4][KC], vraw[FT];
        Pages::Place of_key{}, of_value{};  // chunk col / 4 for the keys, chunk g for the values and the scales
        bool exists = false;
        float key_scale = 0.0f, value_scale = 1.0f;
        auto find = [&](uint32_t block) {
            of_key = pages.find(block * 4u + col / 4u);
            of_value = pages.find(block * 4u + g);
        };
        auto load_keys = [&] {
            const int8_t* k = a.cache.keys + ((static_cast<uint64_t>(pages.page(of_key)) * kv_heads + h) * page_size +
                                              of_key.slot + col % 4u) * d;
            // features that the head does not have: others in their place, which meet zeros of the query
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int kc = 0; kc < KC; ++kc)
                    kraw[t][kc] = *reinterpret_cast<const uint4*>(k + 4u * t * d + min(64u * kc + 16u * g, d - 16u));
        };
        auto load_values = [&] {
            exists = pages.exists(of_value);
            const uint64_t plane = static_cast<uint64_t>(pages.page(of_value)) * kv_heads + h;
            key_scale = a.cache.key_scales[plane];
            value_scale = a.cache.value_scales[plane];
            const int8_t* v = a.cache.values + (plane * d + col) * page_size + of_value.slot;
#pragma unroll
            for (int f = 0; f < FT; ++f)
                vraw[f] = *reinterpret_cast<const uint4*>(v + static_cast<uint64_t>(16u * f) * page_size);
        };
        uint32_t block = first + wave;
        if (block < last) {
            find(block);
            load_keys();
            load_values();
            find(min(block + 4u, last - 1u));
        }

        // the right operand of the scores
        h8 qf[NP][KC][2];
        float factor;  // score = sum * factor, in units of log2
        {
            const E* x = static_cast<const E*>(a.query) + static_cast<uint64_t>(q.begin + token) * a.query_stride +
                         static_cast<uint64_t>(head) * d;
            typedef E V __attribute__((ext_vector_type(16 / sizeof(E))));
            constexpr int kVec = 16 / sizeof(E);
            float v[KC][16];
            float largest = 0.0f;
#pragma unroll
            for (int kc = 0; kc < KC; ++kc)
#pragma unroll
                for (int j = 0; j < 16 / kVec; ++j) {
                    V piece{};
                    if (64u * kc + 16u * g < d) piece = *reinterpret_cast<const V*>(x + 64 * kc + 16 * g + kVec * j);
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        v[kc][kVec * j + i] = static_cast<float>(piece[i]);
                        largest = fmaxf(largest, fabsf(v[kc][kVec * j + i]));
                    }
                }
            largest = over_groups(largest, Larger());
            // up is a power of two; rows of zeros, NaN and infinities stay as they are
            const int e = largest > 0.0f && largest < INFINITY ? 14 - ilogbf(largest) : 0;
            const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
            factor = ldexpf(fabsf(a.scale) * kLog2e, -e);
#pragma unroll
            for (int kc = 0; kc < KC; ++kc)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float y = keep_fp32(ldexpf(v[kc][i], e) * sign);
                    const _Float16 hi = static_cast<_Float16>(y);
                    qf[0][kc][i >> 3][i & 7] = hi;
                    if constexpr (kFloat)
                        qf[1][kc][i >> 3][i & 7] = static_cast<_Float16>(y - static_cast<float>(hi));
                }
        }

        // A wave's last block is apart: registers that are loaded in one branch
        // only are waited for where the branches meet (64 sequences of up to
        // 2048 keys, 16 heads of 64: 44 us with the branch, 38 without).
        auto step = [&](auto more) {
            constexpr bool kMore = decltype(more)::value;
            v4f sc[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                sc[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kc = 0; kc < KC; ++kc) {
                    const h8 k0 = widen(kraw[t][kc].x, kraw[t][kc].y), k1 = widen(kraw[t][kc].z, kraw[t][kc].w);
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[p][kc][0], sc[t], 0, 0, 0);
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[p][kc][1], sc[t], 0, 0, 0);
                    }
                }
            }
            if constexpr (kMore) load_keys();
            float exponent, fraction, inverse;
            const uint32_t key0 = block * 64u + 16u * g;  // of this lane's first score
            // a chunk that the row does not see may have any scale, NaN included
            split_scale(exists && key0 < limit ? value_scale : 1.0f, exponent, fraction, inverse);
            const float c = key_scale * factor;
            const bool whole = (block + 1u) * 64u <= least && __all(exists);
            float largest = kNoScore;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = fmaf(sc[t][r], c, exponent);
                    if (!whole && (!exists || key0 + 4 * t + r >= limit)) x = -INFINITY;
                    sc[t][r] = x;
                    largest = fmaxf(largest, x);
                }
            largest = over_groups(largest, Larger());
            if (__any(largest > maximum)) {
                maximum = fmaxf(maximum, largest);
                const float moved = fabsf(maximum) < kFar ? maximum - kBias : maximum;
                const float keep = __builtin_amdgcn_exp2f(base - moved);
                base = moved;
                sum *= keep;
#pragma unroll
                for (int f = 0; f < FT; ++f) o[f] *= keep;
            }
            // Both parts for every type, as the products are not what bounds this
            // kernel: the error of binary16 rows falls from 3.0e-4 to 2.1e-4, that
            // of rounding the output alone, for 231 -> 232 us in the case above,
            // 38.4 -> 40.2 for 64 sequences of 2048 keys, 16 heads of 64, and 23.4
            // -> 25.3 for 8 tokens each of 8 on 4096 keys, 32 heads of 4 of 128.
            h8 pf[2][2];
            float part = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float w = __builtin_amdgcn_exp2f(sc[t][r] - base);
                    part += w;
                    const float y = keep_fp32(w * fraction);  // hi and lo of one rounded product
                    const _Float16 hi = static_cast<_Float16>(y);
                    pf[0][t >> 1][4 * (t & 1) + r] = hi;
                    pf[1][t >> 1][4 * (t & 1) + r] = static_cast<_Float16>((y - static_cast<float>(hi)) * kSecond);
                }
            sum = fmaf(part, inverse, sum);
#pragma unroll
            for (int f = 0; f < FT; ++f) {
                const h8 v0 = widen(vraw[f].x, vraw[f].y), v1 = widen(vraw[f].z, vraw[f].w);
                o[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[0][0], o[f], 0, 0, 0);
                o[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[0][1], o[f], 0, 0, 0);
                o[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(for_second(v0), pf[1][0], o[f], 0, 0, 0);
                o[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(for_second(v1), pf[1][1], o[f], 0, 0, 0);
            }
            if constexpr (kMore) {
                load_values();
                find(min(block + 8u, last - 1u));
            }
        };
        for (; block + 4u < last; block += 4u) step(std::true_type());
        if (block < last) step(std::false_type());
        sum = over_groups(sum, Plus());

        // join the four waves: lane (col, g), register r of o[f]: feature 16 f + 4 g + r of row col
        __syncthreads();  // the tile before has been read
        if (g == 0) {
            shared_base[wave][col] = base;
            shared_sum[wave][col] = sum;
        }
        __syncthreads();
        float top = kNoScore;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, shared_base[w][col]);
        const float mine = __builtin_amdgcn_exp2f(base - top);
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
            for (int r = 0; r < 4; ++r) joined[wave][(16 * f + 4 * g + r) * kPad + col] = o[f][r] * mine;
        __syncthreads();
        // 16 threads for each of the 16 rows
        const uint32_t out_col = threadIdx.x >> 4, lane16 = threadIdx.x & 15u;
        if (tile * 16u + out_col < rows) {
            float all = kNoScore, total = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) all = fmaxf(all, shared_base[w][out_col]);
#pragma unroll
            for (int w = 0; w < 4; ++w)
                total = fmaf(shared_sum[w][out_col], __builtin_amdgcn_exp2f(shared_base[w][out_col] - all), total);
            uint32_t out_token, out_head;
            of.find(out_col, out_token, out_head);
            out_head += h * group;
            const uint64_t at = static_cast<uint64_t>(q.begin) + out_token;
            const float scale = splits > 1 ? 1.0f : total == 0.0f ? 0.0f : 1.0f / total;
            E* y = static_cast<E*>(a.output) + at * a.output_stride + static_cast<uint64_t>(out_head) * d;
            const uint64_t slot = (at * a.heads + out_head) * splits + split;
            for (uint32_t f = lane16; f < d; f += 16u) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) v += joined[w][f * kPad + out_col];
                if (splits > 1) parts.sums[slot * d + f] = v;
                else y[f] = static_cast<E>(v * scale);
            }
            if (splits > 1 && lane16 == 0) parts.stats[slot] = make_float2(all, total);
        }
    }
}

// Many query rows for a cache head (prompts): bound by the matrix cores, the
// vector units and LDS, each busy for some 40 % of the time. A workgroup has
// 128 or 256 rows of one sequence and cache head, 32 for each of its waves, and
// goes through the keys 64 at a time: codes are widened to binary16 once for
// all waves on their way into LDS (two buffers, one barrier for a tile; the
// next tile's codes are in registers meanwhile, its places in the table a tile
// before). Two prompts' last 2048 of up to 8192 tokens, 32 heads of 8, 128
// features, f16: 451 us, 700 TFLOP/s; 8 times 512 of 4096 750 TFLOP/s; every
// row all keys 800. A tile shared by eight waves instead of four is worth 10 %
// there, the staging and the exponentials written between the matrix
// instructions 8 %. Heads of 64 are held to registers for three waves a SIMD:
// 16 prompts' last 300 of up to 2048 tokens 76 us, 12 % more with four registers
// more. A slack of 6 with a smaller bias (see above) is 1 % faster, the fp32
// mode without its factor of 2^11 5 to 9 %.
//
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16_f16. Lane l holds, for
// query l % 32, the scores of keys 8 (r / 4) + 4 (l / 32) + r % 4 of a 32-key
// block in registers r; registers 8 t .. 8 t + 7 are the right operand of the
// second product's step t if V^T holds its keys in that order, which their
// place in LDS gives them: keys 0-3, 8-11 of a chunk, then 4-7, 12-15. Eight
// registers are one 16-token chunk, so scales are uniform for them.
template <typename E, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, D <= 64 && sizeof(E) == 2 ? 3 : 2)
void cache_tiles_kernel(dav2_attention_cache_i8_args a, uint32_t splits, uint32_t tiles) {
    constexpr bool kFloat = std::is_same_v<E, float>;
    constexpr int HEAD = D <= 64 ? 64 : 128;  // features of a row in LDS
    constexpr int KS = D / 16, FB = (D + 31) / 32, NP = kFloat ? 2 : 1;
    constexpr uint32_t d = D;
    constexpr uint32_t kThreads = 64 * WAVES, kTileRows = 32 * WAVES;
    constexpr int kPieces = HEAD * 4 / kThreads;  // of 16 codes, for each thread and tile: keys, and values
    constexpr int kRow = HEAD * 2;       // bytes of a key row in LDS
    // rescale when a score passes the running maximum by kSlack: most tiles
    // leave the sums alone. Weights (times a fraction in the fp32 mode) stay
    // below 2^15.
    constexpr float kSlack = 2.0f, kBias = kFloat ? 14.0f - kSlack : 15.0f - kSlack;
    __shared__ __attribute__((aligned(16))) int8_t lds_keys[2][64 * kRow];
    __shared__ __attribute__((aligned(16))) int8_t lds_values[2][HEAD * 128];
    __shared__ __attribute__((aligned(16))) v4f lds_scales[2][4];  // of a chunk: key scale, log2 / exponent, inverse, fraction
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col = lane & 31u, hf = lane >> 5;
    const uint32_t kv_heads = a.cache.kv_heads, page_size = a.cache.page_size;
    const uint32_t s = blockIdx.x / kv_heads, h = blockIdx.x - s * kv_heads, group = a.heads / kv_heads;
    const uint32_t split = blockIdx.y % splits;
    const Sequence q = sequence_of(a.starts, a.lengths, s, a.tokens);
    const uint32_t n = static_cast<uint32_t>(q.end - q.begin), rows = n * group;
    const int64_t span = static_cast<int64_t>(a.table_pages) * page_size;
    const Pages pages = pages_of(a, s);
    const Parts parts = parts_of(a, splits);
    const uint32_t row_tiles = (rows + kTileRows - 1u) / kTileRows;
    auto seen = [&](uint32_t i) {
        int64_t t = q.length;
        if (a.causal) t += 1 + static_cast<int64_t>(i) - n;
        return static_cast<uint32_t>(max(min(t, span), int64_t(0)));
    };

    // the last rows first: under a causal mask they see the most keys
    for (uint32_t turn = blockIdx.y / splits; turn < row_tiles; turn += tiles) {
        const uint32_t tile = row_tiles - 1u - turn;
        const uint32_t row0 = tile * kTileRows + wave * 32u;  // of this wave
        const bool any_row = row0 < rows;
        const Rows<32> of(any_row ? row0 : tile * kTileRows, group, rows);
        uint32_t token, head, last_token, last_head;
        of.find(col, token, head);
        of.find(31u, last_token, last_head);
        head += h * group;
        const uint32_t limit = row0 + col < rows ? seen(token) : 0u;
        const uint32_t wave_most = any_row ? seen(last_token) : 0u, wave_least = seen(of.token);
        const uint32_t most = seen((min(tile * kTileRows + kTileRows, rows) - 1u) / group);
        const uint32_t blocks = (most + 63u) / 64u, per = (blocks + splits - 1u) / splits;
        const uint32_t first = split * per, last = min(first + per, blocks);

        // staging
        uint4 key_codes[kPieces], value_codes[kPieces];
        Pages::Place of_key[kPieces]{}, of_value{};
        float key_scale = 0.0f, value_scale = 1.0f;
        bool exists = false;
        const uint32_t key_chunk = threadIdx.x % (HEAD / 16), key_row = threadIdx.x / (HEAD / 16);
        const uint32_t value_chunk = threadIdx.x & 3u, value_row = threadIdx.x >> 2;
        constexpr uint32_t kKeyStep = kThreads / (HEAD / 16), kValueStep = kThreads / 4;
        // features that the head does not have: others in their place, whose
        // copies in LDS meet no query feature and reach no output
        const uint32_t key_feature = 16u * key_chunk < d ? 16u * key_chunk : 0u;
        // Called without a condition, and never past the last block: registers
        // that are loaded in one branch only are waited for where the branches
        // meet.
        auto find = [&](uint32_t block) {
            block = min(block, last - 1u);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) of_key[i] = pages.find(block * 4u + (key_row + kKeyStep * i) / 16u);
            of_value = pages.find(block * 4u + value_chunk);
        };
        auto load_keys = [&] {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint64_t plane = static_cast<uint64_t>(pages.page(of_key[i])) * kv_heads + h;
                key_codes[i] = *reinterpret_cast<const uint4*>(
                    a.cache.keys + (plane * page_size + of_key[i].slot + (key_row + kKeyStep * i) % 16u) * d + key_feature);
            }
        };
        auto load_values = [&] {
            exists = pages.exists(of_value);
            const uint64_t plane = static_cast<uint64_t>(pages.page(of_value)) * kv_heads + h;
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                value_codes[i] = *reinterpret_cast<const uint4*>(
                    a.cache.values + (plane * d + min(value_row + kValueStep * i, d - 1u)) * page_size + of_value.slot);
            key_scale = a.cache.key_scales[plane];
            value_scale = a.cache.value_scales[plane];
        };
        auto store_scales = [&](uint32_t buffer) {
            if (threadIdx.x < 4) {
                float exponent, fraction, inverse;
                split_scale(value_scale, exponent, fraction, inverse);
                v4f c = {key_scale, exponent, inverse, fraction};
                if constexpr (!kFloat) {
                    // the weights take the whole scale, off by half a step of its
                    // logarithm: below 2^-20 of them for scales of 1e-8 and more
                    c[1] = exponent + __builtin_amdgcn_logf(fraction);
                    c[2] = inverse / fraction;
                }
                if (!exists) c = v4f{0.f, 0.f, 0.f, 0.f};
                lds_scales[buffer][threadIdx.x] = c;
            }
        };
        // Bringing a tile in small steps that fit between matrix instructions:
        // the codes loaded before go to LDS, the next ones are loaded, and the
        // places of those after them are looked up.
        constexpr int kStages = 4 * kPieces + 3;
        auto stage = [&](int n, uint32_t buffer, uint32_t block) {
            if (n < 4 * kPieces) {
                const int i = n / 4, half = n & 1;
                if (n & 2) {
                    const uint4 v = value_codes[i];
                    *reinterpret_cast<h8*>(lds_values[buffer] +
                                           swz<128>(value_row + kValueStep * i, 2u * value_chunk + half)) =
                        half ? widen(v.y, v.w) : widen(v.x, v.z);
                } else {
                    const uint4 k = key_codes[i];
                    *reinterpret_cast<h8*>(lds_keys[buffer] + swz<kRow>(key_row + kKeyStep * i, 2u * key_chunk + half)) =
                        half ? widen(k.z, k.w) : widen(k.x, k.y);
                }
            } else if (n == 4 * kPieces) {
                load_keys();
            } else if (n == 4 * kPieces + 1) {
                load_values();
            } else if (n == 4 * kPieces + 2) {
                find(block);
            }
        };
        auto stage_rest = [&](int n, uint32_t buffer, uint32_t block) {
#pragma unroll
            for (int i = 0; i < kStages; ++i)
                if (i >= n) stage(i, buffer, block);
        };
        __syncthreads();  // the row tile before has been read
        if (first < last) {
            find(first);
            load_keys();
            load_values();
            find(first + 1u);
        }

        // the right operand of the scores
        h8 qf[NP][KS];
        float factor;
        {
            const E* x = static_cast<const E*>(a.query) + static_cast<uint64_t>(q.begin + token) * a.query_stride +
                         static_cast<uint64_t>(head) * d + 8u * hf;
            typedef E V __attribute__((ext_vector_type(16 / sizeof(E))));
            constexpr int kVec = 16 / sizeof(E);
            V raw[KS][8 / kVec];
            float largest = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int j = 0; j < 8 / kVec; ++j) {
                    raw[k][j] = *reinterpret_cast<const V*>(x + 16 * k + kVec * j);
#pragma unroll
                    for (int i = 0; i < kVec; ++i) largest = fmaxf(largest, fabsf(static_cast<float>(raw[k][j][i])));
                }
            largest = over_halves(largest, Larger());
            const int e = largest > 0.0f && largest < INFINITY ? 14 - ilogbf(largest) : 0;
            const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
            factor = ldexpf(fabsf(a.scale) * kLog2e, -e);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = keep_fp32(ldexpf(static_cast<float>(raw[k][i / kVec][i % kVec]), e) * sign);
                    const _Float16 hi = static_cast<_Float16>(y);
                    qf[0][k][i] = hi;
                    if constexpr (kFloat) qf[1][k][i] = static_cast<_Float16>(y - static_cast<float>(hi));
                }
        }

        v16f o[FB];
#pragma unroll
        for (int f = 0; f < FB; ++f)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[f][r] = 0.0f;
        float base = kNoScore, sum = 0.0f;  // sum: this lane's keys only
        bool far = false;                   // the same for all lanes

        if (first < last) {
            store_scales(0);
            stage_rest(0, 0, first + 2u);
        }
        __syncthreads();
        for (uint32_t block = first; block < last; ++block) {
            const uint32_t buffer = (block - first) & 1u;
            const uint32_t k0 = block * 64u;
            // behind the last tile that one is brought again, unread
            store_scales(buffer ^ 1u);
            if (k0 >= wave_most) {
                stage_rest(0, buffer ^ 1u, block + 3u);
            } else {
                // A matrix instruction leaves the wave some seven others for
                // free: the order is written out and held.
                v16f sc[2];
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[b][r] = 0.0f;
                {
                    h8 in[2][2];
                    auto read = [&](int k, h8 (&v)[2]) {
                        v[0] = *reinterpret_cast<const h8*>(lds_keys[buffer] + swz<kRow>(col, 2u * k + hf));
                        v[1] = *reinterpret_cast<const h8*>(lds_keys[buffer] + swz<kRow>(col + 32u, 2u * k + hf));
                    };
                    read(0, in[0]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        if (k + 1 < KS) read(k + 1, in[(k + 1) & 1]);
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
#pragma unroll
                            for (int p = 0; p < NP; ++p)
                                sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(in[k & 1][b], qf[p][k], sc[b], 0, 0, 0);
                            stage(2 * k + b, buffer ^ 1u, block + 3u);
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                    stage_rest(2 * KS, buffer ^ 1u, block + 3u);
                }
                h8 vf[2][FB];
                auto read_values = [&](int t, h8 (&v)[FB]) {
#pragma unroll
                    for (int f = 0; f < FB; ++f)
                        v[f] = *reinterpret_cast<const h8*>(lds_values[buffer] + swz<128>(32u * f + col, 2u * t + hf));
                };
                read_values(0, vf[0]);
                __builtin_amdgcn_sched_barrier(0);
                // chunk t of the tile: registers 8 (t % 2) .. of block t / 2
                float c[4], shift[4], inverse[4], fraction[4];
                bool whole = k0 + 64u <= wave_least;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const v4f of_chunk = lds_scales[buffer][t];
                    c[t] = of_chunk[0] * factor;
                    shift[t] = of_chunk[1];
                    inverse[t] = of_chunk[2];
                    fraction[t] = of_chunk[3];
                    whole = whole && of_chunk[3] != 0.0f;  // else the page does not exist
                }
                if (!__all(whole)) {
                    stay_in_branch();
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const bool here = fraction[t] != 0.0f;
#pragma unroll
                        for (int r = 0; r < 8; ++r) {
                            const float x = fmaf(sc[t >> 1][8 * (t & 1) + r], c[t], shift[t]);
                            const uint32_t key = k0 + 16u * t + 8u * (r >> 2) + 4u * hf + (r & 3);
                            sc[t >> 1][8 * (t & 1) + r] = here && key < limit ? x : -INFINITY;
                        }
                        c[t] = 1.0f;
                        shift[t] = 0.0f;
                        // a chunk that the row does not see may have any scale, NaN included
                        if (!here || k0 + 16u * t >= limit) inverse[t] = fraction[t] = 1.0f;
                    }
                }
                float largest = kNoScore;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    float m = sc[t >> 1][8 * (t & 1)];
#pragma unroll
                    for (int r = 1; r < 8; ++r) m = fmaxf(m, sc[t >> 1][8 * (t & 1) + r]);
                    largest = fmaxf(largest, fmaf(m, c[t], shift[t]));
                }
                largest = over_halves(largest, Larger());
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
                if (far) {
                    // a fused score minus the base would keep bits that the base has lost
                    stay_in_branch();
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            sc[t >> 1][8 * (t & 1) + r] = fmaf(sc[t >> 1][8 * (t & 1) + r], c[t], shift[t]);
                        c[t] = 1.0f;
                        shift[t] = 0.0f;
                    }
                }
                // weights of chunk t + 1 between the products of chunk t
                h8 pf[2][NP];
                float part = 0.0f;
                auto weigh = [&](int t, int r) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(sc[t >> 1][8 * (t & 1) + r], c[t], shift[t] - base));
                    part = r ? part + w : w;
                    if constexpr (kFloat) {
                        const float y = keep_fp32(w * fraction[t]);  // hi and lo of one rounded product
                        const _Float16 hi = static_cast<_Float16>(y);
                        pf[t & 1][0][r] = hi;
                        pf[t & 1][1][r] = static_cast<_Float16>((y - static_cast<float>(hi)) * kSecond);
                    } else {
                        pf[t & 1][0][r] = static_cast<_Float16>(w);
                    }
                    if (r == 7) sum = fmaf(part, inverse[t], sum);
                };
#pragma unroll
                for (int r = 0; r < 8; ++r) weigh(0, r);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (t < 3) read_values(t + 1, vf[(t + 1) & 1]);
#pragma unroll
                    for (int f = 0; f < FB; ++f) {
                        o[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[t & 1][f], pf[t & 1][0], o[f], 0, 0, 0);
                        if constexpr (kFloat)
                            o[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(for_second(vf[t & 1][f]), pf[t & 1][1], o[f], 0,
                                                                          0, 0);
                        if (t < 3)
#pragma unroll
                            for (int r = 8 * f / FB; r < 8 * (f + 1) / FB; ++r) weigh(t + 1, r);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
            lds_turn();
        }
        sum = over_halves(sum, Plus());
        // register r of o[f]: feature 32 f + 8 (r / 4) + 4 hf + r % 4 of row col
        if (row0 + col < rows) {
            const uint64_t at = static_cast<uint64_t>(q.begin) + token;
            const uint64_t slot = (at * a.heads + head) * splits + split;
            const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
            typedef E V4 __attribute__((ext_vector_type(4)));
            E* y = static_cast<E*>(a.output) + at * a.output_stride + static_cast<uint64_t>(head) * d;
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
            if (splits > 1 && hf == 0) parts.stats[slot] = make_float2(base, sum);
        }
    }
}

// The splits of the sequences' rows joined.
template <typename E, int FEW>
__global__ __launch_bounds__(256) void cache_join_kernel(dav2_attention_cache_i8_args a, uint32_t splits) {
    join_sequence<E, FEW>(a, parts_of(a, splits), splits);
}

bool valid(const dav2_attention_cache_i8_args& a) {
    const uint64_t row = static_cast<uint64_t>(a.heads) * a.cache.head_dim;
    return valid_pages(a.cache) && a.query && a.output && aligned16(a.query) && aligned16(a.output) && a.page_table &&
           a.starts && a.lengths && a.dtype <= DAV2_DTYPE_BF16 && a.sequences <= 65535u && a.tokens <= 0x7fffffffu &&
           a.table_pages > 0 && a.table_pages <= 0x7fffffffu && a.heads > 0 && a.heads <= 65535u &&
           a.heads % a.cache.kv_heads == 0 && static_cast<uint64_t>(a.tokens) * a.heads <= 0xfffffe00ull &&
           static_cast<uint64_t>(a.sequences) * a.cache.kv_heads <= 0x7fffffull &&
           a.query_stride % 8 == 0 && a.output_stride % 8 == 0 &&
           (a.tokens == 1 || (a.query_stride >= row && a.output_stride >= row));
}

// How a call is dealt out. cache_rows_kernel for up to 32 rows of a cache head,
// or little work: the tiles of cache_tiles_kernel have four times its latency,
// but do the same work in less than two thirds of the time where they fill the
// chip. us, rows against tiles, bf16, causal: 32 rows of 8 cache heads of 128, 8
// sequences of 2048 keys 21 / 25; 64 rows of 4 of 128, 8 of 4096 (2^26) 25 / 31;
// 128 rows of 8 of 64, 2 of 8192 (2^26) 22 / 25; 72 rows of 4 of 128, 32 of 1500
// (2^27) 37 / 32; 100 rows of 16 of 64, 8 of 4096 (2^28) 58 / 41.
// The figures below are from before the weights' bias and second part, which
// cost both sides alike: tiles 2 %, rows 1 to 10 %.
//
// cache_rows_kernel: two workgroups share a CU, so up to 512 all run at once:
// split the keys as far as that goes, down to 128 keys (two waves' blocks) each.
// Beyond it a further split only evens out sequences of different lengths and
// pays for long ones: up to 2048 workgroups of at least 2048 keys. Heads 32 of
// 8, 128 features, us: 40 sequences of 300 keys 13.2 whole, 19.6 in two (640
// workgroups); 8 of 4096 19.5 in 8 (512 workgroups), 24.0 in 16; 32 of up to
// 32768 257 in 2 (512), 244 in 4, 242 in 8; one token over 1370 keys, 16 heads
// of 64, 11.9 in 2, 10.4 in 5, 9.2 in 10.
//
// cache_tiles_kernel: splitting n keys s times costs n / s tiles one after the
// other and s parts to join, so s grows with sqrt(n), as sqrt(n / 32) (128 rows
// of 8 heads, 32768 keys, us: 46; sqrt(n / 64) 56, sqrt(n / 16) 53), and to
// one workgroup of 256 rows or two of 128 a CU. Tiles of 256 rows read and
// widen the keys once for twice the rows (441 us against 493 above, 36 against
// 40 for 8 times 64 tokens), if the head is wide enough that three waves of the
// smaller ones do not fit a SIMD instead (heads of 64, 16 times 1500 tokens:
// 166 against 141), if they add no rows that do not exist (2 times 577 tokens
// 60 against 45), and if there are enough of them: one for each CU, and two
// where a causal mask makes them unequal (4 prompts of 1024 tokens, 16 heads:
// 43 against 38).
struct Plan {
    uint32_t tile;  // rows: 16 of cache_rows_kernel, 128 or 256 of cache_tiles_kernel
    uint32_t tiles, splits;
};
Plan plan_of(const dav2_attention_cache_i8_args& a) {
    Plan p{16, 1, 1};
    if (a.cache.kv_heads == 0 || a.heads < a.cache.kv_heads || a.sequences == 0 || a.max_query == 0) return p;
    const uint64_t rows = static_cast<uint64_t>(std::min(a.max_query, a.tokens)) * (a.heads / a.cache.kv_heads);
    const uint64_t planes = static_cast<uint64_t>(a.cache.kv_heads) * a.sequences;
    const double work = static_cast<double>((rows + 15) / 16 * planes) * a.max_length * a.cache.head_dim;
    if (rows > 32 && work > 67108864.0) {
        uint64_t most = 1;  // splits
        while (most < kMostSplits && (most + 1) * (most + 1) * 32 <= a.max_length) ++most;
        const uint64_t wide = (rows + 255) / 256 * planes;
        const bool unequal = a.causal && a.max_query > a.max_length / 2 && wide < 512;
        p.tile = a.cache.head_dim > 64 && (rows + 127) / 128 % 2 == 0 && wide * most >= 256 && !unequal ? 256 : 128;
        p.tiles = static_cast<uint32_t>(std::min<uint64_t>((rows + p.tile - 1) / p.tile, 512));
        p.splits = static_cast<uint32_t>(
            std::clamp<uint64_t>((p.tile == 256 ? 256 : 512) / std::max<uint64_t>(1, p.tiles * planes), 1, most));
        return p;
    }
    p.tiles = static_cast<uint32_t>(std::min<uint64_t>((rows + 15) / 16, 4096));
    const uint64_t have = std::max<uint64_t>(1, p.tiles * planes);
    const uint64_t resident = std::min<uint64_t>(512 / have, a.max_length / 128);
    const uint64_t even = std::min<uint64_t>(2048 / have, a.max_length / 2048);
    p.splits = static_cast<uint32_t>(std::clamp<uint64_t>(std::max(resident, even), 1, kMostSplits));
    return p;
}

}  // namespace

extern "C" {

int dav2_hip_cache_store_i8(const dav2_cache_store_i8_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_cache_store_i8_args& a = *args;
    if (a.sequences == 0 || a.tokens == 0 || a.max_new == 0) return hipSuccess;
    const uint64_t row = static_cast<uint64_t>(a.cache.kv_heads) * a.cache.head_dim;
    if (!valid_pages(a.cache) || !a.keys || !a.values || !a.page_table || !a.starts || !a.lengths ||
        a.dtype > DAV2_DTYPE_BF16 || a.sequences > 65535u || a.tokens > 0x7fffffffu || a.table_pages == 0 ||
        a.table_pages > 0x7fffffffu || (a.tokens > 1 && (a.key_stride < row || a.value_stride < row)))
        return hipErrorInvalidValue;
    const uint64_t new_most = a.max_new < a.tokens ? a.max_new : a.tokens;
    const uint64_t touched = (new_most + a.cache.page_size - 2) / a.cache.page_size + 1;
    constexpr uint64_t kMostPages = 1u << 22;  // workgroups along x: threads of a launch stay below 2^32
    const dim3 grid(static_cast<uint32_t>(std::min<uint64_t>({touched, a.table_pages, kMostPages})), 2 * a.cache.kv_heads,
                    a.sequences);
    const uint64_t size = dtype_bytes(a.dtype);
    const bool aligned = aligned16(a.keys) && aligned16(a.values) && a.key_stride * size % 16 == 0 &&
                         a.value_stride * size % 16 == 0;
    with_dtype(a.dtype, [&](auto* e) {
        typedef std::remove_pointer_t<decltype(e)> E;
        dispatch(aligned ? cache_store_kernel<E, true> : cache_store_kernel<E, false>, grid, dim3(256), 0,
                 static_cast<hipStream_t>(stream), a);
    });
    return hipGetLastError();
}

uint64_t dav2_hip_attention_cache_i8_scratch_bytes(const dav2_attention_cache_i8_args* args) {
    if (!args) return 0;
    const dav2_attention_cache_i8_args& a = *args;
    const Plan p = plan_of(a);
    if (p.splits == 1) return 0;
    return parts_bytes(static_cast<uint64_t>(a.tokens) * a.heads * p.splits, a.cache.head_dim);
}

int dav2_hip_attention_cache_i8(const dav2_attention_cache_i8_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_attention_cache_i8_args& a = *args;
    if (a.sequences == 0 || a.tokens == 0 || a.max_query == 0) return hipSuccess;
    if (!valid(a)) return hipErrorInvalidValue;
    const uint64_t need = dav2_hip_attention_cache_i8_scratch_bytes(args);
    if (need && (!a.scratch || !aligned16(a.scratch) || a.scratch_bytes < need)) return hipErrorInvalidValue;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const Plan p = plan_of(a);
    const dim3 grid = p.tile > 16 ? dim3(a.cache.kv_heads * a.sequences, p.tiles * p.splits)
                              : dim3(p.tiles * p.splits, a.cache.kv_heads, a.sequences);
    return with_dtype(a.dtype, [&](auto* e) -> int {
        typedef std::remove_pointer_t<decltype(e)> E;
        with_head_dim(a.cache.head_dim, [&](auto dim) {
            constexpr int D = decltype(dim)::value;
            if constexpr (D > 64) {
                if (p.tile == 256) return dispatch(cache_tiles_kernel<E, D, 8>, grid, dim3(512), 0, s, a, p.splits, p.tiles);
            }
            if (p.tile == 128) dispatch(cache_tiles_kernel<E, D, 4>, grid, dim3(256), 0, s, a, p.splits, p.tiles);
            else dispatch(cache_rows_kernel<E, D>, grid, dim3(256), 0, s, a, p.splits, p.tiles);
        });
        if (p.splits > 1) {
            const JoinLaunch j = join_launch(a, p.splits);
            dispatch(j.few == 4   ? cache_join_kernel<E, 4>
                     : j.few == 8 ? cache_join_kernel<E, 8>
                                  : cache_join_kernel<E, 0>,
                     j.grid, dim3(256), 0, s, a, p.splits);
        }
        return hipGetLastError();
    });
}

}  // extern "C"
