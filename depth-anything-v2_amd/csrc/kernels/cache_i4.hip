// The 4-bit key/value cache: storing new tokens, and attention over it.
//
// One scale per token and head, s = max |x| / 7 over its features: a stored
// token is never rounded again, as one in a page with a common scale would be
// whenever that grows, which four bits do not bear.

#include <algorithm>
#include <type_traits>

#include "cache.h"

using namespace dav2k;

namespace {

// 16-byte vectors at addresses that are multiples of less
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4_by8 __attribute__((ext_vector_type(4), aligned(8)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));

// A code as it is held, of the rounded and clamped quotient x / scale; NaN is the lowest.
DAV2_DEV uint32_t nibble(float x, float scale, float inverse) {
    // x * inverse is within 7 (2^-23 + 2^-24 + 2^-47) < 2^-19 of the rounded
    // quotient: where it is that near to a border, the quotient itself decides
    float y = x * inverse;
    if (__builtin_expect(fabsf(y - __builtin_rintf(y)) > 0.5f - 0x1p-18f, 0)) y = div_rn(x, scale);
    return static_cast<uint32_t>(static_cast<int>(fminf(fmaxf(__builtin_rintf(y), -7.0f), 7.0f)) + 8);
}

// A wave for each new row (token, head, side).
template <typename E>
__global__ __launch_bounds__(256) void cache4_scale_kernel(dav2_cache_store_i4_args a) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t h = blockIdx.y >> 1, side = blockIdx.y & 1u, s = blockIdx.z;
    const uint32_t page_size = a.cache.page_size, d = a.cache.head_dim;
    const Sequence q = sequence_of(a.starts, a.lengths, s, a.tokens);
    const int64_t origin = static_cast<int64_t>(q.length) - (q.end - q.begin);
    const int64_t first = max(origin, int64_t(0));
    const int64_t last = min(static_cast<int64_t>(q.length), static_cast<int64_t>(a.table_pages) * page_size);
    const uint64_t stride = side ? a.value_stride : a.key_stride;
    const E* x = static_cast<const E*>(side ? a.values : a.keys) + static_cast<uint64_t>(h) * d;
    // two neighbouring tokens for each wave: their values share bytes
    for (int64_t pair = first / 2 + blockIdx.x * 4u + wave; 2 * pair < last; pair += gridDim.x * 4u) {
        for (int64_t t = max(2 * pair, first); t < min(2 * pair + 2, last); ++t) {
            const int32_t page = a.page_table[static_cast<uint64_t>(s) * a.table_pages + t / page_size];
            if (page < 0 || static_cast<uint32_t>(page) >= a.cache.pages) continue;
            const uint32_t slot = static_cast<uint32_t>(t % page_size);
            const uint64_t plane = static_cast<uint64_t>(page) * a.cache.kv_heads + h;
            const E* row = x + static_cast<uint64_t>(q.begin + (t - origin)) * stride;
            float v0 = 0.0f, v1 = 0.0f;  // features 2 lane, 2 lane + 1
            if (2 * lane < d) {
                v0 = static_cast<float>(row[2 * lane]);
                v1 = static_cast<float>(row[2 * lane + 1]);
            }
            uint32_t bits = max(__float_as_uint(fabsf(v0)), __float_as_uint(fabsf(v1)));  // NaN above all
            for (int o = 32; o > 0; o >>= 1)
                bits = max(bits, static_cast<uint32_t>(__shfl_xor(static_cast<int>(bits), o, kWave)));
            bits = max(__float_as_uint(div_rn(__uint_as_float(bits), 7.0f)), __float_as_uint(1.0e-8f));
            const float scale = __uint_as_float(bits), inverse = div_rn(1.0f, scale);
            if (lane == 0) (side ? a.cache.value_scales : a.cache.key_scales)[plane * page_size + slot] = scale;
            if (2 * lane >= d) continue;
            const uint32_t c0 = nibble(v0, scale, inverse), c1 = nibble(v1, scale, inverse);
            uint8_t* at = (side ? a.cache.values : a.cache.keys) + plane * (page_size / 2u) * d;
            if (side == 0) {
                at[slot * (d / 2u) + lane] = static_cast<uint8_t>(c0 | (c1 << 4));
            } else {
                at += (slot / 16u) * 8u * d + 16u * lane + (slot % 16u) / 2u;
                const uint32_t shift = 4u * (slot & 1u), keep = 0xf0u >> shift;
                at[0] = static_cast<uint8_t>((at[0] & keep) | (c0 << shift));
                at[8] = static_cast<uint8_t>((at[8] & keep) | (c1 << shift));
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Attention over the cache: the products, weights and bases of cache_i8.hip,
// with scales of keys. A score is (q c) times its key's scale, in fp32; a
// value's scale 2^e f goes with the weight of its key: t = s log2(e) + e, w =
// exp2(t - base), O = sum (w f) c, L = sum w 2^-e.

// Eight codes as binary16, the half bytes i and i + 4 side by side: 0, 4, 1, 5,
// 2, 6, 3, 7. A half byte x below the exponent of 1024 is the number 1024 + x,
// four bits further up 1024 + 16 x: x - 8 by one operation each, exactly.
DAV2_DEV h8 widen4(uint32_t w) {
    const h2 down = {static_cast<_Float16>(1032.0f), static_cast<_Float16>(1032.0f)};
    const h2 share = {static_cast<_Float16>(0.0625f), static_cast<_Float16>(0.0625f)};
    const h2 down16 = {static_cast<_Float16>(-72.0f), static_cast<_Float16>(-72.0f)};
    const uint32_t u = w >> 8;
    const h2 a = __builtin_bit_cast(h2, (w & 0x000f000fu) | 0x64006400u) - down;
    const h2 b = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & 0x00f000f0u) | 0x64006400u), share, down16);
    const h2 c = __builtin_bit_cast(h2, (u & 0x000f000fu) | 0x64006400u) - down;
    const h2 d = __builtin_elementwise_fma(__builtin_bit_cast(h2, (u & 0x00f000f0u) | 0x64006400u), share, down16);
    return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
// which of eight the i-th of widen4 is
constexpr int widened(int i) { return (i >> 1) + 4 * (i & 1); }

DAV2_DEV Parts parts_of(const dav2_attention_cache_i4_args& a, uint32_t splits) {
    return parts_at(a.scratch, static_cast<uint64_t>(a.tokens) * a.heads * splits);
}

// Few query rows for a cache head: the split of the work, the tiles and the
// joins of cache_rows_kernel in cache_i8.hip.
//
// Lane l = (col, g) = (l % 16, l / 16) takes F features F g .. of its key for
// the first product (those past the head's width are others, that meet zeros
// of the query), and chunk g's 16 keys of two neighbouring features for the
// second, which so are the even and the odd rows of two tiles.
template <typename E, int D>
__global__ __launch_bounds__(256, 2) void cache4_rows_kernel(dav2_attention_cache_i4_args a, uint32_t splits,
                                                             uint32_t tiles) {
    constexpr bool kFloat = std::is_same_v<E, float>;
    constexpr int F = D > 64 ? 32 : 16, KS = F / 8, FT = D / 16, FP = FT / 2, NP = kFloat ? 2 : 1;
    constexpr uint32_t d = D;
    constexpr int kPad = 17;
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
    const uint32_t rows = n * group;
    const int64_t span = static_cast<int64_t>(a.table_pages) * page_size;
    const Pages pages = pages_of(a, s);
    const Parts parts = parts_of(a, splits);

    for (uint32_t tile = blockIdx.x / splits; tile < (rows + 15u) / 16u; tile += tiles) {
        const Rows<16> of(tile * 16u, group, rows);
        const uint32_t row = tile * 16u + col;
        uint32_t token, head;
        of.find(col, token, head);
        head += h * group;
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
        float maximum = kNoScore, base = kNoScore, sum = 0.0f;

        uint32_t kraw[4][F / 8];
        u4_t vraw[FP > 0 ? FP : 1];
        u2_t vlast{};  // of the last 16 features, where their number is odd
        v4f key_scale[4], value_scale[4];
        Pages::Place of_key{}, of_value{};
        bool exists = false;
        const uint32_t f0 = min(F * g, d - F);  // this lane's features
        auto find = [&](uint32_t block) {
            of_key = pages.find(block * 4u + col / 4u);
            of_value = pages.find(block * 4u + g);
        };
        auto load_keys = [&] {
            const uint8_t* k = a.cache.keys + ((static_cast<uint64_t>(pages.page(of_key)) * kv_heads + h) * page_size +
                                               of_key.slot + col % 4u) * (d / 2u) + f0 / 2u;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if constexpr (F == 32) {
                    const u4_by8 v = *reinterpret_cast<const u4_by8*>(k + 4u * t * (d / 2u));
#pragma unroll
                    for (int i = 0; i < 4; ++i) kraw[t][i] = v[i];
                } else {
                    const u2_t v = *reinterpret_cast<const u2_t*>(k + 4u * t * (d / 2u));
                    kraw[t][0] = v[0], kraw[t][1] = v[1];
                }
            }
        };
        auto load_values = [&] {
            exists = pages.exists(of_value);
            const uint64_t at = (static_cast<uint64_t>(pages.page(of_value)) * kv_heads + h) * page_size + of_value.slot;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                key_scale[t] = *reinterpret_cast<const v4f_any*>(a.cache.key_scales + at + 4 * t);
                value_scale[t] = *reinterpret_cast<const v4f_any*>(a.cache.value_scales + at + 4 * t);
            }
            const uint8_t* v = a.cache.values + at * (d / 2u);
#pragma unroll
            for (int f = 0; f < FP; ++f) vraw[f] = *reinterpret_cast<const u4_t*>(v + 256u * f + 16u * col);
            if constexpr (FT % 2) vlast = *reinterpret_cast<const u2_t*>(v + 256u * FP + 8u * col);
        };
        uint32_t block = first + wave;
        if (block < last) {
            find(block);
            load_keys();
            load_values();
            find(min(block + 4u, last - 1u));
        }

        h8 qf[NP][KS];
        float factor;
        {
            const E* x = static_cast<const E*>(a.query) + static_cast<uint64_t>(q.begin + token) * a.query_stride +
                         static_cast<uint64_t>(head) * d + f0;
            typedef E V __attribute__((ext_vector_type(16 / sizeof(E))));
            constexpr int kVec = 16 / sizeof(E);
            float v[F];
            float largest = 0.0f;
#pragma unroll
            for (int j = 0; j < F / kVec; ++j) {
                const V piece = *reinterpret_cast<const V*>(x + kVec * j);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    // another lane has those before F g
                    v[kVec * j + i] = f0 + kVec * j + i >= F * g ? static_cast<float>(piece[i]) : 0.0f;
                    largest = fmaxf(largest, fabsf(v[kVec * j + i]));
                }
            }
            largest = over_groups(largest, Larger());
            const int e = largest > 0.0f && largest < INFINITY ? 14 - ilogbf(largest) : 0;
            const float sign = a.scale < 0.0f ? -1.0f : 1.0f;
            factor = ldexpf(fabsf(a.scale) * kLog2e, -e);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = keep_fp32(ldexpf(v[8 * k + widened(i)], e) * sign);
                    const _Float16 hi = static_cast<_Float16>(y);
                    qf[0][k][i] = hi;
                    if constexpr (kFloat) qf[1][k][i] = static_cast<_Float16>(y - static_cast<float>(hi));
                }
        }

        auto step = [&](auto more) {
            constexpr bool kMore = decltype(more)::value;
            v4f sc[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                sc[t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    const h8 key = widen4(kraw[t][k]);
#pragma unroll
                    for (int p = 0; p < NP; ++p)
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(key, qf[p][k], sc[t], 0, 0, 0);
                }
            }
            if constexpr (kMore) load_keys();
            const uint32_t key0 = block * 64u + 16u * g;  // of this lane's first score
            const bool whole = (block + 1u) * 64u <= least && __all(exists);
            float fraction[4][4], inverse[4][4];
            float largest = kNoScore;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool here = whole || (exists && key0 + 4 * t + r < limit);
                    float exponent;
                    // a token that the row does not see may have any scale, NaN included
                    split_scale(here ? value_scale[t][r] : 1.0f, exponent, fraction[t][r], inverse[t][r]);
                    const float x = fmaf(sc[t][r], key_scale[t][r] * factor, exponent);
                    sc[t][r] = here ? x : -INFINITY;
                    largest = fmaxf(largest, sc[t][r]);
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
            h8 pf[2][2];
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float w = __builtin_amdgcn_exp2f(sc[t][r] - base);
                    sum = fmaf(w, inverse[t][r], sum);
                    const float y = keep_fp32(w * fraction[t][r]);  // hi and lo of one rounded product
                    const _Float16 hi = static_cast<_Float16>(y);
                    // key 4 t + r of the chunk, in the order of widen4
                    pf[0][t >> 1][2 * r + (t & 1)] = hi;
                    pf[1][t >> 1][2 * r + (t & 1)] = static_cast<_Float16>((y - static_cast<float>(hi)) * kSecond);
                }
            auto add = [&](v4f& sums, uint32_t lo, uint32_t hi) {
                const h8 v0 = widen4(lo), v1 = widen4(hi);
                sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[0][0], sums, 0, 0, 0);
                sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[0][1], sums, 0, 0, 0);
                sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(for_second(v0), pf[1][0], sums, 0, 0, 0);
                sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(for_second(v1), pf[1][1], sums, 0, 0, 0);
            };
#pragma unroll
            for (int f = 0; f < FP; ++f) {
                add(o[2 * f], vraw[f][0], vraw[f][1]);
                add(o[2 * f + 1], vraw[f][2], vraw[f][3]);
            }
            if constexpr (FT % 2) add(o[FT - 1], vlast[0], vlast[1]);
            if constexpr (kMore) {
                load_values();
                find(min(block + 8u, last - 1u));
            }
        };
        for (; block + 4u < last; block += 4u) step(std::true_type());
        if (block < last) step(std::false_type());
        sum = over_groups(sum, Plus());

        // join the four waves
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
            for (int r = 0; r < 4; ++r) {
                // register r of o[f]: row 4 g + r of tile f
                const uint32_t i = 4 * g + r;
                const uint32_t feature = f < 2 * FP ? 32u * (f / 2) + 2u * i + f % 2 : 16u * f + i;
                joined[wave][feature * kPad + col] = o[f][r] * mine;
            }
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

// The splits of the sequences' rows joined.
template <typename E, int FEW>
__global__ __launch_bounds__(256) void cache4_join_kernel(dav2_attention_cache_i4_args a, uint32_t splits) {
    join_sequence<E, FEW>(a, parts_of(a, splits), splits);
}

bool valid(const dav2_cache_i4& c) { return valid_pages(c); }

bool valid(const dav2_attention_cache_i4_args& a) {
    const uint64_t row = static_cast<uint64_t>(a.heads) * a.cache.head_dim;
    return valid(a.cache) && a.query && a.output && aligned16(a.query) && aligned16(a.output) && a.page_table &&
           a.starts && a.lengths && a.dtype <= DAV2_DTYPE_BF16 && a.sequences <= 65535u && a.tokens <= 0x7fffffffu &&
           a.table_pages > 0 && a.table_pages <= 0x7fffffffu && a.heads > 0 && a.heads <= 65535u &&
           a.heads % a.cache.kv_heads == 0 && static_cast<uint64_t>(a.tokens) * a.heads <= 0xfffffe00ull &&
           static_cast<uint64_t>(a.sequences) * a.cache.kv_heads <= 0x7fffffull &&
           a.query_stride % 8 == 0 && a.output_stride % 8 == 0 &&
           (a.tokens == 1 || (a.query_stride >= row && a.output_stride >= row));
}

struct Plan {
    uint32_t tile;  // rows of a workgroup
    uint32_t tiles, splits;
};
Plan plan_of(const dav2_attention_cache_i4_args& a) {
    Plan p{16, 1, 1};
    if (a.cache.kv_heads == 0 || a.heads < a.cache.kv_heads || a.sequences == 0 || a.max_query == 0) return p;
    const uint64_t rows = static_cast<uint64_t>(std::min(a.max_query, a.tokens)) * (a.heads / a.cache.kv_heads);
    const uint64_t planes = static_cast<uint64_t>(a.cache.kv_heads) * a.sequences;
    p.tiles = static_cast<uint32_t>(std::min<uint64_t>((rows + 15) / 16, 4096));
    const uint64_t have = std::max<uint64_t>(1, p.tiles * planes);
    const uint64_t resident = std::min<uint64_t>(512 / have, a.max_length / 128);
    const uint64_t even = std::min<uint64_t>(2048 / have, a.max_length / 2048);
    p.splits = static_cast<uint32_t>(std::clamp<uint64_t>(std::max(resident, even), 1, kMostSplits));
    return p;
}

}  // namespace

extern "C" {

int dav2_hip_cache_store_i4(const dav2_cache_store_i4_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_cache_store_i4_args& a = *args;
    if (a.sequences == 0 || a.tokens == 0 || a.max_new == 0) return hipSuccess;
    const uint64_t row = static_cast<uint64_t>(a.cache.kv_heads) * a.cache.head_dim;
    if (!valid(a.cache) || !a.keys || !a.values || !a.page_table || !a.starts || !a.lengths ||
        a.dtype > DAV2_DTYPE_BF16 || a.sequences > 65535u || a.tokens > 0x7fffffffu || a.table_pages == 0 ||
        a.table_pages > 0x7fffffffu || (a.tokens > 1 && (a.key_stride < row || a.value_stride < row)))
        return hipErrorInvalidValue;
    const uint64_t new_most = std::min(a.max_new, a.tokens);
    const uint64_t pairs = new_most / 2 + 1;
    constexpr uint64_t kMostGroups = 1u << 22;  // workgroups along x: threads of a launch stay below 2^32
    const dim3 grid(static_cast<uint32_t>(std::min<uint64_t>((pairs + 3) / 4, kMostGroups)), 2 * a.cache.kv_heads, a.sequences);
    with_dtype(a.dtype, [&](auto* e) {
        typedef std::remove_pointer_t<decltype(e)> E;
        dispatch(cache4_scale_kernel<E>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
    });
    return hipGetLastError();
}

uint64_t dav2_hip_attention_cache_i4_scratch_bytes(const dav2_attention_cache_i4_args* args) {
    if (!args) return 0;
    const dav2_attention_cache_i4_args& a = *args;
    const Plan p = plan_of(a);
    if (p.splits == 1) return 0;
    return parts_bytes(static_cast<uint64_t>(a.tokens) * a.heads * p.splits, a.cache.head_dim);
}

int dav2_hip_attention_cache_i4(const dav2_attention_cache_i4_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_attention_cache_i4_args& a = *args;
    if (a.sequences == 0 || a.tokens == 0 || a.max_query == 0) return hipSuccess;
    if (!valid(a)) return hipErrorInvalidValue;
    const uint64_t need = dav2_hip_attention_cache_i4_scratch_bytes(args);
    if (need && (!a.scratch || !aligned16(a.scratch) || a.scratch_bytes < need)) return hipErrorInvalidValue;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const Plan p = plan_of(a);
    const dim3 grid(p.tiles * p.splits, a.cache.kv_heads, a.sequences);
    return with_dtype(a.dtype, [&](auto* e) -> int {
        typedef std::remove_pointer_t<decltype(e)> E;
        with_head_dim(a.cache.head_dim, [&](auto dim) {
            constexpr int D = decltype(dim)::value;
            dispatch(cache4_rows_kernel<E, D>, grid, dim3(256), 0, s, a, p.splits, p.tiles);
        });
        if (p.splits > 1) {
            const JoinLaunch j = join_launch(a, p.splits);
            dispatch(j.few == 4   ? cache4_join_kernel<E, 4>
                     : j.few == 8 ? cache4_join_kernel<E, 8>
                                  : cache4_join_kernel<E, 0>,
                     j.grid, dim3(256), 0, s, a, p.splits);
        }
        return hipGetLastError();
    });
}

}  // extern "C"
