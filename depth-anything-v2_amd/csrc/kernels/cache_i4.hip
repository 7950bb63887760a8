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

// vectors, `any` and `by` at addresses that are multiples of less
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v2f_any __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u4_by8 __attribute__((ext_vector_type(4), aligned(8)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));

// Eight codes as they are held, one to a half byte: x / scale rounded, of which
// x * inverse is within 7 (2^-23 + 2^-24 + 2^-47) < 2^-19. Where that is as near
// to a border, which is rare, the quotients themselves decide. Adding 1.5 * 2^23
// rounds to a whole number, and 8 more are the code in its low bits.
DAV2_DEV uint32_t half_bytes(const float (&x)[8], float scale, float inverse) {
    constexpr float kRound = 0x1.8p23f;
    float y[8];
    bool border = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = x[i] * inverse;
        border |= fabsf(y[i] - ((y[i] + kRound) - kRound)) > 0.5f - 0x1p-18f;
    }
    if (__builtin_expect(border, 0))
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = div_rn(x[i], scale);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // no number is 0; |y| is at most 7 (1 + 2^-23)
        const float whole = (y[i] == y[i] ? y[i] : 0.0f) + (kRound + 8.0f);
        word |= (__float_as_uint(whole) & 15u) << (4 * i);
    }
    return word;
}

// The largest over 16 neighbouring lanes, received by all of them.
template <int CTRL>
DAV2_DEV uint32_t larger(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, true)));
}
DAV2_DEV uint32_t largest_of_16(uint32_t v) {
    v = larger<0x121>(v);  // row_ror:1, 2, 4, 8
    v = larger<0x122>(v);
    v = larger<0x124>(v);
    return larger<0x128>(v);
}

// A wave for each chunk of 16 tokens, head and side. Lane (t, f) = (l / 16, l %
// 16) has features 8 f .. of the tokens t, t + 4, t + 8 and t + 12. A key's eight
// codes are a word as they stand. Values are held the other way round: each lane
// puts its codes where its tokens are in the eight bytes of their features, and
// the four lanes of a feature join theirs, each ending with two of the eight
// features and one store. A chunk that has older or later tokens too is read,
// changed and written back; nobody else writes it. Bound by memory and by the
// rounding: 8 prompts of up to 2048 tokens, 8 heads of 128, f16 (46 MB), 19 us,
// 2.4 TB/s (41 with a workgroup for a page that reads its rows twice); a token
// for each of 64 sequences 4.0 us, the call.
template <typename E>
__global__ __launch_bounds__(256) void cache4_store_kernel(dav2_cache_store_i4_args a) {
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t kv_heads = a.cache.kv_heads, page_size = a.cache.page_size, d = a.cache.head_dim;
    const uint32_t plane_of = blockIdx.y * 4u + wave, side = plane_of >= kv_heads, h = plane_of - side * kv_heads;
    if (plane_of >= 2u * kv_heads) return;
    const uint32_t s = blockIdx.z, t0 = lane >> 4, f = lane & 15u;
    const Sequence q = sequence_of(a.starts, a.lengths, s, a.tokens);
    // positions [first, last) are new; in 64 bits, as a length may be anything
    const int64_t origin = static_cast<int64_t>(q.length) - (q.end - q.begin);  // row r has position origin + r - begin
    const int64_t first = max(origin, int64_t(0));
    const int64_t last = min(static_cast<int64_t>(q.length), static_cast<int64_t>(a.table_pages) * page_size);
    // nothing new: the chunk that the next token goes to is left alone, it may be another sequence's by now
    if (first >= last) return;
    const uint64_t stride = side ? a.value_stride : a.key_stride;
    const E* x = static_cast<const E*>(side ? a.values : a.keys) + static_cast<uint64_t>(h) * d + 8u * f;
    const bool feature = 8u * f < d;
    for (int64_t chunk = first / 16 + blockIdx.x; chunk * 16 < last; chunk += gridDim.x) {
        const int64_t base = chunk * 16;
        const int32_t page = a.page_table[static_cast<uint64_t>(s) * a.table_pages + base / page_size];
        if (page < 0 || static_cast<uint32_t>(page) >= a.cache.pages) continue;  // the same for the wave
        const uint32_t slot0 = static_cast<uint32_t>(base % page_size);
        const uint32_t from = static_cast<uint32_t>(max(first - base, int64_t(0)));
        const uint32_t to = static_cast<uint32_t>(min(last - base, int64_t(16)));
        const uint64_t at = (static_cast<uint64_t>(page) * kv_heads + h) * page_size + slot0;  // of the chunk's first token
        float v[4][8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t t = t0 + 4 * i;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
            if (feature && t >= from && t < to) {
                const E* row = x + (q.begin + (base + t - origin)) * static_cast<int64_t>(stride);
#pragma unroll
                for (int j = 0; j < 8; j += Vec<E>::N) {
                    float part[Vec<E>::N];
                    Vec<E>::load(row, j, 8u, part);
#pragma unroll
                    for (int k = 0; k < Vec<E>::N; ++k) v[i][j + k] = part[k];
                }
            }
        }
        uint32_t codes[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            codes[i] = 0;
            if (to <= 4u * i || from >= 4u * i + 4u) continue;  // the same for the wave
            uint32_t bits = 0;  // NaN above all
#pragma unroll
            for (int j = 0; j < 8; ++j) bits = max(bits, __float_as_uint(fabsf(v[i][j])));
            bits = largest_of_16(bits);
            bits = max(__float_as_uint(div_rn(__uint_as_float(bits), 7.0f)), __float_as_uint(1.0e-8f));
            const float scale = __uint_as_float(bits);
            codes[i] = half_bytes(v[i], scale, div_rn(1.0f, scale));
            const uint32_t t = t0 + 4 * i;
            if (f == 0 && t >= from && t < to) (side ? a.cache.value_scales : a.cache.key_scales)[at + t] = scale;
        }
        if (side == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t t = t0 + 4 * i;
                if (feature && t >= from && t < to)
                    *reinterpret_cast<uint32_t*>(a.cache.keys + (at + t) * (d / 2u) + 4u * f) = codes[i];
            }
            continue;
        }
        // words 2 j and 2 j + 1: tokens 0-7 and 8-15 of feature j
        uint32_t words[16];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t a0 = (codes[2 * half] >> (4 * j)) & 15u, a1 = (codes[2 * half + 1] >> (4 * j)) & 15u;
                words[2 * j + half] = (a0 | (a1 << 16)) << (4u * t0);
            }
        // lanes of the upper half end with the upper half of the words, and so on
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const auto p = __builtin_amdgcn_permlane32_swap(words[j], words[j + 8], false, false);
            words[j] = p[0] | p[1];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const auto p = __builtin_amdgcn_permlane16_swap(words[j], words[j + 4], false, false);
            words[j] = p[0] | p[1];
        }
        // features 8 f + 4 (t0 / 2) + 2 (t0 % 2) and the next
        if (!feature) continue;
        u4_t out = {words[0], words[1], words[2], words[3]};
        u4_t* const place = reinterpret_cast<u4_t*>(a.cache.values + at * (d / 2u) + 8u * (8u * f + 2u * t0));
        if (to - from < 16u) {
            const uint64_t mask = ((to < 16u ? 1ull << (4u * to) : 0ull) - (1ull << (4u * from)));
            const uint32_t lo = static_cast<uint32_t>(mask), hi = static_cast<uint32_t>(mask >> 32);
            const u4_t masks = {lo, hi, lo, hi};
            out = (out & masks) | (*place & ~masks);
        }
        *place = out;
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
    // one operation with the constants in registers, which the compiler makes two
    auto below = [](uint32_t x, uint32_t mask) {
        uint32_t y;
        asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(y) : "v"(x), "s"(mask), "v"(0x64006400u));
        return __builtin_bit_cast(h2, y);
    };
    const h2 a = below(w, 0x000f000fu) - down;
    const h2 b = __builtin_elementwise_fma(below(w, 0x00f000f0u), share, down16);
    const h2 c = below(u, 0x000f000fu) - down;
    const h2 d = __builtin_elementwise_fma(below(u, 0x00f000f0u), share, down16);
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
// second, which so are the even and the odd rows of two tiles. Register r of
// score tile t is key_of(t, r) of chunk g, so that a tile's four scores are two
// words of the second product's right operand, in the order of widen4.
//
// A tile has COLS rows of 16 columns. With 4 or 8 the columns behind them would
// have their scores weighed for nothing: the tiles' scores are spread over them
// first, T tiles for each lane, and the weights gathered again. Bound by memory
// where the cache is long: 32 sequences of up to 32768 tokens, 32 heads of 8, 128
// features, bf16 (651 MB) 143 us, 4.6 TB/s, in 4 columns; 179 in 16.
DAV2_DEV constexpr uint32_t key_of(uint32_t t, uint32_t r) { return 8u * (t >> 1) + 2u * (t & 1u) + (r >> 1) + 4u * (r & 1u); }

// Lanes of the banks (of four lanes) in BANKS: x of the lane that CTRL names; the others keep `old`.
template <int CTRL, int BANKS>
DAV2_DEV float moved(float old, float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(x), CTRL, 0xf, BANKS, false));
}
constexpr int kShl4 = 0x104, kShl8 = 0x108, kShl12 = 0x10c, kShr4 = 0x114, kShr8 = 0x118, kShr12 = 0x11c, kRor4 = 0x124,
              kRor8 = 0x128;

// op over the lanes of a query, COLS apart and in all groups.
template <int COLS, typename Op>
DAV2_DEV float over_query(float v, Op op) {
    if constexpr (COLS == 4) v = op(v, moved<kRor4, 0xf>(v, v));
    if constexpr (COLS <= 8) v = op(v, moved<kRor8, 0xf>(v, v));
    return over_groups(v, op);
}

template <typename E, int D, int COLS>
__global__ __launch_bounds__(256, 2) void cache4_rows_kernel(dav2_attention_cache_i4_args a, uint32_t splits,
                                                             uint32_t tiles) {
    constexpr bool kFloat = std::is_same_v<E, float>;
    constexpr int F = D > 64 ? 32 : 16, KS = F / 8, FT = D / 16, FP = FT / 2, NP = kFloat ? 2 : 1;
    constexpr int T = COLS / 4;  // score tiles that a lane weighs
    // The second parts' sums in registers of their own save the multiplications
    // of the codes (see for_second), where that does not cost a wave: 64
    // sequences of up to 2048 keys, 8 heads of 128, 25 for 27 us; 16 heads of 64, fp32, 32.5 for 28.
    constexpr bool kApart = D > 64;
    constexpr uint32_t d = D;
    constexpr int kPad = COLS + 1;
    constexpr float kBias = 14.0f;  // a weight times a fraction stays below 2^15
    __shared__ float joined[4][D * kPad];
    __shared__ float shared_base[4][COLS], shared_sum[4][COLS];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t col = lane & 15u, g = lane >> 4, t0 = T * (col / COLS);  // the lane's first tile
    const uint32_t split = blockIdx.x % splits, h = blockIdx.y, s = blockIdx.z;
    const uint32_t page_size = a.cache.page_size, kv_heads = a.cache.kv_heads;
    const uint32_t group = a.heads / kv_heads;
    const Sequence q = sequence_of(a.starts, a.lengths, s, a.tokens);
    const uint32_t n = static_cast<uint32_t>(q.end - q.begin);
    const uint32_t rows = n * group;
    const int64_t span = static_cast<int64_t>(a.table_pages) * page_size;
    const Pages pages = pages_of(a, s);
    const Parts parts = parts_of(a, splits);

    for (uint32_t tile = blockIdx.x / splits; tile < (rows + COLS - 1u) / COLS; tile += tiles) {
        const Rows<COLS> of(tile * COLS, group, rows);
        const uint32_t row = tile * COLS + col % COLS;
        uint32_t token, head;
        of.find(col % COLS, token, head);
        head += h * group;
        auto seen = [&](uint32_t i) {
            int64_t t = q.length;
            if (a.causal) t += 1 + static_cast<int64_t>(i) - n;
            return static_cast<uint32_t>(max(min(t, span), int64_t(0)));
        };
        const uint32_t limit = row < rows ? seen(token) : 0u;
        uint32_t last_token, last_head;
        of.find(COLS - 1u, last_token, last_head);
        const uint32_t most = seen(last_token), least = seen(of.token);
        const uint32_t blocks = (most + 63u) / 64u, per = (blocks + splits - 1u) / splits;
        const uint32_t first = split * per, last = min(first + per, blocks);

        v4f o[FT], o2[kApart ? FT : 1];  // of the weights' first and second parts
#pragma unroll
        for (int f = 0; f < FT; ++f) o[f] = o2[kApart ? f : 0] = v4f{0.f, 0.f, 0.f, 0.f};
        float maximum = kNoScore, base = kNoScore, sum = 0.0f;

        uint32_t kraw[4][F / 8];
        u4_t vraw[FP > 0 ? FP : 1];
        u2_t vlast{};  // of the last 16 features, where their number is odd
        v4f key_scale[T], value_scale[T];
        Pages::Place of_key{}, of_value{};
        bool exists = false;
        const uint32_t f0 = min(F * g, d - F);  // this lane's features
        auto find = [&](uint32_t block) {
            of_key = pages.find(block * 4u + col / 4u);
            of_value = pages.find(block * 4u + g);
        };
        auto load_keys = [&] {
            const uint8_t* k = a.cache.keys + ((static_cast<uint64_t>(pages.page(of_key)) * kv_heads + h) * page_size +
                                               of_key.slot + key_of(0, col % 4u)) * (d / 2u) + f0 / 2u;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if constexpr (F == 32) {
                    const u4_by8 v = *reinterpret_cast<const u4_by8*>(k + key_of(t, 0) * (d / 2u));
#pragma unroll
                    for (int i = 0; i < 4; ++i) kraw[t][i] = v[i];
                } else {
                    const u2_t v = *reinterpret_cast<const u2_t*>(k + key_of(t, 0) * (d / 2u));
                    kraw[t][0] = v[0], kraw[t][1] = v[1];
                }
            }
        };
        auto load_values = [&] {
            exists = pages.exists(of_value);
            const uint64_t at = (static_cast<uint64_t>(pages.page(of_value)) * kv_heads + h) * page_size + of_value.slot;
            auto four = [&](const float* x) {
                const v2f_any lo = *reinterpret_cast<const v2f_any*>(x), hi = *reinterpret_cast<const v2f_any*>(x + 4);
                return v4f{lo[0], hi[0], lo[1], hi[1]};
            };
#pragma unroll
            for (int t = 0; t < T; ++t) {
                key_scale[t] = four(a.cache.key_scales + at + key_of(t0 + t, 0));
                value_scale[t] = four(a.cache.value_scales + at + key_of(t0 + t, 0));
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
            v4f x[T];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (COLS == 16) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) x[t][r] = sc[t][r];
                } else if constexpr (COLS == 8) {
                    x[0][r] = moved<kShr8, 0xc>(sc[0][r], sc[2][r]);
                    x[1][r] = moved<kShr8, 0xc>(sc[1][r], sc[3][r]);
                } else {
                    x[0][r] = moved<kShr4, 0x2>(sc[0][r], sc[1][r]);
                    x[0][r] = moved<kShr8, 0x4>(x[0][r], sc[2][r]);
                    x[0][r] = moved<kShr12, 0x8>(x[0][r], sc[3][r]);
                }
            }
            const uint32_t key0 = block * 64u + 16u * g;  // of this lane's chunk
            const bool whole = (block + 1u) * 64u <= least && __all(exists);
            float fraction[T][4], inverse[T][4];
            float largest = kNoScore;
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool here = whole || (exists && key0 + key_of(t0 + t, r) < limit);
                    float exponent;
                    // a token that the row does not see may have any scale, NaN included
                    split_scale(here ? value_scale[t][r] : 1.0f, exponent, fraction[t][r], inverse[t][r]);
                    const float y = fmaf(x[t][r], key_scale[t][r] * factor, exponent);
                    x[t][r] = here ? y : -INFINITY;
                    largest = fmaxf(largest, x[t][r]);
                }
            largest = over_query<COLS>(largest, Larger());
            if (__any(largest > maximum)) {
                maximum = fmaxf(maximum, largest);
                const float moved_base = fabsf(maximum) < kFar ? maximum - kBias : maximum;
                const float keep = __builtin_amdgcn_exp2f(base - moved_base);
                base = moved_base;
                sum *= keep;
#pragma unroll
                for (int f = 0; f < FT; ++f) {
                    o[f] *= keep;
                    if constexpr (kApart) o2[f] *= keep;
                }
            }
            // weights, the first parts and the rest of them, as words of the right operand
            float words[T][2][2];
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    h2 hi, lo;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float w = __builtin_amdgcn_exp2f(x[t][r + i] - base);
                        sum = fmaf(w, inverse[t][r + i], sum);
                        const float y = keep_fp32(w * fraction[t][r + i]);  // hi and lo of one rounded product
                        hi[i] = static_cast<_Float16>(y);
                        lo[i] = static_cast<_Float16>((y - static_cast<float>(hi[i])) * kSecond);
                    }
                    words[t][0][r / 2] = __builtin_bit_cast(float, hi);
                    words[t][1][r / 2] = __builtin_bit_cast(float, lo);
                }
            h8 pf[2][2];  // part, half of the chunk
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                v4f half[2];
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        // tile t is with the lane COLS (t / T) further
                        const float own = words[t % T][p][i];
                        constexpr int kNone = 0;
                        const float from = COLS == 16 || t / T == kNone ? own
                                           : COLS == 8 || t / T == 2    ? moved<kShl8, 0xf>(0.0f, own)
                                           : t / T == 1                 ? moved<kShl4, 0xf>(0.0f, own)
                                                                        : moved<kShl12, 0xf>(0.0f, own);
                        half[t >> 1][2 * (t & 1) + i] = from;
                    }
                pf[p][0] = __builtin_bit_cast(h8, half[0]);
                pf[p][1] = __builtin_bit_cast(h8, half[1]);
            }
            auto add = [&](int f, uint32_t lo, uint32_t hi) {
                const h8 v0 = widen4(lo), v1 = widen4(hi);
                v4f& second = kApart ? o2[kApart ? f : 0] : o[f];
                o[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[0][0], o[f], 0, 0, 0);
                second = __builtin_amdgcn_mfma_f32_16x16x32_f16(kApart ? v0 : for_second(v0), pf[1][0], second, 0, 0, 0);
                o[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[0][1], o[f], 0, 0, 0);
                second = __builtin_amdgcn_mfma_f32_16x16x32_f16(kApart ? v1 : for_second(v1), pf[1][1], second, 0, 0, 0);
            };
#pragma unroll
            for (int f = 0; f < FP; ++f) {
                add(2 * f, vraw[f][0], vraw[f][1]);
                add(2 * f + 1, vraw[f][2], vraw[f][3]);
            }
            if constexpr (FT % 2) add(FT - 1, vlast[0], vlast[1]);
            if constexpr (kMore) {
                load_values();
                find(min(block + 8u, last - 1u));
            }
        };
        for (; block + 4u < last; block += 4u) step(std::true_type());
        if (block < last) step(std::false_type());
        sum = over_query<COLS>(sum, Plus());

        // join the four waves
        __syncthreads();  // the tile before has been read
        if (g == 0 && col < COLS) {
            shared_base[wave][col] = base;
            shared_sum[wave][col] = sum;
        }
        __syncthreads();
        float top = kNoScore;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, shared_base[w][col % COLS]);
        const float mine = __builtin_amdgcn_exp2f(base - top);
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                // register r of o[f]: row 4 g + r of tile f
                const uint32_t i = 4 * g + r;
                const uint32_t feature = f < 2 * FP ? 32u * (f / 2) + 2u * i + f % 2 : 16u * f + i;
                if (col < COLS) joined[wave][feature * kPad + col] = (kApart ? fmaf(o2[kApart ? f : 0][r], 1.0f / kSecond, o[f][r]) : o[f][r]) * mine;
            }
        __syncthreads();
        // the threads shared out to the rows
        constexpr uint32_t kShare = 256 / COLS;
        const uint32_t out_col = threadIdx.x / kShare, out_lane = threadIdx.x % kShare;
        if (tile * COLS + out_col < rows) {
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
            for (uint32_t f = out_lane; f < d; f += kShare) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) v += joined[w][f * kPad + out_col];
                if (splits > 1) parts.sums[slot * d + f] = v;
                else y[f] = static_cast<E>(v * scale);
            }
            if (splits > 1 && out_lane == 0) parts.stats[slot] = make_float2(all, total);
        }
    }
}

// Many query rows for a cache head (prompts): the tiles, the order of the work
// and the split of cache_tiles_kernel in cache_i8.hip, with scales of keys: four
// numbers in LDS for each key of a tile, read four keys at a time.
//
// Codes are widened once for all waves: a key's words of eight features in the
// order of widen4, which the query's features are put in too; the tokens 0-3 and
// 8-11 of a chunk, then 4-7 and 12-15, which are what a lane holds scores of.
// A weight is one binary16 number for bf16, whose rounding of the output hides
// 2^-12. For f16 it added as much error as that rounding does (2.7e-4 of the
// output against 64 bits, where a 32-bit softmax has 2.1e-4): two parts, 2^-22 of
// a weight and 2^-38 of the largest at most. The rest needs no factor as in
// for_second: it loses what a single part loses.
//
// Bound by vector units and matrix cores, partly beside one another, and by the
// clock that falls under both: 2 prompts of 2048 tokens at the end of 8192, 32
// heads of 8, 128 features (316 GFLOP), bf16 561 us, 563 TFLOP/s (vector units 53 %
// busy, LDS 39 %, of whose 56 reads of a wave and tile 24 are scales, matrix cores
// 34 %); f16, with half as many products again, 641. With one part for f16: 566,
// 1125 with a scale read for each score, 723 with 64 rows a wave.
template <typename E, int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES, D <= 64 && sizeof(E) == 2 ? 3 : 2)
void cache4_tiles_kernel(dav2_attention_cache_i4_args a, uint32_t splits, uint32_t tiles) {
    constexpr bool kFloat = std::is_same_v<E, float>;
    constexpr int HEAD = D <= 64 ? 64 : 128;  // features of a row in LDS
    constexpr int KS = D / 16, FB = (D + 31) / 32, NP = kFloat ? 2 : 1;
    constexpr int WP = std::is_same_v<E, __bf16> ? 1 : 2;  // parts of a weight
    constexpr bool kPairs = WP == 2 && !kFloat;
    constexpr int kSteps = kFloat ? FB : WP * FB;          // of the second product, for 16 keys
    constexpr uint32_t d = D;
    constexpr uint32_t kThreads = 64 * WAVES, kTileRows = 32 * WAVES;
    constexpr int kPieces = HEAD * 4 / kThreads;  // of 16 codes, for each thread and tile: keys, and values
    constexpr int kRow = HEAD * 2;                // bytes of a key row in LDS
    constexpr float kSlack = 2.0f, kBias = kFloat ? 14.0f - kSlack : 15.0f - kSlack;
    __shared__ __attribute__((aligned(16))) int8_t lds_keys[2][64 * kRow];
    __shared__ __attribute__((aligned(16))) int8_t lds_values[2][HEAD * 128];
    // of a key: its scale, what its value's scale adds to the exponent, the share
    // of its weight in the sum, and the fraction (fp32); whether its page exists
    constexpr int kKinds = kFloat ? 4 : 3;
    __shared__ __attribute__((aligned(16))) float lds_scales[2][kKinds][64];
    __shared__ uint32_t lds_exists[2][4];
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

        // Staging. A wave's pieces of a tile are of one chunk of 16 tokens, so
        // that their places in the table are found once for it.
        u2_t key_codes[kPieces], value_codes[kPieces];
        Pages::Place of_key[kPieces]{}, of_value{}, of_scale{};
        float key_scale = 0.0f, value_scale = 1.0f;
        bool exists = false;
        constexpr uint32_t kLanes = HEAD / 16, kWaveKeys = 64 / kLanes, kKeyStep = WAVES * kWaveKeys;
        constexpr uint32_t kValueStep = kThreads / 4;
        const uint32_t key_chunk = lane % kLanes, key_row = wave * kWaveKeys + lane / kLanes;
        const uint32_t value_chunk = wave & 3u, value_row = lane + 64u * (wave >> 2);
        // features that the head does not have: others in their place, whose
        // copies in LDS meet no query feature and reach no output
        const uint32_t key_feature = 16u * key_chunk < d ? 16u * key_chunk : 0u;
        // Called without a condition, and never past the last block: registers
        // that are loaded in one branch only are waited for where the branches
        // meet.
        auto find = [&](uint32_t block) {
            block = min(block, last - 1u);
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                of_key[i] = pages.find(block * 4u + (wave * kWaveKeys + kKeyStep * i) / 16u);
            of_value = pages.find(block * 4u + value_chunk);
            of_scale = pages.find(block * 4u + lane / 16u);
        };
        auto load_keys = [&] {
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint64_t plane = static_cast<uint64_t>(pages.page(of_key[i])) * kv_heads + h;
                key_codes[i] = *reinterpret_cast<const u2_t*>(
                    a.cache.keys +
                    ((plane * page_size + of_key[i].slot + (key_row + kKeyStep * i) % 16u) * d + key_feature) / 2u);
            }
        };
        auto load_values = [&] {
            const uint64_t plane = static_cast<uint64_t>(pages.page(of_value)) * kv_heads + h;
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                value_codes[i] = *reinterpret_cast<const u2_t*>(a.cache.values + (plane * page_size + of_value.slot) * (d / 2u) +
                                                                8u * min(value_row + kValueStep * i, d - 1u));
            exists = pages.exists(of_scale);
            const uint64_t at = (static_cast<uint64_t>(pages.page(of_scale)) * kv_heads + h) * page_size + of_scale.slot +
                                lane % 16u;
            key_scale = a.cache.key_scales[at];
            value_scale = a.cache.value_scales[at];
        };
        auto store_scales = [&](uint32_t buffer) {
            if (wave == 0) {
                float exponent, fraction, inverse;
                split_scale(value_scale, exponent, fraction, inverse);
                // a scale that is no number shows in the exponent alone: a token
                // that a row does not see adds nothing to its sums
                const bool number = fraction == fraction;
                if (!number) exponent = fraction;
                if constexpr (kFloat) {
                    lds_scales[buffer][3][lane] = number ? fraction : 1.0f;
                } else {
                    // the weights take the whole scale, off by half a step of its
                    // logarithm: below 2^-20 of them for scales of 1e-8 to 2^32,
                    // 2^-18 for any
                    exponent += __builtin_amdgcn_logf(number ? fraction : 1.0f);
                    inverse = inverse / (number ? fraction : 1.0f);
                }
                lds_scales[buffer][0][lane] = exists ? key_scale : 0.0f;
                lds_scales[buffer][1][lane] = exists ? exponent : -INFINITY;
                lds_scales[buffer][2][lane] = number ? inverse : 1.0f;
                if (lane % 16u == 0) lds_exists[buffer][lane / 16u] = exists;
            }
        };
        // Bringing a tile in small steps that fit between matrix instructions.
        constexpr int kStages = 4 * kPieces + 3;
        auto stage = [&](int n, uint32_t buffer, uint32_t block) {
            if (n < 4 * kPieces) {
                const int i = n / 4, half = n & 1;
                if (n & 2) {
                    const u2_t v = value_codes[i];
                    *reinterpret_cast<h8*>(lds_values[buffer] +
                                           swz<128>(value_row + kValueStep * i, 2u * value_chunk + half)) =
                        widen4(__builtin_amdgcn_perm(v[1], v[0], half ? 0x07060302u : 0x05040100u));
                } else {
                    *reinterpret_cast<h8*>(lds_keys[buffer] + swz<kRow>(key_row + kKeyStep * i, 2u * key_chunk + half)) =
                        widen4(key_codes[i][half]);
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
                    const int from = widened(i);
                    const float y = keep_fp32(ldexpf(static_cast<float>(raw[k][from / kVec][from % kVec]), e) * sign);
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
                // four keys of the lane: registers 4 g .. of block b
                auto read_scales = [&](int kind, int b, int g) {
                    return *reinterpret_cast<const v4f*>(&lds_scales[buffer][kind][32 * b + 8 * g + 4 * hf]);
                };
                __builtin_amdgcn_sched_barrier(0);
                float largest = kNoScore;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const v4f c = read_scales(0, b, g), shift = read_scales(1, b, g);
#pragma unroll
                        for (int r = 0; r < 4; ++r) sc[b][4 * g + r] = fmaf(sc[b][4 * g + r], c[r] * factor, shift[r]);
                    }
                const v4i_t pages_exist = *reinterpret_cast<const v4i_t*>(lds_exists[buffer]);
                if (!(k0 + 64u <= wave_least && pages_exist[0] && pages_exist[1] && pages_exist[2] && pages_exist[3])) {
                    stay_in_branch();
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const uint32_t key = k0 + 32u * b + 8u * (r >> 2) + 4u * hf + (r & 3);
                            if (!pages_exist[2 * b + (r >> 3)] || key >= limit) sc[b][r] = -INFINITY;
                        }
                }
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r) largest = fmaxf(largest, sc[b][r]);
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
                // weights of chunk t + 1 between the products of chunk t
                h8 pf[2][WP];
                v4f share[2], fraction[2];
                float before = 0.0f;  // a weight that waits for its neighbour
                auto weigh = [&](int t, int i) {
                    const int r = kPairs ? 4 * (i & 1) + i / 2 : i;
                    if (kPairs ? i < 2 : r % 4 == 0) {
                        share[r / 4] = read_scales(2, t >> 1, 2 * (t & 1) + r / 4);
                        if constexpr (kFloat) fraction[r / 4] = read_scales(3, t >> 1, 2 * (t & 1) + r / 4);
                    }
                    const float w = __builtin_amdgcn_exp2f(sc[t >> 1][8 * (t & 1) + r] - base);
                    sum = fmaf(w, share[r / 4][r % 4], sum);
                    const int to = 2 * (r & 3) + (r >> 2);  // in the order of widen4
                    if constexpr (kFloat) {
                        const float y = keep_fp32(w * fraction[r / 4][r % 4]);  // hi and lo of one rounded product
                        const _Float16 hi = static_cast<_Float16>(y);
                        pf[t & 1][0][to] = hi;
                        pf[t & 1][1][to] = static_cast<_Float16>((y - static_cast<float>(hi)) * kSecond);
                    } else if constexpr (kPairs) {
                        if (i % 2 == 0) {
                            before = w;
                        } else {
                            const h2 hi = __builtin_convertvector((v2f{before, w}), h2);
                            float rest0, rest1;  // w less its first part, in one operation: 641 us for 656 above
                            asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rest0) : "v"(hi), "v"(before));
                            asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
                                : "=v"(rest1)
                                : "v"(hi), "v"(w));
                            const h2 lo = __builtin_convertvector((v2f{rest0, rest1}), h2);
                            pf[t & 1][0][to - 1] = hi[0], pf[t & 1][0][to] = hi[1];
                            pf[t & 1][1][to - 1] = lo[0], pf[t & 1][1][to] = lo[1];
                        }
                    } else {
                        pf[t & 1][0][to] = static_cast<_Float16>(w);
                    }
                };
#pragma unroll
                for (int r = 0; r < 8; ++r) weigh(0, r);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (t < 3) read_values(t + 1, vf[(t + 1) & 1]);
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) {
                        const int f = i % FB;
                        o[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[t & 1][f], pf[t & 1][i / FB], o[f], 0, 0, 0);
                        if constexpr (kFloat)
                            o[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(for_second(vf[t & 1][f]), pf[t & 1][1], o[f], 0,
                                                                          0, 0);
                        if (t < 3)
#pragma unroll
                            for (int r = 8 * i / kSteps; r < 8 * (i + 1) / kSteps; ++r) weigh(t + 1, r);
                        if (!kPairs || i % 2) __builtin_amdgcn_sched_barrier(0);
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

// Which kernel, and how its keys are split. us; 32 heads of 8, 128 features, bf16,
// unless it says otherwise.
//
// Tiles widen a key once for up to 256 rows, and leave waves without rows where
// there are few: rows are faster up to a work of 2^26 (one sequence, 64 tokens
// over 2048 19.0 / 25.1, over 4096 25.8 / 31.5; 4 of 128 over 512 22.1 / 30.1),
// tiles beyond (128 over 8192 49.5 / 68.2).
//
// Rows: as few columns as hold them (32 of up to 4096 keys: 30.5 in 4 columns,
// 38.8 in 16). Two workgroups share a CU, so up to 512 run at once: keys are split as
// far as that goes, to 128 keys each (8 of 4096: 14.5 in 8, 19.9 in 2, 18.8 in 16; one
// token over 1370, 16 heads of 64, f32: 9.2 in 10, 10.0 in 5, 11.3 in 2; 40 of 300: 9.4
// whole, 13.8 in two). Beyond it a split only evens out sequences of different
// lengths, and pays for long ones: up to 2048 workgroups of at least 2048 keys (32
// of up to 32768: 142 in 8, 148 in 4, 159 in 2, 153 in 16).
//
// Tiles: splitting n keys s times costs n / s tiles one after the other and s
// parts to join, so s grows as sqrt(n / 32) (128 tokens over 32768, 8 heads: 56.6;
// sqrt(n / 64) 72.5, sqrt(n / 16) 58.9), and to one workgroup of 256 rows or two
// of 128 a CU. 256 rows widen the keys once for twice the rows (2 of 2048 over
// 8192 561 against 583, f16 641 / 665; 512 over 32768 334 / 361, f16 406 / 438),
// if the head is so wide that three waves of the smaller ones do not fit a SIMD
// instead, if they add no rows that do not exist (2 of 577 tokens, 16 heads of 16:
// 36.0 against 33.8), and if there are enough of them, one for each CU and two
// where a causal mask makes them unequal (4096 tokens, 8 heads of 8: 103.9 against
// 94.8).
struct Plan {
    uint32_t tile;  // rows: 4, 8 or 16 of cache4_rows_kernel, 128 or 256 of cache4_tiles_kernel
    uint32_t tiles, splits;
};
Plan plan_of(const dav2_attention_cache_i4_args& a) {
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
    p.tile = rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
    p.tiles = static_cast<uint32_t>(std::min<uint64_t>((rows + p.tile - 1) / p.tile, 4096));
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
    const uint64_t chunks = (std::min(a.max_new, a.tokens) + 14u) / 16u + 1u;
    constexpr uint64_t kMostGroups = 1u << 22;  // workgroups along x: threads of a launch stay below 2^32
    const dim3 grid(static_cast<uint32_t>(std::min(chunks, kMostGroups)), (2u * a.cache.kv_heads + 3u) / 4u, a.sequences);
    with_dtype(a.dtype, [&](auto* e) {
        typedef std::remove_pointer_t<decltype(e)> E;
        dispatch(cache4_store_kernel<E>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
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
    const dim3 grid = p.tile > 16 ? dim3(a.cache.kv_heads * a.sequences, p.tiles * p.splits)
                                  : dim3(p.tiles * p.splits, a.cache.kv_heads, a.sequences);
    return with_dtype(a.dtype, [&](auto* e) -> int {
        typedef std::remove_pointer_t<decltype(e)> E;
        with_head_dim(a.cache.head_dim, [&](auto dim) {
            constexpr int D = decltype(dim)::value;
            if constexpr (D > 64) {
                if (p.tile == 256) return dispatch(cache4_tiles_kernel<E, D, 8>, grid, dim3(512), 0, s, a, p.splits, p.tiles);
            }
            if (p.tile == 128) dispatch(cache4_tiles_kernel<E, D, 4>, grid, dim3(256), 0, s, a, p.splits, p.tiles);
            else dispatch(p.tile == 4   ? cache4_rows_kernel<E, D, 4>
                          : p.tile == 8 ? cache4_rows_kernel<E, D, 8>
                                        : cache4_rows_kernel<E, D, 16>,
                          grid, dim3(256), 0, s, a, p.splits, p.tiles);
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
