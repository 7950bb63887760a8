// The next token of each row of logits, by a given random number.
//
// The tokens stand in order of their logits, equal ones by index, and what
// min-p, top-k and top-p keep is a prefix of that order, as is what lies below
// the random number: each is a search for the token at which a running count or
// a running sum of weights passes a bound. Weights are whole numbers, 2^s
// exp((l - l_max) / t) rounded, so that sums of any parts in any order are the same
// and a search may go by parts of the row.
//
// A row is read three times, the first time from memory: for its largest logit;
// for what falls into each of kBins bins of the distance to that, how many
// tokens and what weight; and for the tokens of those few bins in which the three
// searches can end, as a list. A workgroup for each row then sorts the list and
// ends them. Where the list has no room (thousands of equal logits), it searches
// the row itself. Long rows of 16 bits without a top-k are counted number by
// number instead, in one pass, and read again for the places of the number drawn.
//
// Bound by one CU's work on its rows, not by memory: a token's count is an atomic
// operation in LDS, its weight a polynomial in 64 bits beside one. 4 rows of
// 32000, fp32, every filter 13.0 us; 256 of 100003, bf16, top-p 35 us (51 MB).

#include <algorithm>

#include "decoder.h"

using namespace dav2k;

namespace {

constexpr uint32_t kThreads = 1024, kWaves = kThreads / 64, kDigits = 2048;
constexpr uint32_t kBins = 2048;        // of a row: 48 powers of two, the last one what is further
constexpr uint32_t kList = 4096;        // tokens of a row's list
// A row of so many is its own list: us, 64 rows of 60 tokens 5.7 against 9.5 with
// bins, of 250 8.9 / 9.5, of 500 16.2 / 9.5, of 4000 41 / 11.
constexpr uint32_t kSorted = 256;
constexpr uint32_t kMostChunks = 64;    // workgroups that share a row
constexpr uint32_t kChunkThreads = 256;
constexpr uint32_t kFew = 2048;         // a top-k up to this many is few

// A logit's place in the order, 0 for the largest number there is: floats as
// whole numbers that grow as they fall. -0 is 0, NaN is -infinity.
DAV2_DEV uint32_t rank_key(float l) {
    l = l != l ? -INFINITY : l + 0.0f;
    const uint32_t b = __float_as_uint(l);
    return ~(b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u));
}
DAV2_DEV float logit_of(uint32_t key) {
    const uint32_t b = ~key;
    return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u : ~b);
}

// What a row asks for.
struct Asked {
    double per_temperature;  // log2(e) / temperature
    double min_p, top_p;
    uint32_t top_k;  // at least 1
    float uniform;
    bool greedy;
    bool few;  // the list has all that top-k leaves, and the bins need no weights
};
DAV2_DEV Asked asked_of(const dav2_sample_args& a, uint32_t row) {
    Asked q;
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    q.greedy = !(t > 0.0f);
    q.per_temperature = 1.4426950408889634 / (q.greedy ? 1.0 : static_cast<double>(t));
    const float min_p = a.min_p ? a.min_p[row] : 0.0f, top_p = a.top_p ? a.top_p[row] : 1.0f;
    q.min_p = min_p > 0.0f && min_p <= 1.0f ? min_p : 0.0;
    q.top_p = top_p < 1.0f ? fmaxf(top_p, 0.0f) : 1.0;  // NaN keeps all
    const int32_t k = a.top_k ? a.top_k[row] : 0;
    q.top_k = q.greedy ? 1u : k > 0 && static_cast<uint32_t>(k) < a.vocabulary ? static_cast<uint32_t>(k) : a.vocabulary;
    q.few = q.top_k <= kFew && q.top_k < a.vocabulary;
    q.uniform = fminf(fmaxf(a.uniform[row], 0.0f), 0x1.fffffep-1f);  // fmaxf drops a NaN
    return q;
}

// 2^x over 2^n for -100 <= x <= 0: x = n + f, |f| <= 1/2, and the Taylor polynomial
// of 2^f of degree 11, whose rest is below 2^-47. n is the low word of x + 1.5 * 2^52.
DAV2_DEV double exp2_of(double x, int& n) {
    constexpr double kLn2 = 0.69314718055994530942, kRound = 0x1.8p52;
    constexpr double c2 = kLn2 * kLn2 / 2, c3 = c2 * kLn2 / 3, c4 = c3 * kLn2 / 4, c5 = c4 * kLn2 / 5,
                     c6 = c5 * kLn2 / 6, c7 = c6 * kLn2 / 7, c8 = c7 * kLn2 / 8, c9 = c8 * kLn2 / 9,
                     c10 = c9 * kLn2 / 10, c11 = c10 * kLn2 / 11;
    const double rounded = x + kRound, f = x - (rounded - kRound);
    double p = fma(c11, f, c10);
    p = fma(p, f, c9);
    p = fma(p, f, c8);
    p = fma(p, f, c7);
    p = fma(p, f, c6);
    p = fma(p, f, c5);
    p = fma(p, f, c4);
    p = fma(p, f, c3);
    p = fma(p, f, c2);
    p = fma(p, f, kLn2);
    n = static_cast<int>(__double2loint(rounded));
    return fma(p, f, 1.0);
}

// exp((l - top) / temperature) in 64 bits. An infinite top has weight 1 and all others none.
DAV2_DEV double weight_of(float l, float top, double per_temperature) {
    if (l == top) return 1.0;
    const double x = (static_cast<double>(l) - static_cast<double>(top)) * per_temperature;
    if (!(x > -100.0)) return 0.0;  // a NaN is infinity less infinity
    int n;
    const double p = exp2_of(x, n);
    return ldexp(p, n);
}
// ... in units of 2^-bits, bits <= 46: the sum with 2^52 is rounded to a whole number, in its low 52 bits
DAV2_DEV uint64_t units_of(double weight, int bits) {
    const double v = weight * __hiloint2double((bits + 1023) << 20, 0) + 0x1p52;
    return static_cast<uint64_t>(__double_as_longlong(v)) & 0xfffffffffffffull;
}

DAV2_DEV uint64_t wave_sum64(uint64_t v) { return lane63(wave_upto(v)); }

// of the search in the row itself
struct Shared {
    uint32_t counts[kDigits];
    unsigned long long sums[kDigits];
    uint64_t of_wave[kWaves];
    uint32_t found;
    uint64_t found_count, found_sum;
};

// The sum over the workgroup, the same for all threads.
DAV2_DEV uint64_t group_sum(uint64_t v, uint64_t* of_wave) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) of_wave[threadIdx.x >> 6] = v;
    __syncthreads();
    waves_before<kWaves>(of_wave, v);
    return v;
}

// The sum over the threads before this one, and over the workgroup.
DAV2_DEV uint64_t group_before(uint64_t v, uint64_t* of_wave, uint64_t& all) {
    const uint64_t upto = wave_upto(v);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    __syncthreads();
    if (lane == 63u) of_wave[wave] = upto;
    __syncthreads();
    return waves_before<kWaves>(of_wave, all) + upto - v;
}

// The sum of weights that the last token of top-p passes: the first at which the
// running sum reaches top_p of the whole.
DAV2_DEV uint64_t share_of(double top_p, uint64_t whole) {
    const uint64_t bound = static_cast<uint64_t>(ceil(top_p * static_cast<double>(whole)));
    return min(bound > 0 ? bound - 1 : 0, whole - 1);
}
// ... that the token drawn passes
DAV2_DEV uint64_t drawn_of(const Asked& q, uint64_t whole) {
    return min(static_cast<uint64_t>(static_cast<double>(q.uniform) * static_cast<double>(whole)), whole - 1);
}

// One row, by a workgroup.
template <typename E>
struct Row {
    const E* logits;
    uint32_t vocabulary;
    int bits;
    float top;  // the largest logit
    Asked q;

    // A place in the order: the tokens before it are those of a smaller key,
    // and those of its key with a smaller index.
    struct Place {
        uint32_t key, index;
        DAV2_DEV bool after(uint32_t k, uint32_t i) const { return k < key || (k == key && i < index); }
    };
    DAV2_DEV float logit(uint32_t i) const { return static_cast<float>(logits[i]); }
    DAV2_DEV uint64_t units(uint32_t key) const {
        const float l = logit_of(key);
        const double w = weight_of(l, top, q.per_temperature);
        return l > -INFINITY && w >= q.min_p ? units_of(w, bits) : 0;
    }

    // units() of any logit under a largest one that is finite: what is below 2^-100
    // or no number rounds to 0 by itself
    struct Weigher {
        double top, per_temperature, least;
        int bits;
        DAV2_DEV uint64_t operator()(float l) const {
            const double x = fmax((static_cast<double>(l) - top) * per_temperature, -100.0);
            int n;
            const double v = ldexp(exp2_of(x, n), n + bits);
            const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v + 0x1p52)) & 0xfffffffffffffull;
            return v >= least ? u : 0;
        }
    };
    DAV2_DEV Weigher weigher() const { return {top, q.per_temperature, ldexp(q.min_p, bits), bits}; }

    // a token's weight over the whole
    DAV2_DEV float share(uint32_t key, uint64_t whole) const {
        return static_cast<float>(weight_of(logit_of(key), top, q.per_temperature) /
                                  ldexp(static_cast<double>(whole), -bits));
    }

    // How a search ends: the token's place, and what lies before it.
    struct Found {
        Place at;
        uint64_t count, sum;
    };
    // The token at which the running count (BY_SUM: the running sum) first passes
    // `bound`, of those before `end`; the whole has to be above it. Three digits
    // of the key one after the other, then the index among equal keys.
    template <bool BY_SUM>
    DAV2_DEV Found search(uint64_t bound, const Place& end, Shared& sh) const {
        uint32_t key = 0, known = 0;  // digits found so far, and the bits they stand in
        uint64_t count = 0, sum = 0;
        for (int level = 0; level < 3; ++level) {
            const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
            const uint32_t digits = level == 2 ? 1024u : 2048u;
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < kDigits; i += kThreads) {
                sh.counts[i] = 0;
                sh.sums[i] = 0;
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < vocabulary; i += kThreads) {
                const uint32_t k = rank_key(logit(i));
                if ((k & known) != key || !end.after(k, i)) continue;
                const uint32_t digit = (k >> shift) & (digits - 1u);
                atomicAdd(&sh.counts[digit], 1u);
                if constexpr (BY_SUM) atomicAdd(&sh.sums[digit], static_cast<unsigned long long>(units(k)));
            }
            __syncthreads();
            // two digits for each thread
            const uint32_t d0 = 2u * threadIdx.x;
            const uint64_t c0 = sh.counts[d0], c1 = sh.counts[d0 + 1], s0 = sh.sums[d0], s1 = sh.sums[d0 + 1];
            uint64_t all;
            const uint64_t count_before = count + group_before(c0 + c1, sh.of_wave, all);
            const uint64_t sum_before = sum + group_before(s0 + s1, sh.of_wave, all);
            const uint64_t before = BY_SUM ? sum_before : count_before;
            const uint64_t a0 = BY_SUM ? s0 : c0, a1 = BY_SUM ? s1 : c1;
            if (before <= bound && bound < before + a0 + a1) {
                const bool second = bound >= before + a0;
                sh.found = d0 + second;
                sh.found_count = count_before + (second ? c0 : 0);
                sh.found_sum = sum_before + (second ? s0 : 0);
            }
            __syncthreads();
            key |= sh.found << shift;
            known |= (digits - 1u) << shift;
            count = sh.found_count;
            sum = sh.found_sum;
        }
        // equal keys have equal weights: which of them it is, then its index
        const uint64_t each = units(key);
        const uint64_t nth = BY_SUM ? (bound - sum) / each : bound - count;
        count += nth;
        sum += nth * each;
        uint64_t left = nth;
        for (uint32_t first = 0; first < vocabulary; first += kThreads) {
            const uint32_t i = first + threadIdx.x;
            const bool is = i < vocabulary && rank_key(logit(i)) == key && end.after(key, i);
            uint64_t all;
            const uint64_t before = group_before(is, sh.of_wave, all);
            if (all > left) {  // the same for all threads
                if (is && before == left) sh.found = i;
                __syncthreads();
                break;
            }
            left -= all;
        }
        return {{key, sh.found}, count, sum};
    }
};

// The three searches in the row itself.
template <typename E>
DAV2_DEV void search_row(const Row<E>& row, Shared& sh, int32_t* token, float* share) {
    typedef typename Row<E>::Place Place;
    // what top-k keeps ends before `end`
    Place end = {~0u, ~0u};
    if (row.q.top_k < row.vocabulary) end = row.template search<false>(row.q.top_k, Place{~0u, ~0u}, sh).at;
    uint64_t whole = 0;
    for (uint32_t i = threadIdx.x; i < row.vocabulary; i += kThreads) {
        const uint32_t k = rank_key(row.logit(i));
        if (end.after(k, i)) whole += row.units(k);
    }
    whole = group_sum(whole, sh.of_wave);
    if (row.q.top_p < 1.0) {
        const auto last = row.template search<true>(share_of(row.q.top_p, whole), end, sh);
        end = {last.at.key, last.at.index + 1u};
        whole = last.sum + row.units(last.at.key);
    }
    const auto found = row.template search<true>(drawn_of(row.q, whole), end, sh);
    if (threadIdx.x == 0) {
        *token = static_cast<int32_t>(found.at.index);
        *share = row.share(found.at.key, whole);
    }
}

// ---- the row by parts ---------------------------------------------------------

// What a row's workgroups tell the next kernel.
struct RowState {
    unsigned long long sums[kBins];
    uint32_t counts[kBins];
    float largest[kMostChunks];
    uint32_t listed, unused[3];
    unsigned long long list[kList];  // rank key, index
};

// f(logit, index, bit) for the elements [begin, end) of a row, by THREADS threads
// and up to 32 elements at a time, and next(c) after these: bit b of a thread is
// the element index_of(c, b, end). Loads behind the end are of the last
// elements instead, so that all are under way together. A row shorter than a
// vector has no bits.
template <typename E, uint32_t THREADS>
struct Elements {
    typedef Vec<E> V;
    static constexpr uint32_t N = V::N, kTogether = 4, kStep = THREADS * N;
    static DAV2_DEV uint32_t index_of(uint32_t c, uint32_t bit, uint32_t end) {
        return min(c + bit / N * kStep, end - N) + bit % N;
    }
    template <typename F, typename G>
    static DAV2_DEV void each(const E* row, uint32_t begin, uint32_t end, F&& f, G&& next) {
        if (end < N) {
            if (threadIdx.x == 0)
                for (uint32_t i = begin; i < end; ++i) f(static_cast<float>(row[i]), i, i);
            return;
        }
        for (uint32_t c0 = begin; c0 < end; c0 += kTogether * kStep) {  // the same for all threads
            const uint32_t c = c0 + threadIdx.x * N;
            float v[kTogether][N];
#pragma unroll
            for (uint32_t t = 0; t < kTogether; ++t) V::load(row, index_of(c, t * N, end), ~0u, v[t]);
            if (c0 + kTogether * kStep <= end) {
#pragma unroll
                for (uint32_t t = 0; t < kTogether; ++t)
#pragma unroll
                    for (uint32_t i = 0; i < N; ++i) f(v[t][i], c + t * kStep + i, t * N + i);
            } else {
#pragma unroll
                for (uint32_t t = 0; t < kTogether; ++t) {
                    if (c0 + t * kStep >= end) break;
#pragma unroll
                    for (uint32_t i = 0; i < N; ++i) {
                        const uint32_t at = index_of(c, t * N + i, end);
                        if (at >= c + t * kStep) f(v[t][i], at, t * N + i);
                    }
                }
            }
            next(c);
        }
    }
};
template <uint32_t THREADS, typename E, typename F>
DAV2_DEV void for_each(const E* row, uint32_t begin, uint32_t end, F&& f) {
    Elements<E, THREADS>::each(row, begin, end, [&](float l, uint32_t i, uint32_t) { f(l, i); }, [](uint32_t) {});
}

struct Chunk {
    uint32_t row, begin, end;
};
DAV2_DEV Chunk chunk_of(const dav2_sample_args& a, uint32_t length) {
    const uint32_t begin = blockIdx.x * length;
    return {blockIdx.y, min(begin, a.vocabulary), min(begin + length, a.vocabulary)};
}
DAV2_DEV unsigned long long list_entry(float l, uint32_t i) { return (static_cast<uint64_t>(rank_key(l)) << 32) | i; }
template <typename E>
DAV2_DEV const E* row_of(const dav2_sample_args& a, uint32_t row) {
    return static_cast<const E*>(a.logits) + row * a.logit_stride;
}
// The largest of the chunks' largest logits; a zero without its sign.
DAV2_DEV float top_of(const RowState& state, uint32_t chunks) {
    return wave_max((threadIdx.x & 63u) < chunks ? state.largest[threadIdx.x & 63u] : -INFINITY) + 0.0f;
}

// The bin of a logit: no larger for a larger one, as each rounding keeps the order.
// What the last one has weighs nothing: 2^-48 rounds to 0 in units of 2^-46. A
// distance is formed as its half, which no two finite numbers take past fp32, and
// counts for something at any temperature: an infinite one stays infinite.
struct Bins {
    float half_top, scale;  // finite, and not 0
    // whose whole part is the bin
    DAV2_DEV float place(float l) const { return fmaf(-0.5f, l, half_top) * scale; }
    DAV2_DEV Bins(float top, const Asked& q)
        : half_top(0.5f * fminf(top, 3.0e38f)),
          scale(fminf(fmaxf(static_cast<float>(q.per_temperature * (2 * kBins / 48.0)), 0x1p-126f), 3.0e38f)) {}
    DAV2_DEV uint32_t operator()(float l) const {
        // NaN is in the last one
        return static_cast<uint32_t>(fmaxf(fminf(place(l), static_cast<float>(kBins - 1u)), 0.0f));
    }
};

template <typename E>
__global__ __launch_bounds__(kChunkThreads) void sample_largest_kernel(dav2_sample_args a, uint32_t length) {
    __shared__ float of_wave[kChunkThreads / 64];
    const Chunk chunk = chunk_of(a, length);
    RowState& state = static_cast<RowState*>(a.scratch)[chunk.row];
    float top = -INFINITY;
    for_each<kChunkThreads>(row_of<E>(a, chunk.row), chunk.begin, chunk.end, [&](float l, uint32_t) { top = fmaxf(top, l); });
    top = wave_max(top);
    if ((threadIdx.x & 63u) == 0) of_wave[threadIdx.x >> 6] = top;
    for (uint32_t b = blockIdx.x * kChunkThreads + threadIdx.x; b < kBins; b += gridDim.x * kChunkThreads) {
        state.counts[b] = 0;
        state.sums[b] = 0;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) state.listed = 0;
    __syncthreads();
    if (threadIdx.x == 0) state.largest[blockIdx.x] = fmaxf(fmaxf(of_wave[0], of_wave[1]), fmaxf(of_wave[2], of_wave[3]));
}

// What the elements [begin, end) of a row add to its bins, in LDS: weights
// where the list may not have all that is kept, counts where there is a top-k.
template <uint32_t THREADS, typename E>
DAV2_DEV void fill_bins(const Row<E>& row, uint32_t begin, uint32_t end, uint32_t* counts, unsigned long long* sums) {
    const Bins bin_of(row.top, row.q);
    if (row.q.few) {
        for_each<THREADS>(row.logits, begin, end, [&](float l, uint32_t) { atomicAdd(&counts[bin_of(l)], 1u); });
        return;
    }
    const bool counted = row.q.top_k < row.vocabulary;
    auto fill = [&](auto&& units) {
        for_each<THREADS>(row.logits, begin, end, [&](float l, uint32_t) {
            const uint32_t b = bin_of(l);
            if (counted) atomicAdd(&counts[b], 1u);
            const uint64_t w = units(l);
            if (w) atomicAdd(&sums[b], static_cast<unsigned long long>(w));
        });
    };
    if (row.top < INFINITY) fill(row.weigher());
    else fill([&](float l) { return l == INFINITY ? 1ull << row.bits : 0ull; });
}

template <typename E>
__global__ __launch_bounds__(kChunkThreads) void sample_bins_kernel(dav2_sample_args a, uint32_t length, int bits) {
    __shared__ uint32_t counts[kBins];
    __shared__ unsigned long long sums[kBins];
    const Chunk chunk = chunk_of(a, length);
    RowState& state = static_cast<RowState*>(a.scratch)[chunk.row];
    const float top = top_of(state, gridDim.x);
    if (!(top > -INFINITY)) return;
    const Row<E> row = {row_of<E>(a, chunk.row), a.vocabulary, bits, top, asked_of(a, chunk.row)};
    for (uint32_t b = threadIdx.x; b < kBins; b += kChunkThreads) {
        counts[b] = 0;
        sums[b] = 0;
    }
    __syncthreads();
    fill_bins<kChunkThreads>(row, chunk.begin, chunk.end, counts, sums);
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < kBins; b += kChunkThreads) {
        if (counts[b]) atomicAdd(&state.counts[b], counts[b]);
        if (sums[b]) atomicAdd(&state.sums[b], sums[b]);
    }
}

// A row's bins in order, THREADS threads with neighbouring ones each, and which of them the list has.
template <uint32_t THREADS>
struct BinScan {
    static constexpr uint32_t N = kBins / THREADS;
    struct Shared {
        uint64_t of_wave[2][THREADS / 64];
        uint32_t found[8];
        uint64_t sums[4];  // before and of bins that were found
    };
    uint32_t counts[N], count_before;
    uint64_t sums[N], sum_before, whole;
    uint32_t low[3], high[3];  // bins of the list, both ends among them

    DAV2_DEV void load(const uint32_t* of_counts, const unsigned long long* of_sums, bool weighed, Shared& sh) {
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        uint64_t count = 0, sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            counts[i] = of_counts[threadIdx.x * N + i];
            sums[i] = weighed ? of_sums[threadIdx.x * N + i] : 0u;
            count += counts[i];
            sum += sums[i];
        }
        uint64_t c = wave_upto(count), s = weighed ? wave_upto(sum) : 0u;
        if (lane == 63u) {
            sh.of_wave[0][wave] = c;
            sh.of_wave[1][wave] = s;
        }
        __syncthreads();
        uint64_t all;
        c += waves_before<THREADS / 64u>(sh.of_wave[0], all) - count;
        whole = 0;
        if (weighed) s += waves_before<THREADS / 64u>(sh.of_wave[1], whole) - sum;
        count_before = static_cast<uint32_t>(c);
        sum_before = s;
    }

    // f(bin, tokens before, tokens, sum before, sum) for this thread's bins
    template <typename F>
    DAV2_DEV void each(F&& f) const {
        uint32_t c = count_before;
        uint64_t s = sum_before;
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            f(threadIdx.x * N + i, c, counts[i], s, sums[i]);
            c += counts[i];
            s += sums[i];
        }
    }

    // Which bins the searches can end in. The first is known by its count; the
    // sums that bound the second and third are known as ranges.
    DAV2_DEV void choose(const Asked& q, uint32_t vocabulary, int bits, Shared& sh) {
        const bool by_count = q.top_k < vocabulary;
        uint64_t lower = whole, upper = whole;  // what top-k leaves
        if (threadIdx.x < 8) sh.found[threadIdx.x] = 0;
        __syncthreads();
        if (by_count) {
            each([&](uint32_t b, uint32_t c, uint32_t n, uint64_t s, uint64_t m) {
                if (c < q.top_k && q.top_k <= c + n) {
                    sh.found[0] = b;
                    sh.sums[0] = s;
                    sh.sums[1] = s + m;
                }
            });
            __syncthreads();
            low[0] = high[0] = sh.found[0];
            if (high[0] == kBins - 1u) high[0] -= 1u;  // where that ends does not matter
            lower = sh.sums[0];
            upper = sh.sums[1];
        } else {
            low[0] = 1;
            high[0] = 0;
        }
        if (q.few) {  // all that top-k keeps
            low[0] = 0;
            low[1] = low[2] = 1;
            high[1] = high[2] = 0;
            return;
        }
        const uint64_t one = 1ull << bits;  // the first token's weight, which always stays
        lower = max(lower, one);
        auto range = [&](uint64_t from, uint64_t to, uint32_t which, bool keep_sums) {
            each([&](uint32_t b, uint32_t, uint32_t, uint64_t s, uint64_t m) {
                if (s <= from && from < s + m) {
                    sh.found[which] = b;
                    if (keep_sums) sh.sums[2] = s;
                }
                if (s <= to && to < s + m) {
                    sh.found[which + 1] = b;
                    if (keep_sums) sh.sums[3] = s + m;
                }
            });
            __syncthreads();
            low[which / 2] = sh.found[which];
            high[which / 2] = sh.found[which + 1];
        };
        low[1] = 1;
        high[1] = 0;
        if (q.top_p < 1.0) {
            range(share_of(q.top_p, lower), share_of(q.top_p, upper), 2, true);
            lower = max(sh.sums[2], one);
            upper = min(sh.sums[3], upper);
        }
        range(drawn_of(q, lower), drawn_of(q, upper), 4, false);
    }
};

// put(place, index) for the elements of [begin, end) that are so, places being
// counted in `listed`. A thread marks which of its elements are, and a wave
// counts for all of its own at once. The row is no shorter than a vector.
template <uint32_t THREADS, typename E, typename Is, typename F>
DAV2_DEV void gather(const E* row, uint32_t begin, uint32_t end, uint32_t* listed, Is&& is, F&& put) {
    typedef Elements<E, THREADS> All;
    uint32_t marks = 0;
    All::each(
        row, begin, end, [&](float l, uint32_t, uint32_t bit) { marks |= is(l) ? 1u << bit : 0u; },
        [&](uint32_t c) {
            if (!__any(marks != 0u)) return;
            const uint32_t count = static_cast<uint32_t>(__popc(marks)), upto = wave_upto32(count);
            uint32_t first = 0;
            if ((threadIdx.x & 63u) == 63u) first = atomicAdd(listed, upto);
            uint32_t at = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(first), 63)) + upto - count;
            for (; marks; marks &= marks - 1u) put(at++, All::index_of(c, static_cast<uint32_t>(__builtin_ctz(marks)), end));
        });
}

// put(place, entry) for the tokens of [begin, end) in those bins.
template <uint32_t THREADS, typename E, typename Scan, typename F>
DAV2_DEV void for_listed(const Row<E>& row, const Scan& scan, uint32_t begin, uint32_t end, uint32_t* listed, F&& put) {
    const Bins bin_of(row.top, row.q);
    // in places of the bins; the last bin, where no number is, is in no list
    float from[3], to[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const bool none = scan.low[i] > scan.high[i];
        // an infinite top is before the first place
        from[i] = none ? INFINITY : scan.low[i] ? static_cast<float>(scan.low[i]) : -INFINITY;
        to[i] = none ? -INFINITY : static_cast<float>(scan.high[i] + 1u);
    }
    auto pass = [&](auto ranges) {
        auto is = [&](float l) {
            const float x = bin_of.place(l);
            bool in = x >= from[0] && x < to[0];
            if constexpr (decltype(ranges)::value > 1) in |= x >= from[2] && x < to[2];
            if constexpr (decltype(ranges)::value > 2) in |= x >= from[1] && x < to[1];
            return in;
        };
        gather<THREADS>(row.logits, begin, end, listed, is,
                        [&](uint32_t at, uint32_t i) { put(at, list_entry(row.logit(i), i)); });
    };
    if (scan.low[1] <= scan.high[1]) pass(std::integral_constant<int, 3>());
    else if (scan.low[2] <= scan.high[2]) pass(std::integral_constant<int, 2>());
    else pass(std::integral_constant<int, 1>());
}

template <typename E>
__global__ __launch_bounds__(kChunkThreads) void sample_list_kernel(dav2_sample_args a, uint32_t length, int bits) {
    __shared__ typename BinScan<kChunkThreads>::Shared sh;
    __shared__ unsigned long long staged[kList];
    __shared__ uint32_t here, first;
    const Chunk chunk = chunk_of(a, length);
    RowState& state = static_cast<RowState*>(a.scratch)[chunk.row];
    const float top = top_of(state, gridDim.x);
    if (!(top > -INFINITY)) return;
    if (threadIdx.x == 0) here = 0;
    const Row<E> row = {row_of<E>(a, chunk.row), a.vocabulary, bits, top, asked_of(a, chunk.row)};
    BinScan<kChunkThreads> scan;
    scan.load(state.counts, state.sums, !row.q.few, sh);
    scan.choose(row.q, a.vocabulary, bits, sh);
    for_listed<kChunkThreads>(row, scan, chunk.begin, chunk.end, &here, [&](uint32_t at, unsigned long long entry) {
        if (at < kList) staged[at] = entry;
    });
    __syncthreads();
    if (here == 0) return;
    if (threadIdx.x == 0) first = atomicAdd(&state.listed, here);
    __syncthreads();
    for (uint32_t i = threadIdx.x; first + i < kList && i < here; i += kChunkThreads) state.list[first + i] = staged[i];
}

// A list sorted into LDS: entry(i) is its i-th, all different.
template <typename F>
DAV2_DEV void sort_list(unsigned long long* list, uint32_t listed, F&& entry) {
    constexpr uint32_t kCounted = 512;
    if (listed <= kCounted) {
        // how many are before it says where a token goes: two or four threads
        // for each, and nothing to wait for between
        typedef unsigned long long U2 __attribute__((ext_vector_type(2)));
        unsigned long long* const raw = list + kList - kCounted;
        if (threadIdx.x < kCounted) raw[threadIdx.x] = entry(threadIdx.x);
        __syncthreads();
        const uint32_t sharing = listed <= kCounted / 2 ? 2u : 1u;  // log2 of the threads
        const uint32_t i = threadIdx.x >> sharing, part = threadIdx.x & ((1u << sharing) - 1u);
        const uint32_t pairs = (((listed + 1u) / 2u) >> sharing) + 1u;  // of each thread
        const unsigned long long mine = raw[i];
        uint32_t before = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < pairs; ++j) {
            // past the last the first again, counted by nobody
            const uint32_t p = part * pairs + j;
            const U2 x = reinterpret_cast<const U2*>(raw)[min(p, kCounted / 2 - 1u)];
            before += (x[0] < mine) & (2u * p < listed);
            before += (x[1] < mine) & (2u * p + 1u < listed);
        }
        before += __shfl_xor(static_cast<int>(before), 1, kWave);
        if (sharing == 2u) before += __shfl_xor(static_cast<int>(before), 2, kWave);
        if (i < listed && part == 0) list[before] = mine;
        __syncthreads();
        return;
    }
    uint32_t size = 2 * kCounted;
    while (size < listed) size *= 2;
    for (uint32_t i = threadIdx.x; i < size; i += kThreads) list[i] = entry(i);
    __syncthreads();
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            for (uint32_t t = threadIdx.x; t < size / 2; t += kThreads) {
                const uint32_t i = 2 * t - (t & (j - 1)), p = i + j;
                const unsigned long long x = list[i], y = list[p];
                if ((x > y) == ((i & k) == 0)) {
                    list[i] = y;
                    list[p] = x;
                }
            }
            __syncthreads();
        }
}

// What a workgroup that ends a row's searches has in LDS; KEYS: with a count for
// each number of 16 bits, two of them to a word.
constexpr uint32_t kKeyWords = 32768;
template <bool KEYS = false>
struct Finish {
    union {
        Shared search;
        unsigned long long list[kList];
        uint32_t keys[KEYS ? kKeyWords : 1];
    };
    unsigned long long sums[kBins];  // of a bin; then before it, less the list's sum there
    uint32_t counts[kBins];
    typename BinScan<kThreads>::Shared bins;
    uint64_t of_wave[kWaves], result[2];
    float tops[kWaves];
    int32_t token;
    float share;
    uint32_t listed;
};

// The searches ended in the row's list, whose i-th token is entry(i). gaps: bins
// lie between those of the list; sums and counts are then those before each bin,
// and whole the sum of all.
template <uint32_t kEach, typename E, typename F>
DAV2_DEV void finish_sorted(const Row<E>& row, F& sh, uint32_t listed, bool gaps, uint64_t whole) {
    const Asked& q = row.q;
    const Bins bin_of(row.top, q);
    // neighbouring tokens for each thread, and the sums before them
    uint64_t w[kEach], sum = 0;
    uint32_t key[kEach], bin[kEach];
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
        const uint32_t i = threadIdx.x * kEach + e;
        key[e] = i < listed ? static_cast<uint32_t>(sh.list[i] >> 32) : ~0u;
        w[e] = i < listed ? row.units(key[e]) : 0;
        bin[e] = gaps && i < listed ? bin_of(logit_of(key[e])) : 0u;
        sum += w[e];
    }
    uint64_t all;
    const uint64_t before = group_before(sum, sh.of_wave, all);
    if (gaps) {
        // a bin's first token says where the bin is in the list
        uint64_t at = before;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) {
            const uint32_t i = threadIdx.x * kEach + e;
            if (i < listed && (i == 0 || bin_of(logit_of(static_cast<uint32_t>(sh.list[i - 1] >> 32))) != bin[e])) {
                sh.sums[bin[e]] -= at;
                sh.counts[bin[e]] -= i;
            }
            at += w[e];
        }
    } else {
        whole = all;
    }
    // where top-k ends in the last bin, the whole is that of all others
    if (threadIdx.x == 0) sh.result[0] = whole;
    __syncthreads();
    // f(token of the list, its rank, the sum before it)
    auto each = [&](auto&& f) {
        uint64_t s = before;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e) {
            const uint32_t i = threadIdx.x * kEach + e;
            if (i < listed) f(e, gaps ? i + sh.counts[bin[e]] : i, gaps ? s + sh.sums[bin[e]] : s);
            s += w[e];
        }
    };
    if (q.top_k < row.vocabulary) {
        each([&](uint32_t e, uint32_t rank, uint64_t s) {
            if (rank == q.top_k - 1u) sh.result[0] = s + w[e];
        });
        __syncthreads();
        whole = sh.result[0];
    }
    if (q.top_p < 1.0) {
        const uint64_t bound = share_of(q.top_p, whole);
        each([&](uint32_t e, uint32_t, uint64_t s) {
            if (s <= bound && bound < s + w[e]) sh.result[1] = s + w[e];
        });
        __syncthreads();
        whole = sh.result[1];
    }
    const uint64_t drawn = drawn_of(q, whole);
    each([&](uint32_t e, uint32_t, uint64_t s) {
        if (s <= drawn && drawn < s + w[e]) {
            sh.token = static_cast<int32_t>(static_cast<uint32_t>(sh.list[threadIdx.x * kEach + e]));
            sh.share = row.share(key[e], whole);
        }
    });
}

template <typename E, typename S, typename F>
DAV2_DEV void finish_row(const Row<E>& row, S& sh, uint32_t listed, bool gaps, uint64_t whole, F&& entry) {
    sort_list(sh.list, listed, entry);
    if (listed <= kThreads) finish_sorted<1>(row, sh, listed, gaps, whole);
    else finish_sorted<kList / kThreads>(row, sh, listed, gaps, whole);
}

// The sums before each bin in the place of those of each.
template <typename F>
DAV2_DEV void put_before(const BinScan<kThreads>& scan, F& sh) {
    scan.each([&](uint32_t b, uint32_t c, uint32_t, uint64_t s, uint64_t) {
        sh.sums[b] = s;
        sh.counts[b] = c;
    });
}

template <typename F>
DAV2_DEV void put_token(const dav2_sample_args& a, const F& sh) {
    __syncthreads();
    if (threadIdx.x != 0) return;
    a.tokens[blockIdx.x] = sh.token;
    if (a.probabilities) a.probabilities[blockIdx.x] = sh.share;
}

// The list of a row whose bins have been filled, and the end of its searches.
template <typename E, typename F>
DAV2_DEV void list_and_finish(const Row<E>& row, F& sh) {
    BinScan<kThreads> scan;
    scan.load(sh.counts, sh.sums, !row.q.few, sh.bins);
    scan.choose(row.q, row.vocabulary, row.bits, sh.bins);
    put_before(scan, sh);
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    for_listed<kThreads>(row, scan, 0u, row.vocabulary, &sh.listed, [&](uint32_t at, unsigned long long entry) {
        if (at < kList) sh.list[at] = entry;
    });
    __syncthreads();
    const uint32_t listed = sh.listed;
    if (listed > kList) return search_row(row, sh.search, &sh.token, &sh.share);
    finish_row(row, sh, listed, !row.q.few, scan.whole, [&](uint32_t i) { return i < listed ? sh.list[i] : ~0ull; });
}

// The end of a row that workgroups have shared.
template <typename E>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(dav2_sample_args a, uint32_t chunks, int bits) {
    __shared__ Finish<> sh;
    const RowState& state = static_cast<const RowState*>(a.scratch)[blockIdx.x];
    const Row<E> row = {row_of<E>(a, blockIdx.x), a.vocabulary, bits, top_of(state, chunks), asked_of(a, blockIdx.x)};
    if (threadIdx.x == 0) {
        sh.token = -1;
        sh.share = 0.0f;
    }
    if (!(row.top > -INFINITY)) return put_token(a, sh);
    const uint32_t listed = state.listed;
    if (listed > kList) {
        __syncthreads();
        search_row(row, sh.search, &sh.token, &sh.share);
        return put_token(a, sh);
    }
    const bool gaps = !row.q.few;
    uint64_t whole = 0;
    if (gaps) {
        BinScan<kThreads> scan;
        scan.load(state.counts, state.sums, true, sh.bins);
        put_before(scan, sh);
        whole = scan.whole;
    }
    finish_row(row, sh, listed, gaps, whole, [&](uint32_t i) { return i < listed ? state.list[i] : ~0ull; });
    put_token(a, sh);
}

// ---- rows of 16-bit logits by how often each number is there -----------------------
//
// Without a top-k a row's bins need every token's weight, but there are only so
// many numbers of 16 bits: they are counted, and weighed once. The searches go
// by the bins, by the numbers of a bin, and by the tokens of a number.

// Numbers in order: 0 .. 32767 are the positive ones from the largest pattern
// down, 32768 .. 65535 the negative ones.
DAV2_DEV uint32_t pattern_of(uint32_t order) { return order < 32768u ? 32767u - order : order; }
template <typename E>
DAV2_DEV float number_of(uint32_t order) {
    return static_cast<float>(__builtin_bit_cast(E, static_cast<uint16_t>(pattern_of(order))));
}

// f(pattern, how often) for the numbers that are there. Neighbouring numbers are
// of neighbouring threads: those of a row lie close together.
template <typename F>
DAV2_DEV void for_keys(const Finish<true>& sh, F&& f) {
    constexpr uint32_t kTogether = 8;
    for (uint32_t i0 = threadIdx.x; i0 < kKeyWords; i0 += kTogether * kThreads) {
        uint32_t word[kTogether];
#pragma unroll
        for (uint32_t j = 0; j < kTogether; ++j) word[j] = sh.keys[i0 + j * kThreads];
#pragma unroll
        for (uint32_t j = 0; j < kTogether; ++j) {
            const uint32_t i = i0 + j * kThreads;
            if (word[j] == 0) continue;
            if (word[j] & 0xffffu) f(2u * i, word[j] & 0xffffu);
            if (word[j] >> 16) f(2u * i + 1u, word[j] >> 16);
        }
    }
}
template <typename E>
DAV2_DEV float number_at(uint32_t pattern) {
    return static_cast<float>(__builtin_bit_cast(E, static_cast<uint16_t>(pattern)));
}

// Whether all were counted: 65536 equal ones overflow their half word, and the
// sum of all counts is then another. The largest logit goes into row.top.
template <typename E>
DAV2_DEV bool count_keys(Row<E>& row, Finish<true>& sh) {
    typedef uint16_t Raw __attribute__((ext_vector_type(8), aligned(2)));
    const uint16_t* const raw = reinterpret_cast<const uint16_t*>(row.logits);
    for (uint32_t i = threadIdx.x; i < kKeyWords / 4u; i += kThreads)
        reinterpret_cast<uint4*>(sh.keys)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    auto add = [&](uint32_t x) { atomicAdd(&sh.keys[x >> 1], 1u << (16u * (x & 1u))); };
    constexpr uint32_t kTogether = 4, kStep = 8 * kThreads;
    uint32_t c = 8u * threadIdx.x;
    for (; c + (kTogether - 1u) * kStep + 8u <= row.vocabulary; c += kTogether * kStep) {
        Raw v[kTogether];
#pragma unroll
        for (uint32_t t = 0; t < kTogether; ++t) v[t] = *reinterpret_cast<const Raw*>(raw + c + t * kStep);
#pragma unroll
        for (uint32_t t = 0; t < kTogether; ++t)
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) add(v[t][i]);
    }
    for (; c < row.vocabulary; c += kStep)
        for (uint32_t i = c; i < min(c + 8u, row.vocabulary); ++i) add(raw[i]);
    __syncthreads();
    uint64_t counted = 0;
    float top = -INFINITY;
    for_keys(sh, [&](uint32_t pattern, uint32_t n) {
        counted += n;
        top = fmaxf(top, number_at<E>(pattern));
    });
    top = wave_max(top);
    if ((threadIdx.x & 63u) == 0) sh.tops[threadIdx.x >> 6] = top;
    const bool all = group_sum(counted, sh.of_wave) == row.vocabulary;
    row.top = wave_max(sh.tops[threadIdx.x & (kWaves - 1u)]) + 0.0f;
    return all;
}

// The bins' sums, a weight for each number.
template <typename E>
DAV2_DEV void weigh_keys(const Row<E>& row, Finish<true>& sh) {
    const Bins bin_of(row.top, row.q);
    for_keys(sh, [&](uint32_t pattern, uint32_t n) {
        const float l = number_at<E>(pattern);
        const uint64_t w = row.units(rank_key(l));
        if (w) atomicAdd(&sh.sums[bin_of(l)], static_cast<unsigned long long>(w * n));
    });
    __syncthreads();
}

// Where the running sum passes `bound`: a number, which of its tokens, and the sum before that one.
struct Passed {
    uint32_t order, nth;
    uint64_t before;
};
template <typename E>
DAV2_DEV Passed search_keys(const Row<E>& row, Finish<true>& sh, const BinScan<kThreads>& scan, uint64_t bound) {
    const Bins bin_of(row.top, row.q);
    scan.each([&](uint32_t b, uint32_t, uint32_t, uint64_t s, uint64_t m) {
        if (s <= bound && bound < s + m) {
            sh.bins.found[0] = b;
            sh.bins.sums[0] = s;
        }
    });
    __syncthreads();
    const uint32_t bin = sh.bins.found[0];
    const uint32_t infinity = 32767u - (sizeof(E) == 2 && std::is_same_v<E, _Float16> ? 0x7c00u : 0x7f80u);
    // the bin's numbers, found by each wave alike
    const uint32_t last = 65535u - infinity;
    auto first_of = [&](uint32_t b) {
        return first_where(infinity, last + 1u, [&](uint32_t o) { return bin_of(number_of<E>(o)) >= b; });
    };
    const uint32_t begin = first_of(bin), end = first_of(bin + 1u);
    // a run of neighbours for each thread: a bin about zero has thousands, few of which are there
    const uint32_t each = (end - begin + kThreads - 1u) / kThreads;
    const uint32_t from = min(begin + threadIdx.x * each, end), to = min(from + each, end);
    auto count = [&](uint32_t o) {
        const uint32_t pattern = pattern_of(o), n = (sh.keys[pattern >> 1] >> (16u * (pattern & 1u))) & 0xffffu;
        // both zeros are one number
        if (pattern == 0u) return n + (sh.keys[0x8000u >> 1] & 0xffffu);
        return pattern == 0x8000u ? 0u : n;
    };
    auto weight = [&](uint32_t o) { return row.units(rank_key(number_of<E>(o))); };
    uint64_t sum = 0;
    for (uint32_t o = from; o < to; ++o)
        if (const uint32_t n = count(o)) sum += n * weight(o);
    uint64_t all;
    uint64_t before = sh.bins.sums[0] + group_before(sum, sh.of_wave, all);
    if (before <= bound && bound < before + sum) {
        for (uint32_t o = from; o < to; ++o) {
            const uint32_t n = count(o);
            if (n == 0) continue;
            const uint64_t w = weight(o);
            if (bound < before + n * w) {
                const uint64_t nth = (bound - before) / w;
                sh.result[0] = before + nth * w;
                sh.bins.found[1] = o;
                sh.bins.found[2] = static_cast<uint32_t>(nth);
                break;
            }
            before += n * w;
        }
    }
    __syncthreads();
    const Passed passed = {sh.bins.found[1], sh.bins.found[2], sh.result[0]};
    __syncthreads();
    return passed;
}

// The index of the nth token of a number: by a list of all of them or, if they
// are many, each wave counting a part of the row.
template <typename E>
DAV2_DEV void find_nth(const Row<E>& row, Finish<true>& sh, float number, uint32_t nth) {
    constexpr uint32_t kMost = 256;
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();  // the keys, in whose place the list is, have been read
    gather<kThreads>(row.logits, 0u, row.vocabulary, &sh.listed, [&](float l) { return l == number; },
                     [&](uint32_t at, uint32_t i) {
                         if (at < kMost) sh.list[at] = i;
                     });
    __syncthreads();
    const uint32_t listed = sh.listed;
    if (listed <= kMost) {
        if (threadIdx.x >= listed) return;
        const unsigned long long mine = sh.list[threadIdx.x];
        uint32_t before_mine = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < listed; ++j) before_mine += sh.list[j] < mine;
        if (before_mine == nth) sh.token = static_cast<int32_t>(mine);
        return;
    }
    typedef Vec<E> V;
    constexpr uint32_t N = V::N, kBlock = 64 * N;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t length = ((row.vocabulary + kWaves - 1u) / kWaves + kBlock - 1u) / kBlock * kBlock;
    const uint32_t begin = min(wave * length, row.vocabulary), end = min(begin + length, row.vocabulary);
    auto count = [&](uint32_t c) {
        uint32_t n = 0;
        if (c + N <= end) {
            float v[N];
            V::load(row.logits, c, ~0u, v);
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) n += v[i] == number;
        } else {
            for (uint32_t i = c; i < end; ++i) n += row.logit(i) == number;
        }
        return n;
    };
    uint32_t n = 0;
#pragma unroll 4
    for (uint32_t c = begin + lane * N; c < end; c += kBlock) n += count(c);
    const uint64_t of_wave = wave_sum64(n);
    __syncthreads();
    if (lane == 0) sh.of_wave[wave] = of_wave;
    __syncthreads();
    uint64_t before = 0;
    for (uint32_t w = 0; w < wave; ++w) before += sh.of_wave[w];
    if (before > nth || nth >= before + of_wave) return;
    // this wave has it
    for (uint32_t c0 = begin; c0 < end; c0 += kBlock) {
        const uint32_t c = c0 + lane * N;
        const uint32_t mine = c < end ? count(c) : 0u;
        const uint64_t upto = wave_upto(mine), from = before + upto - mine;
        if (from <= nth && nth < from + mine) {
            uint32_t left = nth - static_cast<uint32_t>(from);
            for (uint32_t i = c; i < end; ++i)
                if (row.logit(i) == number && left-- == 0) {
                    sh.token = static_cast<int32_t>(i);
                    break;
                }
        }
        before += lane63(upto);
        if (before > nth) break;
    }
}

template <typename E>
DAV2_DEV void finish_keys(const Row<E>& row, Finish<true>& sh) {
    BinScan<kThreads> scan;
    scan.load(sh.counts, sh.sums, true, sh.bins);
    uint64_t whole = scan.whole;
    if (row.q.top_p < 1.0) {
        const Passed last = search_keys(row, sh, scan, share_of(row.q.top_p, whole));
        whole = last.before + row.units(rank_key(number_of<E>(last.order)));
    }
    const Passed drawn = search_keys(row, sh, scan, drawn_of(row.q, whole));
    const float number = number_of<E>(drawn.order);
    if (threadIdx.x == 0) sh.share = row.share(rank_key(number), whole);
    find_nth(row, sh, number, drawn.nth);
}

// A workgroup for each row, from its largest logit to its token: where rows are
// many, and where they are short, which then are their own list.
template <typename E, bool KEYS>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(dav2_sample_args a, int bits) {
    __shared__ Finish<KEYS> sh;
    Row<E> row = {row_of<E>(a, blockIdx.x), a.vocabulary, bits, 0.0f, asked_of(a, blockIdx.x)};
    if (threadIdx.x == 0) {
        sh.token = -1;
        sh.share = 0.0f;
    }
    for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) {
        sh.counts[b] = 0;
        sh.sums[b] = 0;
    }
    if constexpr (KEYS) {
        if (count_keys(row, sh)) {
            if (!(row.top > -INFINITY)) return put_token(a, sh);
            if (row.q.greedy) {
                if (threadIdx.x == 0) sh.share = 1.0f;
                find_nth(row, sh, row.top, 0u);
            } else {
                weigh_keys(row, sh);
                finish_keys(row, sh);
            }
            return put_token(a, sh);
        }
    }
    float top = -INFINITY;
    for_each<kThreads>(row.logits, 0u, a.vocabulary, [&](float l, uint32_t) { top = fmaxf(top, l); });
    top = wave_max(top);
    if ((threadIdx.x & 63u) == 0) sh.tops[threadIdx.x >> 6] = top;
    __syncthreads();
    row.top = wave_max(sh.tops[threadIdx.x & (kWaves - 1u)]) + 0.0f;
    if (!(row.top > -INFINITY)) return put_token(a, sh);
    if (a.vocabulary <= kSorted) {
        finish_row(row, sh, a.vocabulary, false, 0,
                   [&](uint32_t i) { return i < a.vocabulary ? list_entry(row.logit(i), i) : ~0ull; });
        return put_token(a, sh);
    }
    fill_bins<kThreads>(row, 0u, a.vocabulary, sh.counts, sh.sums);
    __syncthreads();
    list_and_finish(row, sh);
    put_token(a, sh);
}

// Weights of 2^bits each, summed over a vocabulary, stay below 2^63.
int weight_bits(uint32_t vocabulary) {
    int log2 = 0;
    while ((1u << log2) < vocabulary) ++log2;
    return std::min(62 - log2, 46);
}

// Rows that workgroups share: few and long ones, and sooner where every token of
// the row is weighed. us, a workgroup for each row against four launches, 1, 4, 16
// and 64 rows: fp32 with top-p alone, 32000 tokens 23 / 21, 23 / 22, 24 / 23, 25 / 31,
// 64000 36 / 22, 37 / 23, 38 / 26, 45 / 43, 100003 51 / 22, 53 / 24, 63 / 38, 63 / 52;
// with top-k 64000 tokens 15 / 16, 18 / 18, 18 / 19, 19 / 24, 100003 20 / 16, 23 / 18,
// 24 / 21, 24 / 27, 200000 32 / 16, 37 / 19, 37 / 24, 44 / 42; bf16 with top-p alone, 1, 4
// and 16 rows, 64000 tokens 24 / 22, 26 / 24, 27 / 30, 100003 26 / 24, 29 / 29, 32 / 39,
// 200000 35 / 24, 40 / 35, 41 / 44, 400000 52 / 33, 86 / 46, 83 / 72.
bool shares_rows(const dav2_sample_args& a, bool top_k) {
    if (top_k) return a.rows <= 64 && a.vocabulary >= 65536u + 2048u * a.rows;
    if (a.dtype == DAV2_DTYPE_F32) return a.rows <= 96 && a.vocabulary >= 28672u + 640u * a.rows;
    return a.rows <= 16 && a.vocabulary >= 65536u + 16384u * a.rows;
}

// Rows whose 16-bit logits are counted by their value.
// us, 64 rows, counted / not: 12000 tokens 23 / 16, 24000 26 / 22, 32000 25 / 26, 64000
// 28 / 48, 100003 32 / 68.
bool by_key(const dav2_sample_args& a) { return !a.top_k && a.vocabulary >= 28672u; }

// Logits of a chunk: 512 workgroups for the call, of 4096 and more each.
uint32_t chunk_length(const dav2_sample_args& a) {
    const uint32_t chunks = std::clamp(512u / a.rows, 1u, std::min(kMostChunks, (a.vocabulary + 4095u) / 4096u));
    return ((a.vocabulary + chunks - 1u) / chunks + 7u) / 8u * 8u;
}

}  // namespace

extern "C" {

uint64_t dav2_hip_sample_scratch_bytes(const dav2_sample_args* args) {
    return args && (shares_rows(*args, false) || shares_rows(*args, true))
               ? static_cast<uint64_t>(args->rows) * sizeof(RowState) : 0;
}

int dav2_hip_sample(const dav2_sample_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_sample_args& a = *args;
    if (a.rows == 0) return hipSuccess;
    const bool shared = shares_rows(a, a.top_k != nullptr);
    const uint64_t need = shared ? static_cast<uint64_t>(a.rows) * sizeof(RowState) : 0;
    if (!a.logits || !a.uniform || !a.tokens || a.rows > 65535u || a.vocabulary == 0 || a.vocabulary > (1u << 20) ||
        a.dtype > DAV2_DTYPE_BF16 || (a.rows > 1 && a.logit_stride < a.vocabulary) ||
        (need && (!a.scratch || !aligned16(a.scratch) || a.scratch_bytes < need)))
        return hipErrorInvalidValue;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int bits = weight_bits(a.vocabulary);
    return with_dtype(a.dtype, [&](auto* e) -> int {
        typedef std::remove_pointer_t<decltype(e)> E;
        if (shared) {
            const uint32_t length = chunk_length(a), chunks = (a.vocabulary + length - 1u) / length;
            const dim3 grid(chunks, a.rows);
            dispatch(sample_largest_kernel<E>, grid, dim3(kChunkThreads), 0, s, a, length);
            dispatch(sample_bins_kernel<E>, grid, dim3(kChunkThreads), 0, s, a, length, bits);
            dispatch(sample_list_kernel<E>, grid, dim3(kChunkThreads), 0, s, a, length, bits);
            dispatch(sample_pick_kernel<E>, dim3(a.rows), dim3(kThreads), 0, s, a, chunks, bits);
        } else {
            if constexpr (sizeof(E) == 2) {
                if (by_key(a)) {
                    dispatch(sample_row_kernel<E, true>, dim3(a.rows), dim3(kThreads), 0, s, a, bits);
                    return hipGetLastError();
                }
            }
            dispatch(sample_row_kernel<E, false>, dim3(a.rows), dim3(kThreads), 0, s, a, bits);
        }
        return hipGetLastError();
    });
}

}  // extern "C"
