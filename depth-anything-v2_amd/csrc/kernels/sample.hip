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
// the row itself.

#include <algorithm>

#include "decoder.h"

using namespace dav2k;

namespace {

constexpr uint32_t kThreads = 1024, kWaves = kThreads / 64, kDigits = 2048;
constexpr uint32_t kBins = 1024;        // of a row: 48 powers of two, the last one what is further
constexpr uint32_t kList = 4096;        // tokens of a row's list
constexpr uint32_t kMostChunks = 64;    // workgroups that share a row
constexpr uint32_t kChunkThreads = 256;
constexpr uint32_t kFew = 2048;         // a top-k up to this many: the list has all of it, and the bins need no weights

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
    q.uniform = fminf(fmaxf(a.uniform[row], 0.0f), 0x1.fffffep-1f);  // fmaxf drops a NaN
    return q;
}

// 2^x for x <= 0: x = n + f, |f| <= 1/2, and the Taylor polynomial of e^(f ln 2) of
// degree 13, whose rest is below 2^-57. Below 2^-100 it is 0.
DAV2_DEV double exp2_of(double x) {
    constexpr double kLn2 = 0.69314718055994530942;
    if (!(x > -100.0)) return 0.0;
    const double n = rint(x), f = (x - n) * kLn2;
    double p = 1.0 / 6227020800.0;
    p = fma(p, f, 1.0 / 479001600.0);
    p = fma(p, f, 1.0 / 39916800.0);
    p = fma(p, f, 1.0 / 3628800.0);
    p = fma(p, f, 1.0 / 362880.0);
    p = fma(p, f, 1.0 / 40320.0);
    p = fma(p, f, 1.0 / 5040.0);
    p = fma(p, f, 1.0 / 720.0);
    p = fma(p, f, 1.0 / 120.0);
    p = fma(p, f, 1.0 / 24.0);
    p = fma(p, f, 1.0 / 6.0);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    return ldexp(p, static_cast<int>(n));
}

// exp((l - top) / temperature) in 64 bits. An infinite top has weight 1 and all others none.
DAV2_DEV double weight_of(float l, float top, double per_temperature) {
    if (l == top) return 1.0;
    if (!(top < INFINITY)) return 0.0;
    return exp2_of((static_cast<double>(l) - static_cast<double>(top)) * per_temperature);
}
// ... in units of 2^-bits, bits <= 62
DAV2_DEV uint64_t units_of(double weight, int bits) {
    const double v = ldexp(weight, bits) + 0.5;
    const uint32_t hi = static_cast<uint32_t>(v * 0x1p-32);
    return (static_cast<uint64_t>(hi) << 32) + static_cast<uint32_t>(fma(static_cast<double>(hi), -0x1p32, v));
}

DAV2_DEV uint64_t wave_sum64(uint64_t v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(static_cast<unsigned long long>(v), o, kWave);
    return v;
}

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
    v = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) v += of_wave[w];
    return v;
}

// The sum over the threads before this one.
DAV2_DEV uint64_t group_before(uint64_t v, uint64_t* of_wave) {
    uint64_t upto = v;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t other = __shfl_up(static_cast<unsigned long long>(upto), o, kWave);
        if (lane >= static_cast<uint32_t>(o)) upto += other;
    }
    __syncthreads();
    if (lane == 63u) of_wave[wave] = upto;
    __syncthreads();
    uint64_t before = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) before += w < wave ? of_wave[w] : 0;
    return before + upto - v;
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
            const uint64_t count_before = count + group_before(c0 + c1, sh.of_wave);
            const uint64_t sum_before = sum + group_before(s0 + s1, sh.of_wave);
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
            const uint64_t before = group_before(is, sh.of_wave);
            const uint64_t all = group_sum(is, sh.of_wave);
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

// f(logit, index) for the elements [begin, end) of a row, by kChunkThreads threads.
template <typename E, typename F>
DAV2_DEV void for_each(const E* row, uint32_t begin, uint32_t end, F&& f) {
    typedef Vec<E> V;
    constexpr uint32_t N = V::N, kTogether = 4;  // loads that are under way together
    for (uint32_t c0 = begin + threadIdx.x * N; c0 < end; c0 += kTogether * kChunkThreads * N) {
        float v[kTogether][N];
#pragma unroll
        for (uint32_t t = 0; t < kTogether; ++t) {
            const uint32_t c = c0 + t * kChunkThreads * N;
            if (c < end) V::load(row, c, end, v[t]);
        }
#pragma unroll
        for (uint32_t t = 0; t < kTogether; ++t) {
            const uint32_t c = c0 + t * kChunkThreads * N;
            if (c >= end) break;
#pragma unroll
            for (uint32_t i = 0; i < N; ++i)
                if (c + i < end) f(v[t][i], c + i);
        }
    }
}

struct Chunk {
    uint32_t row, begin, end;
};
DAV2_DEV Chunk chunk_of(const dav2_sample_args& a, uint32_t length) {
    const uint32_t begin = blockIdx.x * length;
    return {blockIdx.y, min(begin, a.vocabulary), min(begin + length, a.vocabulary)};
}
template <typename E>
DAV2_DEV const E* row_of(const dav2_sample_args& a, uint32_t row) {
    return static_cast<const E*>(a.logits) + row * a.logit_stride;
}
// The largest of the chunks' largest logits; a zero without its sign.
DAV2_DEV float top_of(const RowState& state, uint32_t chunks) {
    return wave_max((threadIdx.x & 63u) < chunks ? state.largest[threadIdx.x & 63u] : -INFINITY) + 0.0f;
}

// The bin of a logit: no larger for a larger one, as each rounding keeps the order.
struct Bins {
    float top, scale;
    DAV2_DEV Bins(float top_, const Asked& q) : top(top_), scale(static_cast<float>(q.per_temperature * (kBins / 48.0))) {}
    DAV2_DEV uint32_t operator()(float l) const {
        if (l == top) return 0u;
        const float x = (top - l) * scale;
        return x < static_cast<float>(kBins - 1u) ? static_cast<uint32_t>(x) : kBins - 1u;  // NaN in the last
    }
};

template <typename E>
__global__ __launch_bounds__(kChunkThreads) void sample_largest_kernel(dav2_sample_args a, uint32_t length) {
    __shared__ float of_wave[kChunkThreads / 64];
    const Chunk chunk = chunk_of(a, length);
    RowState& state = static_cast<RowState*>(a.scratch)[chunk.row];
    float top = -INFINITY;
    for_each(row_of<E>(a, chunk.row), chunk.begin, chunk.end, [&](float l, uint32_t) { top = fmaxf(top, l); });
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

template <typename E>
__global__ __launch_bounds__(kChunkThreads) void sample_bins_kernel(dav2_sample_args a, uint32_t length, int bits) {
    __shared__ uint32_t counts[kBins];
    __shared__ unsigned long long sums[kBins];
    const Chunk chunk = chunk_of(a, length);
    RowState& state = static_cast<RowState*>(a.scratch)[chunk.row];
    const float top = top_of(state, gridDim.x);
    if (!(top > -INFINITY)) return;
    const Asked q = asked_of(a, chunk.row);
    const Row<E> row = {row_of<E>(a, chunk.row), a.vocabulary, bits, top, q};
    const Bins bin_of(top, q);
    for (uint32_t b = threadIdx.x; b < kBins; b += kChunkThreads) {
        counts[b] = 0;
        sums[b] = 0;
    }
    __syncthreads();
    const bool weighed = q.top_k > kFew;
    for_each(row.logits, chunk.begin, chunk.end, [&](float l, uint32_t) {
        const uint32_t b = bin_of(l);
        atomicAdd(&counts[b], 1u);
        if (weighed) {
            const uint64_t w = row.units(rank_key(l));
            if (w) atomicAdd(&sums[b], static_cast<unsigned long long>(w));
        }
    });
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

    DAV2_DEV void load(const RowState& state, Shared& sh) {
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        uint64_t count = 0, sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            counts[i] = state.counts[threadIdx.x * N + i];
            sums[i] = state.sums[threadIdx.x * N + i];
            count += counts[i];
            sum += sums[i];
        }
        uint64_t c = count, s = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t c1 = __shfl_up(static_cast<unsigned long long>(c), o, kWave);
            const uint64_t s1 = __shfl_up(static_cast<unsigned long long>(s), o, kWave);
            if (lane >= static_cast<uint32_t>(o)) {
                c += c1;
                s += s1;
            }
        }
        if (lane == 63u) {
            sh.of_wave[0][wave] = c;
            sh.of_wave[1][wave] = s;
        }
        __syncthreads();
        c -= count;
        s -= sum;
        whole = 0;
#pragma unroll
        for (uint32_t w = 0; w < THREADS / 64u; ++w) {
            if (w < wave) {
                c += sh.of_wave[0][w];
                s += sh.of_wave[1][w];
            }
            whole += sh.of_wave[1][w];
        }
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
        uint64_t least = whole, most = whole;  // what top-k leaves
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
            least = sh.sums[0];
            most = sh.sums[1];
        } else {
            low[0] = 1;
            high[0] = 0;
        }
        if (q.top_k <= kFew) {  // all that top-k keeps
            low[0] = 0;
            low[1] = low[2] = 1;
            high[1] = high[2] = 0;
            return;
        }
        const uint64_t one = 1ull << bits;  // the first token's weight, which always stays
        least = max(least, one);
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
            range(share_of(q.top_p, least), share_of(q.top_p, most), 2, true);
            least = max(sh.sums[2], one);
            most = min(sh.sums[3], most);
        }
        range(drawn_of(q, least), drawn_of(q, most), 4, false);
    }
    // Tokens of those bins.
    DAV2_DEV uint32_t listed(Shared& sh) const {
        each([&](uint32_t b, uint32_t, uint32_t n, uint64_t, uint64_t) {
            if (n && lists(b)) atomicAdd(&sh.found[7], n);
        });
        __syncthreads();
        return sh.found[7];
    }
    DAV2_DEV bool lists(uint32_t b) const {
        return (b >= low[0] && b <= high[0]) || (b >= low[1] && b <= high[1]) || (b >= low[2] && b <= high[2]);
    }
};

template <typename E>
__global__ __launch_bounds__(kChunkThreads) void sample_list_kernel(dav2_sample_args a, uint32_t length, int bits) {
    __shared__ typename BinScan<kChunkThreads>::Shared sh;
    const Chunk chunk = chunk_of(a, length);
    RowState& state = static_cast<RowState*>(a.scratch)[chunk.row];
    const float top = top_of(state, gridDim.x);
    if (!(top > -INFINITY)) return;
    const Asked q = asked_of(a, chunk.row);
    const Bins bin_of(top, q);
    BinScan<kChunkThreads> scan;
    scan.load(state, sh);
    scan.choose(q, a.vocabulary, bits, sh);
    if (scan.listed(sh) > kList) {
        if (blockIdx.x == 0 && threadIdx.x == 0) state.listed = kList + 1u;
        return;
    }
    for_each(row_of<E>(a, chunk.row), chunk.begin, chunk.end, [&](float l, uint32_t i) {
        if (!scan.lists(bin_of(l))) return;
        state.list[atomicAdd(&state.listed, 1u)] = (static_cast<uint64_t>(rank_key(l)) << 32) | i;
    });
}

// The list of a row sorted, and the searches ended in it: a workgroup for each
// row. chunks 0: the row is short enough to be its own list.
template <typename E>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(dav2_sample_args a, uint32_t chunks, int bits) {
    typedef typename Row<E>::Place Place;
    __shared__ union {
        Shared search;
        unsigned long long list[kList];
    } sh;
    __shared__ typename BinScan<kThreads>::Shared bins;
    __shared__ uint64_t sums_before[kBins];  // of a bin, less the list's sum before it
    __shared__ uint32_t counts_before[kBins];
    __shared__ uint64_t of_wave[kWaves], result[2];
    __shared__ int32_t token;
    __shared__ float share;
    constexpr uint32_t kEach = kList / kThreads;
    const uint32_t r = blockIdx.x;
    const RowState* state = chunks ? static_cast<const RowState*>(a.scratch) + r : nullptr;
    Row<E> row = {row_of<E>(a, r), a.vocabulary, bits, 0.0f, asked_of(a, r)};
    const Asked& q = row.q;
    uint32_t listed;
    if (threadIdx.x == 0) {
        token = -1;
        share = 0.0f;
    }
    if (chunks) {
        row.top = top_of(*state, chunks);
        listed = state->listed;
    } else {
        float top = -INFINITY;
        for (uint32_t i = threadIdx.x; i < a.vocabulary; i += kThreads) top = fmaxf(top, row.logit(i));
        top = wave_max(top);
        float* tops = reinterpret_cast<float*>(of_wave);
        if ((threadIdx.x & 63u) == 0) tops[threadIdx.x >> 6] = top;
        __syncthreads();
        for (uint32_t w = 0; w < kWaves; ++w) top = fmaxf(top, tops[w]);
        row.top = top + 0.0f;
        listed = a.vocabulary;
    }
    const Bins bin_of(row.top, q);
    // whether bins lie between those of the list
    const bool gaps = chunks && q.top_k > kFew;
    uint64_t whole = 0;
    __syncthreads();
    if (row.top > -INFINITY && listed > kList) {
        search_row(row, sh.search, &token, &share);
    } else if (row.top > -INFINITY) {
        if (gaps) {
            BinScan<kThreads> scan;
            scan.load(*state, bins);
            scan.each([&](uint32_t b, uint32_t c, uint32_t, uint64_t s, uint64_t) {
                sums_before[b] = s;
                counts_before[b] = c;
            });
            whole = scan.whole;
        }
        uint32_t size = 2;
        while (size < listed) size *= 2;
        for (uint32_t i = threadIdx.x; i < size; i += kThreads)
            sh.list[i] = i >= listed ? ~0ull
                         : chunks    ? state->list[i]
                                     : (static_cast<uint64_t>(rank_key(row.logit(i))) << 32) | i;
        __syncthreads();
        for (uint32_t k = 2; k <= size; k *= 2)
            for (uint32_t j = k / 2; j > 0; j /= 2) {
                for (uint32_t t = threadIdx.x; t < size / 2; t += kThreads) {
                    const uint32_t i = 2 * t - (t & (j - 1)), p = i + j;
                    const unsigned long long x = sh.list[i], y = sh.list[p];
                    if ((x > y) == ((i & k) == 0)) {
                        sh.list[i] = y;
                        sh.list[p] = x;
                    }
                }
                __syncthreads();
            }
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
        uint64_t before = group_before(sum, of_wave);
        const uint64_t all = group_sum(sum, of_wave);
        if (!gaps) whole = all;
        uint64_t at = before;
        if (gaps) {
            // a bin's first token says where the bin is in the list
#pragma unroll
            for (uint32_t e = 0; e < kEach; ++e) {
                const uint32_t i = threadIdx.x * kEach + e;
                if (i < listed && (i == 0 || bin_of(logit_of(static_cast<uint32_t>(sh.list[i - 1] >> 32))) != bin[e])) {
                    sums_before[bin[e]] -= at;
                    counts_before[bin[e]] -= i;
                }
                at += w[e];
            }
            __syncthreads();
        }
        // f(token of the list, its rank, the sum before it)
        auto each = [&](auto&& f) {
            uint64_t s = before;
#pragma unroll
            for (uint32_t e = 0; e < kEach; ++e) {
                const uint32_t i = threadIdx.x * kEach + e;
                if (i < listed) f(e, gaps ? i + counts_before[bin[e]] : i, gaps ? s + sums_before[bin[e]] : s);
                s += w[e];
            }
        };
        if (q.top_k < a.vocabulary) {
            each([&](uint32_t e, uint32_t rank, uint64_t s) {
                if (rank == q.top_k - 1u) result[0] = s + w[e];
            });
            __syncthreads();
            whole = result[0];
        }
        if (q.top_p < 1.0) {
            const uint64_t bound = share_of(q.top_p, whole);
            each([&](uint32_t e, uint32_t, uint64_t s) {
                if (s <= bound && bound < s + w[e]) result[1] = s + w[e];
            });
            __syncthreads();
            whole = result[1];
        }
        const uint64_t drawn = drawn_of(q, whole);
        each([&](uint32_t e, uint32_t, uint64_t s) {
            if (s <= drawn && drawn < s + w[e]) {
                token = static_cast<int32_t>(static_cast<uint32_t>(sh.list[threadIdx.x * kEach + e]));
                share = row.share(key[e], whole);
            }
        });
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        a.tokens[r] = token;
        if (a.probabilities) a.probabilities[r] = share;
    }
}

// Weights of 2^bits each, summed over a vocabulary, stay below 2^63.
int weight_bits(uint32_t vocabulary) {
    int log2 = 0;
    while ((1u << log2) < vocabulary) ++log2;
    return 62 - log2;
}

// Logits of a chunk: 2048 workgroups for the call, of 4096 and more each.
uint32_t chunk_length(const dav2_sample_args& a) {
    const uint32_t chunks = std::clamp(2048u / a.rows, 1u, std::min(kMostChunks, (a.vocabulary + 4095u) / 4096u));
    return ((a.vocabulary + chunks - 1u) / chunks + 7u) / 8u * 8u;
}

}  // namespace

extern "C" {

uint64_t dav2_hip_sample_scratch_bytes(const dav2_sample_args* args) {
    return args && args->vocabulary > kList ? static_cast<uint64_t>(args->rows) * sizeof(RowState) : 0;
}

int dav2_hip_sample(const dav2_sample_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_sample_args& a = *args;
    if (a.rows == 0) return hipSuccess;
    const uint64_t need = dav2_hip_sample_scratch_bytes(args);
    if (!a.logits || !a.uniform || !a.tokens || a.rows > 65535u || a.vocabulary == 0 || a.vocabulary > (1u << 20) ||
        a.dtype > DAV2_DTYPE_BF16 || (a.rows > 1 && a.logit_stride < a.vocabulary) ||
        (need && (!a.scratch || !aligned16(a.scratch) || a.scratch_bytes < need)))
        return hipErrorInvalidValue;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int bits = weight_bits(a.vocabulary);
    return with_dtype(a.dtype, [&](auto* e) -> int {
        typedef std::remove_pointer_t<decltype(e)> E;
        uint32_t chunks = 0;
        if (need) {
            const uint32_t length = chunk_length(a);
            chunks = (a.vocabulary + length - 1u) / length;
            const dim3 grid(chunks, a.rows);
            dispatch(sample_largest_kernel<E>, grid, dim3(kChunkThreads), 0, s, a, length);
            dispatch(sample_bins_kernel<E>, grid, dim3(kChunkThreads), 0, s, a, length, bits);
            dispatch(sample_list_kernel<E>, grid, dim3(kChunkThreads), 0, s, a, length, bits);
        }
        dispatch(sample_pick_kernel<E>, dim3(a.rows), dim3(kThreads), 0, s, a, chunks, bits);
        return hipGetLastError();
    });
}

}  // extern "C"
