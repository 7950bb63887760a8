// The next token of each row of logits, by a given random number.
//
// The tokens stand in order of their logits, equal ones by index, and what
// min-p, top-k and top-p keep is a prefix of that order, as is what lies below
// the random number: each is a search for the token at which a running count or
// a running sum of weights passes a bound. Weights are whole numbers, 2^s
// exp((l - l_max) / t) rounded, so that sums of any parts in any order are the same
// and a search may go by parts of the row.

#include <algorithm>

#include "decoder.h"

using namespace dav2k;

namespace {

constexpr uint32_t kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;

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
    q.per_temperature = 1.4426950408889634 / static_cast<double>(t);
    const float min_p = a.min_p ? a.min_p[row] : 0.0f, top_p = a.top_p ? a.top_p[row] : 1.0f;
    q.min_p = min_p > 0.0f && min_p <= 1.0f ? min_p : 0.0;
    q.top_p = top_p < 1.0f ? fmaxf(top_p, 0.0f) : 1.0;  // NaN keeps all
    const int32_t k = a.top_k ? a.top_k[row] : 0;
    q.top_k = k > 0 && static_cast<uint32_t>(k) < a.vocabulary ? static_cast<uint32_t>(k) : a.vocabulary;
    q.uniform = fminf(fmaxf(a.uniform[row], 0.0f), 0x1.fffffep-1f);  // fmaxf drops a NaN
    return q;
}

// exp((l - top) / temperature) in 64 bits. An infinite top has weight 1 and all others none.
DAV2_DEV double weight_of(float l, float top, double per_temperature) {
    if (l == top) return 1.0;
    if (!(top < INFINITY)) return 0.0;
    return exp2((static_cast<double>(l) - static_cast<double>(top)) * per_temperature);
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

struct Shared {
    uint32_t counts[kBins];
    unsigned long long sums[kBins];
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
            for (uint32_t i = threadIdx.x; i < kBins; i += kThreads) {
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

// A workgroup for each row.
template <typename E>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(dav2_sample_args a, int bits) {
    __shared__ Shared sh;
    __shared__ uint32_t smallest[kWaves];
    const uint32_t r = blockIdx.x;
    Row<E> row;
    row.logits = static_cast<const E*>(a.logits) + r * a.logit_stride;
    row.vocabulary = a.vocabulary;
    row.bits = bits;
    row.q = asked_of(a, r);

    uint32_t key = ~0u;
    for (uint32_t i = threadIdx.x; i < a.vocabulary; i += kThreads) key = min(key, rank_key(row.logit(i)));
    for (int o = 32; o > 0; o >>= 1) key = min(key, static_cast<uint32_t>(__shfl_xor(static_cast<int>(key), o, kWave)));
    if ((threadIdx.x & 63u) == 0) smallest[threadIdx.x >> 6] = key;
    __syncthreads();
    for (uint32_t w = 0; w < kWaves; ++w) key = min(key, smallest[w]);
    row.top = logit_of(key);
    typedef typename Row<E>::Place Place;
    int32_t token = -1;
    float probability = 0.0f;
    if (row.top > -INFINITY) {
        // what top-k keeps ends before `end`
        Place end = {~0u, ~0u};
        const uint32_t keep = row.q.greedy ? 1u : row.q.top_k;
        if (keep < a.vocabulary) end = row.template search<false>(keep, Place{~0u, ~0u}, sh).at;
        uint64_t whole = 0;
        for (uint32_t i = threadIdx.x; i < a.vocabulary; i += kThreads) {
            const uint32_t k = rank_key(row.logit(i));
            if (end.after(k, i)) whole += row.units(k);
        }
        whole = group_sum(whole, sh.of_wave);
        if (row.q.top_p < 1.0) {
            // the last token kept is the first at which the running sum reaches top_p of the whole
            const uint64_t bound = static_cast<uint64_t>(ceil(row.q.top_p * static_cast<double>(whole)));
            const auto last = row.template search<true>(min(bound > 0 ? bound - 1 : 0, whole - 1), end, sh);
            end = {last.at.key, last.at.index + 1u};
            whole = last.sum + row.units(last.at.key);
        }
        const uint64_t drawn = static_cast<uint64_t>(static_cast<double>(row.q.uniform) * static_cast<double>(whole));
        const auto found = row.template search<true>(min(drawn, whole - 1), end, sh);
        token = static_cast<int32_t>(found.at.index);
        probability = static_cast<float>(
            weight_of(logit_of(found.at.key), row.top, row.q.per_temperature) / ldexp(static_cast<double>(whole), -bits));
    }
    if (threadIdx.x == 0) {
        a.tokens[r] = token;
        if (a.probabilities) a.probabilities[r] = probability;
    }
}

// Weights of 2^bits each, summed over a vocabulary, stay below 2^63.
int weight_bits(uint32_t vocabulary) {
    int log2 = 0;
    while ((1u << log2) < vocabulary) ++log2;
    return 62 - log2;
}

}  // namespace

extern "C" {

uint64_t dav2_hip_sample_scratch_bytes(const dav2_sample_args*) { return 0; }

int dav2_hip_sample(const dav2_sample_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_sample_args& a = *args;
    if (a.rows == 0) return hipSuccess;
    const uint64_t need = dav2_hip_sample_scratch_bytes(args);
    if (!a.logits || !a.uniform || !a.tokens || a.rows > 65535u || a.vocabulary == 0 || a.vocabulary > (1u << 20) ||
        a.dtype > DAV2_DTYPE_BF16 || (a.rows > 1 && a.logit_stride < a.vocabulary) ||
        (need && (!a.scratch || !aligned16(a.scratch) || a.scratch_bytes < need)))
        return hipErrorInvalidValue;
    return with_dtype(a.dtype, [&](auto* e) -> int {
        typedef std::remove_pointer_t<decltype(e)> E;
        dispatch(sample_row_kernel<E>, dim3(a.rows), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a,
                 weight_bits(a.vocabulary));
        return hipGetLastError();
    });
}

}  // extern "C"
