// The int8 key/value cache: storing new tokens, and attention over it.
//
// One scale per page and head, s = max over the page of |x| / 127, so a page's
// codes are bounded by its largest value and a scale is read once per page.

#include "decoder.h"

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

// A workgroup per (touched page, head, sequence).
template <typename E>
__global__ __launch_bounds__(256) void cache_store_kernel(dav2_cache_store_i8_args a) {
    __shared__ uint32_t shared[4];
    const uint32_t h = blockIdx.y, s = blockIdx.z, page_size = a.cache.page_size, d = a.cache.head_dim;
    const Sequence q = sequence_of(a.starts, a.lengths, s, a.tokens);
    // positions [first, last) are new; in 64 bits, as a length may be anything
    const int64_t origin = static_cast<int64_t>(q.length) - (q.end - q.begin);  // row r has position origin + r - begin
    const int64_t first = max(origin, int64_t(0));
    const int64_t last = min(static_cast<int64_t>(q.length), static_cast<int64_t>(a.table_pages) * page_size);
    for (int64_t p = first / page_size + blockIdx.x; p * page_size < last; p += gridDim.x) {
        const int32_t page = a.page_table[static_cast<uint64_t>(s) * a.table_pages + p];
        if (page < 0 || static_cast<uint32_t>(page) >= a.cache.pages) continue;  // the same for the whole workgroup
        const int64_t base = p * page_size;
        const uint32_t from = static_cast<uint32_t>(max(first - base, int64_t(0)));
        const uint32_t to = static_cast<uint32_t>(min(last - base, static_cast<int64_t>(page_size)));
        const uint64_t plane = static_cast<uint64_t>(page) * a.cache.kv_heads + h;
        for (int side = 0; side < 2; ++side) {
            const E* x = static_cast<const E*>(side ? a.values : a.keys) + static_cast<uint64_t>(h) * d;
            const uint64_t stride = side ? a.value_stride : a.key_stride;
            int8_t* codes = (side ? a.cache.values : a.cache.keys) + plane * page_size * d;
            float* scale = (side ? a.cache.value_scales : a.cache.key_scales) + plane;
            auto row = [&](uint32_t slot) { return x + static_cast<uint64_t>(q.begin + (base + slot - origin)) * stride; };
            auto place = [&](uint32_t slot, uint32_t f) { return side ? f * page_size + slot : slot * d + f; };
            uint32_t most = 0;
            for (uint32_t i = threadIdx.x; i < (to - from) * d; i += 256u)
                most = max(most, __float_as_uint(fabsf(static_cast<float>(row(from + i / d)[i % d]))));
            most = workgroup_max_bits(most, shared);
            const float old = from ? *scale : 0.0f;
            // fmaxf would drop a NaN: compare bits again
            uint32_t bits = max(__float_as_uint(div_rn(__uint_as_float(most), 127.0f)), __float_as_uint(1.0e-8f));
            bits = max(bits, __float_as_uint(old) & 0x7fffffffu);
            const float now = __uint_as_float(bits);
            __syncthreads();  // every thread has read the old scale
            if (threadIdx.x == 0) *scale = now;
            if (from && now != old)
                for (uint32_t i = threadIdx.x; i < from * d; i += 256u) {
                    int8_t* c = codes + place(i / d, i % d);
                    *c = static_cast<int8_t>(quantize_rne(div_rn(static_cast<float>(*c) * old, now)));
                }
            for (uint32_t i = threadIdx.x; i < (to - from) * d; i += 256u) {
                const uint32_t slot = from + i / d, f = i % d;
                codes[place(slot, f)] =
                    static_cast<int8_t>(quantize_rne(div_rn(static_cast<float>(row(slot)[f]), now)));
            }
        }
    }
}

// One wave per query row and head, 64 keys at a time: lane l scores key l,
// then takes features l and l + 64 of the values.
template <typename E>
__global__ __launch_bounds__(64) void cache_attention_kernel(dav2_attention_cache_i8_args a) {
    __shared__ float qs[128], w[64];
    const uint32_t h = blockIdx.y, s = blockIdx.z, lane = threadIdx.x;
    const uint32_t d = a.cache.head_dim, page_size = a.cache.page_size;
    const uint32_t kvh = h / (a.heads / a.cache.kv_heads);
    const Sequence q = sequence_of(a.starts, a.lengths, s, a.tokens);
    const int64_t span = static_cast<int64_t>(a.table_pages) * page_size;
    for (int32_t row = q.begin + static_cast<int32_t>(blockIdx.x); row < q.end; row += gridDim.x) {
        int64_t seen = q.length;
        if (a.causal) seen = static_cast<int64_t>(q.length) - q.end + 1 + row;
        seen = max(min(seen, span), int64_t(0));
        const E* x = static_cast<const E*>(a.query) + static_cast<uint64_t>(row) * a.query_stride + uint64_t(h) * d;
        __syncthreads();
        for (uint32_t f = lane; f < d; f += 64u) qs[f] = static_cast<float>(x[f]) * a.scale;
        __syncthreads();
        float most = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
        for (int64_t j0 = 0; j0 < seen; j0 += 64) {
            const int64_t j = j0 + lane;
            auto page_of = [&](int64_t t) {
                return a.page_table[static_cast<uint64_t>(s) * a.table_pages + static_cast<uint64_t>(t / page_size)];
            };
            float score = -INFINITY;
            if (j < seen) {
                const int32_t page = page_of(j);
                if (page >= 0 && static_cast<uint32_t>(page) < a.cache.pages) {
                    const uint64_t plane = static_cast<uint64_t>(page) * a.cache.kv_heads + kvh;
                    const int8_t* k = a.cache.keys + (plane * page_size + static_cast<uint64_t>(j % page_size)) * d;
                    float dot = 0.0f;
                    for (uint32_t f = 0; f < d; ++f) dot = fmaf(qs[f], static_cast<float>(k[f]), dot);
                    score = dot * a.cache.key_scales[plane];
                }
            }
            const bool any = __ballot(score != -INFINITY) != 0;
            if (!any) continue;
            const float grown = fmaxf(most, wave_max(score));
            const float keep = most == -INFINITY ? 0.0f : expf(most - grown);
            const float weight = score == -INFINITY ? 0.0f : expf(score - grown);
            most = grown;
            sum = fmaf(sum, keep, wave_sum_tree(weight));
            o0 *= keep;
            o1 *= keep;
            __syncthreads();
            w[lane] = weight;
            __syncthreads();
            const uint32_t n = static_cast<uint32_t>(min(seen - j0, int64_t(64)));
            for (uint32_t i = 0; i < n; ++i) {
                const int32_t page = page_of(j0 + i);
                if (page < 0 || static_cast<uint32_t>(page) >= a.cache.pages) continue;
                const uint64_t plane = static_cast<uint64_t>(page) * a.cache.kv_heads + kvh;
                const int8_t* v = a.cache.values + plane * page_size * d + static_cast<uint64_t>((j0 + i) % page_size);
                const float ws = w[i] * a.cache.value_scales[plane];
                if (lane < d) o0 = fmaf(ws, static_cast<float>(v[lane * page_size]), o0);
                if (lane + 64u < d) o1 = fmaf(ws, static_cast<float>(v[(lane + 64u) * page_size]), o1);
            }
        }
        E* y = static_cast<E*>(a.output) + static_cast<uint64_t>(row) * a.output_stride + uint64_t(h) * d;
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (lane < d) y[lane] = static_cast<E>(o0 * inverse);
        if (lane + 64u < d) y[lane + 64u] = static_cast<E>(o1 * inverse);
    }
}

}  // namespace

extern "C" {

int dav2_hip_cache_store_i8(const dav2_cache_store_i8_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_cache_store_i8_args& a = *args;
    if (a.sequences == 0 || a.tokens == 0 || a.max_new == 0) return hipSuccess;
    const uint64_t row = static_cast<uint64_t>(a.cache.kv_heads) * a.cache.head_dim;
    if (!valid_cache(a.cache) || !a.keys || !a.values || !a.page_table || !a.starts || !a.lengths ||
        a.dtype > DAV2_DTYPE_BF16 || a.sequences > 65535u || a.tokens > 0x7fffffffu || a.table_pages == 0 ||
        a.table_pages > 0x7fffffffu || (a.tokens > 1 && (a.key_stride < row || a.value_stride < row)))
        return hipErrorInvalidValue;
    const uint64_t new_most = a.max_new < a.tokens ? a.max_new : a.tokens;
    uint64_t touched = (new_most + a.cache.page_size - 2) / a.cache.page_size + 1;
    if (touched > a.table_pages) touched = a.table_pages;
    const dim3 grid(static_cast<uint32_t>(touched), a.cache.kv_heads, a.sequences);
    with_dtype(a.dtype, [&](auto* e) {
        dispatch(cache_store_kernel<std::remove_pointer_t<decltype(e)>>, grid, dim3(256), 0,
                 static_cast<hipStream_t>(stream), a);
    });
    return hipGetLastError();
}

uint64_t dav2_hip_attention_cache_i8_scratch_bytes(const dav2_attention_cache_i8_args*) { return 0; }

int dav2_hip_attention_cache_i8(const dav2_attention_cache_i8_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_attention_cache_i8_args& a = *args;
    if (a.sequences == 0 || a.tokens == 0 || a.max_query == 0) return hipSuccess;
    const uint64_t row = static_cast<uint64_t>(a.heads) * a.cache.head_dim;
    if (!valid_cache(a.cache) || !a.query || !a.output || !aligned16(a.query) || !aligned16(a.output) ||
        !a.page_table || !a.starts || !a.lengths || a.dtype > DAV2_DTYPE_BF16 || a.sequences > 65535u ||
        a.tokens > 0x7fffffffu || a.table_pages == 0 || a.table_pages > 0x7fffffffu || a.heads == 0 ||
        a.heads > 65535u || a.heads % a.cache.kv_heads || a.query_stride % 8 || a.output_stride % 8 ||
        (a.tokens > 1 && (a.query_stride < row || a.output_stride < row)))
        return hipErrorInvalidValue;
    const uint64_t need = dav2_hip_attention_cache_i8_scratch_bytes(args);
    if (need && (!a.scratch || !aligned16(a.scratch) || a.scratch_bytes < need)) return hipErrorInvalidValue;
    const dim3 grid(a.max_query < a.tokens ? a.max_query : a.tokens, a.heads, a.sequences);
    with_dtype(a.dtype, [&](auto* e) {
        dispatch(cache_attention_kernel<std::remove_pointer_t<decltype(e)>>, grid, dim3(64), 0,
                 static_cast<hipStream_t>(stream), a);
    });
    return hipGetLastError();
}

}  // extern "C"
