// Shared by the paged caches' kernels (cache_i8.hip, cache_i4.hip): the place of
// a token in its pages, the weights' second part and the values' scales.
#pragma once

#include "decoder.h"

namespace dav2k {

// A score past kFar is rounded to more than the exponentials' range has room
// for, and the weights' bias would be lost beside it: the base is then the
// maximum itself.
constexpr float kFar = 1048576.0f;
constexpr float kSecond = 2048.0f;  // what the second part is multiplied by
DAV2_DEV h8 for_second(h8 codes) { return codes * static_cast<_Float16>(1.0f / kSecond); }

// Page and slot of a 16-token chunk; magic = ceil(2^32 / chunks per page),
// which divides every chunk below 2^28 exactly (2 to 16 chunks per page). For
// one chunk per page that is 0 in 32 bits, and alone adds the chunk itself.
struct Pages {
    const int32_t* table;  // of one sequence
    uint32_t table_pages, pages, per_page, magic, alone;
    struct Place {
        uint32_t index, slot;  // of the page in the table, of the chunk in the page
        int32_t entry;
    };
    // A chunk's place; the entry's load is not waited for here.
    DAV2_DEV Place find(uint32_t chunk) const {
        Place p;
        p.index = __umulhi(chunk, magic) + (chunk & alone);
        p.slot = (chunk - p.index * per_page) * 16u;
        p.entry = table[min(p.index, table_pages - 1u)];
        return p;
    }
    DAV2_DEV bool exists(const Place& p) const {
        return p.index < table_pages && static_cast<uint32_t>(p.entry) < pages;
    }
    // the page, or one that may be read in its place
    DAV2_DEV uint32_t page(const Place& p) const { return exists(p) ? static_cast<uint32_t>(p.entry) : 0u; }
};

template <typename Args>
DAV2_DEV Pages pages_of(const Args& a, uint32_t s) {
    const uint32_t per_page = a.cache.page_size / 16u;
    return {a.page_table + static_cast<uint64_t>(s) * a.table_pages, a.table_pages, a.cache.pages, per_page,
            static_cast<uint32_t>(((1ull << 32) + per_page - 1u) / per_page), per_page == 1 ? ~0u : 0u};
}

// A value scale as 2^e f. Below 2^-80 (zeros with a scale of 0) 2^-80 stands in:
// the sum of w 2^-e, of up to 2^31 weights of 2^15, stays finite. Infinity and
// NaN make f NaN.
DAV2_DEV void split_scale(float scale, float& exponent, float& fraction, float& inverse) {
    const uint32_t bits = max(__float_as_uint(scale) & 0x7fffffffu, 47u << 23);
    const int e = static_cast<int>(bits >> 23) - 127;
    exponent = static_cast<float>(e);
    fraction = bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u)
                                   : __uint_as_float((bits & 0x007fffffu) | 0x3f800000u);
    inverse = ldexpf(1.0f, -e);
}

// The splits of a sequence's rows joined: the sequence blockIdx.y, the rows from blockIdx.x on.
template <typename E, int FEW, typename Args>
DAV2_DEV void join_sequence(const Args& a, const Parts& parts, uint32_t splits) {
    const Sequence q = sequence_of(a.starts, a.lengths, blockIdx.y, a.tokens);
    const uint64_t rows = static_cast<uint64_t>(q.end - q.begin) * a.heads;
    const uint32_t d = a.cache.head_dim, heads = a.heads;
    auto token = [&](uint64_t r) { return q.begin + static_cast<uint64_t>(static_cast<uint32_t>(r) / heads); };
    auto head = [&](uint64_t r) { return static_cast<uint64_t>(static_cast<uint32_t>(r) % heads); };
    auto output = [&](uint64_t r) { return static_cast<E*>(a.output) + token(r) * a.output_stride + head(r) * d; };
    auto slot = [&](uint64_t r) { return (token(r) * heads + head(r)) * splits; };
    if constexpr (FEW > 0) {
        const uint32_t lanes = join_lanes_log2(d), each = 256u >> lanes, f4 = threadIdx.x & ((1u << lanes) - 1u);
        for (uint64_t r = static_cast<uint64_t>(blockIdx.x) * each + (threadIdx.x >> lanes); r < rows;
             r += static_cast<uint64_t>(gridDim.x) * each)
            join_few<FEW>(parts, slot(r), splits, d, f4, output(r));
    } else {
        for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) join_row(parts, slot(r), splits, d, output(r));
    }
}
struct JoinLaunch {
    int few;  // of join_kind
    dim3 grid;
};
template <typename Args>
JoinLaunch join_launch(const Args& a, uint32_t splits) {
    const uint64_t rows = static_cast<uint64_t>(a.max_query < a.tokens ? a.max_query : a.tokens) * a.heads;
    const int few = join_kind(rows * a.sequences, splits);
    const uint64_t each = few ? join_rows(a.cache.head_dim) : 1, groups = (rows + each - 1) / each;
    return {few, dim3(static_cast<uint32_t>(groups < 4096 ? groups : 4096), a.sequences)};
}

}  // namespace dav2k
