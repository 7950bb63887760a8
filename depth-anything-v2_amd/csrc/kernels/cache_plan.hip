// What a step of a paged cache needs, from what its sequences hold and get:
// prefix sums over the sequences, then every row of the step on its own.

#include <algorithm>

#include "decoder.h"

using namespace dav2k;

namespace {

constexpr uint32_t kScanThreads = 1024;
// A step of up to so many sequences and rows is planned by one workgroup in one launch.
constexpr uint32_t kSmallSequences = 128, kSmallRows = 4096;

// What a row has to know of its sequence.
struct Record {
    int32_t held;   // tokens before the step
    int32_t front;  // which free page its first new one is; -1: it is not served
    int32_t given;  // pages that ended sequences before it give back, at most `pages`
    int32_t pages;  // that it gives back itself
};

struct Ring {
    uint32_t first, count, pages;
    DAV2_DEV uint32_t at(uint32_t i) const {  // i <= pages
        const uint32_t p = first + i;         // below 2^32, as pages is below 2^31
        return p >= pages ? p - pages : p;
    }
};
DAV2_DEV Ring ring_of(const dav2_cache_plan_args& a) {
    const uint32_t pages = a.pages;
    return {static_cast<uint32_t>(min(max(a.free_state[0], 0), static_cast<int32_t>(pages) - 1)),
            static_cast<uint32_t>(min(max(a.free_state[1], 0), static_cast<int32_t>(pages))), pages};
}

// The sums of u and v over the threads before this one, and over all THREADS.
template <uint32_t THREADS>
DAV2_DEV void sums_before(int64_t& u, int64_t& v, uint64_t* shared, int64_t& all_u, int64_t& all_v) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const int64_t upto_u = static_cast<int64_t>(wave_upto(static_cast<uint64_t>(u)));
    const int64_t upto_v = static_cast<int64_t>(wave_upto(static_cast<uint64_t>(v)));
    if constexpr (THREADS > 64) {
        __syncthreads();  // the sums before have been read
        if (lane == 63u) {
            shared[wave] = static_cast<uint64_t>(upto_u);
            shared[THREADS / 64u + wave] = static_cast<uint64_t>(upto_v);
        }
        __syncthreads();
        uint64_t all;
        u = static_cast<int64_t>(waves_before<THREADS / 64u>(shared, all)) + upto_u - u;
        all_u = static_cast<int64_t>(all);
        v = static_cast<int64_t>(waves_before<THREADS / 64u>(shared + THREADS / 64u, all)) + upto_v - v;
        all_v = static_cast<int64_t>(all);
    } else {
        all_u = static_cast<int64_t>(lane63(static_cast<uint64_t>(upto_u)));
        all_v = static_cast<int64_t>(lane63(static_cast<uint64_t>(upto_v)));
        u = upto_u - u;
        v = upto_v - v;
    }
}

struct Request {
    int64_t held, added;  // added below 0: the sequence ends
};
DAV2_DEV Request request_of(const dav2_cache_plan_args& a, uint32_t s) {
    return {max(a.held[s], 0), a.added[s]};
}
DAV2_DEV int64_t pages_for(int64_t tokens, uint32_t page_size) { return (tokens + page_size - 1) / page_size; }

// The sequences' sums by THREADS threads (all of a workgroup, or its first wave),
// a run of sequences for each: starts, lengths, held_out and the ring's state,
// and a record for each sequence. Behind them {first, count} of the ring as it
// was, which free_state_out may be. lds_starts: a copy of starts, or NULL.
template <uint32_t THREADS>
DAV2_DEV void plan_sequences(const dav2_cache_plan_args& a, Record* records, uint64_t* shared, int32_t* lds_starts) {
    const Ring ring = ring_of(a);
    const uint32_t per = (a.sequences + THREADS - 1u) / THREADS;
    const uint32_t s0 = min(threadIdx.x * per, a.sequences), s1 = min(s0 + per, a.sequences);
    const int64_t span = min(static_cast<int64_t>(a.table_pages) * a.page_size, int64_t(0x7fffffff));
    const Request only = request_of(a, min(s0, a.sequences - 1u));
    // each is asked for three times
    auto request = [&](uint32_t s) { return per == 1u ? only : request_of(a, s); };
    auto gives = [&](const Request& r) {
        return r.added < 0 ? min(pages_for(r.held, a.page_size), static_cast<int64_t>(a.table_pages)) : int64_t(0);
    };
    // the pages that a sequence needs, if its tokens and its rows fit
    auto needs = [&](const Request& r, int64_t end) -> int64_t {
        if (r.added < 0 || r.held + r.added > span || end > static_cast<int64_t>(a.tokens)) return -1;
        return pages_for(r.held + r.added, a.page_size) - pages_for(r.held, a.page_size);
    };
    int64_t row0 = 0, given = 0, rows_all, given_all;
    for (uint32_t s = s0; s < s1; ++s) {
        const Request r = request(s);
        row0 += max(r.added, int64_t(0));
        given += gives(r);
    }
    sums_before<THREADS>(row0, given, shared, rows_all, given_all);
    int64_t taken = 0, rows = row0, nothing = 0, need_all, none;
    for (uint32_t s = s0; s < s1; ++s) {
        const Request r = request(s);
        rows += max(r.added, int64_t(0));
        taken += max(needs(r, rows), int64_t(0));
    }
    sums_before<THREADS>(taken, nothing, shared, need_all, none);
    rows = row0;
    uint64_t used = 0;  // pages taken after this thread's sequences
    for (uint32_t s = s0; s < s1; ++s) {
        const Request r = request(s);
        const int32_t start = static_cast<int32_t>(min(rows, static_cast<int64_t>(a.tokens)));
        a.starts[s] = start;
        if (lds_starts) lds_starts[s] = start;
        rows += max(r.added, int64_t(0));
        const int64_t n = needs(r, rows);
        const bool served = n == 0 || (n > 0 && taken + n <= ring.count);
        records[s] = {static_cast<int32_t>(r.held), served ? static_cast<int32_t>(min(taken, int64_t(0x7fffffff))) : -1,
                      static_cast<int32_t>(min(given, static_cast<int64_t>(ring.pages))), static_cast<int32_t>(gives(r))};
        if (n > 0) taken += n;
        // all that are served come before any that is not
        if (served && n > 0) used += static_cast<uint64_t>(n);
        given += gives(r);
        a.lengths[s] = served ? static_cast<int32_t>(r.held + r.added) : 0;
        a.held_out[s] = r.added < 0 ? 0 : static_cast<int32_t>(served ? r.held + r.added : r.held);
    }
    int64_t used_before = static_cast<int64_t>(used), used_all;
    sums_before<THREADS>(used_before, nothing, shared, used_all, none);
    if (threadIdx.x == 0) {
        const int32_t end = static_cast<int32_t>(min(rows_all, static_cast<int64_t>(a.tokens)));
        a.starts[a.sequences] = end;
        if (lds_starts) lds_starts[a.sequences] = end;
        records[a.sequences].held = static_cast<int32_t>(ring.first);
        records[a.sequences].front = static_cast<int32_t>(ring.count);
        records[a.sequences].given = static_cast<int32_t>(min(given_all, static_cast<int64_t>(ring.pages)));
        const int64_t room = ring.pages - ring.count;
        a.free_state_out[0] = static_cast<int32_t>((ring.first + used_all) % ring.pages);
        a.free_state_out[1] = static_cast<int32_t>(ring.count - used_all + min(given_all, room));
    }
}

typedef int32_t i4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef int64_t l2_any __attribute__((ext_vector_type(2), aligned(8)));

// Four rows of the step's `end` from `row` on, whose sequences are in [low, high].
// starts and records: of the sequences from `origin` on.
DAV2_DEV void plan_rows(const dav2_cache_plan_args& a, const Ring& ring, const int32_t* starts, const Record* records,
                        uint32_t origin, uint32_t row, uint32_t end, uint32_t low, uint32_t high) {
    low -= origin;
    high -= origin;
    // the last sequence that starts at or before the row
    while (low < high) {
        const uint32_t mid = (low + high + 1u) / 2u;
        if (static_cast<uint32_t>(starts[mid]) <= row) low = mid;
        else high = mid - 1u;
    }
    Record r = records[low];
    uint32_t begin = static_cast<uint32_t>(starts[low]), next = static_cast<uint32_t>(starts[low + 1u]);
    const uint32_t size = a.page_size;
    i4_any position = {0, 0, 0, 0}, owner = {-1, -1, -1, -1};
    int64_t slot[4] = {-1, -1, -1, -1};
    uint32_t within[4];
    bool served[4], fresh[4];
    int32_t *entry[4], page[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        served[i] = fresh[i] = false;
        within[i] = 0;
        entry[i] = a.free_pages;  // what may be read
        if (row + i >= end) continue;
        while (row + i >= next) {
            ++low;
            begin = next;
            next = static_cast<uint32_t>(starts[low + 1u]);
            r = records[low];
        }
        const int64_t at = static_cast<int64_t>(r.held) + (row + i - begin);
        position[i] = static_cast<int32_t>(min(at, int64_t(0x7fffffff)));
        owner[i] = static_cast<int32_t>(low + origin);
        if (r.front < 0) continue;
        const uint32_t p = static_cast<uint32_t>(at), place = p / size;
        const uint32_t owned = (static_cast<uint32_t>(r.held) + size - 1u) / size;
        within[i] = p - place * size;
        served[i] = true;
        fresh[i] = place >= owned;
        entry[i] = fresh[i] ? a.free_pages + ring.at(static_cast<uint32_t>(r.front) + place - owned)
                            : a.page_table + static_cast<uint64_t>(low + origin) * a.table_pages + place;
    }
    // the pages of all four together
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) page[i] = *entry[i];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        if (!served[i]) continue;
        if (fresh[i] && within[i] == 0)
            a.page_table[static_cast<uint64_t>(owner[i]) * a.table_pages + static_cast<uint32_t>(position[i]) / size] = page[i];
        if (page[i] >= 0 && static_cast<uint32_t>(page[i]) < a.pages) slot[i] = static_cast<int64_t>(page[i]) * size + within[i];
    }
    if (row + 4u <= a.tokens) {
        if (a.positions) *reinterpret_cast<i4_any*>(a.positions + row) = position;
        if (a.owners) *reinterpret_cast<i4_any*>(a.owners + row) = owner;
        if (a.slots) {
            *reinterpret_cast<l2_any*>(a.slots + row) = l2_any{slot[0], slot[1]};
            *reinterpret_cast<l2_any*>(a.slots + row + 2) = l2_any{slot[2], slot[3]};
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        if (row + i >= a.tokens) break;
        if (a.positions) a.positions[row + i] = position[i];
        if (a.owners) a.owners[row + i] = owner[i];
        if (a.slots) a.slots[row + i] = slot[i];
    }
}

// What an ended sequence gives back, by a wave.
DAV2_DEV void plan_given(const dav2_cache_plan_args& a, const Ring& ring, const Record& r, uint32_t s, uint32_t lane) {
    const uint32_t room = ring.pages - ring.count, given = static_cast<uint32_t>(r.given);
    const uint32_t n = given >= room ? 0u : min(static_cast<uint32_t>(r.pages), room - given);
    const int32_t* const from = a.page_table + static_cast<uint64_t>(s) * a.table_pages;
    for (uint32_t i0 = lane; i0 < n; i0 += 8u * 64u) {
        int32_t page[8];  // on their way together
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) page[i] = from[min(i0 + 64u * i, n - 1u)];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (i0 + 64u * i < n) a.free_pages[ring.at(ring.count + given + i0 + 64u * i)] = page[i];
    }
}

// Both in one workgroup: the records stay in LDS, and starts beside them for the
// search. Up to 64 sequences are one wave's, which waits for nobody. us, against two
// launches: 48 sequences of a token each 6.2 / 9.4, 16 of 128 rows 5.6 / 9.2, 128 of a
// token 9.7 / 10.0.
constexpr uint32_t kSmallThreads = 512;
template <bool WAVE>
__global__ __launch_bounds__(kSmallThreads) void plan_small_kernel(dav2_cache_plan_args a) {
    __shared__ uint64_t shared[2 * kSmallThreads / 64];
    __shared__ Record records[kSmallSequences + 1];
    __shared__ int32_t starts[kSmallSequences + 1];
    if constexpr (!WAVE) plan_sequences<kSmallThreads>(a, records, shared, starts);
    else if (threadIdx.x < 64u) plan_sequences<64>(a, records, shared, starts);
    __syncthreads();
    const Ring ring = {static_cast<uint32_t>(records[a.sequences].held), static_cast<uint32_t>(records[a.sequences].front),
                       a.pages};
    for (uint32_t row = 4u * threadIdx.x; row < a.tokens; row += 4u * kSmallThreads)
        plan_rows(a, ring, starts, records, 0u, row, static_cast<uint32_t>(starts[a.sequences]), 0u, a.sequences - 1u);
    // page by page, as a wave for each sequence would have them one after the other
    const uint32_t given = min(static_cast<uint32_t>(records[a.sequences].given), ring.pages - ring.count);
    for (uint32_t i = threadIdx.x; i < given; i += kSmallThreads) {
        uint32_t low = 0, high = a.sequences - 1u;  // the last sequence before which no more are given
        while (low < high) {
            const uint32_t mid = (low + high + 1u) / 2u;
            if (static_cast<uint32_t>(records[mid].given) <= i) low = mid;
            else high = mid - 1u;
        }
        a.free_pages[ring.at(ring.count + i)] =
            a.page_table[static_cast<uint64_t>(low) * a.table_pages + i - static_cast<uint32_t>(records[low].given)];
    }
}

__global__ __launch_bounds__(kScanThreads) void plan_sequences_kernel(dav2_cache_plan_args a) {
    __shared__ uint64_t shared[2 * kScanThreads / 64];
    plan_sequences<kScanThreads>(a, static_cast<Record*>(a.scratch), shared, nullptr);
}

// A workgroup has 1024 rows. Two of its waves find their first and last
// sequences, whose starts and records then go into LDS, unless sequences without
// rows make them too many.
__global__ __launch_bounds__(256) void plan_rows_kernel(dav2_cache_plan_args a, uint32_t row_groups) {
    constexpr uint32_t kMost = 1056;
    __shared__ int32_t starts[kMost + 1];
    __shared__ Record held[kMost];
    __shared__ uint32_t ends[2];
    const Record* records = static_cast<const Record*>(a.scratch);
    const Record last = records[a.sequences];
    const Ring ring = {static_cast<uint32_t>(last.held), static_cast<uint32_t>(last.front), a.pages};
    if (blockIdx.x < row_groups) {
        const uint32_t end = static_cast<uint32_t>(a.starts[a.sequences]);
        for (uint64_t row0 = static_cast<uint64_t>(blockIdx.x) * 1024u; row0 < a.tokens;
             row0 += static_cast<uint64_t>(row_groups) * 1024u) {
            const uint32_t first = static_cast<uint32_t>(row0), row = first + 4u * threadIdx.x;
            __syncthreads();  // the rows before are done
            if (first < end && threadIdx.x < 128u) {
                const uint32_t wave = threadIdx.x >> 6, of = wave ? min(first + 1023u, end - 1u) : first;
                const uint32_t s = first_where(0u, a.sequences - 1u, [&](uint32_t i) {
                    return static_cast<uint32_t>(a.starts[i + 1u]) > of;
                });
                if ((threadIdx.x & 63u) == 0) ends[wave] = s;
            } else if (threadIdx.x < 2u) {
                ends[threadIdx.x] = a.sequences - 1u;
            }
            __syncthreads();
            const uint32_t low = ends[0], high = ends[1], n = high - low + 1u;
            if (n > kMost) {
                if (row < a.tokens) plan_rows(a, ring, a.starts, records, 0u, row, end, low, high);
                continue;
            }
            for (uint32_t i = threadIdx.x; i <= n; i += 256u) {
                starts[i] = a.starts[low + i];
                if (i < n) held[i] = records[low + i];
            }
            __syncthreads();
            if (row < a.tokens) plan_rows(a, ring, starts, held, low, row, end, low, high);
        }
    } else {
        const uint32_t s = (blockIdx.x - row_groups) * 4u + (threadIdx.x >> 6);
        if (s < a.sequences) plan_given(a, ring, records[s], s, threadIdx.x & 63u);
    }
}

}  // namespace

extern "C" {

uint64_t dav2_hip_cache_plan_scratch_bytes(const dav2_cache_plan_args* args) {
    return args ? (static_cast<uint64_t>(args->sequences) + 1u) * sizeof(Record) : 0;
}

int dav2_hip_cache_plan(const dav2_cache_plan_args* args, void* stream) {
    if (!args) return hipErrorInvalidValue;
    const dav2_cache_plan_args& a = *args;
    if (a.sequences == 0) return hipSuccess;
    if (!a.held || !a.added || !a.page_table || !a.free_pages || !a.free_state || !a.held_out || !a.free_state_out ||
        !a.starts || !a.lengths || a.sequences > 65535u || a.table_pages == 0 || a.table_pages > 0x7fffffffu ||
        a.tokens > 0x7fffffffu || a.pages == 0 || a.pages > 0x7fffffffu || a.page_size < 16 || a.page_size > 256 ||
        a.page_size % 16 || !a.scratch || !aligned16(a.scratch) ||
        a.scratch_bytes < dav2_hip_cache_plan_scratch_bytes(args))
        return hipErrorInvalidValue;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.sequences <= kSmallSequences && a.tokens <= kSmallRows) {
        dispatch(a.sequences <= 64u ? plan_small_kernel<true> : plan_small_kernel<false>, dim3(1), dim3(kSmallThreads), 0, s, a);
        return hipGetLastError();
    }
    dispatch(plan_sequences_kernel, dim3(1), dim3(kScanThreads), 0, s, a);
    const uint32_t row_groups = static_cast<uint32_t>(std::min<uint64_t>((static_cast<uint64_t>(a.tokens) + 1023u) / 1024u, 1u << 20));
    dispatch(plan_rows_kernel, dim3(row_groups + (a.sequences + 3u) / 4u), dim3(256), 0, s, a, row_groups);
    return hipGetLastError();
}

}  // extern "C"
