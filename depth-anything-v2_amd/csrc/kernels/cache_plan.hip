// What a step of a paged cache needs, from what its sequences hold and get:
// prefix sums over the sequences, then every row of the step on its own.

#include <algorithm>

#include "decoder.h"

using namespace dav2k;

namespace {

constexpr uint32_t kScanThreads = 1024;

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

// The sum of v over the threads before this one, and over all of the workgroup.
DAV2_DEV int64_t sum_before(int64_t v, int64_t* shared, int64_t& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    int64_t upto = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t other = __shfl_up(upto, o, kWave);
        if (lane >= static_cast<uint32_t>(o)) upto += other;
    }
    __syncthreads();  // the sums before have been read
    if (lane == 63u) shared[wave] = upto;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kScanThreads / 64u; ++w) {
        const int64_t of_wave = shared[w];
        before += w < wave ? of_wave : 0;
        total += of_wave;
    }
    return before + upto - v;
}

struct Request {
    int64_t held, added;  // added below 0: the sequence ends
};
DAV2_DEV Request request_of(const dav2_cache_plan_args& a, uint32_t s) {
    return {max(a.held[s], 0), a.added[s]};
}
DAV2_DEV int64_t pages_for(int64_t tokens, uint32_t page_size) { return (tokens + page_size - 1) / page_size; }

// The sequences' sums by one workgroup, a run of sequences for each thread:
// starts, lengths, held_out and the ring's state, and a record for each sequence.
// Behind them {first, count} of the ring as it was, which free_state_out may be.
DAV2_DEV void plan_sequences(const dav2_cache_plan_args& a, Record* records, int64_t* shared) {
    const Ring ring = ring_of(a);
    const uint32_t per = (a.sequences + kScanThreads - 1u) / kScanThreads;
    const uint32_t s0 = min(threadIdx.x * per, a.sequences), s1 = min(s0 + per, a.sequences);
    const int64_t span = static_cast<int64_t>(a.table_pages) * a.page_size;
    int64_t rows = 0, given = 0, rows_all, given_all, need_all;
    auto gives = [&](const Request& r) {
        return r.added < 0 ? min(pages_for(r.held, a.page_size), static_cast<int64_t>(a.table_pages)) : int64_t(0);
    };
    for (uint32_t s = s0; s < s1; ++s) {
        const Request r = request_of(a, s);
        rows += max(r.added, int64_t(0));
        given += gives(r);
    }
    const int64_t row0 = sum_before(rows, shared, rows_all);
    const int64_t given0 = sum_before(given, shared, given_all);
    // the pages that a sequence needs, if its tokens and its rows fit
    auto needs = [&](const Request& r, int64_t end) -> int64_t {
        if (r.added < 0 || r.held + r.added > min(span, int64_t(0x7fffffff)) || end > static_cast<int64_t>(a.tokens))
            return -1;
        return pages_for(r.held + r.added, a.page_size) - pages_for(r.held, a.page_size);
    };
    int64_t need = 0;
    rows = row0;
    for (uint32_t s = s0; s < s1; ++s) {
        const Request r = request_of(a, s);
        rows += max(r.added, int64_t(0));
        need += max(needs(r, rows), int64_t(0));
    }
    int64_t taken = sum_before(need, shared, need_all);
    rows = row0;
    given = given0;
    int64_t used = 0;  // after the last sequence of this thread that is served
    for (uint32_t s = s0; s < s1; ++s) {
        const Request r = request_of(a, s);
        a.starts[s] = static_cast<int32_t>(min(rows, static_cast<int64_t>(a.tokens)));
        rows += max(r.added, int64_t(0));
        const int64_t n = needs(r, rows);
        const bool served = n == 0 || (n > 0 && taken + n <= ring.count);
        records[s] = {static_cast<int32_t>(r.held), served ? static_cast<int32_t>(min(taken, int64_t(0x7fffffff))) : -1,
                      static_cast<int32_t>(min(given, static_cast<int64_t>(ring.pages))), static_cast<int32_t>(gives(r))};
        if (n > 0) taken += n;
        if (served && n > 0) used = taken;
        given += gives(r);
        a.lengths[s] = served ? static_cast<int32_t>(r.held + r.added) : 0;
        a.held_out[s] = r.added < 0 ? 0 : static_cast<int32_t>(served ? r.held + r.added : r.held);
    }
    if (threadIdx.x == 0) {
        a.starts[a.sequences] = static_cast<int32_t>(min(rows_all, static_cast<int64_t>(a.tokens)));
        records[a.sequences].held = static_cast<int32_t>(ring.first);
        records[a.sequences].front = static_cast<int32_t>(ring.count);
    }
    // the pages taken are those up to the last sequence served
    for (int o = 32; o > 0; o >>= 1) used = max(used, __shfl_xor(used, o, kWave));
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) shared[threadIdx.x >> 6] = used;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 0; w < kScanThreads / 64u; ++w) used = max(used, shared[w]);
        const int64_t room = ring.pages - ring.count;
        a.free_state_out[0] = static_cast<int32_t>((ring.first + used) % ring.pages);
        a.free_state_out[1] = static_cast<int32_t>(ring.count - used + min(given_all, room));
    }
}

// One row of the step. starts: of the step's rows.
DAV2_DEV void plan_row(const dav2_cache_plan_args& a, const Ring& ring, const int32_t* starts, const Record* records,
                       uint32_t row, uint32_t low, uint32_t high) {
    int32_t position = 0, owner = -1;
    int64_t slot = -1;
    if (row < static_cast<uint32_t>(starts[a.sequences])) {
        // the last sequence in [low, high] that starts at or before the row
        while (low < high) {
            const uint32_t mid = (low + high + 1u) / 2u;
            if (static_cast<uint32_t>(starts[mid]) <= row) low = mid;
            else high = mid - 1u;
        }
        const Record r = records[low];
        const int64_t at = static_cast<int64_t>(r.held) + (row - static_cast<uint32_t>(starts[low]));
        position = static_cast<int32_t>(min(at, int64_t(0x7fffffff)));
        owner = static_cast<int32_t>(low);
        if (r.front >= 0) {
            const uint32_t p = static_cast<uint32_t>(at), size = a.page_size;
            const uint32_t place = p / size, within = p - place * size;
            const uint32_t owned = (static_cast<uint32_t>(r.held) + size - 1u) / size;
            int32_t* const entry = a.page_table + static_cast<uint64_t>(low) * a.table_pages + place;
            int32_t page;
            if (place >= owned) {
                page = a.free_pages[ring.at(static_cast<uint32_t>(r.front) + place - owned)];
                if (within == 0) *entry = page;
            } else {
                page = *entry;
            }
            if (page >= 0 && static_cast<uint32_t>(page) < a.pages) slot = static_cast<int64_t>(page) * size + within;
        }
    }
    if (a.positions) a.positions[row] = position;
    if (a.owners) a.owners[row] = owner;
    if (a.slots) a.slots[row] = slot;
}

// What an ended sequence gives back, by a wave.
DAV2_DEV void plan_given(const dav2_cache_plan_args& a, const Ring& ring, const Record& r, uint32_t s, uint32_t lane) {
    const uint32_t room = ring.pages - ring.count;
    for (uint32_t i = lane; i < static_cast<uint32_t>(r.pages); i += 64u) {
        const uint32_t to = static_cast<uint32_t>(r.given) + i;
        if (to >= room) break;
        a.free_pages[ring.at(ring.count + to)] = a.page_table[static_cast<uint64_t>(s) * a.table_pages + i];
    }
}

__global__ __launch_bounds__(kScanThreads) void plan_sequences_kernel(dav2_cache_plan_args a) {
    __shared__ int64_t shared[kScanThreads / 64];
    plan_sequences(a, static_cast<Record*>(a.scratch), shared);
}

__global__ __launch_bounds__(256) void plan_rows_kernel(dav2_cache_plan_args a, uint32_t row_groups) {
    const Record* records = static_cast<const Record*>(a.scratch);
    const Record last = records[a.sequences];
    const Ring ring = {static_cast<uint32_t>(last.held), static_cast<uint32_t>(last.front), a.pages};
    if (blockIdx.x < row_groups) {
        for (uint64_t row = static_cast<uint64_t>(blockIdx.x) * 256u + threadIdx.x; row < a.tokens;
             row += static_cast<uint64_t>(row_groups) * 256u)
            plan_row(a, ring, a.starts, records, static_cast<uint32_t>(row), 0u, a.sequences - 1u);
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
    dispatch(plan_sequences_kernel, dim3(1), dim3(kScanThreads), 0, s, a);
    const uint32_t row_groups = static_cast<uint32_t>(std::min<uint64_t>((static_cast<uint64_t>(a.tokens) + 255u) / 256u, 1u << 20));
    dispatch(plan_rows_kernel, dim3(row_groups + (a.sequences + 3u) / 4u), dim3(256), 0, s, a, row_groups);
    return hipGetLastError();
}

}  // extern "C"
