// What the kernels over a paged cache share: the batch's description and how a row of packed tokens finds its sequence
// and its position.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/flash_colsum_b200.h"
#include "sm100_ptx.cuh"

namespace fcs {
namespace paged {

// Sequence b holds lens[b] tokens, of which rows starts[b] .. starts[b + 1] of the packed tokens are the last (without
// `starts`: row b alone).  Page i of sequence b is entry i of row b of the table.
struct Batch {
    const int* table;
    long long table_ld;
    const int* lens;
    const int* starts;          // or nullptr
    int pages, kv_heads, page_shift, dim;
    int sequences, width, tokens;
    int* status;                // or nullptr
};

__device__ __forceinline__ void report(const Batch& c, int code) {
    if (c.status) atomicCAS(c.status, 0, code);
}

// How many of 0 .. n - 1 come before the first for which `before` is false, by a converged warp: 32 of them looked at at a time.
template <typename F>
__device__ __forceinline__ int count_before(int n, F before) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32;
        const long long first = lo + (long long)lane * step;
        const int whole = __popc(__ballot_sync(0xffffffffu, first < hi && before((int)min(first + step, (long long)hi) - 1)));
        lo = min(hi, lo + whole * step);
        if (lo < hi) hi = min(hi, lo + step) - 1;     // (the last of the next ones is not)
    }
    return lo;
}

// Sequence of row `t`, by a converged warp; `sequences` for a row behind the last one.
__device__ __forceinline__ int sequence_of(const Batch& c, int t) {
    if (!c.starts) return t;
    return count_before(c.sequences, [&](int i) { return c.starts[i + 1] <= t; });
}

// Position of row `t` of sequence `b` (negative where lens[b] counts fewer tokens than the sequence has rows).
__device__ __forceinline__ long long position_of(const Batch& c, int b, int t) {
    const long long len = c.lens[b];
    return c.starts ? len - c.starts[b + 1] + t : len - 1;
}

// The page of the pools that holds page `i` of sequence `b`, or -1 (said in the status word) where the table has none.
__device__ __forceinline__ int physical_page(const Batch& c, int b, long long i) {
    if (i >= 0 && i < c.width) {
        const int page = c.table[b * c.table_ld + i];
        if (page >= 0 && page < c.pages) return page;
    }
    report(c, FCS_STATUS_BAD_PAGE);
    return -1;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

}  // namespace paged
}  // namespace fcs
