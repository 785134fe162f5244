// Choosing pages: per query and key/value head the k pages whose bounds promise the largest scores.
//
// The mathematics: over the keys of a page q . k <= sum_d max(q_d low_d, q_d high_d); summed over the queries of a group
// that is p . high - n . low with p = sum max(q, 0) and n = sum max(-q, 0), one product of 2 D terms for the whole
// group.  The first and the last pages of a query are always chosen; of the others the best, the lower page among
// equals.  Which of two pages is the better one must not hang on the order of a sum, so the scores are summed in 64 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.cuh"

namespace fcs {
namespace paged {

struct SelectParams {
    Batch c;
    const uint16_t* query;
    const uint16_t* bounds;         // (pages, kv_heads, 2, dim)
    long long query_st[2];          // token, head
    int group;                      // query heads of a key/value head
    int k, first, last;
    int* chosen;                    // (tokens, kv_heads, k)
    double* scores;                 // (tokens of this launch, kv_heads, width)
    int t0;                         // first token of this launch
    int fill_tail;
};

constexpr int SCORE_THREADS = 256;
constexpr int SCORE_PAGES = 64;     // pages of a CTA: eight of a warp

template <bool BF16>
__device__ __forceinline__ float widen16(uint32_t v) {     // (the low half of v)
    if constexpr (BF16) return __uint_as_float(v << 16);
    return __half2float(__ushort_as_half((unsigned short)v));
}

// Pages that the query at `pos` sees (all of them, whether the table holds them or not).
__device__ __forceinline__ long long pages_seen(const Batch& c, long long pos) {
    return pos < 0 ? 0 : (pos >> c.page_shift) + 1;
}

// grid: (page chunks, kv heads, tokens)
template <bool BF16>
__global__ void __launch_bounds__(SCORE_THREADS) score_kernel(const __grid_constant__ SelectParams p) {
    grid_dependency_wait();
    grid_launch_dependents();
    const Batch& c = p.c;
    const int D = c.dim, h = blockIdx.y, t = p.t0 + (int)blockIdx.z;
    const int b = sequence_of(c, t);
    if (b >= c.sequences) return;
    const long long seen = min(pages_seen(c, position_of(c, b, t)), (long long)c.width);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int base = (int)blockIdx.x * SCORE_PAGES + warp * (SCORE_PAGES / 8);
    if (base >= seen) return;

    // A lane keeps eight of the 2 D features -- the first D meet the lows, the others the highs; 2 D / 8 lanes or
    // the next power of two hold a page, and a warp as many pages at a time as fit.
    const int vectors = D / 4;
    int span = 2;
    while (span < vectors) span *= 2;
    const int v = lane & (span - 1);
    double part[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) part[i] = 0.0;
    if (v < vectors) {
        const bool low = v < vectors / 2;
        const uint16_t* q = p.query + t * p.query_st[0] + (long long)h * p.group * p.query_st[1] + (low ? v : v - vectors / 2) * 8;
        for (int g = 0; g < p.group; ++g, q += p.query_st[1]) {
            const uint4 w = *reinterpret_cast<const uint4*>(q);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double x = widen16<BF16>(i & 1 ? words[i / 2] >> 16 : words[i / 2] & 0xffffu);
                part[i] += (low ? x < 0.0 : !(x < 0.0)) ? x : 0.0;      // (NaN stays)
            }
        }
    }
    double* out = p.scores + ((long long)blockIdx.z * c.kv_heads + h) * c.width;
    const int at_once = 32 / span;
    for (int i = 0; i < SCORE_PAGES / 8; i += at_once) {
        const int page = base + i + lane / span;
        const bool take = page < seen && page < base + SCORE_PAGES / 8;
        const int at = take ? physical_page(c, b, page) : -1;
        double score = 0.0;
        if (at >= 0 && v < vectors) {
            const uint4 w = *reinterpret_cast<const uint4*>(p.bounds + ((long long)at * c.kv_heads + h) * 2 * D + v * 8);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                score += part[e] * (double)widen16<BF16>(e & 1 ? words[e / 2] >> 16 : words[e / 2] & 0xffffu);
        }
        for (int o = span / 2; o > 0; o >>= 1) score += __shfl_xor_sync(0xffffffffu, score, o);
        if (take && v == 0) out[page] = at < 0 ? -INFINITY : score != score ? INFINITY : score;
    }
}

// Larger score, larger key.
__device__ __forceinline__ unsigned long long key_of_score(double s) {
    const long long bits = __double_as_longlong(s == 0.0 ? 0.0 : s);     // (zeros of both signs are equal)
    return bits < 0 ? ~(unsigned long long)bits : (unsigned long long)bits | 0x8000000000000000ull;
}

constexpr int CHOOSE_THREADS = 256;
constexpr int DIGIT_BITS = 11, DIGITS = 1 << DIGIT_BITS;

// Exclusive scan of one count per thread; `total` is the block's.
__device__ __forceinline__ uint32_t scan_block(uint32_t v, uint32_t* warp_sums, uint32_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < CHOOSE_THREADS / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    return before + inc - v;
}

// A CTA per (token, kv head): radix selection over the 64-bit keys of the scores, 11 bits at a time from the top.
__global__ void __launch_bounds__(CHOOSE_THREADS) choose_kernel(const __grid_constant__ SelectParams p) {
    __shared__ uint32_t bins[DIGITS];
    __shared__ uint32_t warp_sums[CHOOSE_THREADS / 32];
    __shared__ uint32_t found[3];
    grid_dependency_wait();
    grid_launch_dependents();
    const Batch& c = p.c;
    const int tid = threadIdx.x, h = blockIdx.x, t = p.t0 + (int)blockIdx.y;
    int* out = p.chosen + ((long long)t * c.kv_heads + h) * p.k;
    const int b = sequence_of(c, t);
    if (b >= c.sequences) {
        if (p.fill_tail)
            for (int i = tid; i < p.k; i += CHOOSE_THREADS) out[i] = -1;
        return;
    }
    const long long seen = pages_seen(c, position_of(c, b, t));
    const int pages = (int)min(seen, (long long)c.width);
    if (pages <= p.k) {
        for (int i = tid; i < p.k; i += CHOOSE_THREADS) out[i] = i < pages ? i : -1;
        return;
    }
    const int lo = min(p.first, pages), hi = (int)max((long long)lo, min((long long)pages, seen - p.last));   // candidates
    uint32_t need = (uint32_t)max(0, p.k - lo - (pages - hi));
    const double* scores = p.scores + ((long long)blockIdx.y * c.kv_heads + h) * c.width;

    // the smallest key chosen, as a prefix of `bits` bits; `need`: how many with exactly that prefix
    unsigned long long prefix = 0;
    int bits = 0;
    uint32_t equal = (uint32_t)(hi - lo);
    while (need < equal && need > 0 && bits < 64) {
        const int width = min(DIGIT_BITS, 64 - bits), shift = 64 - bits - width;
        __syncthreads();
        for (int i = tid; i < DIGITS; i += CHOOSE_THREADS) bins[i] = 0;
        __syncthreads();
        for (int i = lo + tid; i < hi; i += CHOOSE_THREADS) {
            const unsigned long long key = key_of_score(scores[i]);
            if (bits == 0 || key >> (64 - bits) == prefix) atomicAdd(&bins[(uint32_t)(key >> shift) & ((1u << width) - 1)], 1u);
        }
        __syncthreads();
        // from the top: thread i sums the bins of one run
        constexpr int RUN = DIGITS / CHOOSE_THREADS;
        const int top = DIGITS - 1 - tid * RUN;
        uint32_t sum = 0;
#pragma unroll
        for (int i = 0; i < RUN; ++i) sum += bins[top - i];
        uint32_t total;
        uint32_t above = scan_block(sum, warp_sums, total);
        if (above < need && need <= above + sum) {
            int bin = top;
            while (above + bins[bin] < need) above += bins[bin--];
            found[0] = (uint32_t)bin;
            found[1] = need - above;
            found[2] = bins[bin];
        }
        __syncthreads();
        prefix = prefix << width | found[0];
        need = found[1];
        equal = found[2];
        bits += width;
    }
    // chosen: the forced ones, keys above the prefix, and of those with the prefix the first `need`
    uint32_t place = 0, equal_before = 0;
    for (int i0 = 0; i0 < pages; i0 += CHOOSE_THREADS) {
        const int i = i0 + tid;
        bool take = i < pages && (i < lo || i >= hi), same = false;
        if (i >= lo && i < hi && need > 0) {
            const unsigned long long key = bits == 0 ? 0ull : key_of_score(scores[i]) >> (64 - bits);
            take = key > prefix;
            same = key == prefix;
        }
        uint32_t total;
        const uint32_t rank = equal_before + scan_block(same, warp_sums, total);
        equal_before += total;
        if (same && rank < need) take = true;
        const uint32_t at = place + scan_block(take, warp_sums, total);
        if (take && at < (uint32_t)p.k) out[at] = i;
        place += total;
    }
    for (int i = (int)place + tid; i < p.k; i += CHOOSE_THREADS) out[i] = -1;
}

}  // namespace paged
}  // namespace fcs
