// Appending to a paged cache: a step's keys, rotated by their positions, and values go to their pages, the bounds of
// the pages take the new keys in, and the step's queries are rotated on the way.
//
// The mathematics: a pair (x, y) of features at position m becomes (x c - y s, y c + x s) with c, s of row m of two
// tables; products and sums are each rounded to 32 bits, the result once to 16.  The bounds of a page and head are the
// smallest and the largest value of every feature over the keys written since its slot 0 was -- of 16-bit values, so
// they are exact in any order.
//
// Work is cut by pages: a CTA owns what the call writes into one page of one sequence, for a group of heads of one kind
// (keys, values or queries), so that a page's bounds have one writer and need no atomics.  How many tokens the
// sequences have is known on the device only: sequence b gets the CTAs from starts[b] / P + 2 b on, which is at least as many as it
// has pages to write, and the ones it does not need leave at once.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.cuh"

namespace fcs {
namespace paged {

constexpr int APPEND_THREADS = 256;

struct AppendParams {
    Batch c;
    const uint16_t *key, *value, *query;
    uint16_t *key_pages, *value_pages, *query_out, *bounds;
    long long key_st[2], value_st[2], query_st[2], query_out_st[2];   // token, head
    long long key_page_st[3], value_page_st[3];                       // page, head, slot
    const float *cos, *sin;        // (table_rows, rotary / 2)
    const int* positions;          // or nullptr: where the token lies in its sequence
    int q_heads, rotary, interleaved, table_rows;
    int heads_shift;               // heads of a CTA, as a power of two (at most 16)
    int kv_groups;                 // CTAs over the key (and as many over the value) heads
    int fill_tail;
};

struct HalfOps {
    using T2 = __half2;
    static constexpr uint32_t kInf2 = 0x7c007c00u, kNegInf2 = 0xfc00fc00u;
    __device__ static float2 widen(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
    __device__ static uint32_t narrow(float a, float b) {
        const __half2 r = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};
struct Bf16Ops {
    using T2 = __nv_bfloat162;
    static constexpr uint32_t kInf2 = 0x7f807f80u, kNegInf2 = 0xff80ff80u;
    __device__ static float2 widen(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    __device__ static uint32_t narrow(float a, float b) {
        const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};

template <typename Ops>
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    using T2 = typename Ops::T2;
    const T2 r = __hmin2_nan(*reinterpret_cast<T2*>(&a), *reinterpret_cast<T2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename Ops>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    using T2 = typename Ops::T2;
    const T2 r = __hmax2_nan(*reinterpret_cast<T2*>(&a), *reinterpret_cast<T2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename Ops>
__device__ __forceinline__ void take_in(uint4& low, uint4& high, const uint4& l, const uint4& h) {
    low = make_uint4(min2<Ops>(low.x, l.x), min2<Ops>(low.y, l.y), min2<Ops>(low.z, l.z), min2<Ops>(low.w, l.w));
    high = make_uint4(max2<Ops>(high.x, h.x), max2<Ops>(high.y, h.y), max2<Ops>(high.z, h.z), max2<Ops>(high.w, h.w));
}

// (x c - y s, y c + x s), every operation rounded by itself
__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
    const float a = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
    y = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
    x = a;
}

// Eight pairs whose halves lie in two vectors.
template <typename Ops>
__device__ __forceinline__ void turn_halves(uint4& a, uint4& b, const float* cos, const float* sin) {
    uint32_t* wa = reinterpret_cast<uint32_t*>(&a);
    uint32_t* wb = reinterpret_cast<uint32_t*>(&b);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float4 c = reinterpret_cast<const float4*>(cos)[h], s = reinterpret_cast<const float4*>(sin)[h];
        float2 x0 = Ops::widen(wa[2 * h]), x1 = Ops::widen(wa[2 * h + 1]);
        float2 y0 = Ops::widen(wb[2 * h]), y1 = Ops::widen(wb[2 * h + 1]);
        turn(x0.x, y0.x, c.x, s.x);
        turn(x0.y, y0.y, c.y, s.y);
        turn(x1.x, y1.x, c.z, s.z);
        turn(x1.y, y1.y, c.w, s.w);
        wa[2 * h] = Ops::narrow(x0.x, x0.y);
        wa[2 * h + 1] = Ops::narrow(x1.x, x1.y);
        wb[2 * h] = Ops::narrow(y0.x, y0.y);
        wb[2 * h + 1] = Ops::narrow(y1.x, y1.y);
    }
}
// Four pairs side by side in one vector.
template <typename Ops>
__device__ __forceinline__ void turn_neighbours(uint4& a, const float* cos, const float* sin) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&a);
    const float4 c4 = *reinterpret_cast<const float4*>(cos), s4 = *reinterpret_cast<const float4*>(sin);
    const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float2 v = Ops::widen(w[i]);
        turn(v.x, v.y, c[i], s[i]);
        w[i] = Ops::narrow(v.x, v.y);
    }
}

template <typename Ops>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(const __grid_constant__ AppendParams p) {
    __shared__ uint4 sums[APPEND_THREADS][4];
    grid_dependency_wait();
    grid_launch_dependents();
    const Batch& c = p.c;
    const int P = 1 << c.page_shift, D = c.dim, heads_of_cta = 1 << p.heads_shift;
    const int kind = (int)blockIdx.y < p.kv_groups ? 0 : (int)blockIdx.y < 2 * p.kv_groups ? 1 : 2;   // keys, values, queries
    const int h0 = ((int)blockIdx.y - kind * p.kv_groups) << p.heads_shift;
    const int heads = min(heads_of_cta, (kind == 2 ? p.q_heads : c.kv_heads) - h0);

    // the page of this CTA: sequence b, the j-th page that it writes
    int b = (int)blockIdx.x;
    long long j = 0, s0 = b, n = 1;
    if (c.starts) {
        int seen = 0;
        for (int base = 0; base < c.sequences; base += APPEND_THREADS) {
            const int i = base + (int)threadIdx.x + 1;
            seen += __syncthreads_count(i <= c.sequences && (c.starts[i] >> c.page_shift) + 2ll * i <= blockIdx.x);
        }
        b = seen;
        s0 = c.starts[b];
        j = (long long)blockIdx.x - ((s0 >> c.page_shift) + 2ll * b);
        if (b == c.sequences) {     // no sequence: rows behind the last one
            if (kind != 2 || !p.fill_tail) return;
            const long long step = (long long)gridDim.x - blockIdx.x + j;
            for (long long t = max(s0, 0ll) + j; t < c.tokens; t += step)
                for (int i = threadIdx.x; i < heads * (D / 8); i += APPEND_THREADS)
                    *reinterpret_cast<uint4*>(p.query_out + t * p.query_out_st[0] + (h0 + i / (D / 8)) * p.query_out_st[1] +
                                              i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
            return;
        }
        n = (long long)c.starts[b + 1] - s0;
        if (s0 < 0 || n < 0 || s0 + n > c.tokens || j < 0) return;   // (starts that do not ascend within the rows)
    }
    const long long len = c.lens[b], p0 = len - n;
    const long long page_index = (p0 >> c.page_shift) + j;
    const long long first = max(p0, page_index << c.page_shift), end = min(len, (page_index + 1) << c.page_shift);
    if (first >= end) return;
    const int tokens = (int)(end - first), slot0 = (int)(first & (P - 1));
    const long long t0 = s0 + (first - p0);
    const int page = kind == 2 ? 0 : physical_page(c, b, page_index);
    if (page < 0) return;

    const uint16_t* src = kind == 0 ? p.key : kind == 1 ? p.value : p.query;
    const long long* src_st = kind == 0 ? p.key_st : kind == 1 ? p.value_st : p.query_st;
    uint16_t* dst;
    long long dst_head, dst_token;
    if (kind == 2) {
        dst = p.query_out + t0 * p.query_out_st[0];
        dst_token = p.query_out_st[0];
        dst_head = p.query_out_st[1];
    } else {
        const long long* st = kind == 0 ? p.key_page_st : p.value_page_st;
        dst = (kind == 0 ? p.key_pages : p.value_pages) + page * st[0] + slot0 * st[2];
        dst_token = st[2];
        dst_head = st[1];
    }

    // A thread keeps its features and its head: a vector of eight features, or two whose features are pairs.
    const int R = kind == 1 ? 0 : p.rotary;
    const bool halves = R > 0 && !p.interleaved;
    const int pair_units = halves ? R / 16 : 0;
    const int units = pair_units + (D - 16 * pair_units) / 8;
    const int rows = (APPEND_THREADS / units) >> p.heads_shift << p.heads_shift;    // (token, head) pairs at a time
    const int u = (int)threadIdx.x % units, r0 = (int)threadIdx.x / units;
    const int head = r0 & (heads_of_cta - 1), lane = r0 >> p.heads_shift, lanes = rows >> p.heads_shift;
    const bool paired = u < pair_units;
    const int va = paired ? u : u + pair_units, vb = u + pair_units;          // vectors of the row
    const bool mine = r0 < rows && head < heads;
    const bool side_by_side = R > 0 && p.interleaved && va * 8 < R;

    uint4 low[2], high[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        low[i] = make_uint4(Ops::kInf2, Ops::kInf2, Ops::kInf2, Ops::kInf2);
        high[i] = make_uint4(Ops::kNegInf2, Ops::kNegInf2, Ops::kNegInf2, Ops::kNegInf2);
    }
    if (mine) {
        src += t0 * src_st[0] + (h0 + head) * src_st[1];
        dst += (h0 + head) * dst_head;
        for (int tok = lane; tok < tokens; tok += lanes) {
            const uint16_t* row = src + tok * src_st[0];
            uint4 a = *reinterpret_cast<const uint4*>(row + va * 8);
            uint4 bb = paired ? *reinterpret_cast<const uint4*>(row + vb * 8) : make_uint4(0, 0, 0, 0);
            bool good = true;
            if (p.cos) {
                const long long pos = p.positions ? (long long)p.positions[t0 + tok] : first + tok;
                good = pos >= 0 && pos < p.table_rows;
                if (!good) {
                    report(c, FCS_STATUS_BAD_POSITION);
                    a = bb = make_uint4(0, 0, 0, 0);
                } else if (paired) {
                    const long long at = pos * (p.rotary / 2) + va * 8;
                    turn_halves<Ops>(a, bb, p.cos + at, p.sin + at);
                } else if (side_by_side) {
                    const long long at = pos * (p.rotary / 2) + va * 4;
                    turn_neighbours<Ops>(a, p.cos + at, p.sin + at);
                }
            }
            if (kind != 2 && !good) continue;
            uint16_t* out = dst + tok * dst_token;
            *reinterpret_cast<uint4*>(out + va * 8) = a;
            if (paired) *reinterpret_cast<uint4*>(out + vb * 8) = bb;
            take_in<Ops>(low[0], high[0], a, a);
            take_in<Ops>(low[1], high[1], bb, bb);
        }
    }
    if (kind != 0 || !p.bounds) return;
    // the lanes of a head meet, and the first takes in what the page had
    const int busy = min(lanes, tokens);
    if (busy > 1) {
        uint4* own = sums[threadIdx.x];
        own[0] = low[0]; own[1] = high[0]; own[2] = low[1]; own[3] = high[1];
        int s = 1;
        while (2 * s < busy) s *= 2;
        for (; s > 0; s >>= 1) {
            __syncthreads();
            if (mine && lane < s && lane + s < busy) {
                const uint4* other = sums[threadIdx.x + units * (s << p.heads_shift)];
                take_in<Ops>(low[0], high[0], other[0], other[1]);
                take_in<Ops>(low[1], high[1], other[2], other[3]);
                own[0] = low[0]; own[1] = high[0]; own[2] = low[1]; own[3] = high[1];
            }
        }
    }
    if (!mine || lane > 0) return;
    uint16_t* at = p.bounds + ((long long)page * c.kv_heads + h0 + head) * 2 * D;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (i && !paired) break;
        uint4* lo = reinterpret_cast<uint4*>(at + (i ? vb : va) * 8);
        uint4* hi = reinterpret_cast<uint4*>(at + D + (i ? vb : va) * 8);
        if (slot0 > 0) take_in<Ops>(low[i], high[i], *lo, *hi);
        *lo = low[i];
        *hi = high[i];
    }
}

}  // namespace paged
}  // namespace fcs
