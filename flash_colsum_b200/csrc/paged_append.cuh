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
//
// Memory bounds it, half of it reads and half writes: 16384 tokens, 32 query and 8 key/value heads of 128, bf16 (413 MB) 76 us,
// 5.4 TB/s.  Short calls are chains of loads: starts, length, table and rows, 11 us for 1861 tokens in 7 sequences.  Blocks of
// 128 threads, eight per SM: of 256 threads, four per SM, the long call took 98 us.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.cuh"

namespace fcs {
namespace paged {

constexpr int APPEND_THREADS = 128;

struct AppendParams {
    Batch c;
    const uint16_t *key, *value, *query;
    uint16_t *key_pages, *value_pages, *query_out, *bounds;
    long long key_st[2], value_st[2], query_st[2], query_out_st[2];   // token, head
    long long key_page_st[3], value_page_st[3];                       // page, head, slot
    const float *cos, *sin;        // (table_rows, rotary / 2)
    const int* positions;          // or nullptr: where the token lies in its sequence
    int q_heads, rotary, table_rows;
    int heads_shift;               // heads that a CTA has at a time, as a power of two (at most 16)
    int steps;                     // and how often, of values and queries
    int key_groups, value_groups;  // CTAs over the key heads, over the value heads
    int groups;                    // and over all; the CTAs of a page are neighbours, so that rows are read and written whole
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

// The rotation of one token, for eight pairs whose halves lie in two vectors or four pairs side by side in one.
struct Turn {
    float4 c[2], s[2];
    __device__ void load(const float* cos, const float* sin, bool both) {
        c[0] = *reinterpret_cast<const float4*>(cos);
        s[0] = *reinterpret_cast<const float4*>(sin);
        if (both) {
            c[1] = *reinterpret_cast<const float4*>(cos + 4);
            s[1] = *reinterpret_cast<const float4*>(sin + 4);
        }
    }
    template <typename Ops>
    __device__ void halves(uint4& a, uint4& b) const {
        uint32_t* wa = reinterpret_cast<uint32_t*>(&a);
        uint32_t* wb = reinterpret_cast<uint32_t*>(&b);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float2 x0 = Ops::widen(wa[2 * h]), x1 = Ops::widen(wa[2 * h + 1]);
            float2 y0 = Ops::widen(wb[2 * h]), y1 = Ops::widen(wb[2 * h + 1]);
            turn(x0.x, y0.x, c[h].x, s[h].x);
            turn(x0.y, y0.y, c[h].y, s[h].y);
            turn(x1.x, y1.x, c[h].z, s[h].z);
            turn(x1.y, y1.y, c[h].w, s[h].w);
            wa[2 * h] = Ops::narrow(x0.x, x0.y);
            wa[2 * h + 1] = Ops::narrow(x1.x, x1.y);
            wb[2 * h] = Ops::narrow(y0.x, y0.y);
            wb[2 * h + 1] = Ops::narrow(y1.x, y1.y);
        }
    }
    template <typename Ops>
    __device__ void neighbours(uint4& a) const {
        uint32_t* w = reinterpret_cast<uint32_t*>(&a);
        const float cc[4] = {c[0].x, c[0].y, c[0].z, c[0].w}, ss[4] = {s[0].x, s[0].y, s[0].z, s[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 v = Ops::widen(w[i]);
            turn(v.x, v.y, cc[i], ss[i]);
            w[i] = Ops::narrow(v.x, v.y);
        }
    }
};

// ROT: 0 nothing is rotated, 1 pairs are half the rotated part apart, 2 side by side
template <typename Ops, int ROT>
__global__ void __launch_bounds__(APPEND_THREADS, 8) append_kernel(const __grid_constant__ AppendParams p) {
    __shared__ uint4 sums[APPEND_THREADS][4];
    // whether this thread left out the page's first token, whose slot is not written then and the bounds do not begin anew (here, as a
    // register more is one spilled: 16384 tokens 0.5 to 1.2 us)
    __shared__ bool left_out[APPEND_THREADS];
    if (ROT != 0) left_out[threadIdx.x] = false;
    grid_dependency_wait();
    grid_launch_dependents();
    const Batch& c = p.c;
    const int D = c.dim, y = (int)(blockIdx.x % (unsigned)p.groups), segment = (int)(blockIdx.x / (unsigned)p.groups);
    const int kind = y < p.key_groups ? 0 : y < p.key_groups + p.value_groups ? 1 : 2;   // keys, values, queries
    const int steps = kind == 0 ? 1 : p.steps;
    const int h0 = (y - (kind == 0 ? 0 : kind == 1 ? p.key_groups : p.key_groups + p.value_groups)) * (steps << p.heads_shift);
    const int heads = min(steps << p.heads_shift, (kind == 2 ? p.q_heads : c.kv_heads) - h0);

    // the page of this CTA: sequence b, the j-th page that it writes
    int b = segment;
    long long j = 0, s0 = b, n = 1;
    if (c.starts) {
        b = count_before(c.sequences, [&](int i) { return (c.starts[i + 1] >> c.page_shift) + 2ll * (i + 1) <= segment; });
        s0 = c.starts[b];
        j = (long long)segment - ((s0 >> c.page_shift) + 2ll * b);
        if (b == c.sequences) {     // no sequence: rows behind the last one
            if (kind != 2 || !p.fill_tail) return;
            const long long step = (long long)(gridDim.x / (unsigned)p.groups) - segment + j;
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
    const int tokens = (int)(end - first), slot0 = (int)(first & ((1 << c.page_shift) - 1));
    const long long t0 = s0 + (first - p0);
    const int page = kind == 2 ? 0 : physical_page(c, b, page_index);
    if (page < 0) return;

    // A thread keeps its features and its head: a vector of eight features, or two whose features are pairs.
    const int rotary = kind == 1 ? 0 : p.rotary;
    const int pair_units = ROT == 1 ? rotary / 16 : 0;
    const int units = pair_units + (D - 16 * pair_units) / 8;
    const int rows = (APPEND_THREADS / units) >> p.heads_shift << p.heads_shift;    // (token, head) pairs at a time
    const int u = (int)threadIdx.x % units, r0 = (int)threadIdx.x / units;
    const int head = r0 & ((1 << p.heads_shift) - 1), lane = r0 >> p.heads_shift, lanes = rows >> p.heads_shift;
    const bool paired = ROT == 1 && u < pair_units;
    const int va = paired ? u : u + pair_units, apart = paired ? pair_units * 8 : 0;      // the vector, and how far the other is
    const bool side_by_side = ROT == 2 && va * 8 < rotary;
    const bool mine = r0 < rows && head < heads;

    const long long src_token = kind == 0 ? p.key_st[0] : kind == 1 ? p.value_st[0] : p.query_st[0];
    const long long src_head = kind == 0 ? p.key_st[1] : kind == 1 ? p.value_st[1] : p.query_st[1];
    const long long dst_token = kind == 0 ? p.key_page_st[2] : kind == 1 ? p.value_page_st[2] : p.query_out_st[0];
    const long long dst_head = kind == 0 ? p.key_page_st[1] : kind == 1 ? p.value_page_st[1] : p.query_out_st[1];
    const uint16_t* src = (kind == 0 ? p.key : kind == 1 ? p.value : p.query) + (t0 + lane) * src_token + (h0 + head) * src_head + va * 8;
    uint16_t* dst = kind == 2 ? p.query_out + t0 * dst_token
                              : (kind == 0 ? p.key_pages + page * p.key_page_st[0] : p.value_pages + page * p.value_page_st[0]) + slot0 * dst_token;
    dst += lane * dst_token + (h0 + head) * dst_head + va * 8;

    // The rotation of a token is asked for; whether there is one.
    auto turn_of = [&](int tok, Turn& turn) {
        if (ROT == 0) return true;
        const long long pos = p.positions ? (long long)p.positions[t0 + tok] : first + tok;
        if (pos < 0 || pos >= p.table_rows) {
            report(c, FCS_STATUS_BAD_POSITION);
            return false;
        }
        const long long at = pos * (p.rotary / 2) + (ROT == 1 ? va * 8 : va * 4);
        if (paired || side_by_side) turn.load(p.cos + at, p.sin + at, ROT == 1);
        return true;
    };
    auto apply = [&](const Turn& turn, uint4& a, uint4& bb) {
        if (paired) turn.halves<Ops>(a, bb);
        if (side_by_side) turn.neighbours<Ops>(a);
    };

    if (kind != 0) {
        // values and queries: a token's rotation serves its heads, which are asked for in twos
        const long long src_step = src_head << p.heads_shift, dst_step = dst_head << p.heads_shift;
        const int mine_steps = (heads - head + (1 << p.heads_shift) - 1) >> p.heads_shift;
        for (int tok = mine ? lane : tokens; tok < tokens; tok += lanes) {
            const uint16_t* from = src;
            uint16_t* to = dst;
            uint4 a0, b0, a1, b1;
            auto ask = [&](int s, uint4& a, uint4& bb) {
                if (s >= mine_steps) return;
                a = *reinterpret_cast<const uint4*>(from);
                if (paired) bb = *reinterpret_cast<const uint4*>(from + apart);
                from += src_step;
            };
            ask(0, a0, b0);
            ask(1, a1, b1);
            Turn turn;
            const bool good = turn_of(tok, turn);
            auto write = [&](uint4& a, uint4& bb) {
                if (good) apply(turn, a, bb);
                else a = bb = make_uint4(0, 0, 0, 0);
                if (good || kind == 2) {
                    *reinterpret_cast<uint4*>(to) = a;
                    if (paired) *reinterpret_cast<uint4*>(to + apart) = bb;
                }
                to += dst_step;
            };
            for (int s = 0; s < mine_steps; s += 2) {
                if (s > 0) {
                    ask(s, a0, b0);
                    ask(s + 1, a1, b1);
                }
                write(a0, b0);
                if (s + 1 < mine_steps) write(a1, b1);
            }
            src += lanes * src_token;
            dst += lanes * dst_token;
        }
        return;
    }

    uint4 low[2], high[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        low[i] = make_uint4(Ops::kInf2, Ops::kInf2, Ops::kInf2, Ops::kInf2);
        high[i] = make_uint4(Ops::kNegInf2, Ops::kNegInf2, Ops::kNegInf2, Ops::kNegInf2);
    }
    for (int tok = mine ? lane : tokens; tok < tokens; tok += lanes) {
        Turn turn;
        uint4 a = *reinterpret_cast<const uint4*>(src), bb;
        if (paired) bb = *reinterpret_cast<const uint4*>(src + apart);
        if (turn_of(tok, turn)) {
            apply(turn, a, bb);
            *reinterpret_cast<uint4*>(dst) = a;
            take_in<Ops>(low[0], high[0], a, a);
            if (paired) {
                *reinterpret_cast<uint4*>(dst + apart) = bb;
                take_in<Ops>(low[1], high[1], bb, bb);
            }
        } else if (ROT != 0 && tok == 0) {
            left_out[threadIdx.x] = true;
        }
        src += lanes * src_token;
        dst += lanes * dst_token;
    }
    if (!p.bounds) return;
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
    const bool begun = slot0 == 0 && (ROT == 0 || !left_out[threadIdx.x]);
    uint16_t* at = p.bounds + ((long long)page * c.kv_heads + h0 + head) * 2 * D + va * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (i && !paired) break;
        uint4* lo = reinterpret_cast<uint4*>(at + i * apart);
        uint4* hi = reinterpret_cast<uint4*>(at + i * apart + D);
        if (!begun) take_in<Ops>(low[i], high[i], *lo, *hi);
        *lo = low[i];
        *hi = high[i];
    }
}

}  // namespace paged
}  // namespace fcs
