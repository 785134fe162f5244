// Choosing pages: per query and key/value head the k pages whose bounds promise the largest scores.
//
// The mathematics: over the keys of a page q . k <= sum_d max(q_d low_d, q_d high_d); summed over the queries of a group
// that is n . low + p . high with n = sum min(q, 0) and p = sum max(q, 0), one product of 2 D terms for the whole group.
// The first and the last pages of a query are always chosen; of the others the best, the lower page among equals.
//
// Which of two pages is the better one must not hang on the order of a sum: pages are ordered by scores summed in 64 bits.  Few
// need that.  Scores are summed in 32 bits first, which are off by at most
//     E = (c (sum |n| + sum |p|) + c' max(|n|, |p|)) max |bound|,
// c and c' counting the roundings (score_error); with t the k-th largest of them, a page above t + 2 E is chosen and one below t - 2 E is not whatever
// the exact scores are (the k-th largest of numbers each moved by E moves by E at most), and only the pages between are summed
// again, in 64 bits.  Where E is not finite, all are.
//
// Two forms share that.  Few tokens a sequence (select_row_kernel): a cluster per row reads the bounds once, and the first CTA
// chooses.  Many (score_tiles_kernel, choose_kernel): 64 tokens by 64 pages at a time, n and p in two 16-bit pieces each, and a
// warp or a block per row chooses from the scores.
//
// Measured, groups of four heads of 128, pages of 64: one query, 2048 pages (8.4 MB) 11 us, a chain of loads and barriers, 7 of them
// without choosing; 32 sequences x 256 to 512 pages (52 MB) in clusters of two 23 us, 17 of them without choosing; 1021 tokens x
// 512 pages 54 us, 27 of scores (matrix pipe 30 % busy) and 27 of choosing (2100 instructions a row, issue slots 64 % busy).
// With 64-bit sums throughout these were 26, 42 and 1022 us.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include "paged.cuh"
#include "paged_mma.cuh"

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
    double* exact;                  // (tokens of this launch, kv_heads, pitch): sums in 64 bits, where they are needed
    float* scores;                  // the same of sums in 32 bits (not for select_row_kernel)
    float* errors;                  // (tokens of this launch, kv_heads, splits): E
    int pitch, splits;
    int t0, t1;                     // tokens of this launch
    int fill_tail;
    int withhold;                   // 1 (self-test): an arrival that never comes is counted, so that no wait for bounds ends
};

template <bool BF16>
__device__ __forceinline__ float widen16(uint32_t v) {     // (the low half of v)
    if constexpr (BF16) return __uint_as_float(v << 16);
    return __half2float(__ushort_as_half((unsigned short)v));
}
template <bool BF16>
__device__ __forceinline__ float2 widen_pair(uint32_t v) {
    if constexpr (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    return __half22float2(*reinterpret_cast<__half2*>(&v));
}
// Pages that the query at `pos` sees (all of them, whether the table holds them or not).
__device__ __forceinline__ long long pages_seen(const Batch& c, long long pos) {
    return pos < 0 ? 0 : (pos >> c.page_shift) + 1;
}

// Pages of a row: 0 .. pages - 1 are there, lo .. hi - 1 of them compete for `need` places, the rest is chosen.
struct Row {
    int t, h, b;
    int pages, lo, hi;
    uint32_t need;
    bool beyond;                // it sees pages that the table is too narrow for
    __device__ void set(const SelectParams& p, int t_, int h_, int b_, long long pos) {
        t = t_, h = h_, b = b_;
        const long long seen = pages_seen(p.c, pos);
        pages = (int)min(seen, (long long)p.c.width);
        beyond = seen > pages;
        lo = min(p.first, pages);
        hi = (int)max((long long)lo, min((long long)pages, seen - p.last));
        need = (uint32_t)max(0, p.k - lo - (pages - hi));
    }
};

// Order-preserving keys: larger value, larger key; zeros are equal.  No value has key 0 or one above +inf's.  (A score that is NaN
// counts as +inf where it is summed in 64 bits -- as it is, since no error bound of its row is finite.)
__device__ __forceinline__ uint32_t key_of(float s) {
    const int bits = __float_as_int(s + 0.f);
    return min((uint32_t)(bits ^ (bits >> 31 | (int)0x80000000)), 0xff800000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ unsigned long long key_of(double s) {
    const unsigned long long bits = (unsigned long long)__double_as_longlong(s != s ? (double)INFINITY : s == 0.0 ? 0.0 : s);
    return bits >> 63 ? ~bits : bits | 0x8000000000000000ull;
}

__device__ __forceinline__ float log2_near(float x) {      // for guesses
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// E of a row whose parts sum up to `size` in magnitude and are at most `most`, over pages whose bounds reach up to `reach`; the
// scores were formed by matrix instructions, 16 terms at a time from zero, of parts in `pieces` 16-bit pieces.  Of the whole's
// magnitude: roundings of 2^-24, the group's sums and `adds` sums behind the matrix instructions, and what the pieces leave.  Of
// the largest term: in each of D / 8 steps up to 2^-23 for 17 terms, where a tensor core drops what lies below its last bit.  And
// half of fp16's smallest step of every part -- none of which may pass fp16's range, whatever they sum up to.  Sums that may overflow are no sums (NaN likewise), and products that underflow
// lose what no share of the whole covers: 1e-36 is 85 times the smallest normal number.
template <bool BF16>
__device__ __forceinline__ float score_error(const SelectParams& p, float size, float most, float reach, int adds, int pieces) {
    const float left = BF16 ? (pieces == 2 ? 3.9e-6f : 0.f) : (pieces == 2 ? 2.4e-7f : 0.f);
    float error = ((float)(p.group + adds + 2) * 6.1e-8f + left) * size + (float)p.c.dim / 8.f * 17.f * 1.2e-7f * most;
    if (!BF16) error = most < 6e4f ? error + 2.f * p.c.dim * 3e-8f : INFINITY;
    return size * reach < 1e37f ? error * reach + 1e-36f : INFINITY;
}

// The largest magnitude among 16-bit values whose bit patterns, as unsigned and as signed integers, go up to these pairs: the
// one finds the largest negative, the other the largest positive value.  NaN comes out as such or as an infinity.
template <bool BF16>
__device__ __forceinline__ float reach_of(uint32_t as_unsigned, uint32_t as_signed) {
    const uint32_t a = as_unsigned & 0x7fff7fffu, b = as_signed & 0x7fff7fffu;
    // (no negative value: the unsigned maximum is the largest positive one, and the other way round)
    const float2 x = widen_pair<BF16>(a), y = widen_pair<BF16>(b);
    return max_or_nan(max_or_nan(x.x, x.y), max_or_nan(y.x, y.y));
}

// A row's scores in 64 bits, by a warp: a lane has eight of the 2 D parts, the first D of which meet the lows.
template <bool BF16>
struct ExactScores {
    double part[8];
    __device__ ExactScores(const SelectParams& p, const Row& r) {
        const int lane = threadIdx.x & 31, half = p.c.dim / 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) part[i] = 0.0;
        if (lane >= 2 * half) return;
        const bool low = lane < half;
        const uint16_t* q = p.query + r.t * p.query_st[0] + (long long)r.h * p.group * p.query_st[1] + (low ? lane : lane - half) * 8;
#pragma unroll 4
        for (int g = 0; g < p.group; ++g) {
            const uint4 w = *reinterpret_cast<const uint4*>(q + g * p.query_st[1]);
            const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 x = widen_pair<BF16>(words[i]);
                part[2 * i] += (low ? x.x < 0.f : !(x.x < 0.f)) ? (double)x.x : 0.0;      // (NaN stays)
                part[2 * i + 1] += (low ? x.y < 0.f : !(x.y < 0.f)) ? (double)x.y : 0.0;
            }
        }
    }
    // Up to N pages at a time (page < 0: none), whose loads are in flight together.
    template <int N>
    __device__ void operator()(const SelectParams& p, const Row& r, const int (&page)[N], double (&score)[N]) const {
        const Batch& c = p.c;
        const int lane = threadIdx.x & 31;
        int at[N];
        uint4 w[N];
#pragma unroll
        for (int i = 0; i < N; ++i) at[i] = page[i] >= 0 ? c.table[r.b * c.table_ld + page[i]] : -1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool there = at[i] >= 0 && at[i] < c.pages;
            w[i] = there && lane < c.dim / 4 ? *reinterpret_cast<const uint4*>(p.bounds + ((long long)at[i] * c.kv_heads + r.h) * 2 * c.dim + lane * 8)
                                             : make_uint4(0, 0, 0, 0);
            if (!there) at[i] = -1;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            score[i] = 0.0;
            if (lane < c.dim / 4)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 x = widen_pair<BF16>(words[e]);
                    score[i] += part[2 * e] * (double)x.x;
                    score[i] += part[2 * e + 1] * (double)x.y;
                }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i) score[i] += __shfl_xor_sync(0xffffffffu, score[i], o);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at[i] < 0) score[i] = -INFINITY;      // (said in the status word by whoever summed in 32 bits)
    }
};

// Pages around the border, up to 32 of them (shared memory of a team).
struct CloseList {
    unsigned long long key[32];
    int page[32];
};

// ---- who chooses for a row: a block, or a warp.  A thread holds the keys of E consecutive pages (a block goes over more than
// NT E pages in tiles, reading the scores again); key 0 is a page that does not compete.

// (`scores` has places for a multiple of four pages)
template <int E>
__device__ __forceinline__ void load_keys(const Row& r, const float* scores, int first, uint32_t (&keys)[E]) {
    const uint32_t skip = (uint32_t)(r.lo - first), some = (uint32_t)(r.hi - r.lo);
#pragma unroll
    for (int j = 0; j < E; j += 4) {
        const float4 q = first + j < r.pages ? *reinterpret_cast<const float4*>(scores + first + j) : make_float4(0.f, 0.f, 0.f, 0.f);
        keys[j] = j - skip < some ? key_of(q.x) : 0u;
        keys[j + 1] = j + 1 - skip < some ? key_of(q.y) : 0u;
        keys[j + 2] = j + 2 - skip < some ? key_of(q.z) : 0u;
        keys[j + 3] = j + 3 - skip < some ? key_of(q.w) : 0u;
    }
}

__device__ __forceinline__ uint32_t warp_upto(uint32_t n) {       // inclusive sum over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, n, o);
        if ((int)(threadIdx.x & 31) >= o) n += up;
    }
    return n;
}

template <int NT, int E>
struct BlockTeam {
    static constexpr int SIZE = NT, RUN = E;
    const float* scores;
    CloseList* close;            // shared
    uint32_t* room;              // shared: [2][3 * NT / 32]
    int turn = 0;
    uint32_t keys[E];
    __device__ int rank() const { return threadIdx.x; }
    __device__ void sync() const { __syncthreads(); }
    __device__ void load(const Row& r, int base) {
        load_keys<E>(r, scores, base + rank() * E, keys);
    }
    // f(first page of this thread's run), for every tile of the row, by all threads
    template <typename F>
    __device__ void tiles(const Row& r, F f) {
        for (int base = 0; base < r.pages; base += NT * E) {
            if (r.pages > NT * E) load(r, base);
            f(base + rank() * E);
        }
    }
    template <typename Op>
    __device__ void reduce(uint32_t (&v)[3], Op op) {
        uint32_t* mine = room + (turn ^= 1) * (3 * NT / 32);      // (two rooms: one barrier is enough)
#pragma unroll
        for (int j = 0; j < 3; ++j) v[j] = op.warp(v[j]);
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int j = 0; j < 3; ++j) mine[j * (NT / 32) + (threadIdx.x >> 5)] = v[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            v[j] = mine[j * (NT / 32)];
#pragma unroll
            for (int w = 1; w < NT / 32; ++w) v[j] = op(v[j], mine[j * (NT / 32) + w]);
        }
    }
    // the sum of `n` over the threads before this one, and over all
    __device__ uint32_t before(uint32_t n, uint32_t& total) {
        uint32_t* mine = room + (turn ^= 1) * (3 * NT / 32);
        const uint32_t upto = warp_upto(n);
        if ((threadIdx.x & 31) == 31) mine[threadIdx.x >> 5] = upto;
        __syncthreads();
        uint32_t sum = upto - n;
        total = 0;
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) {
            if (w < (int)(threadIdx.x >> 5)) sum += mine[w];
            total += mine[w];
        }
        return sum;
    }
};

template <int E>
struct WarpTeam {
    static constexpr int SIZE = 32, RUN = E;
    const float* scores;
    CloseList* close;            // shared, the warp's own
    uint32_t keys[E];
    __device__ int rank() const { return threadIdx.x & 31; }
    __device__ void sync() const { __syncwarp(); }
    __device__ void load(const Row& r, int) {
        load_keys<E>(r, scores, rank() * E, keys);
    }
    template <typename F>
    __device__ void tiles(const Row&, F f) { f(rank() * E); }
    template <typename Op>
    __device__ void reduce(uint32_t (&v)[3], Op op) const {
#pragma unroll
        for (int j = 0; j < 3; ++j) v[j] = op.warp(v[j]);
    }
    __device__ uint32_t before(uint32_t n, uint32_t& total) const {
        const uint32_t upto = warp_upto(n);
        total = __shfl_sync(0xffffffffu, upto, 31);
        return upto - n;
    }
};

struct Sum {
    __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a + b; }
    __device__ uint32_t warp(uint32_t v) const { return __reduce_add_sync(0xffffffffu, v); }
};
struct Largest {
    __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); }
    __device__ uint32_t warp(uint32_t v) const { return __reduce_max_sync(0xffffffffu, v); }
};

// The `need`-th largest of the 64-bit keys that `each` goes over -- at least `need` are >= low, fewer >= high --, or a key that as
// many as `need` reach: then `clean` is set.
template <typename Team, typename Each>
__device__ unsigned long long kth_wide_key(Team& team, uint32_t need, unsigned long long low, unsigned long long high, bool& clean,
                                           Each each) {
    clean = false;
    while (high - low > 1) {
        const unsigned long long d = high - low, quarter = d / 4;
        const unsigned long long m1 = low + (quarter > 0 ? quarter : 1), m2 = low + d / 2, m3 = low + (quarter > 0 ? 3 * quarter : 1);
        uint32_t n[3] = {0, 0, 0};
        each([&](unsigned long long key) {
            n[0] += key >= m1;
            n[1] += key >= m2;
            n[2] += key >= m3;
        });
        team.reduce(n, Sum());
        if (n[0] == need || n[1] == need || n[2] == need) {
            clean = true;
            return n[2] == need ? m3 : n[1] == need ? m2 : m1;
        }
        if (n[2] > need) low = m3;
        else if (n[1] > need) low = m2, high = m3;
        else if (n[0] > need) low = m1, high = m2;
        else high = m1;
    }
    return low;
}

// Chooses the pages of a row and writes them.  `ends`: the largest key and the complement of the smallest, or zeros.  `error`: E.
// `exact`: the row's memory for sums in 64 bits.
//
// The border is looked for with three guesses at a time, which a straight line through the logarithms of the counts places: the
// tail of a sum of many terms falls about so.  When at most 24 pages are left, they and those within the error of them are listed,
// and a warp ranks the list -- each warp for itself.  Where more are left (equal pages, no finite error) 64 bits decide about all.
// [rows of 2048 and 512 pages: three rounds, where halving takes seven and a histogram of 1024 bins two of twice the time]
template <bool BF16, typename Team>
__device__ void choose(const SelectParams& p, const Row& r, Team& team, uint32_t (&ends)[3], float error, double* exact, int* out) {
    constexpr int E = Team::RUN;
    uint32_t(&keys)[E] = team.keys;
    const int lane = threadIdx.x & 31;
    team.load(r, 0);
    // chosen: keys from `high` on, and of those from `low` on: the listed ones that are `picked`, or (wide) those whose 64-bit key is
    // above `bar`, and the first `equal` at it
    uint32_t low = 0xffffffffu, high = 0xffffffffu, picked = 0, equal = 0;
    unsigned long long bar = 0;
    bool wide = false;
    auto count = [&](uint32_t m0, uint32_t m1, uint32_t m2, uint32_t (&n)[3]) {
        n[0] = n[1] = n[2] = 0;
        team.tiles(r, [&](int) {
#pragma unroll
            for (int j = 0; j < E; ++j) {
                n[0] += keys[j] >= m0;
                n[1] += keys[j] >= m1;
                n[2] += keys[j] >= m2;
            }
        });
        team.reduce(n, Sum());
    };
    if (r.need > 0) {
        if (ends[0] == 0) {
            team.tiles(r, [&](int) {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    ends[0] = max(ends[0], keys[j]);
                    if (keys[j]) ends[1] = max(ends[1], ~keys[j]);
                }
            });
            team.reduce(ends, Largest());
        }
        low = ~ends[1];
        high = ends[0] + 1;
        const bool known = error < INFINITY;
        // at least `need` keys are >= low, fewer are >= high
        uint32_t at_low = (uint32_t)(r.hi - r.lo), at_high = 0, n[3];
        auto narrow = [&](uint32_t m0, uint32_t m1, uint32_t m2) {
            count(m0, m1, m2, n);
            if (n[2] >= r.need) low = m2, at_low = n[2];
            else if (n[1] >= r.need) low = m1, at_low = n[1], high = m2, at_high = n[2];
            else if (n[0] >= r.need) low = m0, at_low = n[0], high = m1, at_high = n[1];
            else high = m0, at_high = n[0];
        };
        while (known && high - low > 1 && at_low - at_high > 24) {
            const float top = log2_near((float)at_low + 0.5f), bottom = log2_near((float)at_high + 0.5f);
            const float f = __fdividef(top - log2_near((float)r.need + 0.5f), top - bottom), d = (float)(high - low);
            const uint32_t last = high - low - 1;
            auto guess = [&](float part) { return low + max(1u, min(last, (uint32_t)(part * d))); };
            narrow(guess(0.5f * f), guess(f), guess(0.5f + 0.5f * f));
        }
        bool listed = false;
        uint32_t above = 0;
        if (known) {     // as far as the errors reach (2.5: the sums here are rounded, too)
            const uint32_t from = key_of(value_of(low) - 2.6f * error);
            const uint32_t upto = high > ends[0] ? high : max(high, key_of(value_of(high) + 2.6f * error) + 1);
            count(from, upto, upto, n);
            listed = n[0] - n[1] <= 32;
            if (listed) low = from, high = upto, above = n[1];
        }
        if (listed) {
            const int m = (int)(n[0] - n[1]);
            const uint32_t want = r.need - above;
            uint32_t slot = 0, total;
            team.tiles(r, [&](int i) {
                uint32_t in = 0;
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (keys[j] >= low && keys[j] < high) in |= 1u << j;
                uint32_t at = slot + team.before(__popc(in), total);
                slot += total;
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (in >> j & 1u) {
                        team.close->key[at] = keys[j];
                        team.close->page[at++] = i + j;
                    }
            });
            team.sync();
            const uint32_t key = lane < m ? (uint32_t)team.close->key[lane] : 0u;
            uint32_t ahead = 0;
            for (int i = 0; i < m; ++i) {
                const uint32_t other = __shfl_sync(0xffffffffu, key, i);
                ahead += other > key || (other == key && i < lane);
            }
            const float v = value_of(key), t = __shfl_sync(0xffffffffu, v, __ffs(__ballot_sync(0xffffffffu, lane < m && ahead + 1 == want)) - 1);
            const uint32_t sure = __ballot_sync(0xffffffffu, lane < m && v > t + 2.5f * error);
            const uint32_t near = __ballot_sync(0xffffffffu, lane < m && !(v > t + 2.5f * error) && v >= t - 2.5f * error);
            const uint32_t left = want - __popc(sure);
            picked = sure | near;
            if ((int)left < __popc(near)) {
                const ExactScores<BF16> score(p, r);
                const int warp = Team::SIZE > 32 ? threadIdx.x >> 5 : 0;
                team.sync();               // (the keys have been read)
                uint32_t todo = near;
                for (int i = 0; todo; ++i) {      // two at a time
                    int at[2], page[2];
                    double s[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        at[j] = __ffs(todo) - 1;
                        todo &= todo - 1;
                        page[j] = at[j] >= 0 ? team.close->page[at[j]] : -1;
                    }
                    if (i % (Team::SIZE / 32) != warp) continue;
                    score(p, r, page, s);
                    if (lane == 0) team.close->key[at[0]] = key_of(s[0]);
                    if (lane == 1 && at[1] >= 0) team.close->key[at[1]] = key_of(s[1]);
                }
                team.sync();
                const unsigned long long mine = team.close->key[lane < m ? lane : 0];
                ahead = 0;
                for (todo = near; todo; todo &= todo - 1) {
                    const int i = __ffs(todo) - 1;
                    const unsigned long long other = team.close->key[i];
                    ahead += other > mine || (other == mine && i < lane);
                }
                picked = sure | __ballot_sync(0xffffffffu, (near >> lane & 1u) && ahead < left);
            }
        } else {
            wide = true;
            while (known && high - low > 1) {
                const uint32_t d = high - low, quarter = max(1u, d / 4);
                narrow(low + quarter, low + max(1u, d / 2), low + max(1u, d / 4 * 3));
            }
            const float t = value_of(low);       // the need-th largest
            low = known ? key_of(t - 2.5f * error) : 1u;
            high = known ? key_of(t + 2.5f * error) + 1 : 0xffffffffu;
            count(low, high, high, n);
            const uint32_t left = r.need - n[1];
            const ExactScores<BF16> score(p, r);
            team.tiles(r, [&](int i) {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    uint32_t todo = __ballot_sync(0xffffffffu, keys[j] >= low && keys[j] < high);
                    while (todo) {
                        int src[4], page[4];
                        double s[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            src[q] = __ffs(todo) - 1;
                            todo &= todo - 1;
                            page[q] = __shfl_sync(0xffffffffu, i, max(src[q], 0)) + j;
                            if (src[q] < 0) page[q] = -1;
                        }
                        score(p, r, page, s);
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            if (lane == src[q]) exact[page[q]] = s[q];
                    }
                }
            });
            team.sync();
            auto over = [&](auto f) {
                team.tiles(r, [&](int i) {
#pragma unroll
                    for (int j = 0; j < E; ++j)
                        if (keys[j] >= low && keys[j] < high) f(key_of(exact[i + j]));
                });
            };
            if (left == n[0] - n[1]) {           // all of them
                bar = 0;
            } else {
                // (within E of sums that are within 2.5 E of t)
                bool clean;
                bar = kth_wide_key(team, left, known ? key_of((double)t - 4.0 * error) : 0ull,
                                   known ? key_of((double)t + 4.0 * error) + 1 : ~0ull, clean, over);
                if (clean) {
                    bar -= 1;
                } else {
                    uint32_t higher[3] = {0, 0, 0};
                    over([&](unsigned long long key) { higher[0] += key > bar; });
                    team.reduce(higher, Sum());
                    equal = left - higher[0];
                }
            }
        }
    }
    uint32_t place = 0, slot = 0, equal_before = 0, total;
    team.tiles(r, [&](int i) {
        uint32_t taken = 0, in = 0, same = 0;     // a bit per page of the run
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if (i + j < r.pages && (keys[j] == 0 || keys[j] >= high)) taken |= 1u << j;
            if (keys[j] >= low && keys[j] < high) in |= 1u << j;
        }
        if (wide) {                               // (the same for all)
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (in >> j & 1u) {
                    const unsigned long long key = key_of(exact[i + j]);
                    if (key > bar) taken |= 1u << j;
                    if (key == bar) same |= 1u << j;
                }
            if (equal > 0) {
                uint32_t rank = equal_before + team.before(__popc(same), total);
                equal_before += total;
                for (; same && rank < equal; ++rank, same &= same - 1) taken |= same & -same;
            }
        } else {
            uint32_t at = slot + team.before(__popc(in), total);
            slot += total;
            for (; in; ++at, in &= in - 1)
                if (picked >> at & 1u) taken |= in & -in;
        }
        uint32_t at = place + team.before(__popc(taken), total);
        for (; taken; ++at, taken &= taken - 1)
            if (at < (uint32_t)p.k) out[at] = i + __ffs(taken) - 1;
        place += total;
    });
    for (uint32_t i = place + team.rank(); i < (uint32_t)p.k; i += Team::SIZE) out[i] = -1;
}

// Whether the table lacks a page of those that a row has without a score: its first `lo` ones, those from `hi` on and those past the
// table's width.  A lane in `size`, each for its own.  (The heads share the table: the first looks it up.  By every head, 256 rows of eight
// heads that take all they see took 7.3 us, by the first alone 5.9, without looking 5.6.)
__device__ __forceinline__ bool lacks(const SelectParams& p, const Row& r, int lo, int hi, int rank, int size) {
    const int* table = p.c.table + r.b * p.c.table_ld;
    bool lacking = r.beyond;
    for (int i = rank; i < lo; i += size) lacking |= (uint32_t)table[i] >= (uint32_t)p.c.pages;
    for (int i = hi + rank; i < r.pages; i += size) lacking |= (uint32_t)table[i] >= (uint32_t)p.c.pages;
    return lacking;
}

// The rows that need no scores: behind the last sequence, or with no more pages than are asked for.  (k may be the largest int: places
// are counted without a sign, a step past it would have none.)
__device__ __forceinline__ bool settled(const SelectParams& p, int b, const Row& r, int* out, int rank, int size) {
    if (b >= p.c.sequences) {
        if (p.fill_tail)
            for (uint32_t i = rank; i < (uint32_t)p.k; i += size) out[i] = -1;
        return true;
    }
    if (r.pages > p.k) return false;
    for (uint32_t i = rank; i < (uint32_t)p.k; i += size) out[i] = i < (uint32_t)r.pages ? (int)i : -1;
    return true;
}

// ------------------------------------------------------------------ few tokens a sequence
constexpr int ROW_THREADS = 128;
// Per SM, by the registers (three of 256 threads take as long, within what two runs differ by).  Shared memory has a score for every
// page of the table's width: at heads of 128 it holds six CTAs up to 350 pages, five at 512, four at 4096, three at 8192.
constexpr int ROW_CTAS = 6;
typedef BlockTeam<ROW_THREADS, 16> RowTeam;

// grid: (CL * tokens, kv heads); shared memory: row_smem.  A warp takes 16 pages at a time, whose bounds bulk copies bring -- it
// asks for the next 16 when it has read these -- as the rows of a matrix instruction: a lane reads eight neighbouring features,
// which serve as those that the instruction wants of it, in the order that the parts are given in as well.  The parts' three
// pieces are three of its eight columns.  (Loads into registers in place of the copies: 32 rows of 256 to 512 pages 26.5 us.)
__host__ __device__ constexpr int row_block_bytes(int dim) { return 16 * (4 * dim + 16); }       // (16: no bank twice)
inline int row_smem(int dim, int pitch) { return ROW_THREADS / 32 * row_block_bytes(dim) + 4 * pitch; }

template <bool BF16, int DP, int CL>
__global__ void __launch_bounds__(ROW_THREADS, ROW_CTAS) select_row_kernel(const __grid_constant__ SelectParams p) {
    constexpr int CHUNKS = DP / 16;               // 32 of the 2 D features
    extern __shared__ __align__(16) uint8_t row_smem_raw[];
    __shared__ __align__(8) unsigned long long arrived[ROW_THREADS / 32];
    __shared__ int abort_flag;
    constexpr int WARPS = ROW_THREADS / 32;
    __shared__ uint32_t of_cta[3][CL];            // the largest key, the complement of the smallest, the reach
    __shared__ uint32_t of_warp[3][WARPS];
    __shared__ float warp_size[WARPS], warp_most[WARPS];
    __shared__ uint32_t room[2 * 3 * WARPS];
    __shared__ CloseList close;
    __shared__ __align__(16) uint16_t parts[4][2 * DP];       // what 16 bits hold, the rest of that and the rest's, zeros
    if (threadIdx.x % 32 == 0) mbar_init(smem_u32(&arrived[threadIdx.x / 32]), 1 + p.withhold);
    if (threadIdx.x == 0) abort_flag = 0;
    mbar_fence_init();
    if constexpr (CL > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    grid_dependency_wait();
    grid_launch_dependents();
    const Batch& c = p.c;
    const int D = c.dim, h = blockIdx.y, rank = (int)(blockIdx.x % CL), t = p.t0 + (int)(blockIdx.x / CL);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row_bytes = 4 * D + 16;
    uint8_t* const block = row_smem_raw + warp * row_block_bytes(D);
    float* const row_scores = reinterpret_cast<float*>(row_smem_raw + WARPS * row_block_bytes(D));
    const uint32_t bar = smem_u32(&arrived[warp]);
    const int b = sequence_of(c, t);
    const long long pos = b < c.sequences ? position_of(c, b, t) : -1;

    // a thread has one or two of the 2 D parts: the first D meet the lows, the others the highs
    {
        float size = 0.f, most = 0.f;
#pragma unroll
        for (int i = tid; i < 2 * DP; i += ROW_THREADS) {
            float part = 0.f;
            if (i < 2 * D && b < c.sequences) {
                const bool low = i < D;
                const uint16_t* q = p.query + t * p.query_st[0] + (long long)h * p.group * p.query_st[1] + (low ? i : i - D);
#pragma unroll 4
                for (int g = 0; g < p.group; ++g) {
                    const float x = widen16<BF16>(q[g * p.query_st[1]]);
                    part += (low ? x < 0.f : !(x < 0.f)) ? x : 0.f;      // (NaN stays)
                }
            }
            float rest, rest2, z;
            parts[0][i] = (uint16_t)round_pair<BF16>(part, 0.f, rest, z);
            parts[1][i] = (uint16_t)round_pair<BF16>(rest, 0.f, rest2, z);
            parts[2][i] = (uint16_t)round_pair<BF16>(rest2, 0.f, z, z);
            parts[3][i] = 0;
            size += fabsf(part);
            most = max_or_nan(most, fabsf(part));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            size += __shfl_xor_sync(0xffffffffu, size, o);
            most = max_or_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        if (lane == 0) warp_size[warp] = size, warp_most[warp] = most;
    }
    Row r = {};
    if (b < c.sequences) r.set(p, t, h, b, pos);
    int* out = p.chosen + ((long long)t * c.kv_heads + h) * p.k;
    if (b >= c.sequences || r.pages <= p.k) {       // (all CTAs of the cluster)
        if (rank == 0) {
            settled(p, b, r, out, tid, ROW_THREADS);
            if (h == 0 && b < c.sequences && lacks(p, r, r.pages, r.pages, tid, ROW_THREADS)) report(c, FCS_STATUS_BAD_PAGE);
        }
        if constexpr (CL > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        return;
    }
    const int per = (r.hi - r.lo + CL - 1) / CL, begin = r.lo + rank * per, end = min(r.hi, begin + per);
    const int* table = c.table + b * c.table_ld;
    int base = begin + warp * 16;
    // This warp's next 16 pages; whether each is one of the pools'.  (For one that is not, page 0 stands in.)
    auto ask = [&](int first, int entry) {
        const int n = min(16, end - first);
        if (n <= 0) return;
        if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(n * 4 * D));
        __syncwarp();
        if (lane < n) {
            const int page = entry >= 0 && entry < c.pages ? entry : 0;
            bulk_load(smem_u32(block + lane * row_bytes), p.bounds + ((long long)page * c.kv_heads + h) * 2 * D, 4 * D, bar);
        }
    };
    auto entry_of = [&](int first) { return lane < 16 && first + lane < end ? table[first + lane] : -1; };
    int entry = entry_of(base);
    __syncwarp();
    ask(base, entry);
    uint32_t high_bits = 0, low_bits = 0x80008000u;       // the largest bit patterns, as unsigned and as signed
    bool lacking = false;
    __syncthreads();
    if constexpr (CL > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");     // the first CTA is there
    uint32_t to = smem_u32(row_scores);
    if constexpr (CL > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(to), "r"(0));
    const int row = lane >> 2, col = lane & 3;
    const uint16_t* columns = parts[min(row, 3)] + col * 8;
    uint32_t ends[3] = {0, 0, 0};
    uint32_t phase = 0;
    while (base < end) {
        const int next = base + WARPS * 16;
        const int ahead = entry_of(next);
        if (!mbar_wait(bar, phase, &abort_flag, c.status, FCS_STATUS_WAIT_CONSUMER)) break;
        phase ^= 1;
        const bool in0 = base + row < end, in1 = base + row + 8 < end;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < CHUNKS; ++s) {
            const bool in = s * 32 + col * 8 < 2 * D;
            const uint8_t* at = block + row * row_bytes + col * 16 + s * 64;
            const uint4 w0 = in0 && in ? *reinterpret_cast<const uint4*>(at) : make_uint4(0, 0, 0, 0);
            const uint4 w1 = in1 && in ? *reinterpret_cast<const uint4*>(at + 8 * row_bytes) : make_uint4(0, 0, 0, 0);
            const uint4 f = *reinterpret_cast<const uint4*>(columns + s * 32);
            // (every instruction starts from zero: see score_error)
            float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
            const uint32_t a0[4] = {w0.x, w1.x, w0.y, w1.y}, a1[4] = {w0.z, w1.z, w0.w, w1.w};
            mma16816<BF16>(x, a0, f.x, f.y);
            mma16816<BF16>(y, a1, f.z, f.w);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += x[i] + y[i];
            high_bits = __vimax3_u16x2(__vimax3_u16x2(high_bits, w0.x, w0.y), w0.z, w0.w);
            high_bits = __vimax3_u16x2(__vimax3_u16x2(high_bits, w1.x, w1.y), w1.z, w1.w);
            low_bits = __vimax3_s16x2(__vimax3_s16x2(low_bits, w0.x, w0.y), w0.z, w0.w);
            low_bits = __vimax3_s16x2(__vimax3_s16x2(low_bits, w1.x, w1.y), w1.z, w1.w);
        }
        __syncwarp();
        ask(next, ahead);
        const int page0 = __shfl_sync(0xffffffffu, entry, row), page1 = __shfl_sync(0xffffffffu, entry, row + 8);
        const bool there0 = page0 >= 0 && page0 < c.pages, there1 = page1 >= 0 && page1 < c.pages;
        entry = ahead;
        // columns 0 to 2 together are the score; lane 4 i has 0 and 1 of pages i and i + 8, lane 4 i + 1 has 2
        const float third0 = __shfl_down_sync(0xffffffffu, acc[0], 1), third1 = __shfl_down_sync(0xffffffffu, acc[2], 1);
        const float second = __shfl_up_sync(0xffffffffu, (acc[2] + acc[3]) + third1, 1);
        if (col < 2) {
            const int i = base + row + 8 * col;
            const bool there = col == 0 ? there0 : there1;
            if (i < end) {
                lacking |= !there;
                const float s = !there ? -INFINITY : col == 0 ? (acc[0] + acc[1]) + third0 : second;
                const uint32_t key = key_of(s);
                ends[0] = max(ends[0], key);
                ends[1] = max(ends[1], ~key);
                if constexpr (CL > 1) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4 * i), "f"(s) : "memory");
                else row_scores[i] = s;
            }
        }
        __syncwarp();
        base = next;
    }
    if (abort_flag) __nanosleep(100000);       // (copies of a warp that gave up may still be landing)
    if (lacking) report(c, FCS_STATUS_BAD_PAGE);
    // (the reach is not negative, or NaN: its bits are in order)
    ends[2] = __float_as_uint(reach_of<BF16>(high_bits, low_bits));
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        ends[i] = __reduce_max_sync(0xffffffffu, ends[i]);
        if (lane == 0) of_warp[i][warp] = ends[i];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int i = 0; i < 3; ++i) ends[i] = __reduce_max_sync(0xffffffffu, lane < WARPS ? of_warp[i][lane] : 0u);
        if (lane < 3) {
            const uint32_t mine = lane == 0 ? ends[0] : lane == 1 ? ends[1] : ends[2];
            uint32_t at = smem_u32(&of_cta[lane][rank]);
            if constexpr (CL > 1) {
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(at), "r"(0));
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(mine) : "memory");
            } else {
                of_cta[lane][rank] = mine;
            }
        }
        __syncwarp();
    }
    if constexpr (CL > 1) {
        cluster_sync();
        if (rank > 0) {       // (the last CTA has time to look up the pages that nobody scored)
            if (h == 0 && rank == CL - 1 && lacks(p, r, r.lo, r.hi, tid, ROW_THREADS)) report(c, FCS_STATUS_BAD_PAGE);
            return;
        }
    } else {
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) ends[i] = __reduce_max_sync(0xffffffffu, lane < CL ? of_cta[i][lane] : 0u);
    float size = lane < WARPS ? warp_size[lane] : 0.f, most = lane < WARPS ? warp_most[lane] : 0.f;
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) {
        size += __shfl_xor_sync(0xffffffffu, size, o);
        most = max_or_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    size = __shfl_sync(0xffffffffu, size, 0);
    most = __shfl_sync(0xffffffffu, most, 0);
    RowTeam team{row_scores, &close, room};
    const float error = score_error<BF16>(p, size, most, __uint_as_float(ends[2]), CHUNKS + 3, 3);
    choose<BF16>(p, r, team, ends, error, p.exact + ((long long)(t - p.t0) * c.kv_heads + h) * p.pitch, out);
    if (CL == 1 && h == 0 && lacks(p, r, r.lo, r.hi, tid, ROW_THREADS)) report(c, FCS_STATUS_BAD_PAGE);
}

// ------------------------------------------------------------------ many tokens a sequence
constexpr int TILE_TOKENS = 64, TILE_PAGES = 64;
constexpr int TILES_THREADS = 256;

inline int tiles_row_bytes(int dim) { return 4 * dim + 16; }     // of a row of 2 D values in shared memory: no bank twice
inline int tiles_smem(int dim) { return 3 * 64 * tiles_row_bytes(dim); }

// 64 tokens of one sequence, a share of the pages that they see.  grid: (token tiles, kv heads, splits); sequence b has the
// tiles from starts[b] / 64 + b on, at least as many as it needs (without starts, tile b alone).
template <bool BF16>
__global__ void __launch_bounds__(TILES_THREADS) score_tiles_kernel(const __grid_constant__ SelectParams p) {
    extern __shared__ __align__(16) uint8_t tiles_smem_raw[];
    __shared__ uint32_t reach_of_warp[TILES_THREADS / 32];
    __shared__ float size_of_token[TILE_TOKENS], most_of_token[TILE_TOKENS];
    __shared__ uint8_t missing[TILE_PAGES];
    grid_dependency_wait();
    grid_launch_dependents();
    const Batch& c = p.c;
    const int D = c.dim, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int b;
    long long s0, s1, first;
    if (c.starts) {
        const long long tile_id = (long long)blockIdx.x + max(0, p.t0 / TILE_TOKENS - 1);
        b = count_before(c.sequences, [&](int i) { return c.starts[i + 1] / TILE_TOKENS + (long long)(i + 1) <= tile_id; });
        if (b >= c.sequences) return;
        s0 = c.starts[b], s1 = c.starts[b + 1];
        first = s0 + (tile_id - (s0 / TILE_TOKENS + b)) * TILE_TOKENS;
    } else {
        b = p.t0 + (int)blockIdx.x;
        s0 = first = b, s1 = b + 1;
    }
    if (s0 < 0 || s1 > c.tokens || first < s0 || first >= s1) return;
    if (first >= p.t1 || first + TILE_TOKENS <= p.t0) return;
    const int tokens = (int)min((long long)TILE_TOKENS, s1 - first), t_first = (int)first;
    // pages that the last token lets compete, cut over the splits in whole tiles
    const long long seen = pages_seen(c, position_of(c, b, t_first + tokens - 1));
    const int pages = (int)max(0ll, min((long long)c.width, seen - p.last));
    const int page_tiles = (pages + TILE_PAGES - 1) / TILE_PAGES, per = (page_tiles + p.splits - 1) / p.splits;
    const int begin = blockIdx.z * per * TILE_PAGES, end = min(pages, begin + per * TILE_PAGES);

    const int row_bytes = 4 * D + 16;
    uint8_t* const hi = tiles_smem_raw;                  // [tokens][2 D]: n and p, what 16 bits hold of them
    uint8_t* const lo = hi + TILE_TOKENS * row_bytes;    // the rest
    uint8_t* const tile = lo + TILE_TOKENS * row_bytes;  // [pages][2 D]
    const int my_row = tid >> 2, my_vec = tid & 3;       // four threads a row
    {
        float size = 0.f, most = 0.f;
#pragma unroll 2
        for (int v = my_vec; v < D / 8; v += 4) {
            float n[8], s[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) n[i] = s[i] = 0.f;
            if (my_row < tokens) {
                const uint16_t* q = p.query + (t_first + my_row) * p.query_st[0] + (long long)h * p.group * p.query_st[1] + v * 8;
#pragma unroll 4
                for (int g = 0; g < p.group; ++g) {
                    const uint4 w = *reinterpret_cast<const uint4*>(q + g * p.query_st[1]);
                    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 x = widen_pair<BF16>(words[i]);
                        n[2 * i] += x.x < 0.f ? x.x : 0.f;
                        n[2 * i + 1] += x.y < 0.f ? x.y : 0.f;
                        s[2 * i] += x.x < 0.f ? 0.f : x.x;
                        s[2 * i + 1] += x.y < 0.f ? 0.f : x.y;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                size += s[i] - n[i];
                most = max_or_nan(most, max_or_nan(s[i], -n[i]));
            }
            uint32_t nh[4], nl[4], sh[4], sl[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float ra, rb, z;
                nh[i] = round_pair<BF16>(n[2 * i], n[2 * i + 1], ra, rb);
                nl[i] = round_pair<BF16>(ra, rb, z, z);
                sh[i] = round_pair<BF16>(s[2 * i], s[2 * i + 1], ra, rb);
                sl[i] = round_pair<BF16>(ra, rb, z, z);
            }
            const int at = my_row * row_bytes + v * 16;
            *reinterpret_cast<uint4*>(hi + at) = make_uint4(nh[0], nh[1], nh[2], nh[3]);
            *reinterpret_cast<uint4*>(lo + at) = make_uint4(nl[0], nl[1], nl[2], nl[3]);
            *reinterpret_cast<uint4*>(hi + at + 2 * D) = make_uint4(sh[0], sh[1], sh[2], sh[3]);
            *reinterpret_cast<uint4*>(lo + at + 2 * D) = make_uint4(sl[0], sl[1], sl[2], sl[3]);
        }
        size += __shfl_xor_sync(0xffffffffu, size, 1);
        size += __shfl_xor_sync(0xffffffffu, size, 2);
        most = max_or_nan(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max_or_nan(most, __shfl_xor_sync(0xffffffffu, most, 2));
        if (my_vec == 0) size_of_token[my_row] = size, most_of_token[my_row] = most;
    }

    const int wm = warp & 3, wn = warp >> 2;
    const uint32_t a_at = smem_u32(hi) + (wm * 16 + (lane & 15)) * row_bytes + (lane >> 4) * 16;
    const uint32_t lo_off = TILE_TOKENS * row_bytes;
    const uint32_t b_at = smem_u32(tile) + (wn * 32 + (lane & 7) + (lane >> 4) * 8) * row_bytes + ((lane >> 3) & 1) * 16;
    uint32_t high_bits = 0, low_bits = 0x80008000u;       // the largest bit patterns, as unsigned and as signed
    uint4 next[8];
    int next_page = -1;
    auto fetch = [&](int base) {        // this thread's pieces of its page of the tile at `base`
        next_page = base + my_row < end ? physical_page(c, b, base + my_row) : -1;
        const uint16_t* at = p.bounds + ((long long)max(next_page, 0) * c.kv_heads + h) * 2 * D;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int v = my_vec + 4 * j;
            next[j] = next_page >= 0 && v < D / 4 ? *reinterpret_cast<const uint4*>(at + v * 8) : make_uint4(0, 0, 0, 0);
        }
    };
    if (begin < end) fetch(begin);
    // (the pages that none of these tokens lets compete are looked up here, by one of the splits; the others are by `fetch`)
    if (blockIdx.z == 0 && h == 0)
        for (long long i = pages + tid; i < seen && i <= c.width; i += TILES_THREADS) physical_page(c, b, i);
    for (int base = begin; base < end; base += TILE_PAGES) {
        __syncthreads();                // the tile before has been read
        if (my_vec == 0) missing[my_row] = next_page < 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int v = my_vec + 4 * j;
            if (v < D / 4) *reinterpret_cast<uint4*>(tile + my_row * row_bytes + v * 16) = next[j];
            high_bits = __vimax3_u16x2(__vimax3_u16x2(high_bits, next[j].x, next[j].y), next[j].z, next[j].w);
            low_bits = __vimax3_s16x2(__vimax3_s16x2(low_bits, next[j].x, next[j].y), next[j].z, next[j].w);
        }
        __syncthreads();
        if (base + TILE_PAGES < end) fetch(base + TILE_PAGES);
        float acc[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
        // Every step starts from zero and is added up by ordinary additions: a tensor core drops what lies below the last
        // bit of its largest term, and a running sum would be that term at every step.
#pragma unroll 4
        for (int k = 0; k < D / 8; ++k) {       // 16 of the 2 D terms
            uint32_t ah[4], al[4], b0[4], b1[4];
            ldmatrix_x4(a_at + k * 32, ah);
            ldmatrix_x4(a_at + lo_off + k * 32, al);
            ldmatrix_x4(b_at + k * 32, b0);
            ldmatrix_x4(b_at + 16 * row_bytes + k * 32, b1);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const uint32_t* f = n < 2 ? b0 : b1;
                float step[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816<BF16>(step, al, f[2 * (n & 1)], f[2 * (n & 1) + 1]);
                mma16816<BF16>(step, ah, f[2 * (n & 1)], f[2 * (n & 1) + 1]);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][i] += step[i];
            }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int col = wn * 32 + n * 8 + (lane & 3) * 2, page = base + col;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = wm * 16 + (lane >> 2) + 8 * half, t = t_first + row;
                if (row < tokens && t >= p.t0 && t < p.t1 && page < end)      // (the pitch is even: the second of a pair has a place)
                    *reinterpret_cast<float2*>(p.scores + ((long long)(t - p.t0) * c.kv_heads + h) * p.pitch + page) =
                        make_float2(missing[col] ? -INFINITY : acc[n][2 * half], missing[col + 1] ? -INFINITY : acc[n][2 * half + 1]);
            }
        }
    }
    float most = reach_of<BF16>(high_bits, low_bits);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = max_or_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (lane == 0) reach_of_warp[warp] = __float_as_uint(most);
    __syncthreads();
    if (tid < tokens && t_first + tid >= p.t0 && t_first + tid < p.t1) {
        for (int w = 0; w < TILES_THREADS / 32; ++w) most = max_or_nan(most, __uint_as_float(reach_of_warp[w]));
        p.errors[((long long)(t_first + tid - p.t0) * c.kv_heads + h) * p.splits + blockIdx.z] =
            score_error<BF16>(p, size_of_token[tid], most_of_token[tid], most, D / 8, 2);
    }
}

constexpr int CHOOSE_THREADS = 128;

// A warp per row, of at most 32 E pages, or (E = 0) a block.
template <bool BF16, int E>
__global__ void __launch_bounds__(CHOOSE_THREADS, E == 16 ? 5 : 3) choose_kernel(const __grid_constant__ SelectParams p) {
    constexpr int ROWS = E > 0 ? CHOOSE_THREADS / 32 : 1;
    typedef BlockTeam<CHOOSE_THREADS, 16> Block;
    typedef WarpTeam<(E > 0 ? E : 4)> Warp;
    __shared__ uint32_t room[2 * 3 * CHOOSE_THREADS / 32];
    __shared__ CloseList close[ROWS];
    grid_dependency_wait();
    grid_launch_dependents();
    const Batch& c = p.c;
    const long long row = (long long)blockIdx.x * ROWS + (E > 0 ? threadIdx.x >> 5 : 0);
    const long long at = row / c.kv_heads;
    const int h = (int)(row % c.kv_heads), t = p.t0 + (int)at;
    if (at >= p.t1 - p.t0) return;
    const int b = sequence_of(c, t);
    Row r = {};
    if (b < c.sequences) r.set(p, t, h, b, position_of(c, b, t));
    int* out = p.chosen + ((long long)t * c.kv_heads + h) * p.k;
    const float* scores = p.scores + row * p.pitch;
    double* exact = p.exact + row * p.pitch;
    if (settled(p, b, r, out, E > 0 ? threadIdx.x & 31 : threadIdx.x, E > 0 ? 32 : CHOOSE_THREADS)) return;
    float error = 0.f;
    for (int s = 0; s < p.splits; ++s) error = max_or_nan(error, p.errors[row * p.splits + s]);
    if (!(error < INFINITY)) error = INFINITY;
    uint32_t ends[3] = {0, 0, 0};
    if constexpr (E > 0) {
        Warp team{scores, &close[threadIdx.x >> 5]};
        choose<BF16>(p, r, team, ends, error, exact, out);
    } else {
        Block team{scores, close, room};
        choose<BF16>(p, r, team, ends, error, exact, out);
    }
}

}  // namespace paged
}  // namespace fcs
