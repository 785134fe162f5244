// Attention of every query over the pages that it chose.
//
// The mathematics: one pass over the chosen pages' keys with a running maximum m and sum l per query,
//     s = scale q . k,   m' = max(m, s),   l' = l 2^(m - m') + 2^(s - m'),   o' = o 2^(m - m') + 2^(s - m') v
// in the log2 domain, and at the end o / l.  The parts that warps and CTAs hold are joined by the same rule.
//
// A row is a token and a key/value head: its group of query heads shares the pages, so that a key is fetched once for
// up to eight (or sixteen) queries.  Keys are the rows of the matrix instructions and queries the columns: S^T = K Q^T and
// O^T = V^T P^T with m16n8k16 -- a group of eight fills them, and a query's statistics are in the threads that hold its
// column of O^T.  S^T becomes the second product's operand by an 8 x 8 transposition in registers (movmatrix).  tcgen05 wants
// 128 rows that share one operand; here every row has pages of its own, one flop a byte and query, and the fetching
// of K and V bounds it, not the products.
//
// A producer warp walks the row's list, finds the pages and has them fetched by TMA into a ring of tiles of 64 keys;
// four warps take 16 keys of every tile each and never meet before the end of the list.  A row with a long list, or
// few rows, are spread over the CTAs of a cluster, which join through distributed shared memory.
//
// Measured, groups of four heads of 128, bf16, pages of 64: 32 sequences x 32 pages (269 MB) 46 us, 5.9 TB/s; 4 sequences x 256
// pages in clusters of eight 47 us; one sequence x 32 pages in clusters of sixteen 7.6 us.  Three tiles of 32 KB in flight per CTA and two CTAs per SM;
// with two tiles and three CTAs the 32 sequences take 53 us, with six tiles and one CTA 49 (and the four sequences 79).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.cuh"
#include "paged_mma.cuh"

namespace fcs {
namespace paged {

constexpr int TILE_KEYS = 64;
constexpr int ATTEND_WARPS = 4;                        // consumers
constexpr int ATTEND_THREADS = (ATTEND_WARPS + 1) * 32;
constexpr int SLAB_BYTES = TILE_KEYS * 128;            // 64 features of a tile's keys

struct AttendParams {
    Batch c;
    const uint16_t* query;
    long long query_st[2], out_st[2];   // token, head
    uint16_t* out;
    float* lse;                    // (tokens, q_heads), or nullptr
    const int* chosen;             // (tokens, kv_heads, k)
    int k, group, q_heads, query_tiles;
    int tile_tokens;               // (attend_shared_kernel) tokens of a CTA
    float c_log2;                  // scale * log2(e)
    int fill_tail;                 // rows behind the last sequence: 1 zeros the output's, 2 sets the sums' to -inf
    int withhold;                  // 1 (self-test): an arrival that never comes is counted, so that no wait for a tile ends
};

template <int DP, int STAGES>
struct AttendLayout {
    static constexpr int SLABS = DP / 64;
    static constexpr int STAGE = 2 * SLABS * SLAB_BYTES;
    static constexpr int OFF_BARS = STAGES * STAGE;                 // full[], empty[]
    static constexpr int OFF_INFO = OFF_BARS + 2 * STAGES * 8;      // visible keys of the four places of a stage's tile
    static constexpr int OFF_FLAG = OFF_INFO + STAGES * 16;
    static constexpr int BYTES = OFF_FLAG + 16 + 1024;              // (1024: alignment of the swizzled tiles)
};

template <bool BF16>
__device__ __forceinline__ uint16_t round_one(float a) {
    if constexpr (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(a));
    return __half_as_ushort(__float2half_rn(a));
}
// The natural logarithm of `sum` weights 2^(s - top + lift).  (A score of +inf makes the weights NaN, not their logarithm.)
__device__ __forceinline__ float lse_of(float top, float sum, float lift) {
    return top == INFINITY ? INFINITY : (top + (log2f(sum) - lift)) * 0.6931471805599453f;
}
__device__ __forceinline__ float ld_peer_f32(uint32_t local_addr, uint32_t rank) {
    uint32_t addr;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(local_addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// What a warp holds of NT * 8 queries: O^T in pieces of 16 features x 8 queries, and per query the reference m of the weights
// 2^(s - m) and their sum (of a thread's keys).  The reference follows the maximum only when a weight would pass 2^8: then all
// weights are scaled anew; a vote in place of six shuffles and D / 2 products for most keys.
template <int KS, int NT, bool BF16>
struct Columns {
    // fp16 has no weights below 2^-25: they are held 2^7 times as large, which leaves 2^8 of its range
    static constexpr float LIFT = BF16 ? 0.f : 7.f, MOST = 8.f;
    float o[NT][KS][4], m[NT][2], l[NT][2];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -FLT_MAX;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
        }
    }

    // 16 keys.  key_at, val_at: this lane's addresses for ldmatrix at feature 0 of the swizzled tiles; q(i, n, b): the queries'
    // operand of step i; seen(n, j): how many of the keys this thread's query sees (none at all where `out` says so); `limit`: keys
    // before it are data; ROWS: whether some of the 16 are not to be seen by some of the queries; USE: the sets of eight columns that
    // take part (in the code, as a branch around every matrix instruction costs more than the instruction).
    template <bool ROWS, int USE, typename Q, typename Out, typename Seen>
    __device__ __forceinline__ void add(uint32_t key_at, uint32_t val_at, float c_log2, int limit, Q q, Out out, Seen seen) {
        const int lane = threadIdx.x & 31, col = lane & 3, row = lane >> 2;
        auto use = [](int n) { return (USE >> n & 1) != 0; };
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            uint32_t a[4], b[2 * NT];
            ldmatrix_x4((key_at ^ ((i & 3) << 5)) + (i / 4) * SLAB_BYTES, a);
            q(i, b);
#pragma unroll
            for (int n = 0; n < NT; ++n)
                if (use(n)) mma16816<BF16>(s[n], a, b[2 * n], b[2 * n + 1]);
        }
        // a thread has keys row, row + 8 of queries 2 col, 2 col + 1
        float x[NT][4];
        bool far = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (!use(n)) continue;
                const float off = out(n, j) ? -INFINITY : LIFT - m[n][j];
                x[n][j] = fmaf(s[n][j], c_log2, off);
                x[n][j + 2] = fmaf(s[n][j + 2], c_log2, off);
                if (ROWS) {
                    if (row >= seen(n, j)) x[n][j] = -INFINITY;
                    if (row + 8 >= seen(n, j)) x[n][j + 2] = -INFINITY;
                }
                far |= fmaxf(x[n][j], x[n][j + 2]) > LIFT + MOST;
            }
        if (__any_sync(0xffffffffu, far)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (!use(n)) continue;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    // (from the scores again: next to the first reference, the lowest number, x says nothing)
                    const bool k0 = x[n][j] != -INFINITY && !out(n, j), k1 = x[n][j + 2] != -INFINITY && !out(n, j);
                    const float y0 = k0 ? s[n][j] * c_log2 : -INFINITY, y1 = k1 ? s[n][j + 2] * c_log2 : -INFINITY;
                    float top = max_or_nan(y0, y1);
                    top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    top = max_or_nan(top, m[n][j]);
                    const float scale = ex2_approx(m[n][j] - top);
                    m[n][j] = top;
                    l[n][j] *= scale;
                    x[n][j] = y0 - (top - LIFT);
                    x[n][j + 2] = y1 - (top - LIFT);
#pragma unroll
                    for (int i = 0; i < KS; ++i) {
                        o[n][i][j] *= scale;
                        o[n][i][j + 2] *= scale;
                    }
                }
            }
        }
        // The weights in 16 bits twice, what the first rounding leaves in the second: one rounding alone would add as much
        // error as the result's own.
        uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (!use(n)) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[n][i] = ex2_approx(x[n][i]);
            l[n][0] += x[n][0] + x[n][2];
            l[n][1] += x[n][1] + x[n][3];
            float r0, r1, r2, r3, z;
            hi[n][0] = transpose8(round_pair<BF16>(x[n][0], x[n][1], r0, r1));
            hi[n][1] = transpose8(round_pair<BF16>(x[n][2], x[n][3], r2, r3));
            lo[n][0] = transpose8(round_pair<BF16>(r0, r1, z, z));
            lo[n][1] = transpose8(round_pair<BF16>(r2, r3, z, z));
        }
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            uint32_t a[4];
            ldmatrix_x4_trans((val_at ^ ((i & 3) << 5)) + (i / 4) * SLAB_BYTES, a);
            if (ROWS) {        // what is not data is anything: 0 times it is not 0
                const int k0 = 2 * col;
                const uint32_t m0 = (k0 < limit ? 0xffffu : 0u) | (k0 + 1 < limit ? 0xffff0000u : 0u);
                const uint32_t m1 = (k0 + 8 < limit ? 0xffffu : 0u) | (k0 + 9 < limit ? 0xffff0000u : 0u);
                a[0] &= m0; a[1] &= m0; a[2] &= m1; a[3] &= m1;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
                if (use(n)) {
                    mma16816<BF16>(o[n][i], a, hi[n][0], hi[n][1]);
                    mma16816<BF16>(o[n][i], a, lo[n][0], lo[n][1]);
                }
        }
    }

    // Into shared memory, for the warps to meet: columns of PITCH floats, references and sums.
    template <int PITCH>
    __device__ __forceinline__ void put(float* part_o, float* part_m, float* part_l) const {
        const int lane = threadIdx.x & 31, col = lane & 3, row = lane >> 2;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float sum = l[n][j];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int at = n * 8 + 2 * col + j;
                if (row == 0) {
                    part_m[at] = m[n][j];
                    part_l[at] = sum;
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    part_o[at * PITCH + i * 16 + row] = o[n][i][j];
                    part_o[at * PITCH + i * 16 + row + 8] = o[n][i][j + 2];
                }
            }
    }
};

// grid: (CL * query tiles * tokens, kv heads); NT * 8 queries of a row's group at a time
template <int DP, int NT, int STAGES, bool BF16, int CL>
__global__ void __launch_bounds__(ATTEND_THREADS)
    attend_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                  const __grid_constant__ AttendParams p) {
    using L = AttendLayout<DP, STAGES>;
    constexpr int KS = DP / 16;       // steps of 16 features
    constexpr float LIFT = Columns<KS, NT, BF16>::LIFT;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t tiles = smem_u32(smem);
    const uint32_t full = tiles + L::OFF_BARS, empty = full + STAGES * 8;
    volatile int* info = reinterpret_cast<volatile int*>(smem + L::OFF_INFO);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_FLAG);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Batch& c = p.c;

    if (tid == 0) {
        prefetch_tensormap(&key_map);
        prefetch_tensormap(&value_map);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full + 8 * s, 1 + p.withhold);
            mbar_init(empty + 8 * s, ATTEND_WARPS);
        }
        *abort_flag = 0;
        mbar_fence_init();
    }
    grid_dependency_wait();
    grid_launch_dependents();
    __syncthreads();

    // neighbouring tokens, which choose many pages in common, run at the same time
    const int rank = (int)(blockIdx.x % CL), tile_q = (int)(blockIdx.x / CL % (unsigned)p.query_tiles);
    const int h = blockIdx.y, t = (int)(blockIdx.x / CL / (unsigned)p.query_tiles);
    const int g0 = tile_q * NT * 8, queries = min(NT * 8, p.group - g0);     // of the group
    const int b = sequence_of(c, t);
    if (b >= c.sequences) {        // (all CTAs of a cluster alike)
        if (rank == 0) {
            if (p.fill_tail & 1)
                for (int i = tid; i < queries * c.dim; i += ATTEND_THREADS)
                    p.out[t * p.out_st[0] + ((long long)h * p.group + g0 + i / c.dim) * p.out_st[1] + i % c.dim] = 0;
            if (p.lse && (p.fill_tail & 2))
                for (int i = tid; i < queries; i += ATTEND_THREADS)
                    p.lse[(long long)t * p.q_heads + h * p.group + g0 + i] = -INFINITY;
        }
        return;
    }
    const long long pos = position_of(c, b, t);
    const int P = 1 << c.page_shift;

    Columns<KS, NT, BF16> have;
    have.clear();

    if (warp == ATTEND_WARPS) {
        // ---- producer: this CTA's share of the list, whole tiles' worth of entries
        const int per_tile = P < TILE_KEYS ? TILE_KEYS / P : 1;      // places of a tile
        const int place_keys = P < TILE_KEYS ? P : TILE_KEYS;
        const int units = (p.k + per_tile - 1) / per_tile;
        const int e0 = min(p.k, (int)((long long)units * rank / CL) * per_tile);
        const int e1 = min(p.k, (int)((long long)units * (rank + 1) / CL) * per_tile);
        const int* list = p.chosen + ((long long)t * c.kv_heads + h) * p.k;
        int stage = 0, phase = 1, place = 0;
        bool fine = true;
        const uint32_t piece = (uint32_t)place_keys * 128u;
        for (int base = e0; base < e1 && fine; base += 32) {
            const int e = base + lane;
            const long long page = e < e1 ? list[e] : -1;
            const long long left = page >= 0 ? pos + 1 - (page << c.page_shift) : 0;
            int visible = left <= 0 ? 0 : left < P ? (int)left : P, at = 0;
            if (visible > 0) {
                at = physical_page(c, b, page);
                if (at < 0) visible = 0;
            }
            uint32_t todo = __ballot_sync(0xffffffffu, visible > 0);
            while (todo && fine) {
                const int src = __ffs(todo) - 1;
                todo &= todo - 1;
                const int my_page = __shfl_sync(0xffffffffu, at, src);
                const int my_visible = __shfl_sync(0xffffffffu, visible, src);
                for (int off = 0; off < my_visible; off += place_keys) {      // (pages of 128 keys are two tiles)
                    if (place == 0) {
                        fine = mbar_wait(empty + 8 * stage, phase, abort_flag, c.status, FCS_STATUS_WAIT_PRODUCER);
                        if (!fine) break;
                        if (lane < 4) info[stage * 4 + lane] = 0;
                        __syncwarp();
                    }
                    if (lane == 0) {
                        info[stage * 4 + place] = my_visible - off;
                        const uint32_t dst = tiles + stage * L::STAGE + place * piece;
#pragma unroll
                        for (int s = 0; s < L::SLABS; ++s) {
                            tma_load_4d(dst + s * SLAB_BYTES, &key_map, full + 8 * stage, s * 64, off, h, my_page);
                            tma_load_4d(dst + (L::SLABS + s) * SLAB_BYTES, &value_map, full + 8 * stage, s * 64, off, h, my_page);
                        }
                    }
                    if (++place == per_tile) {
                        __syncwarp();
                        if (lane == 0) mbar_arrive_expect_tx(full + 8 * stage, (uint32_t)per_tile * 2 * L::SLABS * piece);
                        place = 0;
                        if (++stage == STAGES) stage = 0, phase ^= 1;
                    }
                }
            }
        }
        if (place > 0) {           // (the wait for this stage has passed)
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(full + 8 * stage, (uint32_t)place * 2 * L::SLABS * piece);
            if (++stage == STAGES) stage = 0, phase ^= 1;
        }
        if (fine) fine = mbar_wait(empty + 8 * stage, phase, abort_flag, c.status, FCS_STATUS_WAIT_PRODUCER);
        if (fine) {
            if (lane == 0) {
                info[stage * 4] = -1;      // the end
                mbar_arrive(full + 8 * stage);
            }
        }
    } else {
        // ---- consumers
        const int col = lane & 3, row = lane >> 2;
        uint32_t q[NT][KS][2];     // Q^T: features x queries
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int g = n * 8 + row;
            const uint16_t* src = p.query + t * p.query_st[0] + ((long long)h * p.group + g0 + g) * p.query_st[1];
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int d = i * 16 + half * 8 + col * 2;
                    q[n][i][half] = g < queries && d < c.dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
                }
        }
        const int place_keys = P < TILE_KEYS ? P : TILE_KEYS;
        const int my_place = warp * 16 / place_keys, my_off = warp * 16 % place_keys;
        // addresses of ldmatrix: keys are rows of 128 bytes whose 16-byte pieces are swizzled by the row
        const int key_row = warp * 16 + (lane & 15), val_row = warp * 16 + (lane >> 4) * 8 + (lane & 7);
        const uint32_t key_at = tiles + key_row * 128 + (((lane >> 4) ^ (key_row & 7)) << 4);
        const uint32_t val_at = tiles + L::SLABS * SLAB_BYTES + val_row * 128 + ((((lane >> 3) & 1) ^ (val_row & 7)) << 4);
        constexpr int ALL = (1 << NT) - 1;
        auto query = [&](int i, uint32_t(&f)[2 * NT]) {
#pragma unroll
            for (int n = 0; n < NT; ++n) f[2 * n] = q[n][i][0], f[2 * n + 1] = q[n][i][1];
        };
        auto none = [](int, int) { return false; };
        int stage = 0, phase = 0;
        while (true) {
            if (!mbar_wait(full + 8 * stage, phase, abort_flag, c.status, FCS_STATUS_WAIT_CONSUMER)) break;
            if (info[stage * 4] < 0) break;
            const int visible = info[stage * 4 + my_place] - my_off;       // of this warp's 16 keys
            auto seen = [&](int, int) { return visible; };
            const uint32_t off = stage * L::STAGE;
            if (visible >= 16) have.template add<false, ALL>(key_at + off, val_at + off, p.c_log2, 16, query, none, seen);
            else if (visible > 0) have.template add<true, ALL>(key_at + off, val_at + off, p.c_log2, visible, query, none, seen);
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + 8 * stage);
            if (++stage == STAGES) stage = 0, phase ^= 1;
        }
    }

    // ---- the warps of the CTA meet in the memory of the tiles, which all have been read
    if (*abort_flag) __nanosleep(100000);      // (copies of a CTA that gave up may still be landing)
    __syncthreads();
    constexpr int PITCH = DP + 4;
    float* part_o = reinterpret_cast<float*>(smem);                    // [warps][NT * 8][PITCH]
    float* part_m = part_o + ATTEND_WARPS * NT * 8 * PITCH;            // [warps][NT * 8]
    float* part_l = part_m + ATTEND_WARPS * NT * 8;
    float* cta_o = part_l + ATTEND_WARPS * NT * 8;                     // [NT * 8][PITCH]
    float* cta_m = cta_o + NT * 8 * PITCH;
    float* cta_l = cta_m + NT * 8;
    static_assert((ATTEND_WARPS + 1) * NT * 8 * (PITCH + 2) * 4 <= STAGES * L::STAGE, "the parts fit the tiles' memory");
    if (warp < ATTEND_WARPS)
        have.template put<PITCH>(part_o + warp * NT * 8 * PITCH, part_m + warp * NT * 8, part_l + warp * NT * 8);
    __syncthreads();
    const int items = queries * c.dim;
    for (int i = tid; i < items; i += ATTEND_THREADS) {
        const int query = i / c.dim, d = i % c.dim;
        float top = part_m[query];
#pragma unroll
        for (int w = 1; w < ATTEND_WARPS; ++w) top = max_or_nan(top, part_m[w * NT * 8 + query]);
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < ATTEND_WARPS; ++w) {
            const float scale = ex2_approx(part_m[w * NT * 8 + query] - top);
            sum += part_l[w * NT * 8 + query] * scale;
            acc += part_o[(w * NT * 8 + query) * PITCH + d] * scale;
        }
        if constexpr (CL == 1) {
            const long long head = (long long)h * p.group + g0 + query;
            p.out[t * p.out_st[0] + head * p.out_st[1] + d] = round_one<BF16>(sum == 0.f ? 0.f : acc / sum);
            if (d == 0 && p.lse) p.lse[(long long)t * p.q_heads + head] = lse_of(top, sum, LIFT);
        } else {
            cta_o[query * PITCH + d] = acc;
            if (d == 0) {
                cta_m[query] = top;
                cta_l[query] = sum;
            }
        }
    }
    if constexpr (CL > 1) {
        cluster_sync();
        for (int i = rank * ATTEND_THREADS + tid; i < items; i += CL * ATTEND_THREADS) {
            const int query = i / c.dim, d = i % c.dim;
            float pm[CL], pl[CL], po[CL];
#pragma unroll
            for (int r = 0; r < CL; ++r) {
                pm[r] = ld_peer_f32(smem_u32(&cta_m[query]), r);
                pl[r] = ld_peer_f32(smem_u32(&cta_l[query]), r);
                po[r] = ld_peer_f32(smem_u32(&cta_o[query * PITCH + d]), r);
            }
            float top = pm[0], sum = 0.f, acc = 0.f;
#pragma unroll
            for (int r = 1; r < CL; ++r) top = max_or_nan(top, pm[r]);
#pragma unroll
            for (int r = 0; r < CL; ++r) {
                const float scale = ex2_approx(pm[r] - top);
                sum += pl[r] * scale;
                acc += po[r] * scale;
            }
            const long long head = (long long)h * p.group + g0 + query;
            p.out[t * p.out_st[0] + head * p.out_st[1] + d] = round_one<BF16>(sum == 0.f ? 0.f : acc / sum);
            if (d == 0 && p.lse) p.lse[(long long)t * p.q_heads + head] = lse_of(top, sum, LIFT);
        }
        cluster_sync();       // nobody leaves before its parts have been read
    }
}

// ------------------------------------------------------------------ many tokens a sequence
// Neighbouring tokens choose many pages in common, and what bounds them is the fetching.  So a CTA has several of them, as many as
// fit its sixteen columns: the pages that any of them chose, in a table of token sets, are fetched once, and eight columns
// whose tokens did not choose a page pass over it.  What a token did not choose is masked from its columns -- but 0 times a
// value that is not finite is not 0, so a result that is not finite is formed again from the token's own pages alone, as are
// those of a list that names a page twice.
//
// It is bound by the latency of its chains (ldmatrix, products, exponentials, transposition, products), so that CTAs on an SM
// count: 512 tokens that choose 32 of 512 pages each, half of them in common with their neighbours, groups of four heads: a token
// at a time 284 us and 4.3 GB through L2; 16 columns, four tokens, 2.2 GB and 190 us with three CTAs per SM (two stages of tiles),
// 210 us with two (three stages); 32 columns 240 us and 48 or 64 columns 230 and 236 us, one CTA per SM.  57 tokens in threes, 64
// pages of 16 keys, heads of 64: a token at a time 78 us, in blocks with four CTAs per SM 49.  The table of token sets takes shared
// memory by its width: at heads of 128 three CTAs per SM up to about 1440 pages, two past that (the 512 tokens 225 us).
constexpr int SHARED_NT = 2;
constexpr int SHARED_COLS = SHARED_NT * 8;
constexpr int SHARED_WARPS = 4;                        // consumers
constexpr int SHARED_THREADS = (SHARED_WARPS + 1) * 32;
constexpr int SHARED_PAGES = 8192;                     // of the table of token sets
template <int DP> constexpr int SHARED_CTAS = DP == 128 ? 3 : 4;      // per SM

template <int DP, int STAGES>
struct SharedLayout {
    static constexpr int SLABS = DP / 64;
    static constexpr int STAGE = 2 * SLABS * SLAB_BYTES;
    static constexpr int Q_PITCH = DP * 2 + 16;                                  // bytes of a query: no bank twice
    static constexpr int OFF_Q = STAGES * STAGE;
    static constexpr int OFF_BARS = OFF_Q + SHARED_COLS * Q_PITCH;               // full[], empty[]
    static constexpr int OFF_INFO = OFF_BARS + 2 * STAGES * 8;                   // token set and first position of a stage's four places
    static constexpr int OFF_FLAGS = OFF_INFO + STAGES * 32;
    static constexpr int OFF_SETS = OFF_FLAGS + 16;
    static constexpr int bytes(int pages) { return OFF_SETS + 4 * pages + 1024; }
};

// grid: (CL * token tiles, kv heads); sequence b has the tiles from starts[b] / tile + b on, at least as many as it needs
template <int DP, int STAGES, bool BF16, int CL>
__global__ void __launch_bounds__(SHARED_THREADS, SHARED_CTAS<DP>)
    attend_shared_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                         const __grid_constant__ AttendParams p) {
    using L = SharedLayout<DP, STAGES>;
    constexpr int KS = DP / 16, NT = SHARED_NT;
    constexpr float LIFT = Columns<KS, NT, BF16>::LIFT;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    const uint32_t tiles = smem_u32(smem);
    const uint32_t full = tiles + L::OFF_BARS, empty = full + STAGES * 8;
    volatile int* info = reinterpret_cast<volatile int*>(smem + L::OFF_INFO);
    volatile int* flags = reinterpret_cast<volatile int*>(smem + L::OFF_FLAGS);      // abort, a page twice, not finite
    volatile int* abort_flag = flags;
    uint32_t* sets = reinterpret_cast<uint32_t*>(smem + L::OFF_SETS);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const Batch& c = p.c;

    if (tid == 0) {
        prefetch_tensormap(&key_map);
        prefetch_tensormap(&value_map);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full + 8 * s, 1 + p.withhold);
            mbar_init(empty + 8 * s, SHARED_WARPS);
        }
        flags[0] = flags[1] = flags[2] = 0;
        mbar_fence_init();
    }
    grid_dependency_wait();
    grid_launch_dependents();

    const int rank = (int)(blockIdx.x % CL), tile = (int)(blockIdx.x / CL), h = blockIdx.y, G = p.group;
    const int b = count_before(c.sequences, [&](int i) { return c.starts[i + 1] / p.tile_tokens + (long long)(i + 1) <= tile; });
    const long long s0 = c.starts[b];
    if (b >= c.sequences) {        // (all CTAs of a cluster alike)
        // the tiles that no sequence needs share the rows behind the last one
        const long long rest = tile - (s0 / p.tile_tokens + b), step = gridDim.x / CL - tile + rest;
        if (rank > 0) return;
        for (long long t = max(s0, 0ll) + rest; t < c.tokens; t += step) {
            if (p.fill_tail & 1)
                for (int i = tid; i < G * c.dim; i += SHARED_THREADS)
                    p.out[t * p.out_st[0] + ((long long)h * G + i / c.dim) * p.out_st[1] + i % c.dim] = 0;
            if (p.lse && (p.fill_tail & 2))
                for (int i = tid; i < G; i += SHARED_THREADS) p.lse[t * p.q_heads + h * G + i] = -INFINITY;
        }
        return;
    }
    const long long s1 = c.starts[b + 1], t0 = s0 + (tile - (s0 / p.tile_tokens + b)) * p.tile_tokens;
    if (s0 < 0 || s1 > c.tokens || t0 < s0 || t0 >= s1) return;
    const int tokens = (int)min((long long)p.tile_tokens, s1 - t0);
    // of the first token (no table here is as long, and no block reaches back from there to a key)
    const int pos0 = (int)max(min(position_of(c, b, (int)t0), 1ll << 30), -(1ll << 30));
    const int P = 1 << c.page_shift;
    const int pages = pos0 + tokens <= 0 ? 0 : (pos0 + tokens - 1 >> c.page_shift) + 1;      // that the last token sees

    // the queries, and who chose which page
    for (int i = tid; i < SHARED_COLS * (DP / 8); i += SHARED_THREADS) {
        const int col = i / (DP / 8), d = i % (DP / 8) * 8, tok = col / G;
        uint4 q = make_uint4(0, 0, 0, 0);
        if (tok < tokens && d < c.dim)
            q = *reinterpret_cast<const uint4*>(p.query + (t0 + tok) * p.query_st[0] + ((long long)h * G + col % G) * p.query_st[1] + d);
        *reinterpret_cast<uint4*>(smem + L::OFF_Q + col * L::Q_PITCH + d * 2) = q;
    }
    const int table_pages = min(pages, c.width);
    for (int i = tid; i < table_pages; i += SHARED_THREADS) sets[i] = 0;
    __syncthreads();
    for (int i = tid; i < tokens * p.k; i += SHARED_THREADS) {
        const int tok = i / p.k, page = p.chosen[((t0 + tok) * c.kv_heads + h) * p.k + i % p.k];
        if (page < 0 || pos0 + tok < 0 || page > (pos0 + tok) >> c.page_shift) continue;
        if (page >= c.width) report(c, FCS_STATUS_BAD_PAGE);
        else if (atomicOr(&sets[page], 1u << tok) >> tok & 1u) flags[1] = 1;
    }
    __syncthreads();
    const bool twice = flags[1] != 0;

    // The ring goes on from pass to pass: one over the sets, and if need be one over each token's own list.
    int stage = 0, phase = warp == SHARED_WARPS ? 1 : 0;
    bool fine = true;
    int pass = twice ? 0 : -1;
    while (true) {
        Columns<KS, NT, BF16> have;
        have.clear();
        if (warp == SHARED_WARPS) {
            // ---- producer: of the table or the list this CTA's share
            const int per_tile = P < TILE_KEYS ? TILE_KEYS / P : 1;
            const int place_keys = P < TILE_KEYS ? P : TILE_KEYS;
            const uint32_t piece = (uint32_t)place_keys * 128u;
            const int entries = pass < 0 ? table_pages : p.k;
            const int* list = p.chosen + ((t0 + max(pass, 0)) * c.kv_heads + h) * p.k;
            int place = 0;
            for (int base = 0; base < entries && fine; base += 32 * CL) {
                const int e = base + lane * CL + rank;
                int page = -1, at = 0;
                uint32_t set = 0;
                if (e < entries) {
                    page = pass < 0 ? e : list[e];
                    if (pass < 0) set = sets[e];
                    else if (page >= 0 && page < c.width && pos0 + pass >= 0 && page <= (pos0 + pass) >> c.page_shift) set = 1u << pass;
                }
                if (set) {
                    at = physical_page(c, b, page);
                    if (at < 0) set = 0;
                }
                uint32_t todo = __ballot_sync(0xffffffffu, set != 0);
                while (todo && fine) {
                    const int src = __ffs(todo) - 1;
                    todo &= todo - 1;
                    const int my_at = __shfl_sync(0xffffffffu, at, src), my_page = __shfl_sync(0xffffffffu, page, src);
                    const uint32_t my_set = __shfl_sync(0xffffffffu, set, src);
                    const int first = my_page << c.page_shift, end = pos0 + 32 - __clz(my_set);       // the set's last token sees up to there
                    for (int off = 0; off < P && first + off < end; off += place_keys) {
                        if (place == 0) {
                            fine = mbar_wait(empty + 8 * stage, phase, abort_flag, c.status, FCS_STATUS_WAIT_PRODUCER);
                            if (!fine) break;
                            if (lane < 4) info[stage * 8 + lane] = 0;
                            __syncwarp();
                        }
                        if (lane == 0) {
                            info[stage * 8 + place] = (int)my_set;
                            info[stage * 8 + 4 + place] = first + off;
                            const uint32_t dst = tiles + stage * L::STAGE + place * piece;
#pragma unroll
                            for (int s = 0; s < L::SLABS; ++s) {
                                tma_load_4d(dst + s * SLAB_BYTES, &key_map, full + 8 * stage, s * 64, off, h, my_at);
                                tma_load_4d(dst + (L::SLABS + s) * SLAB_BYTES, &value_map, full + 8 * stage, s * 64, off, h, my_at);
                            }
                        }
                        if (++place == per_tile) {
                            __syncwarp();
                            if (lane == 0) mbar_arrive_expect_tx(full + 8 * stage, (uint32_t)per_tile * 2 * L::SLABS * piece);
                            place = 0;
                            if (++stage == STAGES) stage = 0, phase ^= 1;
                        }
                    }
                }
            }
            if (place > 0) {           // (the wait for this stage has passed)
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(full + 8 * stage, (uint32_t)place * 2 * L::SLABS * piece);
                if (++stage == STAGES) stage = 0, phase ^= 1;
            }
            if (fine) fine = mbar_wait(empty + 8 * stage, phase, abort_flag, c.status, FCS_STATUS_WAIT_PRODUCER);
            if (fine) {
                if (lane == 0) {
                    info[stage * 8 + 4] = -1;      // the end
                    mbar_arrive(full + 8 * stage);
                }
                if (++stage == STAGES) stage = 0, phase ^= 1;
            }
        } else {
            // ---- consumers
            int tok[NT][2];            // of this thread's columns; 31: of nobody
            uint32_t mine[NT];         // the tokens of eight columns
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int k = (n * 8 + 2 * (lane & 3) + j) / G;
                    tok[n][j] = k < tokens ? k : 31;
                }
                mine[n] = __reduce_or_sync(0xffffffffu, 1u << tok[n][0] | 1u << tok[n][1]) & 0x7fffffffu;
            }
            const int place_keys = P < TILE_KEYS ? P : TILE_KEYS;
            const int my_place = warp * 16 / place_keys, my_off = warp * 16 % place_keys;
            const int key_row = warp * 16 + (lane & 15), val_row = warp * 16 + (lane >> 4) * 8 + (lane & 7);
            const uint32_t key_at = tiles + key_row * 128 + (((lane >> 4) ^ (key_row & 7)) << 4);
            const uint32_t val_at = tiles + L::SLABS * SLAB_BYTES + val_row * 128 + ((((lane >> 3) & 1) ^ (val_row & 7)) << 4);
            const uint32_t q_at = tiles + L::OFF_Q + ((lane & 7) + (lane >> 4) * 8) * L::Q_PITCH + ((lane >> 3) & 1) * 16;
            auto query = [&](int i, uint32_t(&f)[2 * NT]) { ldmatrix_x4(q_at + i * 32, f); };
            while (true) {
                if (!mbar_wait(full + 8 * stage, phase, abort_flag, c.status, FCS_STATUS_WAIT_CONSUMER)) {
                    fine = false;
                    break;
                }
                const bool last = info[stage * 8 + 4] < 0;
                const uint32_t set = last ? 0u : (uint32_t)info[stage * 8 + my_place];
                const int first = info[stage * 8 + 4 + my_place] + my_off;          // position of this warp's 16 keys
                const int some = pos0 + 32 - __clz(set) - first;                      // of them that the set's last token sees
                if ((set & (mine[0] | mine[1])) && some > 0) {
                    auto out = [&](int n, int j) { return !(set >> tok[n][j] & 1u); };
                    auto seen = [&](int n, int j) { return pos0 + tok[n][j] + 1 - first; };
                    const uint32_t off = stage * L::STAGE;
                    if (first + 16 > pos0 + 1) have.template add<true, 3>(key_at + off, val_at + off, p.c_log2, some, query, out, seen);
                    else if (!(set & mine[1])) have.template add<false, 1>(key_at + off, val_at + off, p.c_log2, 16, query, out, seen);
                    else if (!(set & mine[0])) have.template add<false, 2>(key_at + off, val_at + off, p.c_log2, 16, query, out, seen);
                    else have.template add<false, 3>(key_at + off, val_at + off, p.c_log2, 16, query, out, seen);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + 8 * stage);
                if (++stage == STAGES) stage = 0, phase ^= 1;
                if (last) break;
            }
        }

        // ---- the warps meet in the memory of the tiles, which all have been read
        if (*abort_flag) __nanosleep(100000);      // (copies of a CTA that gave up may still be landing)
        __syncthreads();
        constexpr int PITCH = DP + 4;
        float* part_o = reinterpret_cast<float*>(smem);                    // [4][columns][PITCH]
        float* part_m = part_o + 4 * SHARED_COLS * PITCH;                  // [4][columns]
        float* part_l = part_m + 4 * SHARED_COLS;
        static_assert(4 * SHARED_COLS * (PITCH + 2) * 4 <= STAGES * L::STAGE, "the parts fit the tiles' memory");
        if (warp < SHARED_WARPS) {
            const int at = warp * SHARED_COLS;
            have.template put<PITCH>(part_o + at * PITCH, part_m + at, part_l + at);
        }
        if constexpr (CL > 1) cluster_sync(); else __syncthreads();
        // what every CTA writes: a share of the columns' pairs of features
        const int half_dim = c.dim / 2, items = tokens * G * half_dim;
        bool odd = false;
        for (int i = rank * SHARED_THREADS + tid; i < items; i += CL * SHARED_THREADS) {
            const int column = i / half_dim, d = i % half_dim * 2, tk = column / G;
            if (pass >= 0 && tk != pass) continue;
            float top = -FLT_MAX, sum = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll
            for (int r = 0; r < 4 * CL; ++r) {
                const float* pm = &part_m[r % 4 * SHARED_COLS + column];
                top = max_or_nan(top, CL == 1 ? *pm : ld_peer_f32(smem_u32(pm), r / 4));
            }
#pragma unroll
            for (int r = 0; r < 4 * CL; ++r) {
                const float* pm = &part_m[r % 4 * SHARED_COLS + column];
                const float* pl = &part_l[r % 4 * SHARED_COLS + column];
                const float* po = &part_o[(r % 4 * SHARED_COLS + column) * PITCH + d];
                const float scale = ex2_approx((CL == 1 ? *pm : ld_peer_f32(smem_u32(pm), r / 4)) - top);
                sum += (CL == 1 ? *pl : ld_peer_f32(smem_u32(pl), r / 4)) * scale;
                a0 += (CL == 1 ? po[0] : ld_peer_f32(smem_u32(po), r / 4)) * scale;
                a1 += (CL == 1 ? po[1] : ld_peer_f32(smem_u32(po + 1), r / 4)) * scale;
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            a0 = sum == 0.f ? 0.f : a0 * inv;
            a1 = sum == 0.f ? 0.f : a1 * inv;
            odd |= !(fabsf(a0) < INFINITY) || !(fabsf(a1) < INFINITY);
            float z;
            const long long head = (long long)h * G + column % G;
            *reinterpret_cast<uint32_t*>(p.out + (t0 + tk) * p.out_st[0] + head * p.out_st[1] + d) = round_pair<BF16>(a0, a1, z, z);
            if (d == 0 && p.lse) p.lse[(t0 + tk) * p.q_heads + head] = lse_of(top, sum, LIFT);
        }
        if (pass < 0) {
            // a result that is not finite, of any CTA: again, token by token
            if (__syncthreads_or(odd) && tid == 0) {
                if constexpr (CL == 1) {
                    flags[2] = 1;
                } else {
#pragma unroll
                    for (int r = 0; r < CL; ++r) {
                        uint32_t at;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(smem + L::OFF_FLAGS + 8)), "r"(r));
                        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(1) : "memory");
                    }
                }
            }
            __syncwarp();
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // (the tiles' memory goes back to the copies)
        if constexpr (CL > 1) cluster_sync(); else __syncthreads();        // the parts have been read
        // (the CTAs of a cluster go on or stop together, also where one of them has given up a wait)
        if (pass < 0 ? flags[2] == 0 : pass + 1 == tokens) break;
        ++pass;
    }
}

}  // namespace paged
}  // namespace fcs
