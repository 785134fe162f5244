// Attention of every query over the pages that it chose.
//
// The mathematics: one pass over the chosen pages' keys with a running maximum m and sum l per query,
//     s = scale q . k,   m' = max(m, s),   l' = l 2^(m - m') + 2^(s - m'),   o' = o 2^(m - m') + 2^(s - m') v
// in the log2 domain, and at the end o / l.  The parts that warps and CTAs hold are joined by the same rule.
//
// A row is a token and a key/value head: its group of query heads shares the pages, so that a key is fetched once for
// up to eight (or sixteen) queries.  Keys are the rows of the matrix instructions and queries the columns: S^T = K Q^T and
// O^T = V^T P^T with m16n8k16 -- a group of eight fills them, and a query's statistics are in the threads that hold its
// column of O^T.  S^T becomes the second product's operand by an 8 x 8 transposition in registers (movmatrix).  tcgen05 needs
// 128 rows that share one operand; here every row has pages of its own, and the fetching of K and V bounds it, not
// the products (DESIGN: 4 flops a byte and query).
//
// A producer warp walks the row's list, finds the pages and has them fetched by TMA into a ring of tiles of 64 keys;
// four warps take 16 keys of every tile each and never meet before the end of the list.  A row with a long list, or
// few rows, are spread over the CTAs of a cluster, which join through distributed shared memory.
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
    float c_log2;                  // scale * log2(e)
    int fill_tail;                 // rows behind the last sequence: 1 zeros the output's, 2 sets the sums' to -inf
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
__device__ __forceinline__ float ld_peer_f32(uint32_t local_addr, uint32_t rank) {
    uint32_t addr;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(local_addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// grid: (CL * query tiles * tokens, kv heads); NT * 8 queries of a row's group at a time
template <int DP, int NT, int STAGES, bool BF16, int CL>
__global__ void __launch_bounds__(ATTEND_THREADS)
    attend_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                  const __grid_constant__ AttendParams p) {
    using L = AttendLayout<DP, STAGES>;
    constexpr int KS = DP / 16;       // steps of 16 features
    // fp16 has no weights below 2^-25: they are held 2^12 times as large
    constexpr float LIFT = BF16 ? 0.f : 12.f;
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
            mbar_init(full + 8 * s, 1);
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

    float o[NT][KS][4];            // O^T: 16 features x 8 queries each
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -FLT_MAX;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

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
        const int key_row = warp * 16 + (lane & 15), key_chunk = lane >> 4;
        const int val_row = warp * 16 + (lane >> 4) * 8 + (lane & 7), val_chunk = (lane >> 3) & 1;
        int stage = 0, phase = 0;
        while (true) {
            if (!mbar_wait(full + 8 * stage, phase, abort_flag, c.status, FCS_STATUS_WAIT_CONSUMER)) break;
            if (info[stage * 4] < 0) break;
            const int visible = info[stage * 4 + my_place] - my_off;       // of this warp's 16 keys
            if (visible > 0) {
                const uint32_t ktile = tiles + stage * L::STAGE, vtile = ktile + L::SLABS * SLAB_BYTES;
                float s[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t a[4];
                    const int chunk = (2 * i + key_chunk) & 7;
                    ldmatrix_x4(ktile + (i / 4) * SLAB_BYTES + key_row * 128 + ((chunk ^ (key_row & 7)) << 4), a);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16816<BF16>(s[n], a, q[n][i][0], q[n][i][1]);
                }
                uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    // a thread has keys row, row + 8 of queries 2 col, 2 col + 1
                    float x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = s[n][i] * p.c_log2;
                    if (row >= visible) x[0] = x[1] = -INFINITY;
                    if (row + 8 >= visible) x[2] = x[3] = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float top = max_or_nan(x[j], x[j + 2]);
                        top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = max_or_nan(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        top = max_or_nan(top, m[n][j]);
                        const float scale = ex2_approx(m[n][j] - top);
                        m[n][j] = top;
                        x[j] = ex2_approx(x[j] - (top - LIFT));
                        x[j + 2] = ex2_approx(x[j + 2] - (top - LIFT));
                        l[n][j] = l[n][j] * scale + (x[j] + x[j + 2]);
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            o[n][i][j] *= scale;
                            o[n][i][j + 2] *= scale;
                        }
                    }
                    // the weights in 16 bits twice, what the first rounding leaves in the second: one rounding alone
                    // would add as much error as the result's own
                    float r0, r1, r2, r3, z;
                    ph[n][0] = transpose8(round_pair<BF16>(x[0], x[1], r0, r1));
                    ph[n][1] = transpose8(round_pair<BF16>(x[2], x[3], r2, r3));
                    pl[n][0] = transpose8(round_pair<BF16>(r0, r1, z, z));
                    pl[n][1] = transpose8(round_pair<BF16>(r2, r3, z, z));
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    uint32_t a[4];
                    const int chunk = (2 * i + val_chunk) & 7;
                    ldmatrix_x4_trans(vtile + (i / 4) * SLAB_BYTES + val_row * 128 + ((chunk ^ (val_row & 7)) << 4), a);
                    if (visible < 16) {        // what lies behind the last token is anything: 0 times it is not 0
                        const int k0 = 2 * col;
                        const uint32_t m0 = (k0 < visible ? 0xffffu : 0u) | (k0 + 1 < visible ? 0xffff0000u : 0u);
                        const uint32_t m1 = (k0 + 8 < visible ? 0xffffu : 0u) | (k0 + 9 < visible ? 0xffff0000u : 0u);
                        a[0] &= m0; a[1] &= m0; a[2] &= m1; a[3] &= m1;
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma16816<BF16>(o[n][i], a, ph[n][0], ph[n][1]);
                        mma16816<BF16>(o[n][i], a, pl[n][0], pl[n][1]);
                    }
                }
            }
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
    if (warp < ATTEND_WARPS) {
        const int col = lane & 3, row = lane >> 2;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float sum = l[n][j];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int query = warp * NT * 8 + n * 8 + 2 * col + j;
                if (row == 0) {
                    part_m[query] = m[n][j];
                    part_l[query] = sum;
                }
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    part_o[query * PITCH + i * 16 + row] = o[n][i][j];
                    part_o[query * PITCH + i * 16 + row + 8] = o[n][i][j + 2];
                }
            }
    }
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
            if (d == 0 && p.lse) p.lse[(long long)t * p.q_heads + head] = (top + (log2f(sum) - LIFT)) * 0.6931471805599453f;
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
            if (d == 0 && p.lse) p.lse[(long long)t * p.q_heads + head] = (top + (log2f(sum) - LIFT)) * 0.6931471805599453f;
        }
        cluster_sync();       // nobody leaves before its parts have been read
    }
}

}  // namespace paged
}  // namespace fcs
