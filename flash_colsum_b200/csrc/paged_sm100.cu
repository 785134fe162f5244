// Entry points over a paged cache: appending to it, choosing pages of it, attending over chosen pages.  The kernels are in
// paged_append.cuh, paged_select.cuh and paged_attend.cuh.
#include <float.h>
#include <math.h>
#include <string.h>

#include "../../include/flash_colsum_b200.h"
#include "host_api.h"
#include "host_common.h"
#include "paged_append.cuh"
#include "paged_attend.cuh"
#include "paged_select.cuh"

namespace fcs {
namespace paged {

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Strides (in elements) of `n` outer axes of a tensor of 16-bit elements whose rows are read in pieces of 16 bytes.
static int check_rows(const char* name, const void* ptr, const int64_t* stride, int n) {
    if (!ptr) return fail(FCS_ERR_INVALID_ARGUMENT, "%s is NULL", name);
    if (!aligned16(ptr)) return fail(FCS_ERR_INVALID_ARGUMENT, "%s must be 16-byte aligned", name);
    for (int i = 0; i < n; ++i)
        if (stride[i] < 0 || stride[i] % 8)
            return fail(FCS_ERR_INVALID_ARGUMENT, "%s strides must not be negative and be multiples of 8 elements", name);
    return FCS_OK;
}

static int check_result(const char* name, const FcsPagedCache* c, int q_heads, const int64_t* stride) {
    const int64_t size[2] = {c->tokens, q_heads};
    if (fcs_rows_apart(2, size, stride, c->dim)) return FCS_OK;
    return fail(FCS_ERR_INVALID_ARGUMENT, "%s strides must keep its rows apart", name);
}

// A pool that is written.
static int check_written(const char* name, const FcsPagedCache* c, const int64_t* stride) {
    const int64_t size[3] = {c->pages, c->kv_heads, c->page_size};
    if (fcs_rows_apart(3, size, stride, c->dim)) return FCS_OK;
    return fail(FCS_ERR_INVALID_ARGUMENT, "%s strides must keep its rows apart", name);
}

static int check_cache(const FcsPagedCache* c, Batch& out, int* status) {
    if (!c) return fail(FCS_ERR_INVALID_ARGUMENT, "cache is NULL");
    if (c->dim % 8 || c->dim < 8 || c->dim > 128)
        return fail(FCS_ERR_UNSUPPORTED, "head dimension must be a multiple of 8 from 8 to 128, got %d", c->dim);
    if (c->dtype != FCS_DTYPE_FP16 && c->dtype != FCS_DTYPE_BF16)
        return fail(FCS_ERR_UNSUPPORTED, "dtype must be FCS_DTYPE_FP16 or FCS_DTYPE_BF16, got %d", c->dtype);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return fail(FCS_ERR_UNSUPPORTED, "page size must be 16, 32, 64 or 128, got %d", c->page_size);
    if (c->pages <= 0 || c->kv_heads <= 0 || c->kv_heads > 65535 || c->sequences <= 0 || c->table_width <= 0 || c->tokens <= 0)
        return fail(FCS_ERR_INVALID_ARGUMENT, "sizes must be positive (pages=%d kv_heads=%d sequences=%d table_width=%d tokens=%d)",
                    c->pages, c->kv_heads, c->sequences, c->table_width, c->tokens);
    if (c->table_width > 1 << 28) return fail(FCS_ERR_UNSUPPORTED, "the table has too many pages a sequence (%d)", c->table_width);
    if (!c->page_table || !c->lens) return fail(FCS_ERR_INVALID_ARGUMENT, "page_table and lens must not be NULL");
    if (c->table_stride < c->table_width && c->sequences > 1)
        return fail(FCS_ERR_INVALID_ARGUMENT, "table_stride (%lld) is smaller than the table's width", (long long)c->table_stride);
    if (!c->starts && c->tokens != c->sequences)
        return fail(FCS_ERR_INVALID_ARGUMENT, "without starts there is one token a sequence, got %d tokens and %d sequences",
                    c->tokens, c->sequences);
    out.table = c->page_table;
    out.table_ld = c->table_stride;
    out.lens = c->lens;
    out.starts = c->starts;
    out.pages = c->pages;
    out.kv_heads = c->kv_heads;
    out.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    out.dim = c->dim;
    out.sequences = c->sequences;
    out.width = c->table_width;
    out.tokens = c->tokens;
    out.status = status;
    return FCS_OK;
}

static int check_group(const FcsPagedCache* c, int q_heads) {
    if (q_heads <= 0 || q_heads % c->kv_heads)
        return fail(FCS_ERR_INVALID_ARGUMENT, "query heads (%d) must be a multiple of the key heads (%d)", q_heads, c->kv_heads);
    return FCS_OK;
}

// Every kernel may start while the one before it in the stream drains (it waits for it before it reads).
template <typename... Params, typename... Args>
static cudaError_t launch(void (*kern)(Params...), dim3 grid, int threads, int smem, int cluster, cudaStream_t stream,
                          const Args&... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = cluster;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <typename F>
static cudaError_t allow_smem(F* kern, int bytes, bool wide_cluster = false) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && wide_cluster) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return e;
}

// Runs `set_up` once per device and instance (`done` is the instance's).
template <typename F>
static cudaError_t once_per_device(bool (&done)[64], F set_up) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev < 64 && done[dev])) return e;
    e = set_up();
    if (e == cudaSuccess && dev < 64) done[dev] = true;
    return e;
}

// Whether the current device can hold a cluster of sixteen CTAs of `kern` (asked once per device; `known` is the instance's: 0 not
// asked, 1 no, 2 yes).
template <typename F>
static bool sixteen_fit(int (&known)[64], F* kern, int threads, int smem) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return false;
    if (known[dev] == 0) {
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof(cfg));
        cfg.gridDim = dim3(16);
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 16;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        const bool fits = allow_smem(kern, smem, true) == cudaSuccess &&
                          cudaOccupancyMaxActiveClusters(&n, kern, &cfg) == cudaSuccess && n > 0;
        if (!fits) cudaGetLastError();
        known[dev] = fits ? 2 : 1;
    }
    return known[dev] == 2;
}

// ------------------------------------------------------------------ append
template <typename Ops>
static cudaError_t launch_append(int rot, dim3 grid, cudaStream_t stream, const AppendParams& p) {
    return rot == 0   ? launch(append_kernel<Ops, 0>, grid, APPEND_THREADS, 0, 1, stream, p)
           : rot == 1 ? launch(append_kernel<Ops, 1>, grid, APPEND_THREADS, 0, 1, stream, p)
                      : launch(append_kernel<Ops, 2>, grid, APPEND_THREADS, 0, 1, stream, p);
}

struct AppendPlan {
    int heads_shift, steps;
};

// A CTA has about 32 rows at a time, the heads of a group times the tokens of a page.  Of long calls it has more of the values
// and queries, whose heads share a token's rotation: 16384 tokens, 32 and 8 heads 121 us with one step, 78 with two, 76 with
// four; 1861 tokens of 7 sequences, 16 and 16 heads, pages of 16 13.2 us with one, 11.2 with two, 12.0 with four.
static AppendPlan append_plan(const FcsPagedCache* cache, int q_heads) {
    AppendPlan a = {0, 1};
    const long long B = cache->sequences, T = cache->tokens, P = cache->page_size;
    const long long each = cache->starts ? (T / B < P ? (T + B - 1) / B : P) : 1;
    while (a.heads_shift < 3 && (each << a.heads_shift) < 32) ++a.heads_shift;
    const long long ctas = T / each * (q_heads + cache->kv_heads) / (1 << a.heads_shift);
    a.steps = ctas >= 32ll * num_sms() ? 4 : ctas >= 8ll * num_sms() ? 2 : 1;
    return a;
}

static int append(const FcsPagedCache* cache, const FcsPagedRows* r, int* status, cudaStream_t stream) {
    AppendParams p;
    memset(&p, 0, sizeof(p));
    int rc = check_cache(cache, p.c, status);
    if (rc != FCS_OK) return rc;
    if (!r) return fail(FCS_ERR_INVALID_ARGUMENT, "rows is NULL");
    if ((rc = check_rows("key", r->key, r->key_stride, 2)) != FCS_OK) return rc;
    if ((rc = check_rows("value", r->value, r->value_stride, 2)) != FCS_OK) return rc;
    if ((rc = check_rows("key_pages", cache->key_pages, cache->key_stride, 3)) != FCS_OK) return rc;
    if ((rc = check_rows("value_pages", cache->value_pages, cache->value_stride, 3)) != FCS_OK) return rc;
    if ((rc = check_written("key_pages", cache, cache->key_stride)) != FCS_OK) return rc;
    if ((rc = check_written("value_pages", cache, cache->value_stride)) != FCS_OK) return rc;
    const bool with_query = r->query != nullptr;
    if (with_query) {
        if ((rc = check_rows("query", r->query, r->query_stride, 2)) != FCS_OK) return rc;
        if ((rc = check_rows("query_out", r->query_out, r->query_out_stride, 2)) != FCS_OK) return rc;
        if ((rc = check_group(cache, r->q_heads)) != FCS_OK) return rc;
        if ((rc = check_result("query_out", cache, r->q_heads, r->query_out_stride)) != FCS_OK) return rc;
        if (r->q_heads > 65535 * 8) return fail(FCS_ERR_UNSUPPORTED, "too many query heads (%d)", r->q_heads);
    }
    if ((r->cos == nullptr) != (r->sin == nullptr)) return fail(FCS_ERR_INVALID_ARGUMENT, "cos and sin go together");
    if (r->cos) {
        if (!aligned16(r->cos) || !aligned16(r->sin)) return fail(FCS_ERR_INVALID_ARGUMENT, "cos and sin must be 16-byte aligned");
        if (r->rotary % 16 || r->rotary < 16 || r->rotary > cache->dim)
            return fail(FCS_ERR_UNSUPPORTED, "the rotated features must be a multiple of 16 up to the head dimension, got %d", r->rotary);
        if (r->table_rows <= 0) return fail(FCS_ERR_INVALID_ARGUMENT, "cos and sin have no rows");
        p.cos = r->cos;
        p.sin = r->sin;
        p.rotary = r->rotary;
        p.table_rows = r->table_rows;
        p.positions = r->positions;
    }
    if (r->bounds && !aligned16(r->bounds)) return fail(FCS_ERR_INVALID_ARGUMENT, "bounds must be 16-byte aligned");
    p.key = static_cast<const uint16_t*>(r->key);
    p.value = static_cast<const uint16_t*>(r->value);
    p.query = static_cast<const uint16_t*>(r->query);
    p.query_out = static_cast<uint16_t*>(r->query_out);
    p.bounds = static_cast<uint16_t*>(r->bounds);
    p.key_pages = static_cast<uint16_t*>(cache->key_pages);
    p.value_pages = static_cast<uint16_t*>(cache->value_pages);
    for (int i = 0; i < 2; ++i) {
        p.key_st[i] = r->key_stride[i];
        p.value_st[i] = r->value_stride[i];
        p.query_st[i] = r->query_stride[i];
        p.query_out_st[i] = r->query_out_stride[i];
    }
    for (int i = 0; i < 3; ++i) {
        p.key_page_st[i] = cache->key_stride[i];
        p.value_page_st[i] = cache->value_stride[i];
    }
    p.q_heads = with_query ? r->q_heads : 0;
    p.fill_tail = r->fill_tail != 0;
    const AppendPlan plan = append_plan(cache, p.q_heads);
    p.heads_shift = plan.heads_shift;
    p.steps = plan.steps;
    const int heads = 1 << p.heads_shift;
    const long long B = cache->sequences, T = cache->tokens, P = cache->page_size;
    p.key_groups = (cache->kv_heads + heads - 1) / heads;
    p.value_groups = (cache->kv_heads + heads * p.steps - 1) / (heads * p.steps);
    const long long segments = cache->starts ? T / P + 2 * B + 1 : B;
    const long long groups = (long long)p.key_groups + p.value_groups + (p.q_heads + heads * p.steps - 1) / (heads * p.steps);
    if (segments * groups > 0x7fffffffll)
        return fail(FCS_ERR_UNSUPPORTED, "the call is too large for one launch (%lld tokens, %d heads)", T, p.q_heads);
    p.groups = (int)groups;
    const dim3 grid((unsigned)(segments * groups));
    const int rot = !p.cos ? 0 : r->interleaved ? 2 : 1;
    const cudaError_t e = cache->dtype == FCS_DTYPE_BF16 ? launch_append<Bf16Ops>(rot, grid, stream, p)
                                                         : launch_append<HalfOps>(rot, grid, stream, p);
    if (e != cudaSuccess) return fail(FCS_ERR_CUDA, "appending failed to launch: %s", cudaGetErrorString(e));
    return FCS_OK;
}

// ------------------------------------------------------------------ select
constexpr int ROW_PAGES = 32768;       // scores that a CTA's shared memory holds beside its pages

// Scores of a row, with a place behind the last.
static long long select_pitch(const FcsPagedCache* c) { return (c->table_width + 4ll) & ~3ll; }
// Many tokens a sequence: the scores of 64 tokens and 64 pages are worth a tile of their own from about eight on.  And rows that
// shared memory does not hold.
static bool select_by_tiles(const FcsPagedCache* c) {
    return (c->starts && c->tokens >= 8ll * c->sequences) || select_pitch(c) > ROW_PAGES;
}

struct SelectPlan {
    bool tiles;
    long long pitch, at_once;      // tokens of a launch: 256 MiB of scratch, and as many as a grid takes
    int splits;
    size_t errors, scores, exact, bytes;     // offsets into the workspace
};

static SelectPlan select_plan(const FcsPagedCache* c) {
    SelectPlan s;
    s.tiles = select_by_tiles(c);
    s.pitch = select_pitch(c);
    const long long row = (s.tiles ? 12 : 8) * (long long)c->kv_heads * s.pitch;
    s.at_once = (256ll << 20) / row;
    s.at_once = s.at_once < 1 ? 1 : s.at_once > c->tokens ? c->tokens : s.at_once;
    s.splits = 1;
    if (s.tiles) {
        const long long ctas = (s.at_once / TILE_TOKENS + 1) * c->kv_heads, most = (c->table_width + 2 * TILE_PAGES - 1) / (2 * TILE_PAGES);
        while (s.splits < most && s.splits < 64 && ctas * s.splits < num_sms()) s.splits *= 2;
    }
    const long long rows = s.at_once * c->kv_heads;
    s.exact = 0;
    s.scores = s.exact + (size_t)rows * s.pitch * 8;
    s.errors = s.scores + (s.tiles ? (size_t)rows * s.pitch * 4 : 0);
    s.bytes = s.errors + (s.tiles ? (size_t)rows * s.splits * 4 : 0);
    return s;
}

template <bool BF16>
static int widest_row_cluster() {
    static int known[64] = {0};
    return sixteen_fit(known, select_row_kernel<BF16, 128, 16>, ROW_THREADS, row_smem(128, ROW_PAGES)) ? 16 : 8;
}

// CTAs of a row (select_row_kernel): as many as the device runs at once, 64 pages for each at least.
static int row_ctas(long long rows, int width, int widest) {
    int cl = 1;
    while (cl < widest && rows * cl * 2 <= (long long)ROW_CTAS * num_sms() && width >= 128 * cl) cl *= 2;
    return cl;
}

template <bool BF16, int DP, int CL>
static cudaError_t launch_select_row(const SelectParams& p, unsigned tokens, cudaStream_t stream) {
    static bool done[64] = {false};
    const cudaError_t e = once_per_device(done, [] { return allow_smem(select_row_kernel<BF16, DP, CL>, row_smem(DP, ROW_PAGES), CL > 8); });
    if (e != cudaSuccess) return e;
    return launch(select_row_kernel<BF16, DP, CL>, dim3(CL * tokens, p.c.kv_heads), ROW_THREADS, row_smem(p.c.dim, p.pitch), CL, stream, p);
}

template <bool BF16, int DP>
static cudaError_t launch_select_cl(int cl, const SelectParams& p, unsigned tokens, cudaStream_t stream) {
    return cl == 16  ? launch_select_row<BF16, DP, 16>(p, tokens, stream)
           : cl == 8 ? launch_select_row<BF16, DP, 8>(p, tokens, stream)
           : cl == 4 ? launch_select_row<BF16, DP, 4>(p, tokens, stream)
           : cl == 2 ? launch_select_row<BF16, DP, 2>(p, tokens, stream)
                     : launch_select_row<BF16, DP, 1>(p, tokens, stream);
}

template <bool BF16>
static cudaError_t launch_select(const SelectParams& p, bool tiles, cudaStream_t stream) {
    const unsigned tokens = (unsigned)(p.t1 - p.t0);
    if (!tiles) {
        const int cl = row_ctas((long long)tokens * p.c.kv_heads, p.c.width, widest_row_cluster<BF16>());
        return p.c.dim > 64 ? launch_select_cl<BF16, 128>(cl, p, tokens, stream) : launch_select_cl<BF16, 64>(cl, p, tokens, stream);
    }
    static bool done[64] = {false};
    cudaError_t e = once_per_device(done, [] { return allow_smem(score_tiles_kernel<BF16>, tiles_smem(128)); });
    if (e != cudaSuccess) return e;
    const int first = p.t0 / TILE_TOKENS - 1 > 0 ? p.t0 / TILE_TOKENS - 1 : 0;
    const dim3 grid(p.c.starts ? (unsigned)((p.t1 - 1) / TILE_TOKENS - first + 1 + p.c.sequences) : tokens, p.c.kv_heads, p.splits);
    e = launch(score_tiles_kernel<BF16>, grid, TILES_THREADS, tiles_smem(p.c.dim), 1, stream, p);
    if (e != cudaSuccess) return e;
    const long long rows = (long long)tokens * p.c.kv_heads;
    const unsigned by_warp = (unsigned)((rows + CHOOSE_THREADS / 32 - 1) / (CHOOSE_THREADS / 32));
    return p.c.width <= 512    ? launch(choose_kernel<BF16, 16>, dim3(by_warp), CHOOSE_THREADS, 0, 1, stream, p)
           : p.c.width <= 1024 ? launch(choose_kernel<BF16, 32>, dim3(by_warp), CHOOSE_THREADS, 0, 1, stream, p)
                               : launch(choose_kernel<BF16, 0>, dim3((unsigned)rows), CHOOSE_THREADS, 0, 1, stream, p);
}

static int select(const FcsPagedCache* cache, const void* query, const int64_t* query_stride, int q_heads, const void* bounds,
                  int k, int first, int last, int* chosen, int fill_tail, void* workspace, size_t workspace_bytes, int* status,
                  cudaStream_t stream, bool withhold = false) {
    SelectParams p;
    memset(&p, 0, sizeof(p));
    int rc = check_cache(cache, p.c, status);
    if (rc != FCS_OK) return rc;
    if (!query_stride) return fail(FCS_ERR_INVALID_ARGUMENT, "query strides are NULL");
    if ((rc = check_rows("query", query, query_stride, 2)) != FCS_OK) return rc;
    if ((rc = check_group(cache, q_heads)) != FCS_OK) return rc;
    if (!bounds || !aligned16(bounds)) return fail(FCS_ERR_INVALID_ARGUMENT, "bounds must be a 16-byte aligned device pointer");
    if (!chosen) return fail(FCS_ERR_INVALID_ARGUMENT, "chosen is NULL");
    if (k < 1 || first < 0 || last < 1 || (long long)first + last > k)
        return fail(FCS_ERR_INVALID_ARGUMENT, "k must hold the first and the last pages (k=%d first=%d last=%d)", k, first, last);
    const SelectPlan plan = select_plan(cache);
    if (withhold && plan.tiles) return fail(FCS_ERR_UNSUPPORTED, "this call has no waits");
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < plan.bytes)
        return fail(FCS_ERR_WORKSPACE, "workspace must be 16-byte aligned and hold %zu bytes, got %zu", plan.bytes, workspace_bytes);
    p.query = static_cast<const uint16_t*>(query);
    p.bounds = static_cast<const uint16_t*>(bounds);
    p.query_st[0] = query_stride[0];
    p.query_st[1] = query_stride[1];
    p.group = q_heads / cache->kv_heads;
    p.k = k;
    p.first = first;
    p.last = last;
    p.chosen = chosen;
    p.exact = reinterpret_cast<double*>(static_cast<char*>(workspace) + plan.exact);
    p.scores = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.scores);
    p.errors = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.errors);
    p.pitch = (int)plan.pitch;
    p.splits = plan.splits;
    p.fill_tail = fill_tail;
    p.withhold = withhold;
    for (long long t0 = 0; t0 < cache->tokens; t0 += plan.at_once) {
        p.t0 = (int)t0;
        p.t1 = (int)(cache->tokens - t0 < plan.at_once ? cache->tokens : t0 + plan.at_once);
        const cudaError_t e = cache->dtype == FCS_DTYPE_BF16 ? launch_select<true>(p, plan.tiles, stream)
                                                             : launch_select<false>(p, plan.tiles, stream);
        if (e != cudaSuccess) return fail(FCS_ERR_CUDA, "choosing pages failed to launch: %s", cudaGetErrorString(e));
    }
    return FCS_OK;
}

// ------------------------------------------------------------------ attend
template <int DP, int NT, bool BF16, int CL>
static cudaError_t launch_attend(const CUtensorMap& km, const CUtensorMap& vm, const AttendParams& p, cudaStream_t stream) {
    constexpr int STAGES = DP == 128 ? 3 : 4;
    using L = AttendLayout<DP, STAGES>;
    auto* kern = attend_kernel<DP, NT, STAGES, BF16, CL>;
    if constexpr (CL == 16) {
        static int known[64] = {0};
        if (!sixteen_fit(known, kern, ATTEND_THREADS, L::BYTES)) return launch_attend<DP, NT, BF16, 8>(km, vm, p, stream);
    } else {
        static bool done[64] = {false};
        const cudaError_t e = once_per_device(done, [&] { return allow_smem(kern, L::BYTES); });
        if (e != cudaSuccess) return e;
    }
    const dim3 grid((unsigned)((long long)CL * p.query_tiles * p.c.tokens), p.c.kv_heads);
    return launch(kern, grid, ATTEND_THREADS, L::BYTES, CL, stream, km, vm, p);
}

template <int DP, int NT, bool BF16>
static cudaError_t launch_attend_cl(int cl, const CUtensorMap& km, const CUtensorMap& vm, const AttendParams& p, cudaStream_t s) {
    return cl == 16  ? launch_attend<DP, NT, BF16, 16>(km, vm, p, s)
           : cl == 8 ? launch_attend<DP, NT, BF16, 8>(km, vm, p, s)
           : cl == 4 ? launch_attend<DP, NT, BF16, 4>(km, vm, p, s)
           : cl == 2 ? launch_attend<DP, NT, BF16, 2>(km, vm, p, s)
                     : launch_attend<DP, NT, BF16, 1>(km, vm, p, s);
}

template <int DP, bool BF16, int CL>
static cudaError_t launch_shared(const CUtensorMap& km, const CUtensorMap& vm, const AttendParams& p, cudaStream_t stream) {
    constexpr int STAGES = DP == 128 ? 2 : 3;
    using L = SharedLayout<DP, STAGES>;
    auto* kern = attend_shared_kernel<DP, STAGES, BF16, CL>;
    static bool done[64] = {false};
    const cudaError_t e = once_per_device(done, [&] { return allow_smem(kern, L::bytes(SHARED_PAGES)); });
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)(CL * ((long long)p.c.tokens / p.tile_tokens + p.c.sequences + 1)), p.c.kv_heads);
    return launch(kern, grid, SHARED_THREADS, L::bytes(p.c.width), CL, stream, km, vm, p);
}

template <int DP, bool BF16>
static cudaError_t launch_shared_cl(int cl, const CUtensorMap& km, const CUtensorMap& vm, const AttendParams& p, cudaStream_t s) {
    return cl == 8   ? launch_shared<DP, BF16, 8>(km, vm, p, s)
           : cl == 4 ? launch_shared<DP, BF16, 4>(km, vm, p, s)
           : cl == 2 ? launch_shared<DP, BF16, 2>(km, vm, p, s)
                     : launch_shared<DP, BF16, 1>(km, vm, p, s);
}

static int pool_map(CUtensorMap* m, const FcsPagedCache* c, const void* base, const int64_t* stride) {
    // (the stride of an axis of one entry says nothing; the contiguous one stands in for it)
    int64_t st[3] = {stride[0], stride[1], stride[2]};
    const int64_t size[3] = {c->pages, c->kv_heads, c->page_size};
    int64_t dense = c->dim;
    for (int i = 2; i >= 0; --i) {
        if (size[i] == 1) st[i] = dense;
        if (st[i] <= 0) return fail(FCS_ERR_INVALID_ARGUMENT, "strides of the pools must be positive");
        dense = st[i] * size[i] > dense ? st[i] * size[i] : dense;
    }
    return make_tensor_map(m, base, c->dtype, c->pages, c->kv_heads, c->page_size, c->dim, st[0], st[1], st[2],
                           c->page_size < TILE_KEYS ? c->page_size : TILE_KEYS);
}

// CTAs that share a row's keys, up to `most`: the device runs `per_sm` CTAs per SM, rounds of them one after the other, and a CTA
// costs about a third of a whole row's work beside its share.
static int cluster_for(long long rows, int per_sm, int most) {
    const long long slots = (long long)per_sm * num_sms();
    int best = 1;
    double least = 1e30;
    for (int cl = 1; cl <= most; cl *= 2) {
        const double cost = (double)((rows * cl + slots - 1) / slots) * (1.0 / cl + 0.3);
        if (cost < least) least = cost, best = cl;
    }
    return best;
}

struct AttendPlan {
    bool shared;             // tokens share their pages (attend_shared_kernel)
    int tile_tokens;         // tokens of a block, then
    int nt, query_tiles;     // a row at a time: sets of eight queries in a CTA, and CTAs over a row's queries
    int cl;                  // CTAs of a block or row
};

// Tokens of a sequence share what they chose in common, where there are enough of them: more than two a sequence, and blocks
// for all SMs or of eight tokens.  Measured, blocks against a token at a time, 32 pages of 64 for groups of four heads: 512
// blocks of two tokens 127 and 121 us; 256 of four 96 and 105, 192 of four 50 and 62; 128 of four 48 and 42 (58 and 52), 64
// of four 34 and 22; heads of their own, 64 of sixteen 53 and 60, 32 of sixteen 29 and 39.  512 tokens of eight key/value heads in
// groups of one 118 and 271, two 151 and 275, four 191 and 283, five (three tokens a block) 221 and 285, eight (two) 245 and 296;
// of four in groups of eight 142 and 148.
static AttendPlan attend_plan(const FcsPagedCache* cache, int group, int k) {
    AttendPlan a;
    const long long T = cache->tokens, B = cache->sequences;
    a.tile_tokens = SHARED_COLS / group;
    const long long blocks = (a.tile_tokens > 0 && T / a.tile_tokens > B ? T / a.tile_tokens : B) * cache->kv_heads;
    const long long together = T / B < a.tile_tokens ? T / B : a.tile_tokens;
    a.shared = cache->starts && T > 2 * B && a.tile_tokens >= 2 && cache->table_width <= SHARED_PAGES &&
               (blocks >= num_sms() || together >= 8);
    a.nt = group > 8 ? 2 : 1;
    a.query_tiles = (group + 8 * a.nt - 1) / (8 * a.nt);
    const long long tiles = ((long long)k * cache->page_size + TILE_KEYS - 1) / TILE_KEYS;
    a.cl = a.shared ? cluster_for(blocks, cache->dim > 64 ? SHARED_CTAS<128> : SHARED_CTAS<64>, 8)
                    : cluster_for(T * cache->kv_heads * a.query_tiles, 2,      // (two tiles of keys for each CTA at least)
                                  tiles >= 32 ? 16 : tiles >= 16 ? 8 : tiles >= 8 ? 4 : tiles >= 4 ? 2 : 1);
    return a;
}

static int attend(const FcsPagedCache* cache, const void* query, const int64_t* query_stride, int q_heads, const int* chosen, int k,
                  float scale, void* out, const int64_t* out_stride, float* lse, int fill_tail, int* status, cudaStream_t stream,
                  bool withhold = false) {
    AttendParams p;
    memset(&p, 0, sizeof(p));
    int rc = check_cache(cache, p.c, status);
    if (rc != FCS_OK) return rc;
    if (!query_stride || !out_stride) return fail(FCS_ERR_INVALID_ARGUMENT, "query or out strides are NULL");
    if ((rc = check_rows("query", query, query_stride, 2)) != FCS_OK) return rc;
    if ((rc = check_rows("out", out, out_stride, 2)) != FCS_OK) return rc;
    if ((rc = check_rows("key_pages", cache->key_pages, cache->key_stride, 3)) != FCS_OK) return rc;
    if ((rc = check_rows("value_pages", cache->value_pages, cache->value_stride, 3)) != FCS_OK) return rc;
    if ((rc = check_group(cache, q_heads)) != FCS_OK) return rc;
    if ((rc = check_result("out", cache, q_heads, out_stride)) != FCS_OK) return rc;
    if (!chosen || k < 1) return fail(FCS_ERR_INVALID_ARGUMENT, "chosen is NULL or has no entries (k=%d)", k);
    // (the kernels count the entries of a block of up to sixteen tokens, and some steps past them, in an int)
    static_assert((long long)SHARED_COLS * FCS_LIST_MAX <= 1 << 30, "the entries of a block");
    if (k > FCS_LIST_MAX) return fail(FCS_ERR_UNSUPPORTED, "a list holds at most %d pages, got %d", FCS_LIST_MAX, k);
    if (scale != scale) return fail(FCS_ERR_INVALID_ARGUMENT, "scale is not a number");
    p.query = static_cast<const uint16_t*>(query);
    p.out = static_cast<uint16_t*>(out);
    for (int i = 0; i < 2; ++i) {
        p.query_st[i] = query_stride[i];
        p.out_st[i] = out_stride[i];
    }
    p.lse = lse;
    p.chosen = chosen;
    p.k = k;
    p.group = q_heads / cache->kv_heads;
    p.q_heads = q_heads;
    p.c_log2 = scale * 1.4426950408889634f;
    p.fill_tail = fill_tail;
    p.withhold = withhold;
    const bool wide = cache->dim > 64, bf16 = cache->dtype == FCS_DTYPE_BF16;
    CUtensorMap km, vm;
    if ((rc = pool_map(&km, cache, cache->key_pages, cache->key_stride)) != FCS_OK) return rc;
    if ((rc = pool_map(&vm, cache, cache->value_pages, cache->value_stride)) != FCS_OK) return rc;
    cudaError_t e;
    const long long T = cache->tokens, B = cache->sequences;
    const AttendPlan plan = attend_plan(cache, p.group, k);
    const int cl = plan.cl;
    if (plan.shared) {
        p.tile_tokens = plan.tile_tokens;
        if (8 * (T / p.tile_tokens + B + 1) > 0x7fffffffll) return fail(FCS_ERR_UNSUPPORTED, "too many tokens (%d) for one launch", cache->tokens);
        e = wide ? (bf16 ? launch_shared_cl<128, true>(cl, km, vm, p, stream) : launch_shared_cl<128, false>(cl, km, vm, p, stream))
                 : (bf16 ? launch_shared_cl<64, true>(cl, km, vm, p, stream) : launch_shared_cl<64, false>(cl, km, vm, p, stream));
        if (e != cudaSuccess) return fail(FCS_ERR_CUDA, "attending failed to launch: %s", cudaGetErrorString(e));
        return FCS_OK;
    }
    const int nt = plan.nt;
    p.query_tiles = plan.query_tiles;
    if (T * p.query_tiles * cl > 0x7fffffffll) return fail(FCS_ERR_UNSUPPORTED, "too many tokens (%d) for one launch", cache->tokens);
    if (wide)
        e = nt == 1 ? (bf16 ? launch_attend_cl<128, 1, true>(cl, km, vm, p, stream) : launch_attend_cl<128, 1, false>(cl, km, vm, p, stream))
                    : (bf16 ? launch_attend_cl<128, 2, true>(cl, km, vm, p, stream) : launch_attend_cl<128, 2, false>(cl, km, vm, p, stream));
    else
        e = nt == 1 ? (bf16 ? launch_attend_cl<64, 1, true>(cl, km, vm, p, stream) : launch_attend_cl<64, 1, false>(cl, km, vm, p, stream))
                    : (bf16 ? launch_attend_cl<64, 2, true>(cl, km, vm, p, stream) : launch_attend_cl<64, 2, false>(cl, km, vm, p, stream));
    if (e != cudaSuccess) return fail(FCS_ERR_CUDA, "attending failed to launch: %s", cudaGetErrorString(e));
    return FCS_OK;
}

// ------------------------------------------------------------------ waits that run out
// `call` under a lower limit of the waits, for the self-tests.
template <typename F>
static int under_limit(double seconds, const int* status, cudaStream_t stream, F call) {
    if (!status) return fail(FCS_ERR_INVALID_ARGUMENT, "status must not be NULL");
    if (!(seconds > 0.0) || seconds > 2.0) return fail(FCS_ERR_INVALID_ARGUMENT, "limit_seconds must be in (0, 2]");
    static long long short_limit, full_limit = kWaitLimitCycles;
    short_limit = (long long)(seconds * 1.9e9);
    cudaError_t e = cudaMemcpyToSymbolAsync(g_wait_limit_cycles, &short_limit, sizeof(long long), 0, cudaMemcpyHostToDevice, stream);
    if (e != cudaSuccess) return fail(FCS_ERR_CUDA, "the limit of the waits could not be set: %s", cudaGetErrorString(e));
    const int rc = call();
    e = cudaMemcpyToSymbolAsync(g_wait_limit_cycles, &full_limit, sizeof(long long), 0, cudaMemcpyHostToDevice, stream);
    if (rc == FCS_OK && e != cudaSuccess) return fail(FCS_ERR_CUDA, "the limit of the waits could not be set back: %s", cudaGetErrorString(e));
    return rc;
}

}  // namespace paged
}  // namespace fcs

extern "C" {

int fcs_append_paged(const FcsPagedCache* cache, const FcsPagedRows* rows, int* status, void* stream) {
    fcs::g_err[0] = 0;
    return fcs::paged::append(cache, rows, status, reinterpret_cast<cudaStream_t>(stream));
}

size_t fcs_select_pages_workspace_bytes(const FcsPagedCache* cache) {
    if (!cache || cache->tokens <= 0 || cache->kv_heads <= 0 || cache->table_width <= 0) return 0;
    return fcs::paged::select_plan(cache).bytes;
}

int fcs_select_pages(const FcsPagedCache* cache, const void* query, const int64_t* query_stride, int q_heads, const void* bounds,
                     int k, int first, int last, int* chosen, int fill_tail, void* workspace, size_t workspace_bytes, int* status,
                     void* stream) {
    fcs::g_err[0] = 0;
    return fcs::paged::select(cache, query, query_stride, q_heads, bounds, k, first, last, chosen, fill_tail, workspace,
                              workspace_bytes, status, reinterpret_cast<cudaStream_t>(stream));
}

int fcs_attend_pages(const FcsPagedCache* cache, const void* query, const int64_t* query_stride, int q_heads, const int* chosen, int k,
                     float scale, void* out, const int64_t* out_stride, float* lse, int fill_tail, int* status, void* stream) {
    fcs::g_err[0] = 0;
    return fcs::paged::attend(cache, query, query_stride, q_heads, chosen, k, scale, out, out_stride, lse, fill_tail, status,
                              reinterpret_cast<cudaStream_t>(stream));
}

int fcs_paged_plan(const FcsPagedCache* cache, int q_heads, int k, FcsPagedPlan* plan) {
    fcs::g_err[0] = 0;
    using namespace fcs::paged;
    Batch unused;
    const int rc = check_cache(cache, unused, nullptr);
    if (rc != FCS_OK) return rc;
    if (!plan || q_heads < 0 || q_heads % cache->kv_heads || k < 1)
        return fcs::fail(FCS_ERR_INVALID_ARGUMENT, "plan is NULL, or bad sizes (q_heads=%d k=%d)", q_heads, k);
    memset(plan, 0, sizeof(*plan));
    const AppendPlan a = append_plan(cache, q_heads);
    plan->append_heads = 1 << a.heads_shift;
    plan->append_steps = a.steps;
    const SelectPlan s = select_plan(cache);
    const long long at_once = s.at_once;
    plan->select_tiles = s.tiles;
    plan->select_launches = (int)((cache->tokens + at_once - 1) / at_once);
    plan->select_ctas = s.tiles ? 1
                                : row_ctas(at_once * cache->kv_heads, cache->table_width,
                                           cache->dtype == FCS_DTYPE_BF16 ? widest_row_cluster<true>() : widest_row_cluster<false>());
    if (q_heads == 0) return FCS_OK;
    const AttendPlan t = attend_plan(cache, q_heads / cache->kv_heads, k);
    plan->attend_tokens = t.shared ? t.tile_tokens : 1;
    plan->attend_queries = t.shared ? SHARED_COLS : 8 * t.nt;
    plan->attend_ctas = t.cl;
    return FCS_OK;
}

int fcs_selftest_wait_expiry_select(const FcsPagedCache* cache, const void* query, const int64_t* query_stride, int q_heads,
                                    const void* bounds, int k, int first, int last, int* chosen, void* workspace,
                                    size_t workspace_bytes, int* status, double limit_seconds, void* stream_v) {
    fcs::g_err[0] = 0;
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
    return fcs::paged::under_limit(limit_seconds, status, stream, [&] {
        return fcs::paged::select(cache, query, query_stride, q_heads, bounds, k, first, last, chosen, 0, workspace, workspace_bytes,
                                  status, stream, true);
    });
}

int fcs_selftest_wait_expiry_attend(const FcsPagedCache* cache, const void* query, const int64_t* query_stride, int q_heads,
                                    const int* chosen, int k, float scale, void* out, const int64_t* out_stride, float* lse,
                                    int* status, double limit_seconds, void* stream_v) {
    fcs::g_err[0] = 0;
    cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_v);
    return fcs::paged::under_limit(limit_seconds, status, stream, [&] {
        return fcs::paged::attend(cache, query, query_stride, q_heads, chosen, k, scale, out, out_stride, lse, 0, status, stream, true);
    });
}

}  // extern "C"
