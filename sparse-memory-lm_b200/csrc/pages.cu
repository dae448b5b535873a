// The pages of a paged key-value cache, managed on the device: extending sequences, forking them (whole pages
// shared, the partly filled last page copied), freeing, trimming to a window, and compacting the pool.
//
// The allocator's whole state is one reference count per page (0 = free), and a page is always taken from the lowest
// numbers that are free, so tables and counts after any sequence of calls are reproducible and nothing has to be
// kept beside them. Every count changes by integer atomics, whose order does not matter.
#include "paged.cuh"

namespace smlm {

constexpr int PLAN_THREADS = 1024;

struct Pages {
    int32_t* table;
    int32_t* lengths;
    int32_t* refcount;
    int64_t table_stride;
    int table_rows, max_blocks, n_pages;
    int* status;
};

__device__ __forceinline__ void release(const Pages& pg, int page) {
    if (page >= pg.n_pages || atomicSub(pg.refcount + page, 1) <= 0) {
        flag(pg.status, SMLM_FLAG_INDEX_RANGE);
        if (page < pg.n_pages) atomicAdd(pg.refcount + page, 1);
    }
}

__device__ __forceinline__ bool row_ok(const Pages& pg, int r) {
    if (r >= 0 && r < pg.table_rows) return true;
    flag(pg.status, SMLM_FLAG_INDEX_RANGE);
    return false;
}

// Takes the entry out of the table (an exchange, so that a row listed twice is released once) and drops the page.
__device__ __forceinline__ void drop_entry(const Pages& pg, int32_t* entry) {
    if (*entry < 0) return;
    const int old = atomicExch(entry, -1);
    if (old >= 0) release(pg, old);
}

__global__ void __launch_bounds__(256) pages_free_kernel(Pages pg, const int32_t* rows) {
    const int r = rows[blockIdx.x];
    if (!row_ok(pg, r)) return;
    for (int j = threadIdx.x; j < pg.max_blocks; j += blockDim.x) drop_entry(pg, pg.table + r * pg.table_stride + j);
    if (threadIdx.x == 0) pg.lengths[r] = 0;
}

// Releases the pages that hold only tokens in [sinks, length - window).
__global__ void __launch_bounds__(256) pages_trim_kernel(Pages pg, const int32_t* rows, int shift, int window,
                                                         int sinks) {
    const int r = rows[blockIdx.x];
    if (!row_ok(pg, r)) return;
    const int64_t first = (((int64_t)sinks + (1 << shift) - 1) >> shift);
    const int64_t last = max((int64_t)pg.lengths[r] - window, (int64_t)0) >> shift;
    for (int64_t j = first + threadIdx.x; j < min(last, (int64_t)pg.max_blocks); j += blockDim.x)
        drop_entry(pg, pg.table + r * pg.table_stride + j);
}

// ------------------------------------------------------------------------------------------------- planning
// Exclusive sum over the block, in thread order; *total receives the sum of all.
__device__ __forceinline__ int block_scan(int v, int* total) {
    __shared__ int part[PLAN_THREADS / 32];
    const int lane = lane_id(), warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(FULL, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) part[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int p = part[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(FULL, p, o);
            if (lane >= o) p += y;
        }
        part[lane] = p;
    }
    __syncthreads();
    *total = part[PLAN_THREADS / 32 - 1];
    return x - v + (warp ? part[warp - 1] : 0);
}

// The free pages in increasing order: list[k] = the k-th free page, for k < most. Returns how many there are. Each
// thread counts a contiguous piece, one scan gives its first rank.
__device__ int list_free(const Pages& pg, int32_t* list, int most) {
    const int per = (pg.n_pages + PLAN_THREADS - 1) / PLAN_THREADS;
    const int a = min(pg.n_pages, (int)threadIdx.x * per), e = min(pg.n_pages, a + per);
    int count = 0, total;
    for (int p = a; p < e; p++) count += __ldcg(pg.refcount + p) == 0;
    int k = block_scan(count, &total);
    for (int p = a; p < e && k < most; p++)
        if (__ldcg(pg.refcount + p) == 0) list[k++] = p;
    __syncthreads();
    return total;
}

// offset[i] = sum of need(0 .. i-1); returns the sum of all. need(i) is called once for each i < n.
template <typename F>
__device__ int scan_needs(int n, int32_t* offset, F need) {
    int sum = 0;
    for (int base = 0; base < n; base += PLAN_THREADS) {
        const int i = base + threadIdx.x;
        int total;
        const int off = block_scan(i < n ? need(i) : 0, &total);
        if (i < n) offset[i] = sum + off;
        sum += total;
        __syncthreads();
    }
    return sum;
}

// lengths[r] += n_new for every listed row, with the pages that takes: rows in order, lowest free pages first. A row
// whose pages are not there, or whose table is too narrow, stays as it is and raises a flag. The lengths are taken by
// an exchange and put back at the end, which finds rows listed twice (the second does nothing).
__global__ void __launch_bounds__(PLAN_THREADS) pages_extend_kernel(Pages pg, const int32_t* rows, int n, int n_new,
                                                                    int shift, int32_t* offset, int32_t* len_of,
                                                                    int32_t* list) {
    constexpr int TAKEN = INT32_MIN;
    const int64_t cap = (int64_t)pg.max_blocks << shift;
    auto blocks = [&](int64_t len) { return (int)((len + (1 << shift) - 1) >> shift); };
    auto fits = [&](int len) { return len >= 0 && (int64_t)len + n_new <= cap; };
    const int wanted = scan_needs(n, offset, [&](int i) {
        const int r = rows[i];
        const int len = r >= 0 && r < pg.table_rows ? atomicExch(pg.lengths + r, TAKEN) : TAKEN;
        len_of[i] = len;
        if (len == TAKEN || !fits(len)) flag(pg.status, SMLM_FLAG_INDEX_RANGE);
        return len != TAKEN && fits(len) ? blocks((int64_t)len + n_new) - blocks(len) : 0;
    });
    const int have = wanted ? list_free(pg, list, wanted) : 0;
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
        const int len = len_of[i];
        if (len == TAKEN) continue;
        bool grow = fits(len);
        const int b0 = blocks(len), need = grow ? blocks((int64_t)len + n_new) - b0 : 0;
        if (need && offset[i] + need > have) {
            flag(pg.status, SMLM_FLAG_NO_PAGES);
            grow = false;
        }
        if (grow)
            for (int m = 0; m < need; m++) {
                const int page = list[offset[i] + m];
                pg.table[rows[i] * pg.table_stride + b0 + m] = page;
                pg.refcount[page] = 1;
            }
        pg.lengths[rows[i]] = grow ? len + n_new : len;
    }
}

struct CopyList {
    int32_t *src, *dst, *tokens;  // page numbers, tokens to copy
    int32_t* count;               // entries (device), or NULL: n
    int n;
};

// Row children[i] becomes a copy of row parents[i] as it was before the call, for all i at once.
__global__ void __launch_bounds__(PLAN_THREADS)
    pages_fork_kernel(Pages pg, const int32_t* parents, const int32_t* children, int n, int shift, int32_t* claim,
                      int32_t* snap, int32_t* snap_len, int32_t* offset, int32_t* list, CopyList cl) {
    const int mb = pg.max_blocks;
    // a child listed twice takes its first parent; out-of-range rows are left out
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
        const int c = children[i];
        if (c >= 0 && c < pg.table_rows) claim[c] = INT32_MAX;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS)
        if (row_ok(pg, children[i]) && row_ok(pg, parents[i])) atomicMin(claim + children[i], i);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
        const int c = children[i], p = parents[i];
        const bool in = c >= 0 && c < pg.table_rows && p >= 0 && p < pg.table_rows;
        const bool mine = in && claim[c] == i;
        if (in && !mine) flag(pg.status, SMLM_FLAG_INDEX_RANGE);
        snap_len[i] = mine && c != p ? min(max(pg.lengths[p], 0), mb << shift) : -1;
    }
    __syncthreads();
    // the parents' entries, one more reference for each whole page; the partly filled ones are held meanwhile
    for (int64_t x = threadIdx.x; x < (int64_t)n * mb; x += PLAN_THREADS) {
        const int i = x / mb, j = x % mb;
        if (snap_len[i] < 0 || ((int64_t)j << shift) >= snap_len[i]) continue;
        int e = pg.table[parents[i] * pg.table_stride + j];
        if (e >= pg.n_pages) {
            flag(pg.status, SMLM_FLAG_INDEX_RANGE);
            e = -1;
        }
        snap[x] = e;
        if (e >= 0) atomicAdd(pg.refcount + e, 1);
    }
    __syncthreads();
    for (int64_t x = threadIdx.x; x < (int64_t)n * mb; x += PLAN_THREADS)
        if (snap_len[x / mb] >= 0) drop_entry(pg, pg.table + children[x / mb] * pg.table_stride + x % mb);
    __syncthreads();
    auto part = [&](int i) {  // tokens in the partly filled last page
        const int len = snap_len[i];
        if (len < 0) return 0;
        const int t = len & ((1 << shift) - 1);
        return t && snap[(int64_t)i * mb + (len >> shift)] >= 0 ? t : 0;
    };
    const int wanted = scan_needs(n, offset, [&](int i) { return part(i) ? 1 : 0; });
    const int have = wanted ? list_free(pg, list, wanted) : 0;
    for (int i = threadIdx.x; i < n; i += PLAN_THREADS) {
        int tokens = part(i);
        if (tokens) {
            const int64_t at = (int64_t)i * mb + (snap_len[i] >> shift);
            const int src = snap[at];
            atomicSub(pg.refcount + src, 1);
            cl.src[i] = src;
            if (offset[i] < have) {
                const int dst = list[offset[i]];
                cl.dst[i] = snap[at] = dst;
                pg.refcount[dst] = 1;
            } else {
                flag(pg.status, SMLM_FLAG_NO_PAGES);
                snap[at] = -1;
                tokens = 0;
            }
        }
        cl.tokens[i] = tokens;
        if (snap_len[i] >= 0) pg.lengths[children[i]] = snap_len[i];
    }
    __syncthreads();
    for (int64_t x = threadIdx.x; x < (int64_t)n * mb; x += PLAN_THREADS) {
        const int i = x / mb, j = x % mb;
        if (snap_len[i] >= 0 && ((int64_t)j << shift) < snap_len[i])
            pg.table[children[i] * pg.table_stride + j] = snap[x];
    }
}

// With L pages in use: the k-th used page numbered L or above moves to the k-th free page below L. to[p] (p >= L) is
// where page p went.
__global__ void __launch_bounds__(PLAN_THREADS) pages_compact_kernel(Pages pg, int32_t* to, int32_t* live_out,
                                                                     CopyList cl) {
    const int per = (pg.n_pages + PLAN_THREADS - 1) / PLAN_THREADS;
    const int a = min(pg.n_pages, (int)threadIdx.x * per), e = min(pg.n_pages, a + per);
    int count = 0, live;
    for (int p = a; p < e; p++) count += pg.refcount[p] > 0;
    const int before = block_scan(count, &live);
    __shared__ int used_below;  // used pages below L
    if (a <= live && live < e) {
        int k = before;
        for (int p = a; p < live; p++) k += pg.refcount[p] > 0;
        used_below = k;
    }
    if (threadIdx.x == 0 && live == pg.n_pages) used_below = live;
    __syncthreads();
    const int below = used_below, moves = live - below;
    int used = before;
    for (int p = a; p < e; p++) {
        const bool u = pg.refcount[p] > 0;
        if (p < live) {
            if (!u) cl.dst[p - used] = p;
        } else {
            if (u) cl.src[used - below] = p;
            else to[p] = p;
        }
        used += u;
    }
    if (threadIdx.x == 0) {
        *cl.count = moves;
        *live_out = live;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < moves; k += PLAN_THREADS) {
        const int s = cl.src[k], d = cl.dst[k];
        pg.refcount[d] = pg.refcount[s];
        pg.refcount[s] = 0;
        to[s] = d;
    }
}

// --------------------------------------------------------------------------------------------------- moving
// The listed pages' tokens in every (layer, k / v) plane: one warp per (entry, plane, head), 16 bytes a lane. With
// `to`, the table's entries follow their pages.
__global__ void __launch_bounds__(256) pages_copy_kernel(char* pool, CopyList cl, int planes, int heads, int n_pages,
                                                         int page_size, int token_bytes, Pages pg, const int32_t* to,
                                                         const int32_t* live) {
    const int64_t thread = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (to) {
        const int first = *live;
        const int64_t entries = (int64_t)pg.table_rows * pg.max_blocks;
        for (int64_t x = thread; x < entries; x += (int64_t)gridDim.x * blockDim.x) {
            int32_t* entry = pg.table + x / pg.max_blocks * pg.table_stride + x % pg.max_blocks;
            const int p = *entry;
            if (p >= pg.n_pages) flag(pg.status, SMLM_FLAG_INDEX_RANGE);
            else if (p >= first) *entry = to[p];
        }
    }
    const int lane = lane_id();
    const int64_t page_bytes = (int64_t)page_size * token_bytes;
    const int64_t units = (int64_t)(cl.count ? *cl.count : cl.n) * planes * heads;
    for (int64_t u = thread >> 5; u < units; u += (int64_t)gridDim.x * blockDim.x >> 5) {
        const int i = u / (planes * heads), ph = u % (planes * heads);
        const int tokens = cl.tokens ? cl.tokens[i] : page_size;
        if (tokens == 0) continue;
        const int64_t plane = ph / heads, h = ph % heads;
        const char* s = pool + ((plane * n_pages + cl.src[i]) * heads + h) * page_bytes;
        char* d = pool + ((plane * n_pages + cl.dst[i]) * heads + h) * page_bytes;
        const int bytes = tokens * token_bytes;
        for (int x = lane * 16; x < bytes; x += 512)
            *reinterpret_cast<int4*>(d + x) = *reinterpret_cast<const int4*>(s + x);
    }
}

static int check_pages(Pages& pg, const char* what, int32_t* table, int64_t table_stride, int64_t table_rows,
                       int64_t max_blocks, int32_t* lengths, int32_t* refcount, int64_t n_pages, int64_t page_size,
                       int* status) {
    SMLM_CHECK_ARG(table && refcount, "%s: null table or reference counts", what);
    SMLM_CHECK_ARG(table_rows >= 1 && table_rows <= INT32_MAX && max_blocks >= 1 && table_stride >= max_blocks,
                   "%s: table of %lld rows, %lld columns (stride %lld)", what, (long long)table_rows,
                   (long long)max_blocks, (long long)table_stride);
    SMLM_CHECK_ARG(n_pages >= 1 && n_pages <= INT32_MAX / 2, "%s: %lld pages", what, (long long)n_pages);
    SMLM_CHECK_ARG(page_size >= 1 && page_size <= 4096 && (page_size & (page_size - 1)) == 0 &&
                       max_blocks * page_size <= INT32_MAX / 2,
                   "%s: page_size %lld (a power of two up to 4096; %lld columns)", what, (long long)page_size,
                   (long long)max_blocks);
    pg = Pages{table, lengths, refcount, table_stride, (int)table_rows, (int)max_blocks, (int)n_pages, status};
    return SMLM_OK;
}

static int log2_of(int64_t x) {
    int s = 0;
    while ((int64_t(1) << s) < x) s++;
    return s;
}

static int check_pool(const char* what, const void* pool, int64_t planes, int64_t heads, int64_t token_bytes) {
    SMLM_CHECK_ARG(pool && (uintptr_t)pool % 16 == 0, "%s: the pool has to be 16-byte aligned", what);
    SMLM_CHECK_ARG(planes >= 1 && heads >= 1 && planes * heads <= (1 << 24) && token_bytes >= 16 &&
                       token_bytes % 16 == 0 && token_bytes <= 4096,
                   "%s: %lld planes, %lld heads, %lld bytes per token and head (a multiple of 16 up to 4096)", what,
                   (long long)planes, (long long)heads, (long long)token_bytes);
    return SMLM_OK;
}

static int copy_grid(int64_t most_units) {
    return (int)std::max<int64_t>(1, std::min<int64_t>((most_units + 7) / 8, (int64_t)sm_count() * 8));
}

}  // namespace smlm

using namespace smlm;

extern "C" int smlm_pages_free(int32_t* table, int64_t table_stride, int64_t table_rows, int64_t max_blocks,
                               int32_t* lengths, int32_t* refcount, int64_t n_pages, const int32_t* rows, int64_t n,
                               int* status, void* stream) {
    if (n == 0) return SMLM_OK;
    Pages pg;
    const int rc = check_pages(pg, "pages_free", table, table_stride, table_rows, max_blocks, lengths, refcount,
                               n_pages, 1, status);
    if (rc != SMLM_OK) return rc;
    SMLM_CHECK_ARG(rows && lengths && n > 0 && n <= INT32_MAX, "pages_free: %lld rows", (long long)n);
    pages_free_kernel<<<(unsigned)n, 256, 0, as_stream(stream)>>>(pg, rows);
    SMLM_LAUNCHED("pages_free");
    return SMLM_OK;
}

extern "C" int smlm_pages_trim(int32_t* table, int64_t table_stride, int64_t table_rows, int64_t max_blocks,
                               int32_t* lengths, int32_t* refcount, int64_t n_pages, int64_t page_size,
                               const int32_t* rows, int64_t n, int64_t window, int64_t sinks, int* status,
                               void* stream) {
    if (n == 0) return SMLM_OK;
    Pages pg;
    const int rc = check_pages(pg, "pages_trim", table, table_stride, table_rows, max_blocks, lengths, refcount,
                               n_pages, page_size, status);
    if (rc != SMLM_OK) return rc;
    SMLM_CHECK_ARG(rows && lengths && n > 0 && n <= INT32_MAX, "pages_trim: %lld rows", (long long)n);
    SMLM_CHECK_ARG(window >= 1 && sinks >= 0, "pages_trim: window %lld (at least 1), sinks %lld", (long long)window,
                   (long long)sinks);
    pages_trim_kernel<<<(unsigned)n, 256, 0, as_stream(stream)>>>(pg, rows, log2_of(page_size),
                                                                  (int)std::min<int64_t>(window, INT32_MAX),
                                                                  (int)std::min<int64_t>(sinks, INT32_MAX));
    SMLM_LAUNCHED("pages_trim");
    return SMLM_OK;
}

extern "C" size_t smlm_pages_extend_workspace(int64_t n, int64_t n_pages) {
    WorkspaceSize ws;
    ws.take<int32_t>(n);
    ws.take<int32_t>(n);
    ws.take<int32_t>(n_pages);
    return ws.used;
}

extern "C" int smlm_pages_extend(int32_t* table, int64_t table_stride, int64_t table_rows, int64_t max_blocks,
                                 int32_t* lengths, int32_t* refcount, int64_t n_pages, int64_t page_size,
                                 const int32_t* rows, int64_t n, int64_t n_new, void* workspace, size_t workspace_bytes,
                                 int* status, void* stream) {
    if (n == 0 || n_new == 0) return SMLM_OK;
    Pages pg;
    const int rc = check_pages(pg, "pages_extend", table, table_stride, table_rows, max_blocks, lengths, refcount,
                               n_pages, page_size, status);
    if (rc != SMLM_OK) return rc;
    SMLM_CHECK_ARG(rows && lengths && n > 0 && n <= 65535, "pages_extend: %lld rows (at most 65535)", (long long)n);
    SMLM_CHECK_ARG(n_new > 0 && n_new <= max_blocks * page_size, "pages_extend: %lld new tokens", (long long)n_new);
    Workspace ws(workspace, workspace_bytes);
    int32_t* offset = ws.take<int32_t>(n);
    int32_t* len_of = ws.take<int32_t>(n);
    int32_t* list = ws.take<int32_t>(n_pages);
    if (!workspace || !ws.ok()) {
        set_error("pages_extend: workspace of %zu bytes, %zu needed", workspace_bytes, ws.used);
        return SMLM_ERR_WORKSPACE;
    }
    pages_extend_kernel<<<1, PLAN_THREADS, 0, as_stream(stream)>>>(pg, rows, (int)n, (int)n_new, log2_of(page_size),
                                                                   offset, len_of, list);
    SMLM_LAUNCHED("pages_extend");
    return SMLM_OK;
}

extern "C" size_t smlm_pages_fork_workspace(int64_t n, int64_t table_rows, int64_t max_blocks, int64_t n_pages) {
    WorkspaceSize ws;
    ws.take<int32_t>(table_rows);
    ws.take<int32_t>(n * max_blocks);
    for (int i = 0; i < 5; i++) ws.take<int32_t>(n);
    ws.take<int32_t>(n_pages);
    return ws.used;
}

extern "C" int smlm_pages_fork(void* pool, int64_t planes, int64_t heads, int64_t token_bytes, int32_t* table,
                               int64_t table_stride, int64_t table_rows, int64_t max_blocks, int32_t* lengths,
                               int32_t* refcount, int64_t n_pages, int64_t page_size, const int32_t* parents,
                               const int32_t* children, int64_t n, void* workspace, size_t workspace_bytes,
                               int* status, void* stream) {
    if (n == 0) return SMLM_OK;
    Pages pg;
    int rc = check_pages(pg, "pages_fork", table, table_stride, table_rows, max_blocks, lengths, refcount, n_pages,
                         page_size, status);
    if (rc == SMLM_OK) rc = check_pool("pages_fork", pool, planes, heads, token_bytes);
    if (rc != SMLM_OK) return rc;
    SMLM_CHECK_ARG(parents && children && lengths && n > 0 && n <= 65535, "pages_fork: %lld pairs (at most 65535)",
                   (long long)n);
    Workspace ws(workspace, workspace_bytes);
    int32_t* claim = ws.take<int32_t>(table_rows);
    int32_t* snap = ws.take<int32_t>(n * max_blocks);
    int32_t* snap_len = ws.take<int32_t>(n);
    int32_t* offset = ws.take<int32_t>(n);
    CopyList cl{};
    cl.src = ws.take<int32_t>(n);
    cl.dst = ws.take<int32_t>(n);
    cl.tokens = ws.take<int32_t>(n);
    cl.n = (int)n;
    int32_t* list = ws.take<int32_t>(n_pages);
    if (!workspace || !ws.ok()) {
        set_error("pages_fork: workspace of %zu bytes, %zu needed", workspace_bytes, ws.used);
        return SMLM_ERR_WORKSPACE;
    }
    pages_fork_kernel<<<1, PLAN_THREADS, 0, as_stream(stream)>>>(pg, parents, children, (int)n, log2_of(page_size),
                                                                 claim, snap, snap_len, offset, list, cl);
    SMLM_LAUNCHED("pages_fork: plan");
    pages_copy_kernel<<<copy_grid(n * planes * heads), 256, 0, as_stream(stream)>>>(
        static_cast<char*>(pool), cl, (int)planes, (int)heads, (int)n_pages, (int)page_size, (int)token_bytes, pg,
        nullptr, nullptr);
    SMLM_LAUNCHED("pages_fork: copy");
    return SMLM_OK;
}

extern "C" size_t smlm_pages_compact_workspace(int64_t n_pages) {
    WorkspaceSize ws;
    for (int i = 0; i < 3; i++) ws.take<int32_t>(n_pages);
    ws.take<int32_t>(2);
    return ws.used;
}

extern "C" int smlm_pages_compact(void* pool, int64_t planes, int64_t heads, int64_t token_bytes, int32_t* table,
                                  int64_t table_stride, int64_t table_rows, int64_t max_blocks, int32_t* refcount,
                                  int64_t n_pages, int64_t page_size, void* workspace, size_t workspace_bytes,
                                  int* status, void* stream) {
    Pages pg;
    int rc = check_pages(pg, "pages_compact", table, table_stride, table_rows, max_blocks, nullptr, refcount, n_pages,
                         page_size, status);
    if (rc == SMLM_OK) rc = check_pool("pages_compact", pool, planes, heads, token_bytes);
    if (rc != SMLM_OK) return rc;
    Workspace ws(workspace, workspace_bytes);
    int32_t* to = ws.take<int32_t>(n_pages);
    CopyList cl{};
    cl.src = ws.take<int32_t>(n_pages);
    cl.dst = ws.take<int32_t>(n_pages);
    cl.count = ws.take<int32_t>(2);
    if (!workspace || !ws.ok()) {
        set_error("pages_compact: workspace of %zu bytes, %zu needed", workspace_bytes, ws.used);
        return SMLM_ERR_WORKSPACE;
    }
    pages_compact_kernel<<<1, PLAN_THREADS, 0, as_stream(stream)>>>(pg, to, cl.count + 1, cl);
    SMLM_LAUNCHED("pages_compact: plan");
    pages_copy_kernel<<<copy_grid(n_pages / 2 * planes * heads), 256, 0, as_stream(stream)>>>(
        static_cast<char*>(pool), cl, (int)planes, (int)heads, (int)n_pages, (int)page_size, (int)token_bytes, pg, to,
        cl.count + 1);
    SMLM_LAUNCHED("pages_compact: copy");
    return SMLM_OK;
}
