// The pages of a paged key-value cache, managed on the device: extending sequences, forking them (whole pages
// shared, the partly filled last page copied), freeing, trimming to a window, and compacting the pool.
//
// The allocator's whole state is one reference count per page (0 = free), and a page is always taken from the lowest
// numbers that are free, so tables and counts after any sequence of calls are reproducible and nothing has to be
// kept beside them. Every count changes by integer atomics, whose order does not matter.
#include "paged.cuh"

namespace smlm {

constexpr int PLAN_THREADS = 1024;
constexpr int COPY_UNROLL = 4;

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

// Whether r is a row; negative numbers pad lists of a fixed length, larger ones are flagged.
__device__ __forceinline__ bool row_ok(const Pages& pg, int r) {
    if (r >= 0 && r < pg.table_rows) return true;
    if (r >= 0) flag(pg.status, SMLM_FLAG_INDEX_RANGE);
    return false;
}

// Whether a row's length is one that the table can hold (flagged if not).
__device__ __forceinline__ bool length_ok(const Pages& pg, int len, int shift) {
    if (len >= 0 && len <= (int64_t)pg.max_blocks << shift) return true;
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
    grid_wait();
    grid_release();
    const int r = rows[blockIdx.x];
    if (!row_ok(pg, r)) return;
    for (int j = threadIdx.x; j < pg.max_blocks; j += blockDim.x) drop_entry(pg, pg.table + r * pg.table_stride + j);
    if (threadIdx.x == 0) pg.lengths[r] = 0;
}

// Releases the pages that hold only tokens in [sinks, length - window).
__global__ void __launch_bounds__(256) pages_trim_kernel(Pages pg, const int32_t* rows, int shift, int window,
                                                         int sinks) {
    grid_wait();
    grid_release();
    const int r = rows[blockIdx.x];
    if (!row_ok(pg, r) || !length_ok(pg, pg.lengths[r], shift)) return;
    const int64_t first = (((int64_t)sinks + (1 << shift) - 1) >> shift);
    const int64_t last = max((int64_t)pg.lengths[r] - window, (int64_t)0) >> shift;
    for (int64_t j = first + threadIdx.x; j < min(last, (int64_t)pg.max_blocks); j += blockDim.x)
        drop_entry(pg, pg.table + r * pg.table_stride + j);
}

// ------------------------------------------------------------------------------------------------- planning
// Exclusive sum over the block, in thread order; *total receives the sum of all.
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* total) {
    __shared__ V part[PLAN_THREADS / 32];
    const int lane = lane_id(), warp = threadIdx.x >> 5;
    V x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(FULL, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) part[warp] = x;
    __syncthreads();
    if (warp == 0) {
        V p = part[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const V y = __shfl_up_sync(FULL, p, o);
            if (lane >= o) p += y;
        }
        part[lane] = p;
    }
    __syncthreads();
    *total = part[PLAN_THREADS / 32 - 1];
    return x - v + (warp ? part[warp - 1] : 0);
}

// The blocks of one cluster that plan together (one to eight): phases that read what others wrote are separated by the
// cluster's barrier, which costs a fraction of a kernel launch. What crosses blocks is read past L1 (__ldcg).
struct Team {
    int rank, size;
    __device__ __forceinline__ Team() {
        asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
        asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    }
    __device__ __forceinline__ void sync() const {
        if (size > 1) cluster_sync();
        else __syncthreads();
    }
    __device__ __forceinline__ int thread() const { return rank * PLAN_THREADS + threadIdx.x; }
    __device__ __forceinline__ int threads() const { return size * PLAN_THREADS; }
};
constexpr int MAX_TEAM = 8;

// Exclusive sum over the team's threads in order, of one value each; totals: MAX_TEAM ints in global memory. Every
// thread of the team calls it; it passes one barrier.
__device__ __forceinline__ int team_scan(const Team& team, int v, int32_t* totals, int* total) {
    int mine;
    const int x = block_scan(v, &mine);
    if (team.size == 1) {
        *total = mine;
        return x;
    }
    if (threadIdx.x == 0) totals[team.rank] = mine;
    team.sync();
    int before = 0, all = 0;
    for (int r = 0; r < team.size; r++) {
        const int c = __ldcg(totals + r);
        before += r < team.rank ? c : 0;
        all += c;
    }
    *total = all;
    return before + x;
}

// A warp's contiguous piece of the pages, 32 at a time: which of them are in use. The first 32 words stay in registers
// (lane i has word i), so up to 32768 pages a block are read once. (A thread with pages of its own, one after the other:
// compacting 100000 pages 24 us instead of 13, 10^6 pages 266 instead of 85.)
struct Piece {
    const int32_t* refcount;
    int n_pages, first, words;  // words of 32 pages from word `first` on
    uint32_t kept = 0;
    __device__ __forceinline__ Piece(const Team& team, const Pages& pg) : refcount(pg.refcount), n_pages(pg.n_pages) {
        const int all = (n_pages + 31) / 32, warps = team.threads() / 32, each = (all + warps - 1) / warps;
        first = min(all, team.thread() / 32 * each);
        words = min(all - first, each);
    }
    // f(first page of the word, its bits) for every word, several loads in flight; pages past the end are not in use
    template <typename F>
    __device__ __forceinline__ void read(F f) {
        constexpr int U = 4;
        const int lane = lane_id();
#pragma unroll 1
        for (int w0 = 0; w0 < words; w0 += U) {
            int v[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int p = (first + w0 + u) * 32 + lane;
                v[u] = w0 + u < words && p < n_pages ? __ldcg(refcount + p) : 0;
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (w0 + u >= words) break;
                const uint32_t used = __ballot_sync(FULL, v[u] > 0);
                if (w0 + u == lane) kept = used;
                f((first + w0 + u) * 32, used);
            }
        }
    }
    // the same again, the first 32 words from the registers
    template <typename F>
    __device__ __forceinline__ void again(F f) {
        const int lane = lane_id();
#pragma unroll 1
        for (int w = 0; w < words; w++) {
            const int p = (first + w) * 32;
            uint32_t used = __shfl_sync(FULL, kept, w & 31);
            if (w >= 32) used = __ballot_sync(FULL, p + lane < n_pages && __ldcg(refcount + p + lane) > 0);
            f(p, used);
        }
    }
    // the bits of pages below n in the word that begins at page p
    static __device__ __forceinline__ uint32_t below(int p, int n) {
        return p + 32 <= n ? FULL : p >= n ? 0u : (1u << (n - p)) - 1;
    }
};

// The sum of one value per warp (the same in its lanes) over the warps before this one; *total: of all.
__device__ __forceinline__ int team_scan_warps(const Team& team, int v, int32_t* totals, int* total) {
    return __shfl_sync(FULL, team_scan(team, lane_id() == 0 ? v : 0, totals, total), 0);
}

// The free pages in increasing order: list[k] = the k-th free page, for k < most. Returns how many there are. Ends with
// a barrier.
__device__ int list_free(const Team& team, const Pages& pg, int32_t* list, int most, int32_t* totals) {
    Piece piece(team, pg);
    const int lane = lane_id();
    const uint32_t lower = (1u << lane) - 1;
    int count = 0, total;
    piece.read([&](int p, uint32_t used) { count += __popc(~used & Piece::below(p, pg.n_pages)); });
    int rank = team_scan_warps(team, count, totals, &total);
    if (rank < most)
        piece.again([&](int p, uint32_t used) {
            const uint32_t free = ~used & Piece::below(p, pg.n_pages);
            const int k = rank + __popc(free & lower);
            if (free >> lane & 1 && k < most) list[k] = p + lane;
            rank += __popc(free);
        });
    team.sync();
    return total;
}

// offset[i] = sum of need(0 .. i-1); returns the sum of all; both at most `most` (the pages there are: more cannot be
// handed out). need(i) is called once for each i < n. One block. V holds the sum of all (65535 rows may want 2^30 each).
template <typename V, typename F>
__device__ int scan_needs(int n, int32_t* offset, int most, F need) {
    V sum = 0;
    for (int base = 0; base < n; base += PLAN_THREADS) {
        const int i = base + threadIdx.x;
        V total;
        const V off = block_scan<V>(i < n ? need(i) : 0, &total);
        if (i < n) offset[i] = (int32_t)min(sum + off, (V)most);
        sum += total;
        __syncthreads();
    }
    return (int)min(sum, (V)most);
}

// lengths[r] += n_new for every listed row, with the pages that takes: rows in order, lowest free pages first. A row
// whose pages are not there, or whose table is too narrow, stays as it is and raises a flag. The lengths are taken by
// an exchange and put back at the end, which finds rows listed twice (the second does nothing). Without a page to
// hand out (most decoding steps) the counts are not read. Eight rows: 4 us, a launch and four dependent accesses.
// grown (or NULL): what each listed row of the table grew by, n_new or 0.
// V: what the wanted pages are summed in; the host takes 32 bits where they cannot pass them (64: 0.2 us more).
template <typename V>
__global__ void __launch_bounds__(PLAN_THREADS) pages_extend_kernel(Pages pg, const int32_t* rows, int n, int n_new,
                                                                    int shift, int32_t* offset, int32_t* len_of,
                                                                    int32_t* list, int32_t* totals, int32_t* grown) {
    constexpr int TAKEN = INT32_MIN;
    grid_wait();
    grid_release();
    const Team team;
    const int64_t cap = (int64_t)pg.max_blocks << shift;
    auto blocks = [&](int64_t len) { return (int)((len + (1 << shift) - 1) >> shift); };
    auto fits = [&](int len) { return len >= 0 && (int64_t)len + n_new <= cap; };
    if (team.rank == 0) {
        const int wanted = scan_needs<V>(n, offset, pg.n_pages, [&](int i) {
            const int r = rows[i];
            const bool ok = row_ok(pg, r);
            const int len = ok ? atomicExch(pg.lengths + r, TAKEN) : TAKEN;
            len_of[i] = len;
            if (ok && (len == TAKEN || !fits(len))) flag(pg.status, SMLM_FLAG_INDEX_RANGE);
            return len != TAKEN && fits(len) ? blocks((int64_t)len + n_new) - blocks(len) : 0;
        });
        if (threadIdx.x == 0) totals[MAX_TEAM] = wanted;
    }
    team.sync();
    const int wanted = __ldcg(totals + MAX_TEAM);
    const int have = wanted ? list_free(team, pg, list, wanted, totals) : 0;
    for (int i = team.thread(); i < n; i += team.threads()) {
        const int len = __ldcg(len_of + i);
        if (len == TAKEN) continue;
        bool grow = fits(len);
        const int b0 = blocks(len), need = grow ? blocks((int64_t)len + n_new) - b0 : 0, off = __ldcg(offset + i);
        if (need && (int64_t)off + need > have) {
            flag(pg.status, SMLM_FLAG_NO_PAGES);
            grow = false;
        }
        if (grow)
            for (int m = 0; m < need; m++) {
                const int page = __ldcg(list + off + m);
                pg.table[rows[i] * pg.table_stride + b0 + m] = page;
                pg.refcount[page] = 1;
            }
        pg.lengths[rows[i]] = grow ? len + n_new : len;
        if (grown) grown[rows[i]] = grow ? n_new : 0;
    }
}

struct CopyList {
    int32_t *src, *dst, *tokens;  // page numbers, tokens to copy
    int32_t* count;               // entries (device), or NULL: n
    int n;
};

// Row children[i] becomes a copy of row parents[i] as it was before the call, for all i at once: the parents' entries
// are read (with a reference more for each whole page, and one that holds the partly filled pages meanwhile) before
// the children's are released, and pages are handed out after that. One warp per pair, lanes over its entries. The
// time is the phases' chains of dependent loads (8 pairs 6 us, 256 pairs of 32 entries 9 us with eight blocks; one block
// with a thread an entry took 23), so each phase leaves what the next ones need side by side (snap_len, cl.tokens,
// cl.src: -1 / 0 where nothing is to be done).
__global__ void __launch_bounds__(PLAN_THREADS)
    pages_fork_kernel(Pages pg, const int32_t* parents, const int32_t* children, int n, int shift, int32_t* claim,
                      int32_t* snap, int32_t* snap_len, int32_t* offset, int32_t* list, int32_t* totals, CopyList cl) {
    grid_wait();
    grid_release();
    const Team team;
    const int mb = pg.max_blocks, lane = lane_id();
    const int warp0 = team.thread() >> 5, warps = team.threads() >> 5;
    auto inside = [&](int r) { return r >= 0 && r < pg.table_rows; };
    // of the pairs that list the same child one remains: the one whose number stays here
    for (int i = team.thread(); i < n; i += team.threads()) {
        const int c = children[i], p = parents[i];
        if (row_ok(pg, c) && row_ok(pg, p)) claim[c] = i;
    }
    team.sync();
    for (int i = warp0; i < n; i += warps) {
        const int c = children[i], p = parents[i];
        int len = -1, tokens = 0;
        if (inside(c) && inside(p)) {
            const int owner = __ldcg(claim + c), held = __ldcg(pg.lengths + p);
            const int32_t* row = pg.table + p * pg.table_stride;
            const int head = lane < mb ? row[lane] : -1;  // not waiting for the length
            if (owner != i) {
                if (lane == 0) flag(pg.status, SMLM_FLAG_INDEX_RANGE);
            } else if (c != p && length_ok(pg, held, shift)) {
                len = held;
                const int used = (len + (1 << shift) - 1) >> shift, rest = len & ((1 << shift) - 1);
                for (int j = lane; j < used; j += 32) {
                    int e = j < 32 ? head : row[j];
                    if (e >= pg.n_pages) {
                        flag(pg.status, SMLM_FLAG_INDEX_RANGE);
                        e = -1;
                    }
                    snap[(int64_t)i * mb + j] = e;
                    if (e >= 0) atomicAdd(pg.refcount + e, 1);
                    if (rest && j == used - 1) {
                        cl.src[i] = e;
                        tokens = e >= 0 ? rest : 0;
                    }
                }
                tokens = __reduce_add_sync(FULL, tokens);
            }
        }
        if (lane == 0) {
            snap_len[i] = len;
            cl.tokens[i] = tokens;
        }
    }
    team.sync();
    if (team.rank == 0) {
        const int wanted = scan_needs<int>(n, offset, pg.n_pages, [&](int i) { return __ldcg(cl.tokens + i) ? 1 : 0; });
        if (threadIdx.x == 0) totals[MAX_TEAM] = wanted;
    }
    for (int i = warp0; i < n; i += warps) {
        const int len = __ldcg(snap_len + i), c = children[i];
        if (!inside(c)) continue;
        for (int j = lane; j < mb; j += 32) {
            int32_t* entry = pg.table + c * pg.table_stride + j;
            const int e = __ldcg(entry);
            if (len < 0 || e < 0) continue;
            *entry = -1;
            if (e < pg.n_pages) atomicSub(pg.refcount + e, 1);
            else flag(pg.status, SMLM_FLAG_INDEX_RANGE);
        }
    }
    team.sync();
    const int wanted = __ldcg(totals + MAX_TEAM);
    const int have = wanted ? list_free(team, pg, list, wanted, totals) : 0;
    for (int i = warp0; i < n; i += warps) {
        const int len = __ldcg(snap_len + i), tokens = __ldcg(cl.tokens + i), src = __ldcg(cl.src + i);
        const int off = __ldcg(offset + i), c = children[i];
        if (len < 0) continue;
        const int page = tokens && off < have ? __ldcg(list + off) : -1;
        for (int j = lane; j << shift < len; j += 32)
            pg.table[c * pg.table_stride + j] =
                tokens && j == len >> shift ? page : __ldcg(snap + (int64_t)i * mb + j);
        if (lane) continue;
        pg.lengths[c] = len;
        if (!tokens) continue;
        atomicSub(pg.refcount + src, 1);
        cl.dst[i] = page;
        if (page >= 0) {
            pg.refcount[page] = 1;
        } else {
            cl.tokens[i] = 0;
            flag(pg.status, SMLM_FLAG_NO_PAGES);
        }
    }
}

// With L pages in use: the k-th used page numbered L or above moves to the k-th free page below L. to[p] (p >= L) is
// where page p went. Two scans give L and the ranks. 6480 pages: 7 us, a chain of reads and barriers.
__global__ void __launch_bounds__(PLAN_THREADS) pages_compact_kernel(Pages pg, int32_t* to, int32_t* live_out,
                                                                     int32_t* totals, CopyList cl) {
    grid_wait();
    grid_release();
    const Team team;
    Piece piece(team, pg);
    const int lane = lane_id();
    const uint32_t lower = (1u << lane) - 1;
    int count = 0, live, below;
    piece.read([&](int, uint32_t used) { count += __popc(used); });
    int rank = team_scan_warps(team, count, totals, &live);  // used pages before the word
    count = 0;  // of them below L
    piece.again([&](int p, uint32_t used) { count += __popc(used & Piece::below(p, live)); });
    team_scan_warps(team, count, totals + MAX_TEAM, &below);
    const int moves = live - below;
    piece.again([&](int p, uint32_t used) {
        const int page = p + lane, before = rank + __popc(used & lower);
        const bool u = used >> lane & 1;
        if (page < live) {
            if (!u) cl.dst[page - before] = page;
        } else if (page < pg.n_pages) {
            if (u) cl.src[before - below] = page;
            else to[page] = page;
        }
        rank += __popc(used);
    });
    if (team.thread() == 0) {
        *cl.count = moves;
        *live_out = live;
    }
    team.sync();
    for (int k = team.thread(); k < moves; k += team.threads()) {
        const int s = __ldcg(cl.src + k), d = __ldcg(cl.dst + k);
        pg.refcount[d] = __ldcg(pg.refcount + s);
        pg.refcount[s] = 0;
        to[s] = d;
    }
}

// --------------------------------------------------------------------------------------------------- moving
// The listed pages' tokens in every (layer, k / v) plane: one warp per (entry, plane, head), 16 bytes a lane and four
// loads in flight before the first store. With `to`, the table's entries follow their pages. Memory bounds it: 1583 pages
// of 147 KB in 72 us, 99% of the measured copy rate; one load at a time took 91 us.
__global__ void __launch_bounds__(256) pages_copy_kernel(char* pool, CopyList cl, int planes, int heads, int n_pages,
                                                         int page_size, int token_bytes, Pages pg, const int32_t* to,
                                                         const int32_t* live) {
    grid_wait();
    grid_release();
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
        for (int x0 = lane * 16; x0 < bytes; x0 += 512 * COPY_UNROLL) {
            int4 v[COPY_UNROLL];
#pragma unroll
            for (int k = 0; k < COPY_UNROLL; k++)
                if (x0 + 512 * k < bytes) v[k] = __ldcs(reinterpret_cast<const int4*>(s + x0 + 512 * k));
#pragma unroll
            for (int k = 0; k < COPY_UNROLL; k++)
                if (x0 + 512 * k < bytes) __stcs(reinterpret_cast<int4*>(d + x0 + 512 * k), v[k]);
        }
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

// Plans with one block for small caches, up to eight for large ones (`entries`: about how many threads it wants).
template <typename... P, typename... A>
static int launch_plan(void (*kernel)(P...), const char* what, int64_t entries, cudaStream_t st, A... args) {
    int size = 1;
    while (size < MAX_TEAM && (int64_t)size * PLAN_THREADS < entries) size *= 2;
    return launch_dependent(kernel, what, size, size, PLAN_THREADS, st, args...);
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
    return launch_dependent(pages_free_kernel, "pages_free", 1, n, 256, as_stream(stream), pg, rows);
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
    return launch_dependent(pages_trim_kernel, "pages_trim", 1, n, 256, as_stream(stream), pg, rows, log2_of(page_size),
                            (int)std::min<int64_t>(window, INT32_MAX), (int)std::min<int64_t>(sinks, INT32_MAX));
}

extern "C" size_t smlm_pages_extend_workspace(int64_t n, int64_t n_pages) {
    WorkspaceSize ws;
    ws.take<int32_t>(n);
    ws.take<int32_t>(n);
    ws.take<int32_t>(n_pages);
    ws.take<int32_t>(2 * MAX_TEAM);
    return ws.used;
}

extern "C" int smlm_pages_extend_grown(int32_t* table, int64_t table_stride, int64_t table_rows, int64_t max_blocks,
                                       int32_t* lengths, int32_t* refcount, int64_t n_pages, int64_t page_size,
                                       const int32_t* rows, int64_t n, int64_t n_new, int32_t* grown, void* workspace,
                                       size_t workspace_bytes, int* status, void* stream) {
    if (n == 0 || (n_new == 0 && !grown)) return SMLM_OK;
    Pages pg;
    const int rc = check_pages(pg, "pages_extend", table, table_stride, table_rows, max_blocks, lengths, refcount,
                               n_pages, page_size, status);
    if (rc != SMLM_OK) return rc;
    SMLM_CHECK_ARG(rows && lengths && n > 0 && n <= 65535, "pages_extend: %lld rows (at most 65535)", (long long)n);
    SMLM_CHECK_ARG(n_new >= 0 && n_new <= max_blocks * page_size, "pages_extend: %lld new tokens", (long long)n_new);
    Workspace ws(workspace, workspace_bytes);
    int32_t* offset = ws.take<int32_t>(n);
    int32_t* len_of = ws.take<int32_t>(n);
    int32_t* list = ws.take<int32_t>(n_pages);
    int32_t* totals = ws.take<int32_t>(2 * MAX_TEAM);
    if (!workspace || !ws.ok()) {
        set_error("pages_extend: workspace of %zu bytes, %zu needed", workspace_bytes, ws.used);
        return SMLM_ERR_WORKSPACE;
    }
    const bool fits = n * (n_new / page_size + 1) <= INT32_MAX;  // a row's need is at most that
    return launch_plan(fits ? pages_extend_kernel<int32_t> : pages_extend_kernel<int64_t>, "pages_extend",
                       std::max(n, n_pages), as_stream(stream), pg, rows, (int)n, (int)n_new, log2_of(page_size), offset,
                       len_of, list, totals, grown);
}

extern "C" int smlm_pages_extend(int32_t* table, int64_t table_stride, int64_t table_rows, int64_t max_blocks,
                                 int32_t* lengths, int32_t* refcount, int64_t n_pages, int64_t page_size,
                                 const int32_t* rows, int64_t n, int64_t n_new, void* workspace, size_t workspace_bytes,
                                 int* status, void* stream) {
    return smlm_pages_extend_grown(table, table_stride, table_rows, max_blocks, lengths, refcount, n_pages, page_size,
                                   rows, n, n_new, nullptr, workspace, workspace_bytes, status, stream);
}

extern "C" size_t smlm_pages_fork_workspace(int64_t n, int64_t table_rows, int64_t max_blocks, int64_t n_pages) {
    WorkspaceSize ws;
    ws.take<int32_t>(table_rows);
    ws.take<int32_t>(n * max_blocks);
    for (int i = 0; i < 5; i++) ws.take<int32_t>(n);
    ws.take<int32_t>(n_pages);
    ws.take<int32_t>(2 * MAX_TEAM);
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
    int32_t* totals = ws.take<int32_t>(2 * MAX_TEAM);
    if (!workspace || !ws.ok()) {
        set_error("pages_fork: workspace of %zu bytes, %zu needed", workspace_bytes, ws.used);
        return SMLM_ERR_WORKSPACE;
    }
    rc = launch_plan(pages_fork_kernel, "pages_fork: plan", std::max(32 * n, n_pages), as_stream(stream), pg,
                     parents, children, (int)n, log2_of(page_size), claim, snap, snap_len, offset, list, totals, cl);
    if (rc != SMLM_OK) return rc;
    return launch_dependent(pages_copy_kernel, "pages_fork: copy", 1, copy_grid(n * planes * heads), 256,
                            as_stream(stream), static_cast<char*>(pool), cl, (int)planes, (int)heads, (int)n_pages,
                            (int)page_size, (int)token_bytes, pg, nullptr, nullptr);
}

extern "C" size_t smlm_pages_compact_workspace(int64_t n_pages) {
    WorkspaceSize ws;
    for (int i = 0; i < 3; i++) ws.take<int32_t>(n_pages);
    ws.take<int32_t>(2);
    ws.take<int32_t>(2 * MAX_TEAM);
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
    int32_t* totals = ws.take<int32_t>(2 * MAX_TEAM);
    if (!workspace || !ws.ok()) {
        set_error("pages_compact: workspace of %zu bytes, %zu needed", workspace_bytes, ws.used);
        return SMLM_ERR_WORKSPACE;
    }
    rc = launch_plan(pages_compact_kernel, "pages_compact: plan", n_pages, as_stream(stream), pg, to, cl.count + 1,
                     totals, cl);
    if (rc != SMLM_OK) return rc;
    return launch_dependent(pages_copy_kernel, "pages_compact: copy", 1, copy_grid(n_pages / 2 * planes * heads), 256,
                            as_stream(stream), static_cast<char*>(pool), cl, (int)planes, (int)heads, (int)n_pages,
                            (int)page_size, (int)token_bytes, pg, to, cl.count + 1);
}
