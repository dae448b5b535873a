// Attention of one new token per sequence over a paged key-value cache, and the append that fills it.
#include <atomic>

#include "paged.cuh"

namespace smlm {

// ------------------------------------------------------------------------------------------------ attention
// out = sum_j p_j v_j / sum_j p_j with p_j = exp(scale <q, k_j> - max) over the visible tokens, in one pass: every key
// and value is read once, with 4 flops per element and query head of its group, so reading them is the time, and the
// kernels are built to keep loads in flight. Each WARP works by itself with no barrier in its loop (Stream): it takes
// tiles of TT tokens straight from global memory into registers with 16-byte loads, in the layout that mma.sync wants:
//   S^T = K q^T     A = keys (16 tokens x k), B = queries (k x 8): a lane's 16 bytes of token lane / 4 are the A
//                   fragments of two k-steps, because the order of k is free as long as q's is the same;
//   O^T += V^T P^T  A = values (16 d x tokens): the 16 bytes of tokens 2t, 2t + 1 are zipped into pairs (prmt) and
//                   feed d = 8 g + 2 i in row g, 8 g + 2 i + 1 in row g + 8; B = P^T, the transposed scores
//                   (movmatrix).
// With queries as the 8 columns, up to 8 query heads of one key head cost the same as one. (mma.sync is enough: the
// tile of queries is 8 wide, and tcgen05's 128-row tiles would be 1/16 full or less.) Running maxima and sums are
// fp32, one per column; the weights enter the second product as a sum of two 16-bit values (hi + lo), so they carry
// 16 bits or more and rounding the output is the only loss that shows. fp16 ends at 2^-24, which weights of at most 1
// pass 17 nats below the maximum, while their fp32 sum keeps them: they are taken 2^15 times as large there (WEIGHT) and
// carry 16 bits down to 2^-24 of the largest weight; what is below 2^-40 of it adds nothing.
// fp32 caches use the same shape with tf32 fragments, each operand split in two and three products kept (2^-21).
//
// The tiles of all (sequence, key head, 8 or 16 query heads) items form one list, cut evenly over all warps of the grid,
// whatever the lengths are (they are on the device); items that were cut are joined by paged_join_kernel
// (paged_split_kernel). With few short sequences a cluster of blocks takes an item (paged_cluster_kernel).
//
// Device time per call, share of the measured copy rate (6570 GB/s) for the bytes of the visible keys and values:
//   64 x 2175 tokens, 6 heads x 64, bf16: 41.6 us, 78%; 1 x 131071, 32 / 8 heads x 128, fp16: 86.8 us, 94%;
//   96 x 0-8191, 32 / 8 x 128, bf16: 67.6 us, 84%; 64 x 1028 seen, 16 / 2 x 128, bf16: 17.3 us (cluster), 59%;
//   1 x 2304, 6 x 64, bf16: 5.9 us (cluster); 8 heads, fp32, 32 x 2048 x 64: 54.7 us, 75%, 16 x 2048 x 128: 53.6, 76%.
// While all warps run, memory delivers 93% of the copy rate; the rest is the start (2.5 us to the first tiles), the
// spread of the last warps (4 us) and the join (3 us).

constexpr int SPLIT_WARPS = 4, SPLIT_THREADS = SPLIT_WARPS * 32;
constexpr int JOIN_THREADS = 256;
constexpr int HEAD = 1;  // what beginning an item costs in the cut, in tiles (measured: 1 and 2 alike, 0 and 4 slower)

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
    if constexpr (std::is_same_v<T, __half>)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// fp32 operands as tf32 hi + lo: x = hi + lo up to 2^-22 of x (KEEP: not to be computed once and held in registers)
template <bool KEEP = false>
struct Split32 {
    uint32_t hi, lo;
    __device__ __forceinline__ explicit Split32(uint32_t bits) {
        if constexpr (KEEP) asm volatile("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(__uint_as_float(bits)));
        else asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(__uint_as_float(bits)));
        lo = __float_as_uint(__uint_as_float(bits) - __uint_as_float(hi));
    }
};
__device__ __forceinline__ void mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c += a b, the small products into `small` (the same array, or one of its own). The tensor cores cut the sum of each
// step off instead of rounding it, so long sums stay out of their accumulators: the scores add up in three, the
// outputs' parts of 16 tokens are added to the sums with rounding.
template <bool KEEP>
__device__ __forceinline__ void mma_split32(float (&c)[4], float (&small)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, const Split32<KEEP>& b0, const Split32<KEEP>& b1) {
    const Split32<> x0(a0), x1(a1), x2(a2), x3(a3);
    mma8(small, x0.lo, x1.lo, x2.lo, x3.lo, b0.hi, b1.hi);
    mma8(small, x0.hi, x1.hi, x2.hi, x3.hi, b0.lo, b1.lo);
    mma8(c, x0.hi, x1.hi, x2.hi, x3.hi, b0.hi, b1.hi);
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float x, float y) {  // x in the low half
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <typename T>
__device__ __forceinline__ float2 unpack16(uint32_t p) {
    if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&p));
    else return make_float2(bf16_bits_to_f32(p & 0xffffu), __uint_as_float(p & 0xffff0000u));
}

template <typename T>
__device__ __forceinline__ void widen16(const uint4& v, float (&f)[16 / sizeof(T)]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            f[i] = __uint_as_float(w[i]);
        } else {
            const float2 p = unpack16<T>(w[i]);
            f[2 * i] = p.x;
            f[2 * i + 1] = p.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 narrow16(const float (&f)[16 / sizeof(T)]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
        else w[i] = pack16<T>(f[2 * i], f[2 * i + 1]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A value in the same place of another block's shared memory (rank in the cluster).
template <typename V>
__device__ __forceinline__ V of_block(const V* p, int rank) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    V v;
    if constexpr (sizeof(V) == 16)
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
    else
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
    return v;
}

// The tiles of one sequence: all of [0, n), or with a window those of the first tokens and of [lo, n).
struct Span {
    int n, lo, sinks, head, skip, tiles;  // tiles [0, head) and, skip further on, the rest
    __device__ __forceinline__ Span(int len, int window, int sink, int tt) : n(len) {
        lo = window && n > window ? n - window : 0;
        sinks = min(sink, lo);
        head = (sinks + tt - 1) / tt;
        skip = max(lo / tt - head, 0);
        tiles = (n + tt - 1) / tt - skip;
    }
    __device__ __forceinline__ int token(int tile, int tt) const { return (tile < head ? tile : tile + skip) * tt; }
    __device__ __forceinline__ bool sees(int t) const { return t < n && (t >= lo || t < sinks); }
};

// Where the pieces of items that were cut lie. A worker has at most two: the one it began inside an item (slot 2 w)
// and the one that holds an item's first tile but not its last (slot 2 w + 1).
struct SplitWork {
    int2* cut;  // (batch, items): the workers of the item's first and last tile; x = -1: not cut
    float* ml;  // (slots, rows, 2): running maximum and sum
    float* o;   // (slots, rows, dp)
    int rows, dp;  // rows = min(group, query heads of an item)
};

// NT: eights of query heads an item has (two where a group has more than eight and the registers allow it).
template <typename T, int DP, int NT>
struct SplitShape {
    static constexpr int ES = sizeof(T);
    static constexpr int CH = 16 / ES;                   // elements of a 16-byte load
    static constexpr int TT = ES == 2 && DP <= 64 && NT == 1 ? 32 : 16;  // tokens per tile: 64 registers
    static constexpr int NS = TT / 16;
    static constexpr int KJ = DP / (4 * CH);             // loads per key row and lane
    static constexpr int VB = DP >= 8 * CH ? DP / (8 * CH) : 1;  // loads per value row and lane
    static constexpr int MT = ES == 2 ? 4 : 2;           // 16-row tiles of O^T per value load
    static constexpr int QT = 8 * NT;
    // rows of more than 256 bytes: queries from shared memory, values loaded after the scores; of 1 KB: keys and
    // values in two halves
    static constexpr bool WIDE = DP * ES > 256, HALVES = DP * ES > 512;
    static constexpr int KK = HALVES ? KJ / 2 : KJ, VR = HALVES ? 2 : 4;
    static constexpr int BLOCKS = DP * ES * NT <= 128 ? 4 : DP * ES * NT <= 256 ? 3 : 2;  // per SM (registers)
    // the larger blocks of paged_cluster_kernel: eight warps up to d 64 (at d 128 they lose: 1 x 2048 tokens 8.3 -> 8.5 us)
    static constexpr int MORE_WARPS = QT * DP <= 512 ? 8 : 4;
};

// Tiles first .. last - 1 of one item by one warp: the sums of its columns. PART: d < DP; SMALL: pages of fewer than
// 16 tokens, whose tokens are looked up one by one.
template <typename T, int DP, int NT, bool PART, bool SMALL>
struct Stream {
    using S = SplitShape<T, DP, NT>;
    static constexpr int CH = S::CH, TT = S::TT, NS = S::NS, KJ = S::KJ, KK = S::KK, VB = S::VB, VR = S::VR, MT = S::MT;
    static constexpr bool WIDE = S::WIDE, HALVES = S::HALVES, F = S::ES == 4;
    // a weight in the second product, and so o, is WEIGHT times what l counts; an exact factor, taken out in values()
    static constexpr float WEIGHT = std::is_same_v<T, __half> ? 32768.f : 1.f;
    // The tile after next goes to L2 where few bytes are in flight otherwise (two eights of queries: 8 warps an SM; d
    // well below DP): 64 x 8192 tokens, 32 heads on one: 107 -> 96 us, d 80: 70 -> 66, fp32 d 128: 58 -> 56. Where the
    // loads alone fill the memory's queues it costs: d 64 40.3 -> 41.9, one of 131071 tokens 86.8 -> 91.9.
    static constexpr bool AHEAD = !SMALL && !HALVES && (NT == 2 || (PART && DP == 128) || (F && DP == 128));
    static constexpr unsigned ALL = TT == 32 ? FULL : 0xffffu;
    struct PagesOf {  // the pages of a tile: SMALL: of token `lane`; else of each 16 tokens (the same in all lanes)
        int p[SMALL ? 1 : NS];
    };

    float o[NT][VB * MT][4];
    float m[NT][2], l[NT][2];  // columns 2 t4 and 2 t4 + 1 of each eight

    // Lane's share of the loads: keys of tokens g, g + 8 of 16; values as value_token says; see the head of this part.
    static __device__ __forceinline__ int value_token(int s, int r) {
        const int t4 = lane_id() & 3;
        return 16 * s + (F ? t4 + 4 * r : 2 * t4 + (r & 1) + 8 * (r >> 1));
    }

    __device__ __forceinline__ void scores(float (&sc)[NT][NS][4], const uint4 (&kr)[NS][2][KK],
                                           const uint4 (&qf)[NT][WIDE ? 1 : KJ], const uint4* qs, int j0) {
        float odd[4] = {0.f, 0.f, 0.f, 0.f}, small[4] = {0.f, 0.f, 0.f, 0.f};  // F: second and third accumulator
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int jj = 0; jj < KK; jj++) {
                const uint4 a = kr[s][0][jj], e = kr[s][1][jj];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    uint4 w;
                    if constexpr (WIDE) w = qs[(n * KJ + j0 + jj) * 32 + lane_id()];
                    else w = qf[n][jj];
                    if constexpr (F) {
                        constexpr bool KEEP = DP > 64;  // the split queries have no registers there
                        mma_split32(sc[n][s], small, a.x, e.x, a.y, e.y, Split32<KEEP>(w.x), Split32<KEEP>(w.y));
                        mma_split32(odd, small, a.z, e.z, a.w, e.w, Split32<KEEP>(w.z), Split32<KEEP>(w.w));
                    } else {
                        mma16<T>(sc[n][s], a.x, e.x, a.y, e.y, w.x, w.y);
                        mma16<T>(sc[n][s], a.z, e.z, a.w, e.w, w.z, w.w);
                    }
                }
            }
        if constexpr (F) {
#pragma unroll
            for (int x = 0; x < 4; x++) sc[0][0][x] += odd[x] + small[x];
        }
    }

    // qs: this warp's shared memory, NT KJ 32 vectors (WIDE)
    __device__ __forceinline__ void run(const PageView& pv, const T* q, float c, const Span& span, int b, int h, int q0,
                                        int first, int last, uint4* qs, int* status) {
        const int lane = lane_id(), g = lane >> 2, t4 = lane & 3, group = pv.hq / pv.hkv;
        const int shift = pv.page_shift, slots = (1 << shift) - 1;
        const uint32_t kpb = pv.kp * S::ES, ktb = pv.kt * S::ES, vpb = pv.vp * S::ES, vtb = pv.vt * S::ES;  // bytes
        const int32_t* row = pv.table + b * pv.table_stride;
        auto entry = [&](int t) {  // the page of token t, or -1 past the end, in a hole or outside the pool
            int p = -1;
            if (t < span.n) {
                p = row[t >> shift];
                if (p >= pv.n_pages) {
                    flag(status, SMLM_FLAG_INDEX_RANGE);
                    p = -1;
                }
            }
            return p;
        };
        auto pages_at = [&](int i) {
            const int t0 = span.token(i, TT);
            PagesOf x;
            if constexpr (SMALL) {
                x.p[0] = lane < TT ? entry(t0 + lane) : -1;
            } else {
#pragma unroll
                for (int s = 0; s < NS; s++) x.p[s] = entry(t0 + 16 * s);
            }
            return x;
        };
        auto seen_of = [&](int i, const PagesOf& x) {  // which of the tile's tokens are seen
            const int t0 = span.token(i, TT);
            bool whole = t0 + TT <= span.n && (t0 >= span.lo || t0 + TT <= span.sinks);
            if constexpr (!SMALL) {
#pragma unroll
                for (int s = 0; s < NS; s++) whole = whole && x.p[s] >= 0;
                if (whole) return ALL;
                const int p = lane < 16 ? x.p[0] : x.p[NS - 1];
                return __ballot_sync(FULL, lane < TT && p >= 0 && span.sees(t0 + lane));
            } else {
                return __ballot_sync(FULL, x.p[0] >= 0 && span.sees(t0 + lane));
            }
        };
        PagesOf pages = pages_at(first), pages_next;
        const T* qp = q + ((int64_t)b * pv.hq + h * group) * pv.d;
        uint4 qf[NT][WIDE ? 1 : KJ];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < KJ; j++) {
                const int d0 = (t4 + 4 * j) * CH, qrow = q0 + 8 * n + g;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (qrow < group && (!PART || d0 < pv.d)) v = load16(qp + (int64_t)qrow * pv.d + d0);
                if constexpr (WIDE) qs[(n * KJ + j) * 32 + lane] = v;  // read back by the same lane only
                else qf[n][j] = v;
            }
        const char* kp = reinterpret_cast<const char*>(static_cast<const T*>(pv.k) + h * pv.kh + t4 * CH);
        const char* vp = reinterpret_cast<const char*>(static_cast<const T*>(pv.v) + h * pv.vh);
        uint4 kr[NS][2][KK], vr[NS][VR][VB];
        // Tokens that are not seen are loaded all the same, from their own page or page 0 (mapped memory), and masked.
        auto load_keys = [&](int i, const PagesOf& x, int j0) {
            const int t0 = span.token(i, TT);
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const char* base = kp;
                if constexpr (!SMALL)
                    base += (uint64_t)(uint32_t)max(x.p[s], 0) * kpb + (uint64_t)(uint32_t)((t0 + 16 * s) & slots) * ktb +
                            (uint64_t)(uint32_t)g * ktb;
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const char* src;
                    if constexpr (SMALL) {
                        const int y = 16 * s + 8 * r + g;
                        const int p = max(__shfl_sync(FULL, x.p[0], y), 0);
                        src = kp + (uint64_t)(uint32_t)p * kpb + (uint64_t)(uint32_t)((t0 + y) & slots) * ktb;
                    } else {
                        src = base + (uint64_t)(8 * r) * ktb;
                    }
#pragma unroll
                    for (int j = 0; j < KK; j++) {
                        if (!PART || (t4 + 4 * (j0 + j)) * CH < pv.d) kr[s][r][j] = load16(src + 64 * (j0 + j));
                        else kr[s][r][j] = make_uint4(0, 0, 0, 0);
                    }
                }
            }
        };
        auto load_values = [&](int i, const PagesOf& x, int first_row) {
            const int t0 = span.token(i, TT);
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const char* base = vp;
                if constexpr (!SMALL)
                    base += (uint64_t)(uint32_t)max(x.p[s], 0) * vpb + (uint64_t)(uint32_t)((t0 + 16 * s) & slots) * vtb +
                            (uint64_t)(uint32_t)(F ? t4 : 2 * t4) * vtb;
#pragma unroll
                for (int rr = 0; rr < VR; rr++) {
                    const int r = first_row + rr;
                    const char* src;
                    if constexpr (SMALL) {
                        const int y = value_token(s, r);
                        const int p = max(__shfl_sync(FULL, x.p[0], y), 0);
                        src = vp + (uint64_t)(uint32_t)p * vpb + (uint64_t)(uint32_t)((t0 + y) & slots) * vtb;
                    } else {
                        src = base + (uint64_t)(F ? 4 * r : (r & 1) + 8 * (r >> 1)) * vtb;
                    }
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) {
                        const int d0 = (g + 8 * vb) * CH;  // columns past d are not stored
                        const bool in = (!PART && DP >= 8 * CH) || d0 < pv.d;
                        vr[s][rr][vb] = load16(src + (in ? 16 * g + 128 * vb : 0));
                    }
                }
            }
        };
        auto clear_unseen = [&](unsigned seen, int first_row) {  // 0 * (a stale infinity or NaN) is not 0
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int r = 0; r < VR; r++)
                    if (!(seen >> value_token(s, first_row + r) & 1)) {
#pragma unroll
                        for (int vb = 0; vb < VB; vb++) vr[s][r][vb] = make_uint4(0, 0, 0, 0);
                    }
        };

#pragma unroll
        for (int n = 0; n < NT; n++) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < VB * MT; i++) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
        }
        auto prefetch = [&](int i, const PagesOf& x) {
            if constexpr (AHEAD) {
                const int t0 = span.token(i, TT);
                const bool is_k = lane < 16;
                const char* base = reinterpret_cast<const char*>(is_k ? static_cast<const T*>(pv.k) + h * pv.kh
                                                                      : static_cast<const T*>(pv.v) + h * pv.vh);
                const uint32_t pb = is_k ? kpb : vpb, tb = is_k ? ktb : vtb;
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    const char* src = base + (uint64_t)(uint32_t)max(x.p[s], 0) * pb +
                                      (uint64_t)(uint32_t)(((t0 + 16 * s) & slots) + (lane & 15)) * tb;
#pragma unroll
                    for (int k = 0; k < (DP * S::ES + 127) / 128; k++)
                        if (!PART || 128 * k < pv.d * S::ES)
                            asm volatile("prefetch.global.L2 [%0];" ::"l"(src + 128 * k));
                }
            }
        };
        PagesOf pages_far;
        load_keys(first, pages, 0);
        if (!WIDE) load_values(first, pages, 0);
        if (first + 1 < last) pages_next = pages_at(first + 1);
        if (AHEAD && first + 2 < last) pages_far = pages_at(first + 2);
        for (int i = first; i < last; i++) {
            float sc[NT][NS][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int s = 0; s < NS; s++) sc[n][s][0] = sc[n][s][1] = sc[n][s][2] = sc[n][s][3] = 0.f;
            scores(sc, kr, qf, qs, 0);
            if constexpr (HALVES) {
                load_keys(i, pages, KK);
                scores(sc, kr, qf, qs, KK);
            }
            if constexpr (F) {  // inf - inf in a split operand of a token that is seen? Then once more, product by product
                const bool odd0 = !(sc[0][0][0] == sc[0][0][0] && sc[0][0][1] == sc[0][0][1]);
                const bool odd1 = !(sc[0][0][2] == sc[0][0][2] && sc[0][0][3] == sc[0][0][3]);
                bool again = __any_sync(FULL, odd0 || odd1);
                if (again) {  // (not for what lies beside the sequence: its bits would decide how the others round)
                    const unsigned at = seen_of(i, pages) >> g;
                    again = __any_sync(FULL, (odd0 && at & 1) || (odd1 && at >> 8 & 1));
                }
                if (again) {
                    const int t0 = span.token(i, TT);
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const int y = g + 8 * (x >> 1), col = q0 + 2 * t4 + (x & 1);
                        int p = pages.p[0];
                        if constexpr (SMALL) p = __shfl_sync(FULL, p, y);
                        const T* src = static_cast<const T*>(pv.k) + h * pv.kh + max(p, 0) * pv.kp +
                                       ((t0 + y) & slots) * pv.kt;
                        float sum = 0.f;
                        if (col < group) {
#pragma unroll 1
                            for (int d = 0; d < pv.d; d++) sum = fmaf(src[d], qp[(int64_t)col * pv.d + d], sum);
                        }
                        sc[0][0][x] = sum;
                    }
                }
            }
            if (WIDE) load_values(i, pages, 0);
            const unsigned seen = seen_of(i, pages);
            if (!WIDE && i + 1 < last) load_keys(i + 1, pages_next, 0);
            if (seen != ALL && !WIDE) clear_unseen(seen, 0);
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int s = 0; s < NS; s++)
#pragma unroll
                    for (int x = 0; x < 4; x++) sc[n][s][x] *= c;
                if (seen != ALL) {
#pragma unroll
                    for (int s = 0; s < NS; s++)
#pragma unroll
                        for (int r = 0; r < 2; r++)
                            if (!(seen >> (16 * s + 8 * r + g) & 1)) sc[n][s][2 * r] = sc[n][s][2 * r + 1] = -INFINITY;
                }
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int s = 0; s < NS; s++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        x0 = fmaxf(x0, sc[n][s][2 * r]);
                        x1 = fmaxf(x1, sc[n][s][2 * r + 1]);
                    }
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) {
                    x0 = fmaxf(x0, __shfl_xor_sync(FULL, x0, w));
                    x1 = fmaxf(x1, __shfl_xor_sync(FULL, x1, w));
                }
                if (__any_sync(FULL, x0 > m[n][0] || x1 > m[n][1])) {
                    const float n0 = fmaxf(m[n][0], x0), n1 = fmaxf(m[n][1], x1);
                    const float f0 = m[n][0] == n0 ? 1.f : ex2(m[n][0] - n0);
                    const float f1 = m[n][1] == n1 ? 1.f : ex2(m[n][1] - n1);
                    m[n][0] = n0;
                    m[n][1] = n1;
                    l[n][0] *= f0;
                    l[n][1] *= f1;
#pragma unroll
                    for (int x = 0; x < VB * MT; x++) {
                        o[n][x][0] *= f0;
                        o[n][x][1] *= f1;
                        o[n][x][2] *= f0;
                        o[n][x][3] *= f1;
                    }
                }
                const float z0 = m[n][0] == -INFINITY ? 0.f : m[n][0], z1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
                for (int s = 0; s < NS; s++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        sc[n][s][2 * r] = ex2(sc[n][s][2 * r] - z0);
                        sc[n][s][2 * r + 1] = ex2(sc[n][s][2 * r + 1] - z1);
                        l[n][0] += sc[n][s][2 * r];
                        l[n][1] += sc[n][s][2 * r + 1];
                    }
            }
            if (WIDE && seen != ALL) clear_unseen(seen, 0);
            if constexpr (F) {
                // P^T: weight of token 8 r + t4 (+ 4) for query g, from lane (token, query / 2)
                auto weight = [&](int r, int up) {
                    const int from = 4 * t4 + (g >> 1) + up;
                    const float a = __shfl_sync(FULL, sc[0][0][2 * r], from);
                    const float e = __shfl_sync(FULL, sc[0][0][2 * r + 1], from);
                    return Split32<>(__float_as_uint(g & 1 ? e : a));
                };
                const Split32<> p00 = weight(0, 0), p01 = weight(0, 16), p10 = weight(1, 0), p11 = weight(1, 16);
                auto add = [&](float (&to)[4], const float (&x)[4]) {
#pragma unroll
                    for (int k = 0; k < 4; k++) to[k] += x[k];
                };
#pragma unroll
                for (int vb = 0; vb < VB; vb++) {
                    float e[4] = {0.f, 0.f, 0.f, 0.f}, f[4] = {0.f, 0.f, 0.f, 0.f};
                    const uint4 x = vr[0][0][vb], y = vr[0][1][vb];
                    mma_split32(e, e, x.x, x.y, y.x, y.y, p00, p01);
                    mma_split32(f, f, x.z, x.w, y.z, y.w, p00, p01);
                    if constexpr (!HALVES) {
                        const uint4 z = vr[0][2 % VR][vb], w = vr[0][3 % VR][vb];
                        mma_split32(e, e, z.x, z.y, w.x, w.y, p10, p11);
                        mma_split32(f, f, z.z, z.w, w.z, w.w, p10, p11);
                    }
                    add(o[0][vb * MT], e);
                    add(o[0][vb * MT + 1], f);
                }
                if constexpr (HALVES) {
                    load_values(i, pages, 2);
                    if (seen != ALL) clear_unseen(seen, 2);
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) {
                        float e[4] = {0.f, 0.f, 0.f, 0.f}, f[4] = {0.f, 0.f, 0.f, 0.f};
                        const uint4 z = vr[0][0][vb], w = vr[0][1][vb];
                        mma_split32(e, e, z.x, z.y, w.x, w.y, p10, p11);
                        mma_split32(f, f, z.z, z.w, w.z, w.w, p10, p11);
                        add(o[0][vb * MT], e);
                        add(o[0][vb * MT + 1], f);
                    }
                }
            } else {
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    uint32_t hi[NT][2], lo[NT][2];  // P^T: tokens 0 .. 7 and 8 .. 15 of the 16
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            const float x = sc[n][s][2 * r] * WEIGHT, y = sc[n][s][2 * r + 1] * WEIGHT;
                            const uint32_t w = pack16<T>(x, y);
                            const float2 u = unpack16<T>(w);
                            hi[n][r] = transpose8x8(w);
                            lo[n][r] = transpose8x8(pack16<T>(x - u.x, y - u.y));
                        }
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) {
                        const uint4 x = vr[s][0][vb], y = vr[s][1][vb], z = vr[s][2 % VR][vb], w = vr[s][3 % VR][vb];
                        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
                        const uint32_t zs[4] = {z.x, z.y, z.z, z.w}, ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t a0 = __byte_perm(xs[k], ys[k], 0x5410);
                            const uint32_t a1 = __byte_perm(xs[k], ys[k], 0x7632);
                            const uint32_t a2 = __byte_perm(zs[k], ws[k], 0x5410);
                            const uint32_t a3 = __byte_perm(zs[k], ws[k], 0x7632);
#pragma unroll
                            for (int n = 0; n < NT; n++) {
                                mma16<T>(o[n][vb * MT + k], a0, a1, a2, a3, lo[n][0], lo[n][1]);
                                mma16<T>(o[n][vb * MT + k], a0, a1, a2, a3, hi[n][0], hi[n][1]);
                            }
                        }
                    }
                }
            }
            if (i + 1 < last) {
                if (WIDE) load_keys(i + 1, pages_next, 0);
                else load_values(i + 1, pages_next, 0);
                pages = pages_next;
                if (AHEAD && i + 2 < last) {
                    prefetch(i + 2, pages_far);
                    pages_next = pages_far;
                    if (i + 3 < last) pages_far = pages_at(i + 3);
                } else if (i + 2 < last) {
                    pages_next = pages_at(i + 2);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) {
                l[n][0] += __shfl_xor_sync(FULL, l[n][0], w);
                l[n][1] += __shfl_xor_sync(FULL, l[n][1], w);
            }
    }

    // CH consecutive values, (g + 8 vb) CH and on, of column 2 t4 + x of eight n
    __device__ __forceinline__ void values(int n, int x, int vb, float scale, float (&v)[CH]) const {
        scale *= 1.f / WEIGHT;
#pragma unroll
        for (int k = 0; k < MT; k++) {
            v[2 * k] = o[n][vb * MT + k][x] * scale;
            v[2 * k + 1] = o[n][vb * MT + k][2 + x] * scale;
        }
    }
};

// The list: as many blocks as fit, each warp the same number of tiles (beginning an item counts as one). Its first and
// last pieces of cut items go to the workspace, whole items straight to the output.
template <typename T, int DP, int NT, bool PART, bool SMALL>
__global__ void __launch_bounds__(SPLIT_THREADS, SplitShape<T, DP, NT>::BLOCKS)
    paged_split_kernel(PageView pv, const T* q, float c, int window, int sinks, T* __restrict__ out, float* __restrict__ lse,
                       SplitWork wk, int* status) {
    using S = SplitShape<T, DP, NT>;
    constexpr int CH = S::CH, TT = S::TT, VB = S::VB, QT = S::QT;
    __shared__ int4 pre[SPLIT_THREADS / 4];
    __shared__ int part[SPLIT_WARPS];
    __shared__ uint4 qs[S::WIDE ? SPLIT_WARPS * NT * S::KJ * 32 : 1];
    grid_wait();
    grid_release();

    const int lane = lane_id(), warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    const int group = pv.hq / pv.hkv, gt = (group + QT - 1) / QT, items = pv.hkv * gt;

    // what the items of row r take in the list (its length fits 31 bits: the host checks)
    auto cost = [&](int r, int* st) {
        const int tiles = Span(row_length(pv, r, st), window, sinks, TT).tiles;
        return tiles ? items * (tiles + HEAD) : 0;
    };
    auto inclusive = [&](int x) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(FULL, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    // The sequence, the item and the place in it where this worker starts, and how much it does. Up to 128 rows: each
    // warp for itself, a lane up to four rows (1.1 us after the start instead of 2.0); more: a thread has `chunk` rows,
    // and the warp looks for its start in the block's sums and then among the rows.
    const int workers = gridDim.x * SPLIT_WARPS, worker = warp * gridDim.x + blockIdx.x;  // one warp per SM first
    int b = 0, off, left;
    auto cut = [&](int total) {  // the first total % workers pieces are one tile longer
        const int per = (uint32_t)total / (uint32_t)workers, extra = total - per * workers;
        left = per + (worker < extra);
        off = worker * per + min(worker, extra);
    };
    auto among = [&](int x, int w) {  // x: inclusive sums, w: what lane's row takes
        const unsigned beyond = __ballot_sync(FULL, x > off);
        const int at = beyond ? __ffs(beyond) - 1 : 31;
        off -= __shfl_sync(FULL, beyond ? x - w : x, at);
        b += beyond ? at : 32;
        return beyond != 0;
    };
    if (pv.batch <= 128) {
        const int each = (pv.batch + 31) / 32;
        int w[4], sum = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int r = lane * each + k;
            w[k] = k < each && r < pv.batch ? cost(r, status) : 0;
            sum += w[k];
        }
        const int x = inclusive(sum);
        cut(__shfl_sync(FULL, x, 31));
        if (left <= 0) return;
        const int at = __ffs(__ballot_sync(FULL, x > off)) - 1;
        off -= __shfl_sync(FULL, x - sum, at);
        b = at * each;
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const int wk = __shfl_sync(FULL, w[k], at);
            if (off < wk) break;
            off -= wk;
            b++;
        }
    } else {
        const int chunk = (pv.batch + SPLIT_THREADS - 1) / SPLIT_THREADS;
        const int r0 = min(pv.batch, (int)threadIdx.x * chunk), r1 = min(pv.batch, r0 + chunk);
        int x = 0;
        for (int r = r0; r < r1; r++) x += cost(r, status);
        x = inclusive(x);
        if (lane == 31) part[warp] = x;
        __syncthreads();
        for (int w = 0; w < warp; w++) x += part[w];
        reinterpret_cast<int*>(pre)[threadIdx.x] = x;
        __syncthreads();
        const int4 sums = pre[lane];  // of threads 4 lane .. 4 lane + 3
        cut(__shfl_sync(FULL, sums.w, 31));
        if (left <= 0) return;
        // threads whose sum does not pass the start lie before it
        const int before = (sums.x <= off) + (sums.y <= off) + (sums.z <= off) + (sums.w <= off);
        const int skip = __reduce_add_sync(FULL, before);
        b = skip * chunk;
        off -= skip ? reinterpret_cast<const int*>(pre)[skip - 1] : 0;
        if (chunk > 1) {
            while (true) {
                const int w = b + lane < pv.batch ? cost(b + lane, nullptr) : 0;
                if (among(inclusive(w), w)) break;
            }
        }
    }
    int item, place;
    {
        const uint32_t each = Span(row_length(pv, b, nullptr), window, sinks, TT).tiles + HEAD;
        item = (uint32_t)off / each;
        place = (uint32_t)off - item * each;
    }

    Stream<T, DP, NT, PART, SMALL> st;
    while (true) {
        const Span span(row_length(pv, b, nullptr), window, sinks, TT);
        if (span.tiles == 0) {  // an empty sequence (paged_join_kernel writes its output)
            b++;
            continue;
        }
        const int stop = min(span.tiles + HEAD, place + left);
        const int first = max(place - HEAD, 0), last = max(stop - HEAD, 0);
        const int bb = b, at = item;
        left -= stop - place;
        place = 0;
        if (++item == items) {
            item = 0;
            b++;
        }
        if (first < last) {
            const int h = at / gt, q0 = at % gt * QT;
            st.run(pv, q, c, span, bb, h, q0, first, last, qs + (S::WIDE ? warp * NT * S::KJ * 32 : 0), status);
            const bool whole = first == 0 && last == span.tiles;
            const int64_t slot = 2 * (int64_t)worker + (first == 0);
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int col = 8 * n + 2 * t4 + x;
                    if (q0 + col >= group) continue;
                    const float l = st.l[n][x], m = st.m[n][x];
                    const int64_t head = (int64_t)bb * pv.hq + h * group + q0 + col;
                    const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
                    if (g == 0) {
                        if (!whole)
                            *reinterpret_cast<float2*>(wk.ml + 2 * (slot * wk.rows + col)) = make_float2(m, l);
                        else if (lse)
                            lse[head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994530942f;
                    }
#pragma unroll
                    for (int vb = 0; vb < VB; vb++) {
                        const int d0 = (g + 8 * vb) * CH;
                        if (d0 >= pv.d) continue;
                        float v[CH];
                        st.values(n, x, vb, inv, v);
                        if (whole) {
                            *reinterpret_cast<uint4*>(out + head * pv.d + d0) = narrow16<T>(v);
                        } else {
                            float* dst = wk.o + (slot * wk.rows + col) * wk.dp + d0;
#pragma unroll
                            for (int k = 0; k < CH; k += 4)
                                *reinterpret_cast<float4*>(dst + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                        }
                    }
                }
            if (lane == 0) {
                int2* cut_at = wk.cut + (int64_t)bb * items + at;
                if (first == 0) cut_at->x = whole ? -1 : worker;
                if (last == span.tiles) cut_at->y = worker;
            }
        }
        if (left == 0) return;
    }
}

// Few short sequences: one cluster of blocks per item, its tiles divided among the cluster's warps and joined through
// the blocks' shared memory, so that the call is one launch and nothing goes through global memory in between. One
// sequence of 64 / 1024 tokens (6 heads x 64): 3.5 / 4.9 us, a launch and a chain of four dependent loads (cluster_size
// says when, with the list's times).
template <typename T, int DP, int NT, bool PART, bool SMALL, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, SplitShape<T, DP, NT>::BLOCKS * 4 / WARPS)
    paged_cluster_kernel(PageView pv, const T* q, float c, int window, int sinks, T* __restrict__ out,
                         float* __restrict__ lse, int* status) {
    using S = SplitShape<T, DP, NT>;
    constexpr int CH = S::CH, TT = S::TT, VB = S::VB, QT = S::QT, FOURS = DP / 4;
    __shared__ float4 so[WARPS][QT][FOURS];  // before it a warp's queries, in the wide shapes
    static_assert(!S::WIDE || sizeof(so[0]) >= NT * S::KJ * 32 * sizeof(uint4), "a warp's queries fit in its results");
    __shared__ float2 sml[WARPS][QT], joined[QT];
    grid_wait();
    grid_release();
    const int lane = lane_id(), warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    const int group = pv.hq / pv.hkv, gt = (group + QT - 1) / QT, items = pv.hkv * gt;
    uint32_t rank, size;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const int unit = blockIdx.x / size, b = unit / items, h = unit % items / gt, q0 = unit % items % gt * QT;
    const int cols = min(QT, group - q0);
    const Span span(row_length(pv, b, rank == 0 ? status : nullptr), window, sinks, TT);
    const int workers = size * WARPS, worker = rank * WARPS + warp;
    const int first = span.tiles * worker / workers, last = span.tiles * (worker + 1) / workers;
    if (first < last) {
        Stream<T, DP, NT, PART, SMALL> st;
        st.run(pv, q, c, span, b, h, q0, first, last, reinterpret_cast<uint4*>(so[warp]), status);
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int col = 8 * n + 2 * t4 + x;
                if (col >= cols) continue;
                if (g == 0) sml[warp][col] = make_float2(st.m[n][x], st.l[n][x]);
#pragma unroll
                for (int vb = 0; vb < VB; vb++) {
                    if (DP < 8 * CH && g * CH >= DP) continue;
                    float v[CH];
                    st.values(n, x, vb, 1.f, v);
#pragma unroll
                    for (int k = 0; k < CH; k += 4)
                        so[warp][col][((g + 8 * vb) * CH + k) / 4] = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                }
            }
    } else if (lane < QT) {
        sml[warp][lane] = make_float2(-INFINITY, 0.f);
    }
    __syncthreads();
    // pieces (maximum and sum ml(i), values o(i)) added up; those that saw nothing are not read
    auto add_up = [](int n, auto ml, auto o, float4& acc) {
        float m = -INFINITY, l = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < n; i++) m = fmaxf(m, ml(i).x);
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll 8
        for (int i = 0; i < n; i++) {
            const float2 p = ml(i);
            if (p.x == -INFINITY && p.y == 0.f) continue;
            const float e = ex2(p.x - base);
            const float4 v = o(i);
            l = fmaf(p.y, e, l);
            acc.x = fmaf(v.x, e, acc.x);
            acc.y = fmaf(v.y, e, acc.y);
            acc.z = fmaf(v.z, e, acc.z);
            acc.w = fmaf(v.w, e, acc.w);
        }
        return make_float2(m, l);
    };
    float4 acc;
    for (int e = threadIdx.x; e < cols * FOURS; e += WARPS * 32) {
        const int col = e / FOURS, f = e % FOURS;
        const float2 ml =
            add_up(WARPS, [&](int w) { return sml[w][col]; }, [&](int w) { return so[w][col][f]; }, acc);
        so[0][col][f] = acc;
        if (f == 0) joined[col] = ml;
    }
    cluster_sync();
    for (int e = rank * WARPS * 32 + threadIdx.x; e < cols * FOURS; e += size * WARPS * 32) {
        const int col = e / FOURS, f = e % FOURS;
        const float2 ml = add_up((int)size, [&](int r) { return of_block(&joined[col], r); },
                                 [&](int r) { return of_block(&so[0][col][f], r); }, acc);
        const int64_t head = (int64_t)b * pv.hq + h * group + q0 + col;
        const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
        if (4 * f < pv.d) {
            T* dst = out + head * pv.d + 4 * f;
            dst[0] = narrow<T>(acc.x * inv);
            dst[1] = narrow<T>(acc.y * inv);
            dst[2] = narrow<T>(acc.z * inv);
            dst[3] = narrow<T>(acc.w * inv);
        }
        if (lse && f == 0) lse[head] = ml.y == 0.f ? -INFINITY : (ml.x + log2f(ml.y)) * 0.69314718055994530942f;
    }
    cluster_sync();  // no block leaves while another reads its memory
}

// For each 32 columns of each (sequence, query head): the pieces of an item that was cut, each scaled to the largest
// maximum, in an order that only the lengths decide (the same sums on every run); rows that see nothing become 0.
// Eight lanes take a piece's 128 bytes, four pieces a warp go at a time and every lane has eight of them in flight:
// what this kernel costs is a chain of dependent loads (where the pieces are; the pieces), not their bytes. W warps
// share a head: all eight of a block where there are few heads with many pieces each, one where there are many
// (more blocks than fit at once would cost 1.5 us a wave: 37 us instead of 20 at 1024 heads).
template <typename T, int TT, int QT, int W>
__global__ void __launch_bounds__(JOIN_THREADS) paged_join_kernel(PageView pv, int window, int sinks, int columns,
                                                                  T* __restrict__ out, float* __restrict__ lse,
                                                                  SplitWork wk) {
    constexpr int SETS = 4 * W, U = 8, UNITS = JOIN_THREADS / 32 / W;
    grid_release();
    const int lane = lane_id(), warp = threadIdx.x / 32 % W;
    const uint32_t unit = blockIdx.x * UNITS + threadIdx.x / (32 * W);  // (sequence, query head, 32 columns)
    if (unit >= (uint32_t)pv.batch * pv.hq * columns) return;
    const int col = unit % columns, hq = unit / columns % pv.hq, b = unit / columns / pv.hq;
    const int group = pv.hq / pv.hkv, gt = (group + QT - 1) / QT, qi = hq % group;
    const int tiles = Span(row_length(pv, b, nullptr), window, sinks, TT).tiles;
    const int64_t head = (int64_t)b * pv.hq + hq;
    const int set = 4 * warp + lane / 8, x = col * 32 + lane % 8 * 4;
    T* dst = out + head * pv.d + x;
    const bool mine = set == 0 && x < pv.d, logs = lse && set == 0 && lane == 0 && col == 0;
    grid_wait();
    if (tiles == 0) {
        if (mine) dst[0] = dst[1] = dst[2] = dst[3] = narrow<T>(0.f);
        if (logs) lse[head] = -INFINITY;
        return;
    }
    const int2 cut = wk.cut[((int64_t)b * pv.hkv + hq / group) * gt + qi / QT];
    if (cut.x < 0) return;
    const int pieces = cut.y - cut.x + 1;
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float f, const float4& o) {
        acc.x = fmaf(o.x, f, acc.x);
        acc.y = fmaf(o.y, f, acc.y);
        acc.z = fmaf(o.z, f, acc.z);
        acc.w = fmaf(o.w, f, acc.w);
    };
    auto rescale = [&](float mn) {  // to the maximum mn; returns what is subtracted from exponents
        const float base = mn == -INFINITY ? 0.f : mn, a = ex2(m - base);
        l *= a;
        acc = make_float4(acc.x * a, acc.y * a, acc.z * a, acc.w * a);
        m = mn;
        return base;
    };
    for (int k0 = set; k0 < pieces; k0 += SETS * U) {
        float2 ml[U];
        float4 o[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = k0 + u * SETS;
            ml[u] = make_float2(-INFINITY, 0.f);
            o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k < pieces) {
                // the first piece is the last of its worker, the others the first of theirs
                const int64_t r = (int64_t)(2 * (cut.x + k) + (k == 0)) * wk.rows + qi % QT;
                ml[u] = *reinterpret_cast<const float2*>(wk.ml + 2 * r);
                o[u] = *reinterpret_cast<const float4*>(wk.o + r * wk.dp + x);  // columns past d are not stored
            }
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < U; u++) mn = fmaxf(mn, ml[u].x);
        const float base = rescale(mn);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float e = ex2(ml[u].x - base);
            l = fmaf(ml[u].y, e, l);
            add(e, o[u]);
        }
    }
    // the four sets of a warp, then the warps
    float mn = fmaxf(m, __shfl_xor_sync(FULL, m, 8));
    mn = fmaxf(mn, __shfl_xor_sync(FULL, mn, 16));
    rescale(mn);
#pragma unroll
    for (int w = 8; w < 32; w <<= 1) {
        l += __shfl_xor_sync(FULL, l, w);
        acc.x += __shfl_xor_sync(FULL, acc.x, w);
        acc.y += __shfl_xor_sync(FULL, acc.y, w);
        acc.z += __shfl_xor_sync(FULL, acc.z, w);
        acc.w += __shfl_xor_sync(FULL, acc.w, w);
    }
    if constexpr (W > 1) {
        __shared__ float2 sm[W];
        __shared__ float4 so[W][8];
        if (lane == 0) sm[warp] = make_float2(m, l);
        if (lane < 8) so[warp][lane] = acc;
        __syncthreads();
        if (set) return;
        mn = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; w++) mn = fmaxf(mn, sm[w].x);
        const float base = mn == -INFINITY ? 0.f : mn;
        l = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float e = ex2(sm[w].x - base);
            l = fmaf(sm[w].y, e, l);
            add(e, so[w][lane]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (mine) {
        dst[0] = narrow<T>(acc.x * inv);
        dst[1] = narrow<T>(acc.y * inv);
        dst[2] = narrow<T>(acc.z * inv);
        dst[3] = narrow<T>(acc.w * inv);
    }
    if (logs) lse[head] = l == 0.f ? -INFINITY : (mn + log2f(l)) * 0.69314718055994530942f;
}

// ---------------------------------------------------------------------------------------------------- append
// Rotary positions on the queries and keys of a fused projection, keys and values into their pages: every byte is read
// once and written once. A thread handles 16 bytes of a head's first half and the 16 bytes they are paired with in its
// second half (value i with i + d / 2), for U of a token's heads: those loads go out first, then the position, and
// from it the page and the cos and sin that the heads share. Nothing is exchanged between threads.
// Token t of row b is at position lengths[b] - T + t; a negative one is the padding before a shorter chunk, and with
// grown (or NULL) so are all but the row's last grown[b] tokens.
// Memory bounds it. 16 x 2048 tokens of 18 heads x 64, bf16: 29.7 us, 82% of the copy rate (heads a thread: two 31.3,
// three 30.3, four 35.2, six 30.8; blocks of 256 threads 30.6; a thread for each pair, with the block's positions looked
// up once into shared memory behind a barrier, 34.2); 3 x 777 tokens of 48 heads x 128, fp32: 17.4 us, 97%.
constexpr int APPEND_THREADS = 128, APPEND_HEADS = 3;

template <typename T, int U>
__global__ void __launch_bounds__(APPEND_THREADS)
    paged_append_kernel(PageView pv, const T* qkv, int tokens, const float* cosb, const float* sinb, int max_pos,
                        const int32_t* grown, T* __restrict__ q_out, int groups, int per_block, uint32_t all,
                        int* status) {
    constexpr int CH = 16 / sizeof(T);
    grid_wait();
    grid_release();
    const int half = pv.d / 2, lanes = half / CH, heads = pv.hq + 2 * pv.hkv, rot = pv.hq + pv.hkv;
    const int threads = lanes * groups, tk = threadIdx.x / threads;  // threads of a token
    const uint32_t token = blockIdx.x * per_block + tk;
    if (tk >= per_block || token >= all) return;
    const int r = threadIdx.x - tk * threads, g = r / lanes, c = (r - g * lanes) * CH;
    const T* src = qkv + (int64_t)token * heads * pv.d + c;
    uint4 xs[U], ys[U];
    float cs[CH], sn[CH];
    int state = 0, pos = 0;  // 1: stored, 0: only its queries, -1: beyond the rotary table, skipped
    int64_t k_at = 0, v_at = 0;
    for (int h0 = g; h0 < heads; h0 += U * groups) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int hd = h0 + u * groups;
            if (hd >= heads) break;
            xs[u] = load16(src + hd * pv.d);
            ys[u] = load16(src + hd * pv.d + half);
        }
        if (h0 == g) {
            const int b = token / (uint32_t)tokens, t = token - (uint32_t)b * tokens;
            pos = row_length(pv, b, status) - tokens + t;
            if (grown && tokens - t > grown[b]) pos = -1;
            if (pos >= 0) {
                const int page = page_of(pv, b, pos, status);
                if (cosb && pos < max_pos) {
                    const float* cp = cosb + (int64_t)pos * half + c;
                    const float* sp = sinb + (int64_t)pos * half + c;
#pragma unroll
                    for (int k = 0; k < CH; k += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(cp + k);
                        const float4 y = *reinterpret_cast<const float4*>(sp + k);
                        cs[k] = x.x, cs[k + 1] = x.y, cs[k + 2] = x.z, cs[k + 3] = x.w;
                        sn[k] = y.x, sn[k + 1] = y.y, sn[k + 2] = y.z, sn[k + 3] = y.w;
                    }
                }
                const int64_t slot = pos & ((1 << pv.page_shift) - 1);
                state = page >= 0;
                k_at = page * pv.kp + slot * pv.kt + c;
                v_at = page * pv.vp + slot * pv.vt + c;
                if (page < 0) flag(status, SMLM_FLAG_NO_PAGES);
                if (cosb && pos >= max_pos) {
                    flag(status, SMLM_FLAG_INDEX_RANGE);
                    state = -1;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int hd = h0 + u * groups;
            if (hd >= heads) break;
            uint4 xo = xs[u], yo = ys[u];
            T* dst;
            if (hd < pv.hq) {
                dst = q_out + ((int64_t)token * pv.hq + hd) * pv.d + c;
                if (pos < 0 || state < 0) xo = yo = make_uint4(0, 0, 0, 0);
            } else {
                if (state <= 0) continue;
                if (hd < rot) dst = static_cast<T*>(const_cast<void*>(pv.k)) + k_at + (hd - pv.hq) * pv.kh;
                else dst = static_cast<T*>(const_cast<void*>(pv.v)) + v_at + (hd - rot) * pv.vh;
            }
            if (cosb && hd < rot && pos >= 0 && state >= 0) {
                float x[CH], y[CH];
                widen16<T>(xo, x);
                widen16<T>(yo, y);
#pragma unroll
                for (int k = 0; k < CH; k++) {
                    const float e = x[k], f = y[k];
                    x[k] = e * cs[k] - f * sn[k];
                    y[k] = f * cs[k] + e * sn[k];
                }
                xo = narrow16<T>(x);
                yo = narrow16<T>(y);
            }
            *reinterpret_cast<uint4*>(dst) = xo;
            *reinterpret_cast<uint4*>(dst + half) = yo;
        }
    }
}

static int element_bytes(int dtype) { return dtype == SMLM_F32 ? 4 : 2; }

static int fill_view(PageView& pv, const char* what, const void* k, const void* v, int dtype, const int64_t* strides,
                     const int32_t* table, int64_t table_stride, const int32_t* lengths, int64_t batch, int64_t hq,
                     int64_t hkv, int64_t d, int64_t n_pages, int64_t page_size, int64_t max_blocks) {
    SMLM_CHECK_ARG(dtype == SMLM_F32 || dtype == SMLM_BF16 || dtype == SMLM_F16,
                   "%s: dtype %d (fp32, bf16 or fp16)", what, dtype);
    SMLM_CHECK_ARG(k && v && strides && table && lengths, "%s: null cache, table or lengths", what);
    SMLM_CHECK_ARG(batch >= 0 && batch <= 65535, "%s: batch %lld (at most 65535)", what, (long long)batch);
    SMLM_CHECK_ARG(hkv >= 1 && hq >= 1 && hq <= 4096 && hq % hkv == 0,
                   "%s: %lld query heads over %lld key heads (a multiple, at most 4096)", what, (long long)hq,
                   (long long)hkv);
    SMLM_CHECK_ARG(d >= 16 && d <= 256 && d % 16 == 0, "%s: head dimension %lld (a multiple of 16 up to 256)", what,
                   (long long)d);
    SMLM_CHECK_ARG(page_size >= 1 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
                   "%s: page_size %lld (a power of two up to 4096)", what, (long long)page_size);
    SMLM_CHECK_ARG(n_pages >= 1 && n_pages <= INT32_MAX && max_blocks >= 1 && table_stride >= max_blocks &&
                       max_blocks * page_size <= INT32_MAX / 2,
                   "%s: %lld pages, %lld table columns (stride %lld)", what, (long long)n_pages,
                   (long long)max_blocks, (long long)table_stride);
    const int es = element_bytes(dtype);
    for (int i = 0; i < 6; i++) {
        SMLM_CHECK_ARG(strides[i] >= 0 && strides[i] * es % 16 == 0,
                       "%s: page, head and token strides are multiples of 16 bytes", what);
        SMLM_CHECK_ARG(i % 3 == 1 || strides[i] <= UINT32_MAX / es, "%s: page and token strides below 4 GiB", what);
    }
    SMLM_CHECK_ARG(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "%s: the pages are not 16-byte aligned", what);
    pv = PageView{k, v, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], table, lengths,
                  table_stride, (int)batch, (int)hq, (int)hkv, (int)d, (int)n_pages, 0, (int)max_blocks};
    while ((1 << pv.page_shift) < page_size) pv.page_shift++;
    return SMLM_OK;
}

template <typename F>
static int by_dtype(int dtype, F f) {
    if (dtype == SMLM_F32) return f(float());
    if (dtype == SMLM_F16) return f(__half());
    return f(__nv_bfloat16());
}

static int64_t padded_d(int64_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256; }
// Two eights of query heads where a group has more than eight: each key and value is then read half as often. Rows of
// more than 256 bytes have no registers for it (and fp32 none from 64 on).
static int eights(int64_t group, int64_t dp, int64_t es) { return group > 8 && es == 2 && dp <= 128 ? 2 : 1; }
static int split_blocks(int64_t es, int64_t dp, int nt) { return es * dp * nt <= 128 ? 4 : es * dp * nt <= 256 ? 3 : 2; }

// Carves the workspace (sizes only without one).
template <typename W>
static void split_work(W& ws, SplitWork& wk, int64_t batch, int64_t hq, int64_t hkv, int64_t d, int64_t es) {
    const int64_t dp = padded_d(d), group = hq / std::max<int64_t>(hkv, 1);
    const int nt = eights(group, dp, es);
    const int64_t slots = 2 * (int64_t)sm_count() * split_blocks(es, dp, nt) * SPLIT_WARPS;
    const int64_t items = batch * hkv * ((group + 8 * nt - 1) / (8 * nt));
    wk.rows = (int)std::min<int64_t>(group, 8 * nt);
    wk.dp = (int)dp;
    const auto take = [&](auto*& p, int64_t n) {
        using E = std::remove_reference_t<decltype(*p)>;
        if constexpr (std::is_same_v<W, Workspace>) p = ws.template take<E>(n);
        else ws.template take<E>(n);
    };
    take(wk.cut, items);
    take(wk.ml, 2 * slots * wk.rows);
    take(wk.o, slots * wk.rows * dp);
}

// How many clusters of `size` blocks of the kernel run at once on the current device (asked once per kernel, size and
// device, and more than the portable eight blocks allowed then): fewer than the blocks that fit, because a cluster lies
// in one part of the card.
template <auto kernel, int WARPS>
static int64_t clusters_at_once(int size) {
    static std::atomic<int> known[64][17];  // the answer + 1
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (dev < 64) n = known[dev][size].load();
    if (n) return n - 1;
    if (size > 8 && cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(WARPS * 32);
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = size;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (dev < 64) known[dev][size].store(n + 1);
    return n;
}

// The blocks per item of paged_cluster_kernel, 0: the list and the join. A cluster is faster while its warps have a few
// tiles each and all clusters run at once. Measured, list and join -> clusters:
//   6 heads x 64: 1 x 64 tokens 6.3 -> 3.5 us, 1 x 1024 7.1 -> 4.9, 16 x 256 7.2 -> 5.3;
//   32 / 8 heads x 128: 4 x 2048 15.5 -> 12.0 (eight blocks, four tiles a warp), 16 x 512 13.0 -> 10.4 (three, 2.7);
//   in fives with 3.6 tiles 15.4 -> 15.2 for even sequences and 8.9 -> 10.6 for uneven ones (16 x up to 2304, 6 x 64):
//   the list evens out what the table could hold and the sequences do not;
//   more clusters than run at once 15.4 -> 22.5 (16 x 2304 in sixes).
// Up to six tiles a warp with a window, under which long sequences do the same work (64 x 1028 seen: 20.3 -> 17.3).
// Sixteen blocks find room slowly where several share an SM (fp32, 4 x 2048: 11.7 -> 17.5), so they are for calls of at
// most a block per SM, and then of eight warps for more tiles than 64 (1 x 2304: list 7.3, sixteen blocks of four warps
// 6.9, of eight 5.9; eight warps everywhere would cost 5% on average: 1 x 1024 4.9 -> 5.9).
struct Cluster {
    int size, warps;  // blocks per item (0: the list), warps of a block
};
template <typename V>
static Cluster cluster_size(const PageView& pv, int64_t window, int64_t sinks) {
    constexpr int QT = V::S::QT, TT = V::S::TT, MORE = V::S::MORE_WARPS, W = 4;
    int64_t most = (int64_t)pv.max_blocks << pv.page_shift;  // tokens that any sequence can see
    if (window) most = std::min(most, window + sinks + 2 * TT);
    const int64_t tiles = (most + TT - 1) / TT, items = (int64_t)pv.batch * pv.hkv * ((pv.hq / pv.hkv + QT - 1) / QT);
    const auto at_once = [](int size) { return clusters_at_once<V::cluster, W>(size); };
    if (tiles <= W) return {items <= 2 * at_once(1), W};  // blocks alone: two rounds are as fast
    if (tiles > 8 * W && items * 16 <= sm_count()) {
        if (tiles <= 16 * W && items <= at_once(16)) return {16, W};
        if (tiles <= 16 * MORE * 2 && items <= clusters_at_once<V::cluster_more, MORE>(16)) return {16, MORE};
    }
    for (int size = (int)std::min<int64_t>(8, (tiles + W - 1) / W); size >= 1; size--) {
        if (tiles > size * W * (window ? 6 : size == 8 ? 4 : 3)) break;
        if (items <= at_once(size)) return {size, W};
    }
    return {0, W};
}

// The kernels' template arguments for a call.
template <typename T_, int DP_, int NT_, bool PART_, bool SMALL_>
struct Variant {
    using T = T_;
    using S = SplitShape<T_, DP_, NT_>;
    static constexpr int DP = DP_, NT = NT_;
    static constexpr auto cluster = paged_cluster_kernel<T_, DP_, NT_, PART_, SMALL_, 4>;
    static constexpr auto cluster_more = paged_cluster_kernel<T_, DP_, NT_, PART_, SMALL_, S::MORE_WARPS>;
    static constexpr auto split = paged_split_kernel<T_, DP_, NT_, PART_, SMALL_>;
};

template <typename F>
static int with_variant(const PageView& pv, int dtype, F f) {
    return by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        const auto of = [&](auto dp, auto nt) {
            constexpr int DP = decltype(dp)::value, NT = decltype(nt)::value;
            if (pv.page_shift < 4) return f(Variant<T, DP, NT, true, true>());
            if (pv.d < DP) return f(Variant<T, DP, NT, true, false>());
            return f(Variant<T, DP, NT, false, false>());
        };
        const auto go = [&](auto dp) {
            if constexpr (sizeof(T) == 2 && decltype(dp)::value <= 128)
                if (eights(pv.hq / pv.hkv, decltype(dp)::value, sizeof(T)) == 2)
                    return of(dp, std::integral_constant<int, 2>());
            return of(dp, std::integral_constant<int, 1>());
        };
        if (pv.d <= 32) return go(std::integral_constant<int, 32>());
        if (pv.d <= 64) return go(std::integral_constant<int, 64>());
        if (pv.d <= 128) return go(std::integral_constant<int, 128>());
        return go(std::integral_constant<int, 256>());
    });
}

struct AttentionArgs {
    const void* q;
    float scale;
    int window, sinks;
    void* out;
    float* lse;
    int* status;
    cudaStream_t st;
};

template <typename V>
static int launch_cluster(V, const PageView& pv, const Cluster& c, const AttentionArgs& a) {
    using T = typename V::T;
    const int64_t items = (int64_t)pv.batch * pv.hkv * ((pv.hq / pv.hkv + V::S::QT - 1) / V::S::QT);
    return launch_dependent(c.warps == 4 ? V::cluster : V::cluster_more, "paged_attention", c.size, c.size * items,
                            c.warps * 32, a.st, pv,
                            static_cast<const T*>(a.q), a.scale * 1.4426950408889634074f, a.window, a.sinks,
                            static_cast<T*>(a.out), a.lse, a.status);
}

template <typename V>
static int launch_list(V, const PageView& pv, const SplitWork& wk, const AttentionArgs& a) {
    using T = typename V::T;
    using S = typename V::S;
    const int blocks = sm_count() * S::BLOCKS;
    const int rc = launch_dependent(V::split, "paged_attention", 1, blocks, SPLIT_THREADS, a.st, pv,
                                    static_cast<const T*>(a.q), a.scale * 1.4426950408889634074f, a.window, a.sinks,
                                    static_cast<T*>(a.out), a.lse, wk, a.status);
    if (rc != SMLM_OK) return rc;
    const int columns = (pv.d + 31) / 32;
    const int64_t units = (int64_t)pv.batch * pv.hq * columns;
    const int64_t items = (int64_t)pv.batch * pv.hkv * ((pv.hq / pv.hkv + S::QT - 1) / S::QT);
    const bool shared = (int64_t)blocks * SPLIT_WARPS > 32 * items;  // over 32 pieces an item: a block for each
    return launch_dependent(shared ? paged_join_kernel<T, S::TT, S::QT, 8> : paged_join_kernel<T, S::TT, S::QT, 1>,
                            "paged_attention: join", 1, shared ? units : (units + 7) / 8, JOIN_THREADS, a.st, pv,
                            a.window, a.sinks, columns, static_cast<T*>(a.out), a.lse, wk);
}

static int clamp_window(int64_t window) { return (int)std::min<int64_t>(window, INT32_MAX); }
static int clamp_sinks(int64_t sinks) { return (int)std::min<int64_t>(sinks, INT32_MAX / 2); }

}  // namespace smlm

using namespace smlm;

extern "C" size_t smlm_paged_attention_workspace(int64_t batch, int64_t hq, int64_t hkv, int64_t d, int dtype,
                                                 int64_t page_size, int64_t max_blocks, int64_t window, int64_t sinks) {
    // (any addresses: the checks look at them, nothing is read)
    static const int64_t strides[6] = {};
    void* some = reinterpret_cast<void*>(uintptr_t(16));
    PageView pv;
    if (batch <= 0 || window < 0 || sinks < 0 ||
        fill_view(pv, "paged_attention", some, some, dtype, strides, static_cast<int32_t*>(some), max_blocks,
                  static_cast<int32_t*>(some), batch, hq, hkv, d, 1, page_size, max_blocks) != SMLM_OK)
        return 0;
    const int win = clamp_window(window), snk = clamp_sinks(sinks);
    if (with_variant(pv, dtype, [&](auto v) {
            using V = decltype(v);
            return cluster_size<V>(pv, win, snk).size;
        }))
        return 0;
    WorkspaceSize ws;
    SplitWork wk;
    split_work(ws, wk, batch, hq, hkv, d, element_bytes(dtype));
    return ws.used;
}

extern "C" int smlm_paged_attention(const void* q, const void* k_pages, const void* v_pages, int dtype,
                                    const int64_t* strides, const int32_t* table, int64_t table_stride,
                                    const int32_t* lengths, int64_t batch, int64_t hq, int64_t hkv, int64_t d,
                                    int64_t n_pages, int64_t page_size, int64_t max_blocks, float scale, int64_t window,
                                    int64_t sinks, void* out, float* lse, void* workspace, size_t workspace_bytes,
                                    int* status, void* stream) {
    if (batch == 0) return SMLM_OK;
    PageView pv;
    const int rc = fill_view(pv, "paged_attention", k_pages, v_pages, dtype, strides, table, table_stride, lengths,
                             batch, hq, hkv, d, n_pages, page_size, max_blocks);
    if (rc != SMLM_OK) return rc;
    SMLM_CHECK_ARG(q && out && ((uintptr_t)q | (uintptr_t)out) % 16 == 0,
                   "paged_attention: q and out have to be 16-byte aligned");
    SMLM_CHECK_ARG(window >= 0 && sinks >= 0, "paged_attention: window %lld, sinks %lld", (long long)window,
                   (long long)sinks);
    const AttentionArgs args{q, scale, clamp_window(window), clamp_sinks(sinks), out, lse, status, as_stream(stream)};
    return with_variant(pv, dtype, [&](auto v) {
        using V = decltype(v);
        const Cluster c = cluster_size<V>(pv, args.window, args.sinks);
        if (c.size) return launch_cluster(v, pv, c, args);
        // the list of tiles is counted in 31 bits
        constexpr int TT = V::S::TT, QT = V::S::QT;
        const int64_t items = batch * hkv * ((hq / hkv + QT - 1) / QT);
        int64_t tiles = (max_blocks * page_size + TT - 1) / TT;
        if (args.window) tiles = std::min<int64_t>(tiles, args.window / TT + args.sinks / TT + 3);  // Span's at most
        SMLM_CHECK_ARG(items * (tiles + HEAD) <= INT32_MAX,
                       "paged_attention: %lld sequences x %lld heads x up to %lld tokens: fewer rows a call",
                       (long long)batch, (long long)hq, (long long)(max_blocks * page_size));
        Workspace ws(workspace, workspace_bytes);
        SplitWork wk;
        split_work(ws, wk, batch, hq, hkv, d, element_bytes(dtype));
        if (!workspace || !ws.ok()) {
            set_error("paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes, ws.used);
            return SMLM_ERR_WORKSPACE;
        }
        return launch_list(v, pv, wk, args);
    });
}

extern "C" int smlm_paged_append_grown(const void* qkv, void* k_pages, void* v_pages, int dtype, const int64_t* strides,
                                       const int32_t* table, int64_t table_stride, const int32_t* lengths, int64_t batch,
                                       int64_t tokens, int64_t hq, int64_t hkv, int64_t d, int64_t n_pages,
                                       int64_t page_size, int64_t max_blocks, const float* cos, const float* sin,
                                       int64_t max_pos, const int32_t* grown, void* q_out, int* status, void* stream) {
    if (batch == 0 || tokens == 0) return SMLM_OK;
    PageView pv;
    const int rc = fill_view(pv, "paged_append", k_pages, v_pages, dtype, strides, table, table_stride, lengths, batch,
                             hq, hkv, d, n_pages, page_size, max_blocks);
    if (rc != SMLM_OK) return rc;
    SMLM_CHECK_ARG(tokens > 0 && tokens <= INT32_MAX / 2, "paged_append: %lld tokens", (long long)tokens);
    SMLM_CHECK_ARG(qkv && q_out && ((uintptr_t)qkv | (uintptr_t)q_out) % 16 == 0,
                   "paged_append: qkv and the query output have to be 16-byte aligned");
    SMLM_CHECK_ARG((cos == nullptr) == (sin == nullptr) && (!cos || max_pos > 0),
                   "paged_append: cos and sin come together");
    SMLM_CHECK_ARG(!cos || ((uintptr_t)cos | (uintptr_t)sin) % 16 == 0, "paged_append: cos and sin have to be 16-byte "
                   "aligned");
    // A few tokens: a thread a head (a decoding step's time is one token's); many: several heads a thread.
    const int64_t all = batch * tokens, heads = hq + 2 * hkv, lanes = d / 2 * element_bytes(dtype) / 16;
    const int64_t each = all * heads * lanes < (int64_t)sm_count() * APPEND_THREADS * 4 ? 1 : APPEND_HEADS;
    const int64_t groups = std::min<int64_t>((heads + each - 1) / each, APPEND_THREADS / lanes);
    const int64_t fill = APPEND_THREADS / (lanes * groups);
    const int64_t per_block = each == 1 ? std::min<int64_t>(fill, std::max<int64_t>(1, all / (sm_count() * 4))) : fill;
    const int64_t grid = (all + per_block - 1) / per_block;
    SMLM_CHECK_ARG(all <= INT32_MAX && heads * d <= (1 << 20),
                   "paged_append: %lld tokens of %lld values (at most 2^31 - 1 of 2^20)", (long long)all,
                   (long long)(heads * d));
    return by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return launch_dependent(each == 1 ? paged_append_kernel<T, 1> : paged_append_kernel<T, APPEND_HEADS>,
                                "paged_append", 1, grid, APPEND_THREADS, as_stream(stream), pv,
                                static_cast<const T*>(qkv), (int)tokens, cos, sin,
                                (int)std::min<int64_t>(max_pos, INT32_MAX), grown, static_cast<T*>(q_out), (int)groups,
                                (int)per_block, (uint32_t)all, status);
    });
}

extern "C" int smlm_paged_append(const void* qkv, void* k_pages, void* v_pages, int dtype, const int64_t* strides,
                                 const int32_t* table, int64_t table_stride, const int32_t* lengths, int64_t batch,
                                 int64_t tokens, int64_t hq, int64_t hkv, int64_t d, int64_t n_pages, int64_t page_size,
                                 int64_t max_blocks, const float* cos, const float* sin, int64_t max_pos, void* q_out,
                                 int* status, void* stream) {
    return smlm_paged_append_grown(qkv, k_pages, v_pages, dtype, strides, table, table_stride, lengths, batch, tokens, hq,
                                   hkv, d, n_pages, page_size, max_blocks, cos, sin, max_pos, nullptr, q_out, status,
                                   stream);
}
