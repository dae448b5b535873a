// Shared by the paged key-value cache kernels (paged_attn.cu, pages.cu): the shape of a cache as kernels see it.
#pragma once

#include "common.cuh"

namespace smlm {

// Programmatic dependent launch: a kernel that was launched while its predecessor runs waits for that one's end and
// memory before it touches anything the predecessor wrote; grid_release lets the successor be launched. What a kernel
// reads may thus be written while it already runs (before grid_wait returns), so no load here is a non-coherent one.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;"); }

// Barrier of the blocks of a cluster; what a block wrote before it is seen by the others after it.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Launches while the stream's previous kernel may still run (the kernel calls grid_wait before anything else), in
// clusters of `cluster` blocks.
template <typename... P, typename... A>
inline int launch_dependent(void (*kernel)(P...), const char* what, int cluster, int64_t grid, int threads,
                            cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    return e == cudaSuccess ? SMLM_OK : cuda_status(e, what);
}

// One layer's pages. Token t of a sequence lies in page table[row][t >> page_shift], slot t & (page - 1); its key of
// head h starts at k + page * kp + h * kh + slot * kt (64-bit element offsets: a long cache passes 2^31 elements).
struct PageView {
    const void* k;
    const void* v;
    int64_t kp, kh, kt, vp, vh, vt;
    const int32_t* table;
    const int32_t* lengths;
    int64_t table_stride;
    int batch, hq, hkv, d, n_pages, page_shift, max_blocks;
};

// Tokens of row b. A length outside the table is flagged and the row left out, as if it were empty: a length cut to the
// table's end would place an append on the tokens that are there.
__device__ __forceinline__ int row_length(const PageView& pv, int b, int* status) {
    const int n = pv.lengths[b];
    if (n < 0 || n > (int64_t)pv.max_blocks << pv.page_shift) {
        flag(status, SMLM_FLAG_INDEX_RANGE);
        return 0;
    }
    return n;
}

// The page that holds token t of row b, or -1: a hole (entry -1) or an entry outside the pool (flagged).
__device__ __forceinline__ int page_of(const PageView& pv, int b, int t, int* status) {
    const int p = pv.table[b * pv.table_stride + (t >> pv.page_shift)];
    if (p >= pv.n_pages) {
        flag(status, SMLM_FLAG_INDEX_RANGE);
        return -1;
    }
    return p < 0 ? -1 : p;
}

template <typename T>
__device__ __forceinline__ float widen(T x) {
    if constexpr (std::is_same_v<T, float>) return x;
    else if constexpr (std::is_same_v<T, __half>) return __half2float(x);
    else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T narrow(float x) {
    if constexpr (std::is_same_v<T, float>) return x;
    else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}

}  // namespace smlm
