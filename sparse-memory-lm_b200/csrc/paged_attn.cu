// Attention of one new token per sequence over a paged key-value cache, and the append that fills it.
#include "paged.cuh"

namespace smlm {

// One warp's share of one (sequence, query head): tokens warp, warp + WARPS, ...; the four warps' running maxima,
// sums and outputs are joined at the end.
template <typename T>
__global__ void __launch_bounds__(128) paged_attention_kernel(PageView pv, const T* q, float scale, int window,
                                                              int sinks, T* out, float* lse, int* status) {
    constexpr int WARPS = 4, PER = 8;  // d <= 256: at most 8 values per lane
    const int b = blockIdx.y, hq = blockIdx.x, h = hq / (pv.hq / pv.hkv);
    const int lane = lane_id(), warp = threadIdx.x >> 5;
    const int n = row_length(pv, b, status);
    const int first = window ? max(n - window, 0) : 0;
    float qv[PER], acc[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int c = lane + 32 * i;
        qv[i] = c < pv.d ? widen(q[((int64_t)b * pv.hq + hq) * pv.d + c]) * scale : 0.f;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int t = warp; t < n; t += WARPS) {
        if (t < first && t >= sinks) continue;
        const int p = page_of(pv, b, t, status);
        if (p < 0) continue;
        const int slot = t & ((1 << pv.page_shift) - 1);
        const T* k = static_cast<const T*>(pv.k) + p * pv.kp + h * pv.kh + slot * pv.kt;
        const T* v = static_cast<const T*>(pv.v) + p * pv.vp + h * pv.vh + slot * pv.vt;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane + 32 * i < pv.d) s += qv[i] * widen(k[lane + 32 * i]);
        s = warp_sum(s);
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
        const float c = expf(m - base), e = expf(s - base);
        l = l * c + e;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane + 32 * i < pv.d) acc[i] = acc[i] * c + e * widen(v[lane + 32 * i]);
        m = mn;
    }
    __shared__ float sm[WARPS], sl[WARPS], so[WARPS][256];
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) so[warp][lane + 32 * i] = acc[i];
    __syncthreads();
    float mx = -INFINITY, sum = 0.f;
    for (int w = 0; w < WARPS; w++) mx = fmaxf(mx, sm[w]);
    const float base = mx == -INFINITY ? 0.f : mx;
    for (int w = 0; w < WARPS; w++) sum += sl[w] * expf(sm[w] - base);
    for (int c = threadIdx.x; c < pv.d; c += 128) {
        float o = 0.f;
        for (int w = 0; w < WARPS; w++) o += so[w][c] * expf(sm[w] - base);
        out[((int64_t)b * pv.hq + hq) * pv.d + c] = narrow<T>(sum == 0.f ? 0.f : o / sum);
    }
    if (lse && threadIdx.x == 0) lse[(int64_t)b * pv.hq + hq] = sum == 0.f ? -INFINITY : mx + logf(sum);
}

// Rotary positions on the queries and keys of a fused projection, keys and values into their pages. One thread per
// pair (i, i + d / 2) of one head of one token; token t of row b is at position lengths[b] - T + t (negative: the
// padding before a shorter chunk, whose queries become 0).
template <typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(PageView pv, const T* qkv, int tokens, const float* cosb,
                                                           const float* sinb, int max_pos, T* q_out, int* status) {
    const int heads = pv.hq + 2 * pv.hkv, half = pv.d / 2;
    const int64_t all = (int64_t)pv.batch * tokens * heads * half;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        const int c = i % half, hd = (i / half) % heads;
        const int64_t tok = i / ((int64_t)half * heads);
        const int b = tok / tokens, t = tok % tokens;
        const int pos = row_length(pv, b, status) - tokens + t;
        const T* src = qkv + (tok * heads + hd) * pv.d;
        float x = widen(src[c]), y = widen(src[c + half]);
        if (hd < pv.hq + pv.hkv && cosb && pos >= 0) {
            if (pos >= max_pos) {
                flag(status, SMLM_FLAG_INDEX_RANGE);
                continue;
            }
            const float co = cosb[(int64_t)pos * half + c], si = sinb[(int64_t)pos * half + c];
            const float a = x;
            x = a * co - y * si;
            y = y * co + a * si;
        }
        T* dst;
        if (hd < pv.hq) {
            dst = q_out + (tok * pv.hq + hd) * pv.d;
            if (pos < 0) x = y = 0.f;
        } else {
            if (pos < 0) continue;
            const int p = page_of(pv, b, pos, status);
            if (p < 0) {
                flag(status, SMLM_FLAG_NO_PAGES);
                continue;
            }
            const int slot = pos & ((1 << pv.page_shift) - 1);
            if (hd < pv.hq + pv.hkv)
                dst = static_cast<T*>(const_cast<void*>(pv.k)) + p * pv.kp + (hd - pv.hq) * pv.kh + slot * pv.kt;
            else
                dst = static_cast<T*>(const_cast<void*>(pv.v)) + p * pv.vp + (hd - pv.hq - pv.hkv) * pv.vh +
                      slot * pv.vt;
        }
        dst[c] = narrow<T>(x);
        dst[c + half] = narrow<T>(y);
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
    for (int i = 0; i < 6; i++)
        SMLM_CHECK_ARG(strides[i] >= 0 && strides[i] * es % 16 == 0,
                       "%s: page, head and token strides are multiples of 16 bytes", what);
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

}  // namespace smlm

using namespace smlm;

extern "C" size_t smlm_paged_attention_workspace(int64_t batch, int64_t hq, int64_t d) { return 0; }

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
    const int win = (int)std::min<int64_t>(window, INT32_MAX), snk = (int)std::min<int64_t>(sinks, INT32_MAX);
    return by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        paged_attention_kernel<T><<<dim3(hq, batch), 128, 0, as_stream(stream)>>>(
            pv, static_cast<const T*>(q), scale, win, snk, static_cast<T*>(out), lse, status);
        SMLM_LAUNCHED("paged_attention");
        return SMLM_OK;
    });
}

extern "C" int smlm_paged_append(const void* qkv, void* k_pages, void* v_pages, int dtype, const int64_t* strides,
                                 const int32_t* table, int64_t table_stride, const int32_t* lengths, int64_t batch,
                                 int64_t tokens, int64_t hq, int64_t hkv, int64_t d, int64_t n_pages, int64_t page_size,
                                 int64_t max_blocks, const float* cos, const float* sin, int64_t max_pos, void* q_out,
                                 int* status, void* stream) {
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
    const int64_t all = batch * tokens * (hq + 2 * hkv) * (d / 2);
    const int grid = (int)std::min<int64_t>((all + 255) / 256, (int64_t)sm_count() * 32);
    return by_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        paged_append_kernel<T><<<grid, 256, 0, as_stream(stream)>>>(
            pv, static_cast<const T*>(qkv), (int)tokens, cos, sin, (int)std::min<int64_t>(max_pos, INT32_MAX),
            static_cast<T*>(q_out), status);
        SMLM_LAUNCHED("paged_append");
        return SMLM_OK;
    });
}
