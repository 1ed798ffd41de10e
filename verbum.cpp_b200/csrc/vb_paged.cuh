// vb_paged.cuh -- what the paged-cache kernels share: the device view of a
// page pool and a ragged batch, the search for a row's sequence, and the
// checks that keep every access inside the pool.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>

#include "vb_common.cuh"

namespace vb {

struct PagedView {
    const char* k;
    const char* v;
    int num_pages, page_size, kv_heads;
    int page_shift;  // log2(page_size), or -1
    int64_t stride_page, stride_pos, stride_head;  // bytes
    int batch, tokens, max_new, max_len;
    const int* q_start;
    const int* lens;
    const int* table;
    int table_stride;
    int* status;
};

// Sizes in bytes of VB_F32 / VB_F16 / VB_BF16; 0 for anything else.
inline int paged_elem_bytes(int dtype) { return dtype == VB_F32 ? 4 : dtype == VB_F16 || dtype == VB_BF16 ? 2 : 0; }

// Checks of what the host can see; fills the view (vb_paged_attn.cu).
vb_status paged_view(const vb_paged_cache* cache, const vb_paged_batch* batch, int io, int heads, const char* who,
                     PagedView* out);
inline bool paged_words(std::initializer_list<const void*> p) {  // addresses (or NULL) of 4-byte elements
    uintptr_t bits = 0;
    for (const void* x : p) bits |= reinterpret_cast<uintptr_t>(x);
    return (bits & 3u) == 0;
}
inline bool paged_aligned(const void* p, int64_t row, int64_t head, int elem) {
    return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(row * elem) | (uintptr_t)(head * elem)) & 15u) == 0;
}

#ifdef __CUDACC__
__device__ __forceinline__ void paged_report(const PagedView& p, int bit) {
    if (p.status) atomicOr(p.status, bit);
}

// The last sequence whose rows start at or before t (the one that holds row t
// when the starts ascend), found by the whole warp: 32 probes a step.
__device__ __forceinline__ int paged_find_seq(const int* q_start, int batch, int t, int lane) {
    int lo = 0, hi = batch;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) >> 5;
        const int at = lo + lane * step;
        const bool below = at < hi && q_start[at] <= t;
        const int c = __popc(__ballot_sync(0xffffffffu, below));
        lo += (c > 0 ? c - 1 : 0) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// Rows and length of sequence b after the checks the interface promises.
struct PagedSeq {
    int start, n, len;
    bool ok;  // its rows can be computed
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedView& p, int b) {
    PagedSeq s;
    s.start = p.q_start[b];
    const int end = p.q_start[b + 1];
    s.len = p.lens[b];
    s.ok = s.start >= 0 && end >= s.start && end <= p.tokens && end - s.start <= p.max_new;
    s.n = s.ok ? end - s.start : 0;
    if (!s.ok) paged_report(p, VB_PAGED_BAD_ROWS);
    if (s.len < 0 || s.len > p.max_len) {
        paged_report(p, VB_PAGED_BAD_LEN);
        s.len = 0;
    }
    return s;
}

__device__ __forceinline__ int paged_page_of(const PagedView& p, int pos) {
    return p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
}

// Byte offset of (position pos of sequence b, KV head 0); -1 for a bad page.
// 0 <= pos < the sequence's checked length, so the table entry exists.
__device__ __forceinline__ int64_t paged_offset(const PagedView& p, int b, int pos) {
    const int pg = paged_page_of(p, pos);
    const int id = p.table[(size_t)b * p.table_stride + pg];
    if ((unsigned)id >= (unsigned)p.num_pages) {
        paged_report(p, VB_PAGED_BAD_PAGE);
        return -1;
    }
    return (int64_t)id * p.stride_page + (int64_t)(pos - pg * p.page_size) * p.stride_pos;
}

// Eight elements at once: 16 bytes of a 16-bit type, 32 of f32.
template <typename T>
struct Eight;
template <>
struct Eight<float> {
    static __device__ __forceinline__ void load(const void* p, float* x) {
        const float4 a = static_cast<const float4*>(p)[0], b = static_cast<const float4*>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
        x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    }
    static __device__ __forceinline__ void store(void* p, const float* x) {
        static_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        static_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
};
template <>
struct Eight<__half> {
    static __device__ __forceinline__ void load(const void* p, float* x) {
        const uint4 u = *static_cast<const uint4*>(p);
        const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(h[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void store(void* p, const float* x) {
        uint4 u;
        __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        *static_cast<uint4*>(p) = u;
    }
};
template <>
struct Eight<__nv_bfloat16> {
    static __device__ __forceinline__ void load(const void* p, float* x) {
        const uint4 u = *static_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void store(void* p, const float* x) {
        uint4 u;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        *static_cast<uint4*>(p) = u;
    }
};
#endif  // __CUDACC__

}  // namespace vb
