// vb_logits.cu -- penalties for repeated tokens, biases and grammar masks on
// the logits a sampler reads (Sampler::sample, generate.cpp:197-252, takes the
// raw row; this runs before it).
//
// Bound by memory: a logit is read once and written once.  A CTA owns a slice
// of one row's vocabulary.  Its logits are requested first; while they are on
// their way it counts, in shared memory, how often the slice's tokens stand in
// the row's history (integer atomics: their order changes nothing) and sums
// the slice's biases (a token's biases always by the same warp and in the
// order of the list, so the sum is the same every time).
// 64 rows of 151,936 f32 logits: 26.4 us with histories of up to 4096 tokens, 64
// biases and masks (3.0 TB/s, 0.46 of the measured copy rate), 16 without rules: what
// is between is instructions, the history above all, which each of a row's 38 CTAs
// scans.
#include "vb_kernels.cuh"
#include "vb_paged.cuh"

namespace vb {
namespace {

constexpr int kLgThreads = 256;
constexpr int kLgSlice = 16 * kLgThreads;  // tokens of a CTA: 16 values in each thread's registers

struct LogitsArgs {
    const char* in;
    char* out;
    int64_t stride_in, stride_out;  // bytes
    int64_t vocab;
    int slices;
    vb_logits_rules r;
};

__device__ __forceinline__ float lg_load(const float* p) { return *p; }
__device__ __forceinline__ float lg_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float lg_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void lg_store(float* p, float x) { *p = x; }
__device__ __forceinline__ void lg_store(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void lg_store(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// Lists [start[r], start[r + 1]) kept within 0..total.
__device__ __forceinline__ void lg_range(const int* start, int64_t total, int row, int& lo, int& hi) {
    const int top = (int)min(total, (int64_t)0x7fffffff);
    lo = min(max(start[row], 0), top);
    hi = min(max(start[row + 1], lo), top);
}

// The rules of one row.
struct RowRules {
    float rep, freq, pres;
    bool has_rep;
};
// c: top bit set where the token stands in the prompt, the rest its count behind it
__device__ __forceinline__ float lg_penalty(const RowRules& w, float x, uint32_t c) {
    if (w.has_rep) x = x > 0.f ? __fdiv_rn(x, w.rep) : __fmul_rn(x, w.rep);
    const uint32_t n = c & 0x7fffffffu;
    if (n) x = __fsub_rn(__fsub_rn(x, __fmul_rn(w.freq, (float)n)), w.pres);
    return x;
}

template <typename T>
__global__ void __launch_bounds__(kLgThreads) logits_process_kernel(const __grid_constant__ LogitsArgs a) {
    constexpr int E = 16 / (int)sizeof(T);  // logits of a 16-byte access
    constexpr int NV = 16 / E;              // accesses of a thread
    // by token of the slice, moved so that an access's tokens start at a multiple of 4
    __shared__ __align__(16) uint32_t seen[kLgSlice + E];
    __shared__ __align__(16) float bias[kLgSlice + E];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int row = blockIdx.x / a.slices;
    const int v0 = (int)(blockIdx.x % a.slices) * kLgSlice;
    const int n = (int)min((int64_t)kLgSlice, a.vocab - v0);
    const T* in = reinterpret_cast<const T*>(a.in + row * a.stride_in) + v0;
    T* out = reinterpret_cast<T*>(a.out + row * a.stride_out) + v0;
    // tokens before the first 16-byte boundary; all of them where the two rows' boundaries differ
    const uintptr_t mis = reinterpret_cast<uintptr_t>(in) & 15u;
    const bool wide = mis == (reinterpret_cast<uintptr_t>(out) & 15u);
    const int head = wide ? min(n, (int)((16u - mis) & 15u) / (int)sizeof(T)) : n;
    const int vecs = (n - head) / E, tail = head + vecs * E;
    const int shift = (E - head % E) % E;
    uint4 x[NV];
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (k * kLgThreads + t < vecs) x[k] = reinterpret_cast<const uint4*>(in + head)[k * kLgThreads + t];

    const uint32_t* mask = a.r.mask ? a.r.mask + row * a.r.mask_stride : nullptr;
    // the words with the bits of each access's tokens: one, or two (shifted where they are used:
    // here the shift would wait for them)
    uint32_t lo[NV], hi[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int j = k * kLgThreads + t, tok = v0 + head + j * E;
        const bool real = mask && j < vecs;
        lo[k] = real ? mask[tok >> 5] : 0u;
        hi[k] = real && (tok & 31) > 32 - E ? mask[(tok >> 5) + 1] : 0u;
    }
    int h0 = 0, h1 = 0, b0 = 0, b1 = 0;
    if (a.r.hist_start) lg_range(a.r.hist_start, a.r.hist_total, row, h0, h1);
    if (a.r.bias_start) lg_range(a.r.bias_start, a.r.bias_total, row, b0, b1);
    const bool count = h1 > h0, add = b1 > b0;
    // the first of the history, too, before the shared memory is ready for it
    constexpr int NH = 4;
    int id[NH];
#pragma unroll
    for (int k = 0; k < NH; k++) {
        const int i = h0 + k * kLgThreads + t;
        id[k] = i < h1 ? a.r.hist_ids[i] : -1;
    }
    int tok0 = b0 + lane < b1 ? a.r.bias_ids[b0 + lane] : -1;  // and of the biases
    RowRules w{1.f, 0.f, 0.f, false};
    if (count) {
        w.has_rep = a.r.repetition != nullptr;
        w.rep = w.has_rep ? a.r.repetition[row] : 1.f;
        w.freq = a.r.frequency ? a.r.frequency[row] : 0.f;
        w.pres = a.r.presence ? a.r.presence[row] : 0.f;
        for (int i = t; i < (kLgSlice + E) / 4; i += kLgThreads) reinterpret_cast<uint4*>(seen)[i] = make_uint4(0, 0, 0, 0);
    }
    if (add)
        for (int i = t; i < (kLgSlice + E) / 4; i += kLgThreads)
            reinterpret_cast<float4*>(bias)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    __syncthreads();
    if (count) {
        const int answer = h0 + (a.r.prompt_len ? min(max(a.r.prompt_len[row], 0), h1 - h0) : 0);
        for (int i0 = h0; i0 < h1; i0 += NH * kLgThreads) {
            int next[NH];
#pragma unroll
            for (int k = 0; k < NH; k++) {
                const int i = i0 + (NH + k) * kLgThreads + t;
                next[k] = i < h1 ? a.r.hist_ids[i] : -1;
            }
#pragma unroll
            for (int k = 0; k < NH; k++) {
                const unsigned at = (unsigned)id[k] - (unsigned)v0;  // (an id of -1 is at no slice)
                if (id[k] >= 0 && at < (unsigned)n) {
                    if (i0 + k * kLgThreads + t < answer)
                        atomicOr(&seen[at + shift], 0x80000000u);
                    else
                        atomicAdd(&seen[at + shift], 1u);
                }
                id[k] = next[k];
            }
        }
    }
    if (add) {
        // warp w sums the tokens whose number in the slice is w mod 8
        for (int i0 = b0; i0 < b1; i0 += 32) {
            const int i = i0 + lane, tok = tok0;
            tok0 = i + 32 < b1 ? a.r.bias_ids[i + 32] : -1;
            const unsigned at = (unsigned)tok - (unsigned)v0;
            const bool mine = tok >= 0 && at < (unsigned)n && (int)(at & 7) == warp;
            unsigned left = __ballot_sync(0xffffffffu, mine);
            if (!left) continue;
            const float val = mine ? a.r.bias_vals[i] : 0.f;
            const unsigned same = __match_any_sync(0xffffffffu, mine ? (int)at : -1 - lane);
            while (left) {  // the first entry of each token that is left, until none is
                const bool turn = ((left >> lane) & 1u) && !(same & left & ((1u << lane) - 1u));
                if (turn) bias[at + shift] = __fadd_rn(bias[at + shift], val);
                __syncwarp();
                left &= ~__ballot_sync(0xffffffffu, turn);
            }
        }
    }
    __syncthreads();
    auto single = [&](int i) {
        float v = lg_load(in + i);
        if (count && seen[i + shift]) v = lg_penalty(w, v, seen[i + shift]);
        if (add) v = __fadd_rn(v, bias[i + shift]);
        const int tok = v0 + i;
        if (mask && !((mask[tok >> 5] >> (tok & 31)) & 1u)) v = -INFINITY;
        lg_store(out + i, v);
    };
    for (int i = t; i < head; i += kLgThreads) single(i);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int j = k * kLgThreads + t;
        if (j >= vecs) break;
        const int i = head + j * E;
        float v[E];
#pragma unroll
        for (int c = 0; c < E; c++) v[c] = lg_load(reinterpret_cast<const T*>(&x[k]) + c);
        if (count) {
#pragma unroll
            for (int q = 0; q < E; q += 4) {
                const uint4 c = *reinterpret_cast<const uint4*>(&seen[i + shift + q]);
                if (c.x | c.y | c.z | c.w) {
                    if (c.x) v[q] = lg_penalty(w, v[q], c.x);
                    if (c.y) v[q + 1] = lg_penalty(w, v[q + 1], c.y);
                    if (c.z) v[q + 2] = lg_penalty(w, v[q + 2], c.z);
                    if (c.w) v[q + 3] = lg_penalty(w, v[q + 3], c.w);
                }
            }
        }
        if (add) {
#pragma unroll
            for (int q = 0; q < E; q += 4) {
                const float4 c = *reinterpret_cast<const float4*>(&bias[i + shift + q]);
                v[q] = __fadd_rn(v[q], c.x), v[q + 1] = __fadd_rn(v[q + 1], c.y);
                v[q + 2] = __fadd_rn(v[q + 2], c.z), v[q + 3] = __fadd_rn(v[q + 3], c.w);
            }
        }
        if (mask) {
            const uint32_t bits = __funnelshift_r(lo[k], hi[k], (v0 + i) & 31);
#pragma unroll
            for (int c = 0; c < E; c++) v[c] = (bits >> c) & 1u ? v[c] : -INFINITY;
        }
        uint4 y;
#pragma unroll
        for (int c = 0; c < E; c++) lg_store(reinterpret_cast<T*>(&y) + c, v[c]);
        reinterpret_cast<uint4*>(out + head)[j] = y;
    }
    for (int i = tail + t; i < n; i += kLgThreads) single(i);
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" vb_status vb_logits_process(const void* logits, int64_t stride_in, void* out, int64_t stride_out, int dtype,
                                       int rows, int64_t vocab, const vb_logits_rules* rules, void* stream) {
    const int es = paged_elem_bytes(dtype);
    if (!es) return fail(VB_ERR_ARG, "logits_process: unknown element type");
    if (rows < 0 || vocab <= 0) return fail(VB_ERR_ARG, "logits_process: non-positive shape");
    if (vocab > 0x7fffffffll) return fail(VB_ERR_UNSUPPORTED, "logits_process: token ids are 32-bit");
    if (rows == 0) return VB_OK;
    if (!logits || !out || !rules) return fail(VB_ERR_ARG, "null pointer");
    if (rows > 1 && (stride_in < vocab || stride_out < vocab))
        return fail(VB_ERR_ARG, "logits_process: rows overlap");
    if (logits == out && rows > 1 && stride_in != stride_out)
        return fail(VB_ERR_ARG, "logits_process: in place needs equal strides");
    const vb_logits_rules& r = *rules;
    if (r.hist_total < 0 || r.bias_total < 0) return fail(VB_ERR_ARG, "logits_process: negative size");
    if (r.hist_total > 0x70000000ll || r.bias_total > 0x70000000ll)
        return fail(VB_ERR_UNSUPPORTED, "logits_process: lists are counted in 32 bits");
    if ((r.repetition || r.frequency || r.presence) && !r.hist_start)
        return fail(VB_ERR_ARG, "logits_process: penalties need a history");
    if ((r.hist_start && r.hist_total && !r.hist_ids) ||
        (r.bias_start && r.bias_total && (!r.bias_ids || !r.bias_vals)))
        return fail(VB_ERR_ARG, "null pointer");
    if (r.mask && rows > 1 && r.mask_stride < (vocab + 31) / 32)
        return fail(VB_ERR_ARG, "logits_process: mask rows overlap");
    if ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) % es ||
        !paged_words({r.hist_start, r.hist_ids, r.prompt_len, r.repetition, r.frequency, r.presence, r.bias_start, r.bias_ids,
                      r.bias_vals, r.mask}))
        return fail(VB_ERR_UNSUPPORTED, "logits_process: arrays aligned to their elements required");
    LogitsArgs a{};
    a.in = static_cast<const char*>(logits);
    a.out = static_cast<char*>(out);
    a.stride_in = stride_in * es;
    a.stride_out = stride_out * es;
    a.vocab = vocab;
    a.slices = (int)((vocab + kLgSlice - 1) / kLgSlice);
    a.r = r;
    const int64_t grid = (int64_t)a.slices * rows;
    if (grid > 0x7fffffffll) return fail(VB_ERR_UNSUPPORTED, "logits_process: too many rows");
    cudaStream_t s = as_stream(stream);
    cudaError_t e;
    if (dtype == VB_F32)
        e = launch_pdl(logits_process_kernel<float>, dim3((unsigned)grid), dim3(kLgThreads), 0, s, a);
    else if (dtype == VB_F16)
        e = launch_pdl(logits_process_kernel<__half>, dim3((unsigned)grid), dim3(kLgThreads), 0, s, a);
    else
        e = launch_pdl(logits_process_kernel<__nv_bfloat16>, dim3((unsigned)grid), dim3(kLgThreads), 0, s, a);
    if (e != cudaSuccess) return cuda_fail(e, "logits_process_kernel");
    VB_LAUNCH_CHECK("logits_process_kernel");
    return VB_OK;
}
