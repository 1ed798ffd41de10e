// vb_paged_append.cu -- new keys and values into a paged cache, with the
// per-head RMS norm and the position rotation on the way; q rotated in the
// same launch (kernels/cuda_ops.cu's rope and cache_append, and
// generate.cpp:52-64, for a ragged batch).
//
// Bound by memory: q, k, v are read and q, K, V written once, nothing else is
// moved but the rotation's angles.  A thread takes 16 elements of a head row at a
// time -- the 8 + 8 whose pairs rotate together -- so a row's norm is a sum over
// D / 16 neighbouring lanes and every access is 16 bytes or two of them.  It goes
// through four rows of its token, the next one's elements already asked for: with
// one row a thread the way from a token to its page and angles, three loads one
// after the other and half of all instructions, was walked for every row (21 us
// where this takes 16: four prompts of up to 2048 tokens, 16/8 heads, bf16, 59 MB;
// 3.6 TB/s, 0.55 of the measured copy rate).
#include "vb_kernels.cuh"
#include "vb_paged.cuh"

namespace vb {
namespace {

struct AppendArgs {
    PagedView p;
    vb_paged_rope rope;
    const char *q, *kn, *vn;
    char* qo;
    int64_t q_row, q_head, qo_row, qo_head, k_row, k_head, v_row, v_head;  // bytes
    int heads;      // 0: no q
    int row_units;  // threads of one token
};

constexpr int kAppendThreads = 256;
constexpr int kHeads = 4;  // head rows of a thread, one after the other

// Eight elements as they lie in memory.
template <typename T>
struct Raw {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const char* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) v[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void to(float* x) const { Eight<T>::load(v, x); }
};

template <typename IO, typename KV, int D>
__global__ void __launch_bounds__(kAppendThreads, 4) paged_append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int U = D / 16;  // threads of a head row
    pdl_wait();
    pdl_trigger();
    if (a.p.status && blockIdx.x == 0)  // the sequences that no row leads to are reported too
        for (int i = threadIdx.x; i < a.p.batch; i += kAppendThreads) paged_seq(a.p, i);
    const int lane = threadIdx.x & 31, nk = a.p.kv_heads, rot = a.rope.rot;
    const unsigned g = blockIdx.x * (unsigned)kAppendThreads + threadIdx.x;  // (the host keeps it in 32 bits)
    const int t = (int)(g / (unsigned)a.row_units);
    const int unit = (int)(g - (unsigned)t * (unsigned)a.row_units);
    const int t0 = __shfl_sync(0xffffffffu, t, 0);
    if (t0 >= a.p.tokens) return;  // the whole warp is behind the last token
    const int u = unit % U, first = unit / U * kHeads, rows = a.heads + 2 * nk;
    // the two chunks of 8 elements: pairs that turn together, or neighbours (v's always)
    const bool turns = 16 * u < rot, split = turns && !a.rope.interleaved;
    const int c0 = split ? 8 * u : 16 * u, c1 = split ? rot / 2 + 8 * u : 16 * u + 8;
    Raw<IO> xn, yn;
    auto fetch = [&](int row) {
        if (t < a.p.tokens && row < rows) {
            const int k = row - a.heads, v = k - nk;
            const char* src = k < 0   ? a.q + t * a.q_row + row * a.q_head
                              : v < 0 ? a.kn + t * a.k_row + k * a.k_head
                                      : a.vn + t * a.v_row + v * a.v_head;
            xn.load(src + c0 * sizeof(IO));
            yn.load(src + c1 * sizeof(IO));
        }
    };
    // asked for before the token's sequence and position are known: neither says where it is
    fetch(first);
    // the warp's first token's sequence by a warp-wide search; later tokens are a few sequences on
    int b = paged_find_seq(a.p.q_start, a.p.batch, t0, lane);
    while (b + 1 < a.p.batch && a.p.q_start[b + 1] <= t) b++;
    const PagedSeq s = paged_seq(a.p, b);
    const int pos = s.len - s.n + (t - s.start);
    const bool live = t < a.p.tokens && s.ok && t >= s.start && t < s.start + s.n && pos >= 0;
    float c[8], sn[8];
    int64_t off = -1;
    if (live) {
        if (turns) {
            Eight<float>::load(a.rope.cos_tab + (size_t)pos * rot + 8 * u, c);
            Eight<float>::load(a.rope.sin_tab + (size_t)pos * rot + 8 * u, sn);
        }
        if (first + kHeads > a.heads) off = paged_offset(a.p, b, pos);
    }
#pragma unroll 1
    for (int row = first; row < first + kHeads; row++) {
        float x[8], y[8];
        xn.to(x);
        yn.to(y);
        if (row + 1 < first + kHeads) fetch(row + 1);
        const int k = row - a.heads, v = k - nk;
        const float* w = k < 0 ? a.rope.q_norm : v < 0 ? a.rope.k_norm : nullptr;
        if (a.rope.q_norm || a.rope.k_norm) {  // every lane takes part in the sum
            float ss[4] = {};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                ss[e & 1] = fmaf(x[e], x[e], ss[e & 1]);
                ss[2 + (e & 1)] = fmaf(y[e], y[e], ss[2 + (e & 1)]);
            }
            float sum = (ss[0] + ss[1]) + (ss[2] + ss[3]);
#pragma unroll
            for (int o = U / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (w) {
                const float sc = __frsqrt_rn(__fadd_rn(__fmul_rn(sum, 1.0f / D), a.rope.eps));
                float z[8];
                Eight<float>::load(w + c0, z);
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = __fmul_rn(__fmul_rn(x[e], sc), z[e]);
                Eight<float>::load(w + c1, z);
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = __fmul_rn(__fmul_rn(y[e], sc), z[e]);
            }
        }
        if (!live || v >= nk) continue;
        if (turns && v < 0) {
            if (!a.rope.interleaved) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float lo = __fsub_rn(__fmul_rn(x[e], c[e]), __fmul_rn(y[e], sn[e]));
                    y[e] = __fadd_rn(__fmul_rn(y[e], c[e]), __fmul_rn(x[e], sn[e]));
                    x[e] = lo;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float p = __fsub_rn(__fmul_rn(x[e], c[e / 2]), __fmul_rn(x[e + 1], sn[e / 2]));
                    x[e + 1] = __fadd_rn(__fmul_rn(x[e + 1], c[e / 2]), __fmul_rn(x[e], sn[e / 2]));
                    x[e] = p;
                    const float q = __fsub_rn(__fmul_rn(y[e], c[4 + e / 2]), __fmul_rn(y[e + 1], sn[4 + e / 2]));
                    y[e + 1] = __fadd_rn(__fmul_rn(y[e + 1], c[4 + e / 2]), __fmul_rn(y[e], sn[4 + e / 2]));
                    y[e] = q;
                }
            }
        }
        if (k < 0) {
            char* dst = a.qo + t * a.qo_row + row * a.qo_head;
            Eight<IO>::store(dst + c0 * sizeof(IO), x);
            Eight<IO>::store(dst + c1 * sizeof(IO), y);
        } else if (off >= 0) {
            char* dst = const_cast<char*>(v < 0 ? a.p.k : a.p.v) + off + (v < 0 ? k : v) * a.p.stride_head;
            Eight<KV>::store(dst + c0 * sizeof(KV), x);
            Eight<KV>::store(dst + c1 * sizeof(KV), y);
        }
    }
}

template <typename IO, typename KV>
vb_status launch_append(const AppendArgs& a, int D, unsigned grid, cudaStream_t s) {
    const cudaError_t e =
        D == 128 ? launch_pdl(paged_append_kernel<IO, KV, 128>, dim3(grid), dim3(kAppendThreads), 0, s, a)
                 : launch_pdl(paged_append_kernel<IO, KV, 64>, dim3(grid), dim3(kAppendThreads), 0, s, a);
    if (e != cudaSuccess) return cuda_fail(e, "paged_append_kernel");
    VB_LAUNCH_CHECK("paged_append_kernel");
    return VB_OK;
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" vb_status vb_paged_append(const vb_paged_cache* cache, const vb_paged_batch* batch,
                                     const vb_paged_rope* rope, int io, int heads, const void* q, int64_t q_row,
                                     int64_t q_head, void* q_out, int64_t qo_row, int64_t qo_head, const void* k,
                                     int64_t k_row, int64_t k_head, const void* v, int64_t v_row, int64_t v_head,
                                     void* stream) {
    AppendArgs a{};
    if ((q == nullptr) != (q_out == nullptr)) return fail(VB_ERR_ARG, "paged_append: q and q_out come together");
    const vb_status st = paged_view(cache, batch, io, q ? heads : cache ? cache->kv_heads : 0, "paged_append", &a.p);
    if (st) return st;
    if (batch->tokens == 0 || batch->batch == 0) return VB_OK;
    if (!k || !v) return fail(VB_ERR_ARG, "paged_append: null pointer");
    const int es = paged_elem_bytes(io), D = cache->head_dim;
    if ((q && (!paged_aligned(q, q_row, q_head, es) || !paged_aligned(q_out, qo_row, qo_head, es))) ||
        !paged_aligned(k, k_row, k_head, es) || !paged_aligned(v, v_row, v_head, es))
        return fail(VB_ERR_UNSUPPORTED, "paged_append: 16-byte alignment required");
    if (q == q_out && q && (q_row != qo_row || q_head != qo_head))
        return fail(VB_ERR_ARG, "paged_append: q in place needs equal strides");
    if (rope) a.rope = *rope;
    if (a.rope.rot) {
        if (a.rope.rot < 0 || a.rope.rot % 16 || a.rope.rot > D)
            return fail(VB_ERR_UNSUPPORTED, "paged_append: rot must be a multiple of 16, at most head_dim");
        if (!a.rope.cos_tab || !a.rope.sin_tab) return fail(VB_ERR_ARG, "paged_append: null rotation table");
        if (!paged_aligned(a.rope.cos_tab, 0, 0, 4) || !paged_aligned(a.rope.sin_tab, 0, 0, 4))
            return fail(VB_ERR_UNSUPPORTED, "paged_append: 16-byte alignment required");
        if (batch->max_len > a.rope.rope_positions) return fail(VB_ERR_ROPE, "position is outside the rope table");
    }
    if (!paged_aligned(a.rope.q_norm, 0, 0, 4) || !paged_aligned(a.rope.k_norm, 0, 0, 4))
        return fail(VB_ERR_UNSUPPORTED, "paged_append: 16-byte alignment required");
    a.q = static_cast<const char*>(q);
    a.qo = static_cast<char*>(q_out);
    a.kn = static_cast<const char*>(k);
    a.vn = static_cast<const char*>(v);
    a.q_row = q_row * es, a.q_head = q_head * es, a.qo_row = qo_row * es, a.qo_head = qo_head * es;
    a.k_row = k_row * es, a.k_head = k_head * es, a.v_row = v_row * es, a.v_head = v_head * es;
    a.heads = q ? heads : 0;
    a.row_units = (a.heads + 2 * a.p.kv_heads + kHeads - 1) / kHeads * (D / 16);
    const int64_t blocks = ((int64_t)batch->tokens * a.row_units + kAppendThreads - 1) / kAppendThreads;
    if (blocks * kAppendThreads > 0x7fffffffll) return fail(VB_ERR_UNSUPPORTED, "paged_append: too many rows");
    cudaStream_t s = as_stream(stream);
    const unsigned grid = (unsigned)blocks;
    if (io == VB_F32 && cache->dtype == VB_F32) return launch_append<float, float>(a, D, grid, s);
    if (io == VB_F32) return launch_append<float, __nv_bfloat16>(a, D, grid, s);
    if (io == VB_F16) return launch_append<__half, __half>(a, D, grid, s);
    return launch_append<__nv_bfloat16, __nv_bfloat16>(a, D, grid, s);
}
