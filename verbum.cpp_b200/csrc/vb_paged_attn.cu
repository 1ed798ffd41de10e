// vb_paged_attn.cu -- causal attention of each sequence's new tokens over its
// pages (generate.cpp:73-105 applied at every new position of a ragged batch).
//
// For the rows of one KV head (new tokens x the G query heads that share it)
// s_j = q . k_j, m = max s, l = sum e^(s_j - m), out = sum e^(s_j - m) v_j / l,
// kept as a running (m, l, sum) while one pass goes over the keys, so K and V
// are read once for all G heads.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "vb_kernels.cuh"
#include "vb_paged.cuh"
#include "vb_pipe.cuh"
#include "vb_tc.cuh"

namespace vb {

vb_status paged_view(const vb_paged_cache* c, const vb_paged_batch* b, int io, int heads, const char* who,
                     PagedView* out) {
    const auto refuse = [who](vb_status code, const char* msg) { return fail(code, std::string(who) + ": " + msg); };
    if (!c || !b || !c->k || !c->v) return refuse(VB_ERR_ARG, "null pointer");
    const int es = paged_elem_bytes(c->dtype);
    if (!es || !paged_elem_bytes(io)) return refuse(VB_ERR_ARG, "unknown element type");
    if (io != c->dtype && !(io == VB_F32 && c->dtype == VB_BF16))
        return refuse(VB_ERR_UNSUPPORTED, "rows have the cache's type, or f32 with a bf16 cache");
    if (c->head_dim != 64 && c->head_dim != 128) return refuse(VB_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    if (c->num_pages <= 0 || c->page_size <= 0 || c->kv_heads <= 0) return refuse(VB_ERR_ARG, "non-positive shape");
    if (heads <= 0 || heads % c->kv_heads) return refuse(VB_ERR_ARG, "heads must be a multiple of kv_heads");
    if (c->stride_page < 0 || c->stride_pos < 0 || c->stride_head < 0) return refuse(VB_ERR_ARG, "negative stride");
    if (!paged_aligned(c->k, c->stride_pos, c->stride_head, es) || !paged_aligned(c->v, c->stride_page, 0, es))
        return refuse(VB_ERR_UNSUPPORTED, "16-byte alignment required");
    if (b->batch < 0 || b->tokens < 0 || b->max_new < 0 || b->max_len < 0 || b->table_stride < 0)
        return refuse(VB_ERR_ARG, "negative size");
    if (!paged_words({b->q_start, b->lens, b->table, b->status}))
        return refuse(VB_ERR_UNSUPPORTED, "4-byte alignment required");
    if (b->batch && b->tokens) {
        if (!b->q_start || !b->lens || (b->max_len && !b->table)) return refuse(VB_ERR_ARG, "null pointer");
        if (b->max_len > (int64_t)b->table_stride * c->page_size)
            return refuse(VB_ERR_ARG, "max_len is more than the table's pages hold");
    }
    PagedView& p = *out;
    p.k = static_cast<const char*>(c->k);
    p.v = static_cast<const char*>(c->v);
    p.num_pages = c->num_pages;
    p.page_size = c->page_size;
    p.kv_heads = c->kv_heads;
    p.page_shift = (c->page_size & (c->page_size - 1)) == 0 ? __builtin_ctz((unsigned)c->page_size) : -1;
    p.stride_page = c->stride_page * es;
    p.stride_pos = c->stride_pos * es;
    p.stride_head = c->stride_head * es;
    p.batch = b->batch;
    p.tokens = b->tokens;
    p.max_new = std::min(b->max_new, b->tokens);
    p.max_len = b->max_len;
    p.q_start = b->q_start;
    p.lens = b->lens;
    p.table = b->table;
    p.table_stride = b->table_stride;
    p.status = b->status;
    return VB_OK;
}

namespace {

// How a kernel cuts its work: rows of a tile, and the splits of a tile's keys, which
// start at a multiple of `align`.
struct Cut {
    int rows, splits, len, align;
};

struct AttnView {
    PagedView p;
    const char* q;
    char* out;
    int64_t q_row, q_head, o_row, o_head;  // bytes
    float* lse;
    int heads, group;   // group: query heads per KV head
    float scale_log2;   // scale * log2(e): the softmax runs in base 2
    int window;
    int few_rows;       // sequences with at most this many rows a KV head run in the few-rows kernel
    Cut few, many;
    int stream;         // blocks that share all keys of the few-rows kernel evenly; 0: clusters of blocks, one a tile
    bool redo;          // single tokens of a type whose products do not treat what is seen as the formula does:
                        // no last pass, the few-rows kernel and its join look at their own rows
    bool after_many;    // the few-rows kernel of this call follows its many-rows kernel
    unsigned* ready;    // then: 1 once what came before the call can be read, by the many-rows kernel; else NULL
    int box;            // rows of a page that one TMA copy brings (many rows); 0: no tensor maps
    bool stall;         // test hook (vb_debug_arm_fault): block 0 of the many-rows kernel never has all of its q
    int* hint;          // calls of many rows: [sequence][KV head] where a row that was taken again met a NaN (redo_row)
    float* part;        // [split][token][head][D] sums of a split, relative to its maximum
    float2* part_ml;    // [split][token][head] (maximum in base 2, sum of weights)
    float* strm;        // the same of the shared keys: [block][2][tile row][D]
    float2* strm_ml;    // [block][2][tile row]
};

// The keys that the tile's rows r0 .. r0 + cut.rows - 1 (of n * G) of a sequence see.
struct KeyRange {
    int lo, hi;  // positions lo .. hi - 1
    int base;    // lo rounded down: where the first split starts
};
__device__ __forceinline__ KeyRange key_range(const AttnView& a, const PagedSeq& s, int r0, const Cut& cut) {
    const int r1 = min(r0 + cut.rows, s.n * a.group) - 1;
    const int p0 = s.len - s.n + r0 / a.group, p1 = s.len - s.n + r1 / a.group;
    KeyRange k;
    k.hi = max(p1 + 1, 0);
    k.lo = a.window > 0 ? max(p0 - a.window + 1, 0) : 0;
    k.lo = min(k.lo, k.hi);
    k.base = k.lo & -cut.align;
    return k;
}
// Sharing out the keys of the few-rows kernel's tiles.  A tile (sequence, KV head) is
// units of 64 keys, one at least; the units of all sequences follow one another, KV heads
// within a sequence, and block c of N <= W takes units [c W / N, (c + 1) W / N).
constexpr int kUnit = 64;
__device__ __forceinline__ int stream_units(const AttnView& a, int b) {
    const int start = a.p.q_start[b], end = a.p.q_start[b + 1];
    PagedSeq s;
    s.len = a.p.lens[b];
    s.n = end - start;
    if (s.len < 0 || s.len > a.p.max_len) s.len = 0;
    const KeyRange k = key_range(a, s, 0, a.few);
    const bool ok = start >= 0 && end > start && end <= a.p.tokens && s.n <= a.p.max_new &&
                    (int64_t)s.n * a.group <= a.few_rows;
    return ok ? max(1, (k.hi - k.base + kUnit - 1) / kUnit) : 0;
}
// Units of all sequences, and of those before sequence b; by the whole block of WARPS warps.
// (The host sees to it that they fit 32 bits.)
template <int WARPS>
__device__ __forceinline__ void stream_sums(const AttnView& a, int b, int& all, int& before) {
    __shared__ int2 sums[WARPS];
    int x = 0, y = 0;
    for (int i = threadIdx.x; i < a.p.batch; i += WARPS * 32) {
        const int u = stream_units(a, i);
        x += u;
        if (i < b) y += u;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = make_int2(x, y);
    __syncthreads();
    x = y = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) x += sums[w].x, y += sums[w].y;
    all = x * a.p.kv_heads;
    before = y * a.p.kv_heads;
}
__device__ __forceinline__ int splits_used(const Cut& c, const KeyRange& k) {
    return max(1, (k.hi - k.base + c.len - 1) / c.len);
}

__device__ __forceinline__ void cp_async16(unsigned dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(unsigned addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(unsigned addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ float4 lds128(unsigned addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// d (16 x 8, f32) += a (16 x 16) b (16 x 8)
template <typename T>
__device__ __forceinline__ void mma16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__half>(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d (16 x 8, f32) += a (16 x 8) b (8 x 8), tf32 operands
__device__ __forceinline__ void mma8(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A pair of f32 as NT bf16 pairs whose sum it is: three hold all 24 bits of an
// f32 (8 each), so products with bf16 values lose nothing.
template <typename T, int NT>
__device__ __forceinline__ void split_terms(float a, float b, uint32_t* t) {
    t[0] = pack2<T>(a, b);
    if constexpr (NT > 1) {
#pragma unroll
        for (int i = 1; i < NT; i++) {
            a -= __uint_as_float(t[i - 1] << 16);
            b -= __uint_as_float(t[i - 1] & 0xffff0000u);
            t[i] = pack2<T>(a, b);
        }
    }
}
// x = hi + lo with hi a tf32 number (nearest) and lo the rest; the tensor core
// reads the first 11 bits of lo.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    lo = __float_as_uint(x - __uint_as_float(hi));
}

// The transpose of a matrix of 8 x 8 16-bit values spread over the warp
__device__ __forceinline__ uint32_t mat_t(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// Weights are e^(s - reference); f16 ones take a reference so far (in powers of two) below the
// maximum, for f16 has no normal numbers under 2^-14: a weight of 2^-14 of the largest would
// lose bits that show where the largest one's v is small.  lse and the joins see the
// reference, whatever it is.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 6.f : 0.f;

// ------------------------------------------------------------- rows taken again
// N neighbouring elements of a row
template <typename T, int N>
struct __align__(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Few {
    T v[N];
};

// base + off, or zeros where off is negative (without a branch between an unrolled loop's loads)
template <typename T, int N>
__device__ __forceinline__ Few<T, N> row_or_zeros(const char* base, int64_t off) {
    Few<T, N> x = *reinterpret_cast<const Few<T, N>*>(base + max(off, (int64_t)0));
#pragma unroll
    for (int e = 0; e < N; e++) x.v[e] = off < 0 ? (T)0.f : x.v[e];
    return x;
}

// Places of keys key0 .. key0 + 31 of sequence b, one a lane; -1 beyond `last` and on a bad page.
__device__ __forceinline__ int64_t places(const AttnView& a, int b, int key0, int last, int lane) {
    return key0 + lane <= last ? paged_offset(a.p, b, key0 + lane) : -1;
}

// The rows of those keys (zeros where there is no place), 16 bytes a lane, through f: a lane has
// dims kDims * (lane % kLanes) .. of every row it sees.
template <typename KV, int D>
struct Chunks {
    static constexpr int kDims = 16 / (int)sizeof(KV), kLanes = D / kDims, kRows = 32 / kLanes;
    template <typename F>
    static __device__ __forceinline__ void each(const char* base, int64_t off, int lane, F f) {
#pragma unroll
        for (int j = 0; j < 32 / kRows; j++) {
            const int64_t o = __shfl_sync(0xffffffffu, off, j * kRows + lane / kLanes);
            f(row_or_zeros<KV, kDims>(base + lane % kLanes * 16, o));
        }
    }
    template <typename F>  // bit e: test(element e)
    static __device__ __forceinline__ unsigned bits(const Few<KV, kDims>& x, F test) {
        unsigned m = 0;
#pragma unroll
        for (int e = 0; e < kDims; e++) m |= test((float)x.v[e]) ? 1u << e : 0u;
        return m;
    }
};

// The products treat what a row sees as the formula does: bf16 weights are 0 only where f32's are.
template <typename IO>
constexpr bool kAsSeen = std::is_same<IO, __nv_bfloat16>::value;

// Takes a row with NaN again, by the block's WARPS (an even number, at least 4) warps, each 32
// keys at a time over what the row sees, in 32 bits as the formula has it: an infinity that is seen
// stays one, where the products of terms (f32) or of f16 weights made it NaN.  Other elements stay.
//
// What is NaN for good is found soon.  The first and the last 32 keys are looked at before all else
// (a bad prefix has its NaN there, a sequence that went wrong at the row's own position), and those
// where another row of the sequence and KV head met its NaN (`hint`, verified like the others: any
// value will do); further keys come from both ends by turns, and the block leaves when the sum of the
// weights is NaN or every element in question is.  And bf16 products treat what a row sees as the
// formula does, so a bf16 row is not taken again unless a v of its tile that it does not see is the
// cause.
// 16/8 heads, a call without NaN -> with one in the v of (a) the first of 4096 positions of a prompt,
// (b) one of the last, which 2000 rows of its tile do not see, (c) the middle of 65536 under a chunk of
// 512: bf16 0.10 -> 0.62, 1.05, 0.38 -> 0.70 ms; f16 0.10 -> 0.58, 1.02, 0.38 -> 20; f32 0.43 -> 0.84,
// 0.90, 1.7 -> 19 (each row walked by a warp, a key at a time: (a) 36, 36 and 21).  What is left is a row's
// way through all its keys, 0.3 us a key, paid once a KV head; by every row in an f32 call that sees
// an infinity and no NaN.
template <typename IO, typename KV, int D, int WARPS>
__device__ __forceinline__ void redo_row(const AttnView& a, int token, int head, float (*sums)[D], float2* ml, int* done) {
    constexpr int E = D / 32;
    using C = Chunks<KV, D>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = paged_find_seq(a.p.q_start, a.p.batch, token, lane);
    const PagedSeq s = paged_seq(a.p, b);
    const int pos = s.len - s.n + token - s.start;
    if (!s.ok || token < s.start || token >= s.start + s.n || pos < 0) return;  // not a row of this call, or an empty one
    const int lo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
    const int64_t head_off = (int64_t)(head / a.group) * a.p.stride_head, th = (int64_t)token * a.heads + head;
    const bool need_l = a.lse && isnan(a.lse[th]);
    IO* const row = reinterpret_cast<IO*>(a.out + token * a.o_row + head * a.o_head);
    Few<IO, E> out = *reinterpret_cast<const Few<IO, E>*>(row + lane * E);
    const Few<IO, C::kDims> part = *reinterpret_cast<const Few<IO, C::kDims>*>(row + lane % C::kLanes * C::kDims);
    unsigned bad = 0, bad_c = 0;  // elements that are NaN: of `out`, and of the chunk
#pragma unroll
    for (int e = 0; e < E; e++) bad |= isnan((float)out.v[e]) ? 1u << e : 0u;
#pragma unroll
    for (int e = 0; e < C::kDims; e++) bad_c |= isnan((float)part.v[e]) ? 1u << e : 0u;
    if (!__any_sync(0xffffffffu, bad != 0)) return;  // (an infinity in a sum is a seen one's)
    int* const hint = a.hint ? a.hint + b * a.p.kv_heads + head / a.group : nullptr;

    bool nan_for_good = false;
    const int met = hint ? *(volatile int*)hint : -1;
    for (int i = warp; i < 6; i += WARPS) {  // v and k of the first keys, of the last ones, of those from `met` on
        const int key0 = i < 2 ? lo : i < 4 ? max(lo, pos - 31) : met;
        if (key0 < lo || key0 > pos) continue;
        unsigned seen = 0;
        C::each((i & 1 ? a.p.k : a.p.v) + head_off, places(a, b, key0, pos, lane), lane,
                [&](const auto& x) { seen |= C::bits(x, [](float y) { return isnan(y); }); });
#pragma unroll
        for (int o = C::kLanes; o < 32; o <<= 1) seen |= __shfl_xor_sync(0xffffffffu, seen, o);
        nan_for_good |= i & 1 ? __any_sync(0xffffffffu, seen != 0) : !need_l && __all_sync(0xffffffffu, (bad_c & ~seen) == 0);
    }
    auto leave_nan = [&] {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (bad >> e & 1) out.v[e] = (IO)nanf("");
        if (warp == 0) *reinterpret_cast<Few<IO, E>*>(row + lane * E) = out;
    };
    if (__syncthreads_or(nan_for_good)) {
        leave_nan();
        return;
    }
    if constexpr (kAsSeen<IO>) {
        const int rows = s.n * a.group, r = (token - s.start) * a.group + head % a.group;
        const KeyRange kr =
            rows > a.few_rows ? key_range(a, s, r / a.many.rows * a.many.rows, a.many) : key_range(a, s, 0, a.few);
        bool hit = false;
        auto unseen = [&](int first, int last) {
            for (int key0 = first + warp * 32; key0 <= last && !hit; key0 += WARPS * 32) {
                C::each(a.p.v + head_off, places(a, b, key0, last, lane), lane,
                        [&](const auto& x) { hit |= (C::bits(x, [](float y) { return !isfinite(y); }) & bad_c) != 0; });
                hit = __any_sync(0xffffffffu, hit);
            }
        };
        unseen(pos + 1, kr.hi - 1);
        unseen(kr.lo, lo - 1);
        if (!__syncthreads_or(hit)) return;
    }
    const Few<IO, E> q8 = *reinterpret_cast<const Few<IO, E>*>(a.q + token * a.q_row + head * a.q_head + lane * E * sizeof(IO));
    float q[E], o[E] = {}, m = -INFINITY, l = 0.f;  // l: of this lane's keys
#pragma unroll
    for (int e = 0; e < E; e++) q[e] = (float)q8.v[e];
    if (threadIdx.x == 0) *done = 0;
    __syncthreads();
    const int n = (pos - lo) / 32 + 1;
    for (int i = warp; i < n; i += WARPS) {
        if (*(volatile int*)done) break;
        const int key0 = lo + 32 * (i & 1 ? n - 1 - (i >> 1) : i >> 1);
        const int64_t off = places(a, b, key0, pos, lane);
        const int64_t mine = head_off + (int64_t)lane * E * sizeof(KV);
        float x = 0.f;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float d[16];
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int64_t at = __shfl_sync(0xffffffffu, off, 16 * h + j);
                const Few<KV, E> k = row_or_zeros<KV, E>(a.p.k + mine, at);
                d[j] = 0.f;
#pragma unroll
                for (int e = 0; e < E; e++) d[j] = fmaf(q[e], (float)k.v[e], d[j]);
            }
            const float sum = __shfl_sync(0xffffffffu, warp_sum_scatter<16>(d, lane), 2 * (lane & 15));
            if (lane >> 4 == h) x = sum;
        }
        x = key0 + lane <= pos ? x * a.scale_log2 : -INFINITY;
        const float mn = fmaxf(m, warp_max(x)), mb = mn == -INFINITY ? 0.f : mn;
        const float f = ex2_approx(m - mb), w = ex2_approx(x - mb);
        m = mn;
        l = fmaf(l, f, w);
#pragma unroll
        for (int e = 0; e < E; e++) o[e] *= f;
#pragma unroll 16
        for (int j = 0; j < 32; j++) {
            const int64_t at = __shfl_sync(0xffffffffu, off, j);
            const float wj = __shfl_sync(0xffffffffu, w, j);
            const Few<KV, E> v = row_or_zeros<KV, E>(a.p.v + mine, at);
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = fmaf(wj, (float)v.v[e], o[e]);
        }
        bool open = need_l;
#pragma unroll
        for (int e = 0; e < E; e++) open |= (bad >> e & 1) && !isnan(o[e]);
        if (__any_sync(0xffffffffu, isnan(l)) || !__any_sync(0xffffffffu, open)) {
            if (lane == 0) {
                *(volatile int*)done = 1;
                if (hint) *(volatile int*)hint = key0;
            }
            break;
        }
    }
    l = warp_sum(l);
    if (lane == 0) ml[warp] = make_float2(m, l);
#pragma unroll
    for (int e = 0; e < E; e++) sums[warp][lane * E + e] = o[e];
    __syncthreads();
    if (*done) {
        leave_nan();
    } else if (warp == 0) {
        float M = -INFINITY, L = 0.f, y[E] = {};
        for (int x = 0; x < WARPS; x++) M = fmaxf(M, ml[x].x);
        for (int x = 0; x < WARPS; x++) {
            const float w = ex2_approx(ml[x].x - (M == -INFINITY ? 0.f : M));
            L = fmaf(ml[x].y, w, L);
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = fmaf(w, sums[x][lane * E + e], y[e]);
        }
#pragma unroll
        for (int e = 0; e < E; e++)
            if (bad >> e & 1) out.v[e] = (IO)(L == 0.f ? 0.f : y[e] / L);
        *reinterpret_cast<Few<IO, E>*>(row + lane * E) = out;
        if (need_l && lane == 0)
            a.lse[th] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945309f;
    }
    __syncthreads();  // the shared memory is free for the next row
}

// The same out of line, for kernels that have their registers for something else.
template <typename IO, typename KV, int D, int WARPS>
__device__ __noinline__ void redo_row_apart(const AttnView& a, int token, int head, float (*sums)[D], float2* ml, int* done) {
    redo_row<IO, KV, D, WARPS>(a, token, head, sums, ml, done);
}

// ------------------------------------------------------------- few rows
// The same by cutting the bits off: cheaper, for the operand whose other one is rounded
// (the product of two cut-off rests would be of one sign, and add up).
__device__ __forceinline__ void cut_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
constexpr int kBK = 16;  // keys a warp takes at a time

template <typename KV, int D, int NR>
struct FewCfg {
    static constexpr int kRows = 8 * NR;
    static constexpr int kWarps = sizeof(KV) == 4 && D == 128 ? 6 : 4;
    static constexpr int kRowBytes = D * (int)sizeof(KV);
    static constexpr int kBlockBytes = kBK * kRowBytes;  // K or V of a block
    // 64 KB of ring per CTA and three CTAs on an SM, or (f32, D = 128) 192 KB, six warps and one.  (A third
    // stage and two CTAs moved less: a piece's end and the next one's start leave a CTA without
    // loads in flight, and more of the others' fill in.)
    static constexpr int kStages = kRowBytes == 128 ? 4 : 2;
    static constexpr int kWarpBytes = kStages * 2 * kBlockBytes;
    static constexpr int kLd = D + 4;  // row of the warps' sums, floats
    static constexpr int kMerge = kWarps * kRows * kLd * 4;
    static constexpr int kSmem = kWarps * kWarpBytes > kMerge ? kWarps * kWarpBytes : kMerge;
};

// Where a piece of a tile's keys leaves its rows: the output, or sums to be joined.
struct Sink {
    bool last;       // the piece is the whole tile: the output
    bool keep;       // the sums stay in shared memory, row `row` at row * (D + 4), its (m, l) in kept
    float* part;     // else: row `row`'s sums at part + row * D, its (m, l) at ml + row
    float2* ml;
};

// Attention of 8 NR rows of a KV head by the warps of a block.  They share the rows and
// take turns at blocks of 16 keys, each with a ring of its own in shared memory
// (no barrier in the loop); at the end they join their (m, l, sum).
//
// Bound by memory when a tile holds all rows of its KV head (decoding), so the
// products are turned round: the 16 keys (then the 16 dims of V) are the M of
// m16n8k16 and the query rows its N, of which eight are enough -- with the rows
// as M, half of every product of a head group of 8 or fewer was padding.
//   S^T (16 keys x 8 rows) = K Q^T,  O^T (D x 8 rows) += V^T P^T.
// A thread holds the scores, maxima and sums of rows 2 t4 and 2 t4 + 1.
// f32 rows over a bf16 cache: q and the weights as three bf16 terms.  f32 cache:
// hi/lo tf32 pairs, three products.  Where the result is f32 a block's V^T P^T is
// summed apart and added to the running sum by an FMA: the tensor core's own
// accumulation truncates, which over thousands of keys would show.  16-bit rows: the
// weights are rounded to the cache's type (what the tensor cores take; half a step of
// each, relative, and of both signs), their sum is not.
// 64 sequences of up to 4096 keys, bf16, 16/8 heads: 92 us, 5.3 TB/s, 0.81 of the measured
// copy rate; 64 x 2112 f32 191-207 us from card to card, 0.82-0.88; 2 x up to 131072 f16 74-77 us, 0.84-0.87.
//
// The rows of KV head kvh of sequence b over keys k_begin .. k_end - 1, by the block.
template <typename IO, typename KV, int D, int NR>
__device__ __forceinline__ void few_piece(const AttnView& a, const PagedSeq& s, int b, int kvh, const KeyRange& kr,
                                          int k_begin, int k_end, const Sink& sink, char* smem,
                                          float2 (*ml)[8 * NR], float2* kept = nullptr) {
    using C = FewCfg<KV, D, NR>;
    constexpr bool kF32 = sizeof(KV) == 4;
    constexpr bool kExact = sizeof(IO) == 4;
    constexpr int NT = !kF32 && kExact ? 3 : 1;  // bf16 terms of an f32 operand
    constexpr int NK = D / 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int rows = s.n * a.group;
    const int blocks = max(0, (k_end - k_begin + kBK - 1) / kBK);
    const int mine = blocks > warp ? (blocks - warp + C::kWarps - 1) / C::kWarps : 0;  // blocks warp, warp + kWarps, ...

    const unsigned ring = smem_addr(smem) + warp * C::kWarpBytes;
    const int64_t head_off = (int64_t)kvh * a.p.stride_head;
    // lane l looks up the place of key l % 16 of a block; -1: outside, read as zeros
    auto look_up = [&](int i) -> int64_t {
        const int key = k_begin + (warp + i * C::kWarps) * kBK + (lane & 15);
        return i < mine && key >= kr.lo && key < k_end ? paged_offset(a.p, b, key) : -1;
    };
    // 16-byte chunk c of row r sits at chunk c ^ swz(r): no load below meets a bank twice, be it
    // 8 rows at one chunk (16 bits), 2 rows x 4 chunks (K) or 4 rows x 2 chunks (V)
    auto swz = [](int r) { return kF32 ? (((r & 1) << 1) | ((r >> 1) & 1)) << 1 : r & 7; };
    auto fetch = [&](int i, int64_t off) {
        if (i < mine) {
            constexpr int RC = C::kRowBytes / 16, RPI = 32 / RC;
            const unsigned st = ring + (unsigned)(i % C::kStages) * 2 * C::kBlockBytes;
#pragma unroll
            for (int it = 0; it < kBK / RPI; it++) {
                const int r = it * RPI + lane / RC, c = lane % RC;
                const int64_t o = __shfl_sync(0xffffffffu, off, r);
                const unsigned dst = st + r * C::kRowBytes + ((c ^ swz(r)) << 4);
                const int64_t at = o < 0 ? 0 : o + head_off + c * 16;
                cp_async16(dst, a.p.k + at, o >= 0);
                cp_async16(dst + C::kBlockBytes, a.p.v + at, o >= 0);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < C::kStages - 1; i++) fetch(i, look_up(i));
    int64_t next = look_up(C::kStages - 1);

    // q, the N operand: row 8 n + g of the tile.  f32 cache: dims 16 kk + 4 t4 .. + 3 (the order
    // of the dims inside a product is free as long as K's is the same); 16 bits: dims
    // 16 kk + 2 t4, + 1, + 8, + 9.
    float qf[kF32 ? NR : 1][NK][4];
    uint32_t qh[kF32 ? 1 : NR][NK][NT][2];
#pragma unroll
    for (int n = 0; n < NR; n++) {
        const int r = min(8 * n + g, rows - 1);
        const char* qp = a.q + (int64_t)(s.start + r / a.group) * a.q_row + (int64_t)(kvh * a.group + r % a.group) * a.q_head;
#pragma unroll
        for (int kk = 0; kk < NK; kk++) {
            if constexpr (kF32) {
                const float4 x = *reinterpret_cast<const float4*>(qp + (16 * kk + 4 * t4) * 4);
                qf[n][kk][0] = x.x, qf[n][kk][1] = x.y, qf[n][kk][2] = x.z, qf[n][kk][3] = x.w;
            } else {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const char* x = qp + (16 * kk + 2 * t4 + 8 * e) * sizeof(IO);
                    if constexpr (kExact) {
                        const float2 f = *reinterpret_cast<const float2*>(x);
                        uint32_t tt[NT];
                        split_terms<KV, NT>(f.x, f.y, tt);
#pragma unroll
                        for (int i = 0; i < NT; i++) qh[n][kk][i][e] = tt[i];
                    } else {
                        qh[n][kk][0][e] = *reinterpret_cast<const uint32_t*>(x);
                    }
                }
            }
        }
    }
    // rows 8 n + 2 t4 + e: position, running maximum and sum
    int pos[NR][2];
    float m[NR][2], l[NR][2];
    float o[NR][D / 16][4];
#pragma unroll
    for (int n = 0; n < NR; n++) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 8 * n + 2 * t4 + e;
            pos[n][e] = r < rows ? s.len - s.n + r / a.group : -1;
            m[n][e] = -INFINITY;
            l[n][e] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[n][i][e] = 0.f;
    }

    for (int i = 0; i < mine; i++) {
        cp_async_wait<C::kStages - 2>();
        __syncwarp();
        fetch(i + C::kStages - 1, next);
        next = look_up(i + C::kStages);
        const unsigned kb = ring + (unsigned)(i % C::kStages) * 2 * C::kBlockBytes, vb = kb + C::kBlockBytes;
        const int key0 = k_begin + (warp + i * C::kWarps) * kBK;
        // scores: keys g (e 0, 1) and g + 8 (e 2, 3), rows 2 t4 + (e & 1); the small terms apart
        float sc[NR][4] = {}, sl[NR][4] = {}, sm[kF32 ? NR : 1][4] = {};
        if constexpr (kF32) {
#pragma unroll
            for (int kk = 0; kk < NK; kk++) {
                uint32_t kh[2][4], kl[2][4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int r = 8 * h + g;
                    const float4 x = lds128(kb + r * C::kRowBytes + (((4 * kk + t4) ^ swz(r)) << 4));
                    cut_tf32(x.x, kh[h][0], kl[h][0]);
                    cut_tf32(x.y, kh[h][1], kl[h][1]);
                    cut_tf32(x.z, kh[h][2], kl[h][2]);
                    cut_tf32(x.w, kh[h][3], kl[h][3]);
                }
#pragma unroll
                for (int n = 0; n < NR; n++)
#pragma unroll
                    for (int h = 0; h < 4; h += 2) {
                        uint32_t qhi[2], qlo[2];
                        split_tf32(qf[n][kk][h], qhi[0], qlo[0]);
                        split_tf32(qf[n][kk][h + 1], qhi[1], qlo[1]);
                        const uint32_t ah[4] = {kh[0][h], kh[1][h], kh[0][h + 1], kh[1][h + 1]};
                        const uint32_t al[4] = {kl[0][h], kl[1][h], kl[0][h + 1], kl[1][h + 1]};
                        mma8(sc[n], ah, qhi[0], qhi[1]);
                        mma8(sl[n], al, qhi[0], qhi[1]);
                        mma8(sm[n], ah, qlo[0], qlo[1]);
                    }
            }
#pragma unroll
            for (int n = 0; n < NR; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) sl[n][e] += sm[n][e];
        } else {
            const int r = lane & 15, cc = lane >> 4;
#pragma unroll
            for (int kk = 0; kk < NK; kk++) {
                uint32_t kx[4];
                ldsm4(kb + r * C::kRowBytes + (((2 * kk + cc) ^ swz(r)) << 4), kx);
#pragma unroll
                for (int n = 0; n < NR; n++) {
                    mma16<KV>(sc[n], kx, qh[n][kk][0][0], qh[n][kk][0][1]);
#pragma unroll
                    for (int x = 1; x < NT; x++) mma16<KV>(sl[n], kx, qh[n][kk][x][0], qh[n][kk][x][1]);
                }
            }
        }
        float alpha[NR][2];
#pragma unroll
        for (int n = 0; n < NR; n++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int key = key0 + g + 8 * (e >> 1), p = pos[n][e & 1];
                const float x = (sc[n][e] + sl[n][e]) * a.scale_log2;
                sc[n][e] = key > p || key >= k_end || (a.window > 0 && key <= p - a.window) ? -INFINITY : x;
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float mx = fmaxf(sc[n][e], sc[n][e + 2]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                mx = fmaxf(mx - kLift<KV>, m[n][e]);
                const float mb = mx == -INFINITY ? 0.f : mx;
                alpha[n][e] = ex2_approx(m[n][e] - mb);
                m[n][e] = mx;
                sc[n][e] = ex2_approx(sc[n][e] - mb);
                sc[n][e + 2] = ex2_approx(sc[n][e + 2] - mb);
                l[n][e] = fmaf(l[n][e], alpha[n][e], sc[n][e] + sc[n][e + 2]);
            }
        }
        if constexpr (kF32) {
            // product kt sums keys 8 kt + t4 (k = t4) and + 4 (k = t4 + 4): a row's weights come from
            // the lanes that hold those keys.  The M rows g and g + 8 of product (np, j) are dims
            // 64 np + 4 g + j and + 32.
            uint32_t ph[NR][2][2], pl[NR][2][2];
#pragma unroll
            for (int n = 0; n < NR; n++)
#pragma unroll
                for (int kt = 0; kt < 2; kt++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int src = 4 * (t4 + 4 * h) + (g >> 1);
                        const float x0 = __shfl_sync(0xffffffffu, sc[n][2 * kt], src);
                        const float x1 = __shfl_sync(0xffffffffu, sc[n][2 * kt + 1], src);
                        split_tf32(g & 1 ? x1 : x0, ph[n][kt][h], pl[n][kt][h]);
                    }
#pragma unroll
            for (int np = 0; np < D / 64; np++) {
                float pv[NR][4][4] = {};
#pragma unroll
                for (int kt = 0; kt < 2; kt++) {
                    // v[2 h + x]: key 8 kt + t4 + 4 h, dims 64 np + 32 x + 4 g ..
                    uint32_t vh[4][4], vl[4][4];
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const int r = 8 * kt + t4 + 4 * (y >> 1);
                        const float4 x = lds128(vb + r * C::kRowBytes + (((16 * np + 8 * (y & 1) + g) ^ swz(r)) << 4));
                        cut_tf32(x.x, vh[y][0], vl[y][0]);
                        cut_tf32(x.y, vh[y][1], vl[y][1]);
                        cut_tf32(x.z, vh[y][2], vl[y][2]);
                        cut_tf32(x.w, vh[y][3], vl[y][3]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t ah[4] = {vh[0][j], vh[1][j], vh[2][j], vh[3][j]};
                        const uint32_t al[4] = {vl[0][j], vl[1][j], vl[2][j], vl[3][j]};
#pragma unroll
                        for (int n = 0; n < NR; n++) {
                            mma8(pv[n][j], al, ph[n][kt][0], ph[n][kt][1]);
                            mma8(pv[n][j], ah, pl[n][kt][0], pl[n][kt][1]);
                            mma8(pv[n][j], ah, ph[n][kt][0], ph[n][kt][1]);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < NR; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            o[n][4 * np + j][e] = fmaf(o[n][4 * np + j][e], alpha[n][e & 1], pv[n][j][e]);
            }
        } else {
            // weights to the N operand's layout: keys 2 t4, + 1 (+ 8) of row g
            uint32_t ph[NR][NT][2];
#pragma unroll
            for (int n = 0; n < NR; n++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t tt[NT];
                    split_terms<KV, NT>(sc[n][2 * h], sc[n][2 * h + 1], tt);
#pragma unroll
                    for (int x = 0; x < NT; x++) ph[n][x][h] = mat_t(tt[x]);
                }
            const int r = (lane & 7) + ((lane >> 4) << 3), cc = (lane >> 3) & 1;
#pragma unroll
            for (int i2 = 0; i2 < D / 16; i2++) {
                uint32_t vx[4];
                ldsm4_t(vb + r * C::kRowBytes + (((2 * i2 + cc) ^ swz(r)) << 4), vx);
#pragma unroll
                for (int n = 0; n < NR; n++) {
                    if constexpr (kExact) {
                        float pv[4] = {};
#pragma unroll
                        for (int x = NT - 1; x >= 0; x--) mma16<KV>(pv, vx, ph[n][x][0], ph[n][x][1]);
#pragma unroll
                        for (int e = 0; e < 4; e++) o[n][i2][e] = fmaf(o[n][i2][e], alpha[n][e & 1], pv[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) o[n][i2][e] *= alpha[n][e & 1];
                        mma16<KV>(o[n][i2], vx, ph[n][0][0], ph[n][0][1]);
                    }
                }
            }
        }
    }
    cp_async_wait<0>();
    // join the warps: every warp's sums to shared memory, then all threads over (row, dims)
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
            l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
            if (g == 0) ml[warp][8 * n + 2 * t4 + e] = make_float2(m[n][e], l[n][e]);
        }
    __syncthreads();  // the rings are free
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int n = 0; n < NR; n++)
#pragma unroll
        for (int i = 0; i < D / 16; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int d = kF32 ? 64 * (i >> 2) + 32 * (e >> 1) + 4 * g + (i & 3) : 16 * i + 8 * (e >> 1) + g;
                sums[(warp * C::kRows + 8 * n + 2 * t4 + (e & 1)) * C::kLd + d] = o[n][i][e];
            }
    __syncthreads();
    for (int it = threadIdx.x; it < C::kRows * (D / 8); it += C::kWarps * 32) {
        const int row = it / (D / 8), d = it % (D / 8) * 8;
        if (row >= rows) break;
        float M = -INFINITY, L = 0.f;
        float y[8] = {};
#pragma unroll
        for (int x = 0; x < C::kWarps; x++) M = fmaxf(M, ml[x][row].x);
#pragma unroll
        for (int x = 0; x < C::kWarps; x++) {
            const float w = ex2_approx(ml[x][row].x - (M == -INFINITY ? 0.f : M));
            L = fmaf(ml[x][row].y, w, L);
            float z[8];
            Eight<float>::load(sums + (x * C::kRows + row) * C::kLd + d, z);
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = fmaf(w, z[e], y[e]);
        }
        const int token = s.start + row / a.group, head = kvh * a.group + row % a.group;
        const int64_t th = (int64_t)token * a.heads + head;
        if (sink.keep) {
            Eight<float>::store(sums + row * C::kLd + d, y);  // (over what this thread alone has read)
            if (d == 0) kept[row] = make_float2(M, L);
        } else if (sink.last) {
            const float inv = 1.f / L;
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = L == 0.f ? 0.f : y[e] * inv;  // (a sum that is NaN stays one)
            Eight<IO>::store(a.out + token * a.o_row + head * a.o_head + d * sizeof(IO), y);
            if (d == 0 && a.lse) a.lse[th] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945309f;
        } else {
            Eight<float>::store(sink.part + row * D + d, y);
            if (d == 0) sink.ml[row] = make_float2(M, L);
        }
    }
}

__device__ __forceinline__ float4 cl_ld4(unsigned addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// A call's two kernels beside each other.  The few-rows kernel of a mixed call must not wait for
// the many-rows kernel (griddepcontrol.wait would), but reads what came before the call, and only
// a wait, or an acquire of what was released behind one, makes that visible.  So the word `ready`
// is cleared by a launch of its own (a workspace has no contents to count on), set by the
// many-rows kernel behind its wait, and acquired by each block of the few-rows kernel; a block that
// finds it clear waits for the many-rows kernel after all.
__global__ void paged_attn_clear_kernel(unsigned* ready) {
    pdl_wait();
    pdl_trigger();
    *ready = 0;
}
// (By the many-rows kernel: a loop in the few-rows kernel, reached or not, cost every call of it 4 us.)
__device__ __forceinline__ void clear_hints(const AttnView& a) {
    if (a.hint && blockIdx.x == 0)
        for (int i = threadIdx.x; i < a.p.batch * a.p.kv_heads; i += blockDim.x) a.hint[i] = -1;
}
__device__ __forceinline__ void release_ready(const AttnView& a) {
    if (a.ready && blockIdx.x == 0 && threadIdx.x == 0)
        asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(a.ready), "r"(1u) : "memory");
}

// CLUSTER: a cluster of 8 blocks for a tile (sequence, KV head), which join their pieces
// through each other's shared memory (no second launch).  Else the keys of all tiles are
// shared out evenly over the blocks.
constexpr int kCl = 8;

template <typename IO, typename KV, int D, int NR, bool CLUSTER>
__global__ void __launch_bounds__(FewCfg<KV, D, NR>::kWarps * 32) paged_attn_few_kernel(const __grid_constant__ AttnView a) {
    using C = FewCfg<KV, D, NR>;
    extern __shared__ __align__(1024) char smem[];
    __shared__ float2 ml[C::kWarps][C::kRows];
    // Behind the many-rows kernel of the same call nothing here reads what that one writes, so
    // the order that `ready` gives is enough.  The wait at the end keeps it for what follows.
    if (a.after_many) {
        __shared__ unsigned ready;
        if (threadIdx.x == 0) ready = ld_acquire(a.ready);
        __syncthreads();
        if (ready != 1) pdl_wait();
    } else {
        pdl_wait();
    }
    pdl_trigger();
    struct AtEnd {
        bool wait;
        __device__ ~AtEnd() {
            if (wait) pdl_wait();
        }
    } at_end{a.after_many};
    if constexpr (CLUSTER) {
        __shared__ float2 kept[C::kRows];
        __shared__ int again_done;
        const int rank = (int)cl_rank(), tile = (int)blockIdx.x / kCl;
        const int kvh = tile % a.p.kv_heads, b = tile / a.p.kv_heads;
        const PagedSeq s = paged_seq(a.p, b);
        const int rows = s.n * a.group;
        if (rows == 0 || rows > a.few_rows) return;  // (the whole cluster)
        const KeyRange kr = key_range(a, s, 0, a.few);
        const int n = (kr.hi - kr.base + kBK - 1) / kBK;  // blocks of 16 keys
        const int k_begin = kr.base + n * rank / kCl * kBK, k_end = min(kr.base + n * (rank + 1) / kCl * kBK, kr.hi);
        const Sink sink{false, true, nullptr, nullptr};
        few_piece<IO, KV, D, NR>(a, s, b, kvh, kr, k_begin, k_end, sink, smem, ml, kept);
        cluster_sync_all();
        bool again = false;
        for (int it = rank * C::kWarps * 32 + threadIdx.x; it < C::kRows * (D / 4); it += kCl * C::kWarps * 32) {
            const int row = it / (D / 4), d = it % (D / 4) * 4;
            if (row >= rows) break;
            float2 q[kCl];
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int c = 0; c < kCl; c++) {
                const unsigned at = cl_map(smem_addr(&kept[row]), c);
                q[c] = make_float2(cl_ld(at), cl_ld(at + 4));
                M = fmaxf(M, q[c].x);
            }
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < kCl; c++) {
                const float w = ex2_approx(q[c].x - (M == -INFINITY ? 0.f : M));
                const float4 z = cl_ld4(cl_map(smem_addr(smem) + (row * C::kLd + d) * 4, c));
                L = fmaf(q[c].y, w, L);
                y.x = fmaf(w, z.x, y.x), y.y = fmaf(w, z.y, y.y), y.z = fmaf(w, z.z, y.z), y.w = fmaf(w, z.w, y.w);
            }
            const float inv = 1.f / L;
            if (L == 0.f) y = make_float4(0.f, 0.f, 0.f, 0.f);
            const int token = s.start + row / a.group, head = kvh * a.group + row % a.group;
            IO* dst = reinterpret_cast<IO*>(a.out + token * a.o_row + head * a.o_head) + d;
            if (L != 0.f) y.x *= inv, y.y *= inv, y.z *= inv, y.w *= inv;
            dst[0] = (IO)y.x, dst[1] = (IO)y.y, dst[2] = (IO)y.z, dst[3] = (IO)y.w;
            again |= isnan(y.x + y.y + y.z + y.w);
            if (d == 0 && a.lse)
                a.lse[(int64_t)token * a.heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945309f;
        }
        cluster_sync_all();  // no block leaves while others read its shared memory
        if constexpr (!kAsSeen<IO>) {
            constexpr int kBlockRows = C::kWarps * 128 / D;  // rows of a block in each turn of the loop
            if (a.redo && __syncthreads_or(again))
                for (int i = rank * kBlockRows; i < rows; i += kCl * kBlockRows)
                    for (int row = i; row < min(i + kBlockRows, rows); row++)
                        redo_row_apart<IO, KV, D, C::kWarps>(a, s.start + row / a.group, kvh * a.group + row % a.group,
                                                       reinterpret_cast<float(*)[D]>(smem), ml[0], &again_done);
        }
    } else {
        // this block's units, piece by piece: a piece is what it has of one tile
        const int lane = threadIdx.x & 31;
        if (a.p.status && blockIdx.x == 0)  // the sequences that get no units are reported too
            for (int i = threadIdx.x; i < a.p.batch; i += C::kWarps * 32) paged_seq(a.p, i);
        int all, unused;
        stream_sums<C::kWarps>(a, 0, all, unused);
        const int blocks = min(a.stream, all);  // no block between others is empty
        const int c = (int)blockIdx.x;
        if (c >= blocks) return;
        // c * all / blocks in 32 bits
        const int per = all / blocks, more = all % blocks;
        int u = per * c + more * c / blocks;
        const int u_end = per * (c + 1) + more * (c + 1) / blocks;
        // the sequence of unit u: 32 sequences a step
        int b = 0, off = u;  // u's number within sequence b
        for (int b0 = 0; b0 < a.p.batch; b0 += 32) {
            const int mine = b0 + lane < a.p.batch ? stream_units(a, b0 + lane) * a.p.kv_heads : 0;
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += x;
            }
            const unsigned past = __ballot_sync(0xffffffffu, sum > off);
            if (past) {
                const int l = __ffs(past) - 1;
                off -= __shfl_sync(0xffffffffu, sum - mine, l);
                b = b0 + l;
                break;
            }
            off -= __shfl_sync(0xffffffffu, sum, 31);
        }
        while (u < u_end) {
            const int n = stream_units(a, b);  // units of a tile
            if (n == 0 || off >= n * a.p.kv_heads) {
                off -= n * a.p.kv_heads;
                if (++b >= a.p.batch) return;  // (the lengths changed under the kernel)
                continue;
            }
            const PagedSeq s = paged_seq(a.p, b);
            const KeyRange kr = key_range(a, s, 0, a.few);
            const int kvh = off / n, first = off % n, take = min(n - first, u_end - u);
            const int slot = first > 0 ? 0 : 1;  // a tile begun by an earlier block; begun here
            const int64_t at = ((int64_t)blockIdx.x * 2 + slot) * C::kRows;
            const Sink sink{take == n, false, a.strm + at * D, a.strm_ml + at};
            const int k_begin = kr.base + first * kUnit;
            few_piece<IO, KV, D, NR>(a, s, b, kvh, kr, k_begin, min(k_begin + take * kUnit, kr.hi), sink, smem, ml);
            u += take;
            off += take;
            __syncthreads();  // the shared memory is free for the next piece
        }
    }
}

// ------------------------------------------------------------ many rows
// Attention of 256 rows of a KV head on the 5th-generation tensor cores: two
// tiles of 128 rows, so that one tile's softmax runs while the other's products
// do.  Keys come 128 at a time.
//   warps 0-7, 8-15  softmax of tile 0 / 1: two threads share a row, 64 keys each.
//                    They read their scores from tensor memory, agree on the
//                    maximum through shared memory, and write their weights (16
//                    bits) back over the scores as the A operand of P.V.  (With
//                    one thread a row its chain of load, maximum, exponentials and
//                    store was longer than the products of the other tile.)
//   warp 16          one thread issues the products: for each key tile and row
//                    tile P.V, then the next key tile's Q.K.  They run in order, so
//                    a finished Q.K says that the P.V before it is finished too,
//                    and a row's thread may rescale its sums then.
//   warps 17-19      producers: the tiles' rows from their pages into the
//                    128-byte-swizzled layout the products read, by TMA or
//                    16-byte cp.async; K and V take turns in a ring of four stages.
// The running maximum is raised, and the sums rescaled, only when a score
// exceeds it by more than 2^8: weights stay below 256 (f16: 2^14), which changes
// no rounding (they are relative), and rescaling is rare.  The weights are rounded
// to the cache's 16 bits as the products take them, their sum is not.
// Of the two tiles' 128 x 128 scores the exponentials take 2048 clocks (16 a
// clock on an SM) and, at D = 128, the products as many.  A prompt of 8192
// tokens, 16/8 heads, bf16: 287 us (293 with the last pass: 938 TFLOP/s, 0.57 of the
// measured bf16 rate), at 1700 MHz under the power cap; bound by the chain scores ->
// weights -> P.V -> next scores of one tile.
constexpr int kTcThreads = 640;
constexpr int kTcProducers = 96;
constexpr int kTcRows = 256;
constexpr int kTcStages = 4;

template <int D>
struct TcCfg {
    static constexpr int kHalf = 128 * 128;             // 128 rows of 64 elements
    static constexpr int kTile = kHalf * (D / 64);      // Q, K or V of 128 rows
    static constexpr int kOffKV = 2 * kTile;
    static constexpr int kSmem = kOffKV + kTcStages * kTile + 1024;  // + alignment
    static constexpr int kO = 256;                      // tensor-memory columns: S0, S1, O0, O1
};

// Shared-memory descriptors, 128-byte swizzle, 1024 bytes from 8 rows to the next.  The
// low word holds the address / 16 and, for V, the 16 KB from 64 elements of N to the next
// (V's rows are keys, the summed dimension: its operand is N-major).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kDescK = 1u << 16, kDescV = ((128u * 128u) >> 4) << 16;

__device__ __forceinline__ unsigned elect_one() {
    unsigned r;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
    return r;
}
// The lane with `leader` set issues; addr: a descriptor's address / 16.
// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void mma_ss(unsigned leader, unsigned tmem, unsigned a, unsigned b, uint32_t idesc, bool acc) {
    asm volatile(
        "{ .reg .pred p, q; .reg .b64 da, db; setp.ne.u32 p, %4, 0; setp.ne.u32 q, %5, 0;"
        " mov.b64 da, {%1, %6}; mov.b64 db, {%2, %6};"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p; }" ::"r"(tmem),
        "r"(a | kDescK), "r"(b | kDescK), "r"(idesc), "r"((unsigned)acc), "r"(leader), "r"(kDescHi)
        : "memory");
}
// D[tmem] (+)= A[tmem] B[smem], B N-major
__device__ __forceinline__ void mma_ts(unsigned leader, unsigned tmem, unsigned a, unsigned b, uint32_t desc, uint32_t idesc,
                                       bool acc) {
    asm volatile(
        "{ .reg .pred p, q; .reg .b64 db; setp.ne.u32 p, %4, 0; setp.ne.u32 q, %5, 0; mov.b64 db, {%2, %6};"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p; }" ::"r"(tmem),
        "r"(a), "r"(b | desc), "r"(idesc), "r"((unsigned)acc), "r"(leader), "r"(kDescHi)
        : "memory");
}
__device__ __forceinline__ void commit_one(unsigned leader, unsigned mbar) {
    asm volatile(
        "{ .reg .pred q; setp.ne.u32 q, %1, 0;"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(mbar),
        "r"(leader)
        : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ f2 f2add(f2 a, f2 b) {
    f2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void tma_load_4d(unsigned dst, const CUtensorMap* map, int x, int y, int z, int w, unsigned mbar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(mbar)
        : "memory");
}
// Arrives at an mbarrier once this thread's cp.asyncs so far have landed.  The
// thread that waits for it puts the proxy fence between them and its products.
__device__ __forceinline__ void cp_async_arrive(unsigned bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// 16 columns of this warp's 32 lanes
__device__ __forceinline__ void tmem_ld16(unsigned taddr, float* v) {
    unsigned* r = reinterpret_cast<unsigned*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16]; "
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(unsigned taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(unsigned taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Bounded wait for a phase of an mbarrier: gives up after 2 s, or when another
// wait of this CTA did (failed; NULL: waits on regardless).  Inline: a call
// would hold the softmax threads to the registers of the launch.
__device__ __forceinline__ bool tc_wait(unsigned bar, unsigned parity, volatile int* failed) {
    if (mbar_try(bar, parity)) return true;
    const unsigned long long t0 = now_ns();
    for (unsigned it = 1;; it++) {
        if (mbar_try(bar, parity)) return true;
        if ((it & 63u) == 0 && ((failed && *failed) || now_ns() - t0 > kWaitNs)) {
            if (failed) *failed = 1;
            return false;
        }
    }
}

// Where the many-rows kernel runs without the other (one sequence), it reports what gets no tile.
__device__ __forceinline__ void report_one(const AttnView& a) {
    if (a.few_rows == 0 && blockIdx.x == 0 && threadIdx.x == 0 && a.p.status) paged_seq(a.p, 0);
}

// Sequence and tile of the idx-th of all tiles of `rows` rows (sequences with more than
// a.few_rows rows only), the last ones -- which see most keys -- first; b = -1: none.
__device__ __forceinline__ void find_tile(const AttnView& a, int64_t idx, int rows, int lane, int& b, int& tile) {
    // from the last sequence to the first
    b = -1;
    tile = 0;
    for (int hi = a.p.batch; hi > 0; hi -= 32) {
        const int i = hi - 1 - lane;
        int n = 0;
        if (i >= 0) {
            // (a sequence whose rows are not all there has no tiles: the grid counts those of `tokens` rows)
            const int start = a.p.q_start[i], end = a.p.q_start[i + 1];
            const int64_t d = (int64_t)end - start;
            n = start >= 0 && end <= a.p.tokens && d > 0 && d <= a.p.max_new && d * a.group > a.few_rows
                    ? (int)((d * a.group + rows - 1) / rows)
                    : 0;
        }
        int sum = n;  // tiles of lanes 0..lane
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, sum > idx);
        if (past) {
            const int l = __ffs(past) - 1;
            const int before = __shfl_sync(0xffffffffu, sum - n, l), count = __shfl_sync(0xffffffffu, n, l);
            b = hi - 1 - l;
            tile = count - 1 - (int)(idx - before);
            return;
        }
        idx -= __shfl_sync(0xffffffffu, sum, 31);
    }
}

// The producers of a block: K and V of key tiles of 128 into a ring of stages, by 96 threads.
// Key tiles that lie wholly inside the range come by TMA, a box of rows of one page by one
// thread; at its edges, where places outside must read as zeros (weights of 0 do not silence
// a NaN), and where pages do not tile 128 keys, by 16-byte cp.async.  Every push is 96
// arrivals at its stage's barrier.
template <int D, int STAGES>
struct KvFeed {
    static constexpr int kHalf = 128 * 128, kTile = kHalf * (D / 64);
    static constexpr int RC = D / 8, RPP = kTcProducers / RC;  // 16-byte chunks of a row, rows a pass takes
    const AttnView& a;
    const CUtensorMap *mk, *mv;
    int64_t (*place)[128];
    volatile int* failed;
    unsigned ring, full, empty;  // shared addresses: first stage, its two barriers (8 bytes a stage)
    int b, kvh, lo, k_begin, k_end, n, pt, boxes;
    int page0, page1, row0, row1;  // of tiles j & 1: page and position of box pt
    int x = 0;            // pushes so far
    bool ok = true;

    // chunk c of row r in a tile: half c / 8, swizzled inside its 128 bytes
    static __device__ __forceinline__ unsigned at(int r, int c) {
        return (unsigned)((c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4));
    }
    __device__ __forceinline__ bool by_tma(int j) const {
        const int k0 = k_begin + j * 128;
        return boxes > 0 && k0 >= lo && k0 + 128 <= k_end;
    }
    // asks for the pages of tile j (a tile ahead of its first push)
    __device__ __forceinline__ void look(int j) {
        if (j >= n || pt >= boxes || !by_tma(j)) return;
        const int key = k_begin + j * 128 + pt * a.box, pg = key >> a.p.page_shift;
        int id = a.p.table[(size_t)b * a.p.table_stride + pg];
        if ((unsigned)id >= (unsigned)a.p.num_pages) {
            paged_report(a.p, VB_PAGED_BAD_PAGE);
            id = a.p.num_pages;  // beyond the map: zeros
        }
        const int at = key - (pg << a.p.page_shift);
        if (j & 1)
            page1 = id, row1 = at;
        else
            page0 = id, row0 = at;
    }
    // before the first push of tile j: the places of an edge's rows, -1: zeros
    __device__ __forceinline__ void begin(int j) {
        if (by_tma(j)) return;
        asm volatile("bar.sync 1, %0;" ::"n"(kTcProducers) : "memory");  // the readers of the last such tile are done
        for (int r = pt; r < 128; r += kTcProducers) {
            const int key = k_begin + j * 128 + r;
            place[j & 1][r] = key >= lo && key < k_end ? paged_offset(a.p, b, key) : -1;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kTcProducers) : "memory");
    }
    __device__ __forceinline__ void push(int j, bool v) {
        const int st = x % STAGES;
        const unsigned bar = full + 8 * st, dst = ring + st * kTile;
        if (x >= STAGES) ok = tc_wait(empty + 8 * st, (unsigned)(x / STAGES - 1) & 1u, failed) && ok;
        x++;
        if (by_tma(j)) {
            // all arrivals by one thread, with the bytes that are on their way
            if (pt == 0) {
                if (ok) mbar_expect_tx(bar, kTile);
                mbar_arrive(bar, ok ? kTcProducers - 1 : kTcProducers);
            }
            if (pt < boxes && ok) {
#pragma unroll
                for (int h = 0; h < D / 64; h++)
                    tma_load_4d(dst + h * kHalf + pt * a.box * 128, v ? mv : mk, 64 * h, j & 1 ? row1 : row0, kvh,
                                j & 1 ? page1 : page0, bar);
            }
        } else {
            const int pr = pt / RC, pc = pt % RC;
            const char* src = (v ? a.p.v : a.p.k) + (int64_t)kvh * a.p.stride_head + pc * 16;
            if (ok) {
#pragma unroll 4
                for (int r = pr; r < 128; r += RPP) {
                    const int64_t o = place[j & 1][r];
                    cp_async16(dst + at(r, pc), o < 0 ? a.p.k : src + o, o >= 0);
                }
            }
            cp_async_arrive(bar);
        }
    }
    // nothing in flight when the block ends: the products waited for every TMA copy, unless a wait gave up
    __device__ __forceinline__ void end() {
        if (*failed)
            for (int i = max(0, x - STAGES); i < x; i++) tc_wait(full + 8 * (i % STAGES), (unsigned)(i / STAGES) & 1u, nullptr);
        cp_async_commit();
        cp_async_wait<0>();
    }
};

template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 1) paged_attn_tc_kernel(const __grid_constant__ AttnView a,
                                                                      const __grid_constant__ CUtensorMap mk,
                                                                      const __grid_constant__ CUtensorMap mv) {
    using C = TcCfg<D>;
    constexpr int NH = D / 64;
    constexpr uint32_t kFmt = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0u : 1u;
    // kind::f16: f32 accumulator, A and B of type kFmt; B's rows along the sum for P.V
    constexpr uint32_t kIdS = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t kIdPV =
        (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
    extern __shared__ char smem_raw[];
    __shared__ __align__(8) unsigned long long q_full, kv_full[kTcStages], kv_empty[kTcStages], s_full[2],
        p_full[2][2], o_full[2];
    __shared__ unsigned tmem_slot;
    __shared__ int failed;
    __shared__ int64_t place[2][128];
    __shared__ float xch[2][2][128];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, wg = t >> 7;
    pdl_wait();
    release_ready(a);
    pdl_trigger();
    clear_hints(a);
    int64_t idx = blockIdx.x;
    const int split = (int)(idx % a.many.splits);
    idx /= a.many.splits;
    const int kvh = (int)(idx % a.p.kv_heads);
    idx /= a.p.kv_heads;
    int b, tile;
    report_one(a);
    find_tile(a, idx, kTcRows, lane, b, tile);
    if (b < 0) return;
    const PagedSeq s = paged_seq(a.p, b);
    const int rows = s.n * a.group, r0 = tile * kTcRows;
    if (r0 >= rows) return;
    const KeyRange kr = key_range(a, s, r0, a.many);
    if (split >= splits_used(a.many, kr)) return;
    const int k_begin = kr.base + split * a.many.len, k_end = min(k_begin + a.many.len, kr.hi);
    // key tiles of each row tile
    int nt[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int last = min(r0 + 128 * (i + 1), rows) - 1;
        const int top = r0 + 128 * i < rows ? min(s.len - s.n + last / a.group + 1, k_end) : k_begin;
        nt[i] = max(0, (top - k_begin + 127) / 128);
    }
    const int nmax = max(nt[0], nt[1]);

    const unsigned sb = (smem_addr(smem_raw) + 1023u) & ~1023u;
    if (t == 0) {
        mbar_init(smem_addr(&q_full), 512);
        for (int i = 0; i < kTcStages; i++) {
            mbar_init(smem_addr(&kv_full[i]), kTcProducers);
            mbar_init(smem_addr(&kv_empty[i]), 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_addr(&s_full[i]), 1);
            mbar_init(smem_addr(&p_full[i][0]), 8);
            mbar_init(smem_addr(&p_full[i][1]), 8);
            mbar_init(smem_addr(&o_full[i]), 1);
        }
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tm = tmem_slot;

    if (wg < 4) {
        // ------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const int i = wg >> 1, hf = wg & 1;  // row tile; half of the keys (scores, weights) and of the dims (sums)
        const int row = t & 127, r = r0 + 128 * i + row;
        const bool live = r < rows;
        const int pos = live ? s.len - s.n + r / a.group : -1;
        const unsigned lanes = (unsigned)(32 * (warp & 3)) << 16;
        const unsigned tS = tm + 128u * i + lanes, tO = tm + C::kO + 128u * i + (D / 2) * hf + lanes;
        // q: this half's chunks of 16 bytes of its tile's rows (rows behind the last one: zeros)
        if (nt[i] > 0) {
            constexpr int RC = D / 8;
            for (int x = hf * 128 + row; x < 128 * RC; x += 256) {
                const int qr = x / RC, c = x % RC, y = r0 + 128 * i + qr;
                const bool real = y < rows;
                const int z = real ? y : 0;
                cp_async16(sb + i * C::kTile + KvFeed<D, kTcStages>::at(qr, c),
                           a.q + (int64_t)(s.start + z / a.group) * a.q_row +
                               (int64_t)(kvh * a.group + z % a.group) * a.q_head + c * 16,
                           real);
            }
        }
        if (!(a.stall && blockIdx.x == 0 && t == 0)) cp_async_arrive(smem_addr(&q_full));
        const float sc = fabsf(a.scale_log2);
        const bool flip = a.scale_log2 < 0.f;
        float m = -INFINITY, l = 0.f;  // m: the maximum the sums are relative to; l: this half's sum
        const int n = nt[i], pair = 2 + 4 * i + (warp & 3);
        // what the row's other thread says of it (the two warps of 32 rows meet)
        auto other = [&](float v) {
            xch[i][hf][row] = v;
            asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
            return xch[i][hf ^ 1][row];
        };
        bool ok = true;
        // (no way out of the loop when a wait fails: the other warp of the pair counts on this one)
        for (int j = 0; j < n; j++) {
            // columns this row sees: lo .. hi
            const int k0 = k_begin + j * 128 + 64 * hf;
            const int hi = min(pos, k_end - 1) - k0, lo = a.window > 0 ? pos - a.window + 1 - k0 : 0;
            const bool edge = __any_sync(0xffffffffu, hi < 63 || lo > 0);
            ok = tc_wait(smem_addr(&s_full[i]), (unsigned)j & 1u, &failed) && ok;
            __syncwarp();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float x[64];
            tmem_ld64(tS + 64 * hf, x);
            if (flip) {
#pragma unroll
                for (int c = 0; c < 64; c++) x[c] = -x[c];
            }
            if (edge) {
#pragma unroll
                for (int c = 0; c < 64; c++) x[c] = c <= hi && c >= lo ? x[c] : -INFINITY;
            }
            float mx[4] = {fmaxf(x[0], x[1]), fmaxf(x[2], x[3]), fmaxf(x[4], x[5]), fmaxf(x[6], x[7])};
#pragma unroll
            for (int c = 8; c < 64; c += 8)
#pragma unroll
                for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], x[c + 2 * e], x[c + 2 * e + 1]);
            float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc;
            top = fmaxf(top, other(top));
            top -= kLift<T>;
            const bool raise = top > m + 8.f || (m == -INFINITY && top > m);
            if (__any_sync(0xffffffffu, raise)) {  // in both warps of the pair alike
                const float mn = raise ? top : m;
                const float f = m == -INFINITY ? 0.f : ex2_approx(m - mn);
                l *= f;
                m = mn;
                if (j > 0) {
#pragma unroll
                    for (int c = 0; c < D / 2; c += 16) {
                        float o[16];
                        tmem_ld16(tO + c, o);
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] *= f;
                        tmem_st16(tO + c, reinterpret_cast<const uint32_t*>(o));
                    }
                }
            }
            const float mb = m == -INFINITY ? 0.f : m;
            f2 sum[2] = {0ull, 0ull};
            const f2 sc2 = f2pack(sc, sc), mb2 = f2pack(-mb, -mb);
            // the scores of both halves have been read (other() above): the weights may go over them
            // 16 keys a step.  The products of the first 32 (of each half) may start while the others
            // are made; their stores are waited for a step later, when they have long landed.
            auto publish = [&](int h) {
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_addr(&p_full[i][h]), 1);
            };
#pragma unroll
            for (int h = 0; h < 4; h++) {
                uint32_t w[8];
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                    const f2 y = f2fma(f2pack(x[16 * h + c], x[16 * h + c + 1]), sc2, mb2);
                    float p0, p1;
                    f2unpack(y, p0, p1);
                    p0 = ex2_approx(p0);
                    p1 = ex2_approx(p1);
                    sum[(c >> 1) & 1] = f2add(sum[(c >> 1) & 1], f2pack(p0, p1));
                    w[c / 2] = pack2<T>(p0, p1);
                }
                if (h == 2) publish(0);
                tmem_st8(tS + 32 * hf + 8 * h, w);
            }
            publish(1);
            l += f2sum(sum[0]) + f2sum(sum[1]);
        }
        if (n > 0) ok = tc_wait(smem_addr(&o_full[i]), 0u, &failed) && ok;
        ok = ok && !*(volatile int*)&failed;  // (where another wait gave up the products behind it were left out)
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");  // the last maximum has been read
        l += other(ok ? l : nanf(""));  // rows of which a wait gave up are NaN, not what the output held
        if (!ok) l = nanf("");
        cp_async_wait_all();  // q's, had nobody waited for them
        const bool last = a.many.splits == 1;
        const float inv = last ? 1.f / l : 1.f;
        const int rr = min(r, rows - 1);
        const int token = s.start + rr / a.group, head = kvh * a.group + rr % a.group;
        const int64_t th = (int64_t)token * a.heads + head;
        const int64_t pth = (int64_t)split * a.p.tokens * a.heads + th;
#pragma unroll
        for (int c = 0; c < D / 2; c += 32) {
            float o[32];
            if (n > 0) {
                tmem_ld32(tO + c, o);
            } else {
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = 0.f;
            }
            if (live) {
                const int d = (D / 2) * hf + c;
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = l == 0.f ? 0.f : o[e] * inv;
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    if (last)
                        Eight<T>::store(a.out + token * a.o_row + head * a.o_head + (d + e) * sizeof(T), o + e);
                    else
                        Eight<float>::store(a.part + pth * D + d + e, o + e);
                }
            }
        }
        if (live && hf == 0) {
            if (!last)
                a.part_ml[pth] = make_float2(l == 0.f ? -INFINITY : m, l);
            else if (a.lse)
                a.lse[th] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 16) {
            // ------------------------------------------------- products
            // The whole warp runs this, one lane's instructions count: what the products take
            // (descriptors, addresses) then stays in uniform registers.  A single lane's branch
            // moved every operand there first and issued at half the tensor cores' pace.
            const unsigned leader = elect_one();
            const unsigned utm = __shfl_sync(0xffffffffu, tm, 0);
            const int n0 = __shfl_sync(0xffffffffu, nt[0], 0), n1 = __shfl_sync(0xffffffffu, nt[1], 0);
            const int nm = max(n0, n1);
            const int k_lo = __shfl_sync(0xffffffffu, kr.lo - k_begin, 0), k_hi = __shfl_sync(0xffffffffu, k_end - k_begin, 0);
            const unsigned q_d = (sb & 0x3FFFFu) >> 4, kv_d = q_d + (C::kOffKV >> 4);
            bool ok = nm > 0 && tc_wait(smem_addr(&q_full), 0u, &failed);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            auto wait_kv = [&](int push) {
                ok = ok && tc_wait(smem_addr(&kv_full[push % kTcStages]), (unsigned)(push / kTcStages) & 1u, &failed);
                // rows that came by cp.async, not TMA
                const int k0 = (push >> 1) * 128;
                if (!a.box || k0 < k_lo || k0 + 128 > k_hi) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                ok = __all_sync(0xffffffffu, ok);
            };
            auto qk = [&](int i, int j) {
                if (ok) {
                    const unsigned qd = q_d + i * (C::kTile >> 4), kd = kv_d + (2 * j % kTcStages) * (C::kTile >> 4);
#pragma unroll
                    for (int h = 0; h < NH; h++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            mma_ss(leader, utm + 128u * i, qd + h * (C::kHalf >> 4) + 2 * k, kd + h * (C::kHalf >> 4) + 2 * k,
                                   kIdS, h > 0 || k > 0);
                }
                commit_one(leader, smem_addr(&s_full[i]));
            };
            if (nm > 0) {
                wait_kv(0);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (n0 > 0) qk(0, 0);
                if (n1 > 0) qk(1, 0);
                commit_one(leader, smem_addr(&kv_empty[0]));
            }
            if (nm > 0) wait_kv(1);
            if (nm > 1) wait_kv(2);
            for (int j = 0; j < nm; j++) {
                const unsigned vd = kv_d + ((2 * j + 1) % kTcStages) * (C::kTile >> 4);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int ni = i ? n1 : n0;
                    if (j >= ni) continue;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        ok = ok && tc_wait(smem_addr(&p_full[i][h]), (unsigned)j & 1u, &failed);
                        ok = __all_sync(0xffffffffu, ok);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (!ok) continue;
                        // keys 32 h .. and 64 + 32 h ..
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            const int k = 2 * h + (y & 1) + 4 * (y >> 1);
                            mma_ts(leader, utm + C::kO + 128u * i, utm + 128u * i + 8u * k, vd + 128 * k, kDescV, kIdPV,
                                   j > 0 || h > 0 || y > 0);
                        }
                    }
                    if (j + 1 < ni)
                        qk(i, j + 1);
                    else
                        commit_one(leader, smem_addr(&o_full[i]));
                }
                commit_one(leader, smem_addr(&kv_empty[(2 * j + 1) % kTcStages]));
                if (j + 1 < nm) {
                    commit_one(leader, smem_addr(&kv_empty[(2 * j + 2) % kTcStages]));
                    // the next key tile's V and the K after it, asked after while these products run
                    wait_kv(2 * j + 3);
                    if (j + 2 < nm) wait_kv(2 * j + 4);
                }
            }
            // every product has landed before the tensor memory goes
            if (n0 > 0) tc_wait(smem_addr(&o_full[0]), 0u, nullptr);
            if (n1 > 0) tc_wait(smem_addr(&o_full[1]), 0u, nullptr);
        } else {
            // ------------------------------------------------- producers
            const int pt = t - (kTcThreads - kTcProducers);
            KvFeed<D, kTcStages> feed{a, &mk, &mv, place, &failed, sb + C::kOffKV, smem_addr(kv_full), smem_addr(kv_empty),
                      b, kvh, kr.lo, k_begin, k_end, nmax, pt, a.box ? 128 / a.box : 0};
            feed.look(0);
            for (int j = 0; j < nmax; j++) {
                feed.begin(j);
                feed.look(j + 1);
                feed.push(j, false);
                feed.push(j, true);
            }
            feed.end();
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 16)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512) : "memory");
    if (t == 0 && failed) paged_report(a.p, VB_PAGED_TIMEOUT);
}

// The same for f32 rows, with f32's precision: one tile of 128 rows, q and the weights as
// three bf16 terms (all 24 bits).  Over a bf16 cache a product is three; over an f32 cache
// K and V are three terms too, made by the producers, and a product is the six that reach
// 24 bits (high x high down to the pairs of weight 2^-16).  The scores of two key tiles
// take turns in tensor memory, so that one's softmax runs while the products of the
// other's do: 1536 clocks each for Q.K and P.V of 128 keys at D = 128 (bf16 cache) against
// about 1500 of softmax.  P.V of a key tile is summed apart and added to the running sums,
// which the softmax threads hold, by FMAs: the tensor cores' own accumulation cuts bits off.
// Tensor memory: scores 2 x 128 columns, over which the high and middle terms of the
// weights go; P.V 128; the low terms 2 x 64.
// A prompt of 4096 tokens, 16/8 heads: f32 cache 400 us (3214 us by 16-row tiles of the
// few-rows kernel), bf16 cache 180.  Two chunks of 512 beside 31 decodes, bf16 cache: 125 us in all (348).
constexpr int kExRows = 128;

template <typename KV, int D>
struct ExCfg {
    static constexpr bool kF32 = sizeof(KV) == 4;
    static constexpr int kKeys = kF32 ? 64 : 128;       // of a tile
    static constexpr int kThreads = kF32 ? 512 : 384;   // 8 warps of softmax, one of products, the rest producers
    static constexpr int kProducers = kThreads - 288;
    static constexpr int kStages = kF32 ? 2 : 3;
    static constexpr int kQ = 128 * 128 * (D / 64);     // a term of q
    static constexpr int kHalf = kKeys * 128;           // 64 dims of K's or V's rows
    static constexpr int kTerm = kHalf * (D / 64);      // a term of K or V
    static constexpr int kStage = kTerm * (kF32 ? 3 : 1);
    static constexpr int kOffKV = 3 * kQ;
    static constexpr int kSmem = kOffKV + kStages * kStage + 1024;
    static constexpr int kPV = 256, kLow = 384;
    // which terms of the left and the right operand make a product, the small ones first
    static constexpr int kProducts = kF32 ? 6 : 3;
    static __device__ __forceinline__ constexpr int left(int i) {
        return kF32 ? (i == 0 ? 2 : i == 2 || i == 3 ? 1 : 0) : 2 - i;
    }
    static __device__ __forceinline__ constexpr int right(int i) {
        return kF32 ? (i == 1 ? 2 : i == 2 || i == 4 ? 1 : 0) : 0;
    }
};
static_assert(ExCfg<float, 128>::kProducers == 224 && ExCfg<__nv_bfloat16, 128>::kProducers == kTcProducers, "warps");

// KvFeed's counterpart for an f32 cache: rows of the pages, eight elements at a time, through
// registers into three bf16 tiles.
template <int D>
struct SplitFeed {
    using C = ExCfg<float, D>;
    const AttnView& a;
    int64_t (*place)[128];
    volatile int* failed;
    unsigned ring, full, empty;
    int b, kvh, lo, k_begin, k_end, n, pt;
    int x = 0;
    bool ok = true;

    __device__ __forceinline__ void look(int) {}
    __device__ __forceinline__ void begin(int j) {
        asm volatile("bar.sync 1, %0;" ::"n"(C::kProducers) : "memory");  // the readers of tile j - 2 are done
        if (pt < C::kKeys) {
            const int key = k_begin + j * C::kKeys + pt;
            place[j & 1][pt] = key >= lo && key < k_end ? paged_offset(a.p, b, key) : -1;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(C::kProducers) : "memory");
    }
    __device__ __forceinline__ void push(int j, bool v) {
        constexpr int RC = D / 8, ITEMS = C::kKeys * RC, PER = (ITEMS + C::kProducers - 1) / C::kProducers;
        const int st = x % C::kStages;
        const char* src = (v ? a.p.v : a.p.k) + (int64_t)kvh * a.p.stride_head;
        float f[PER][8];
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int it = i * C::kProducers + pt, r = it / RC, c = it % RC;
            const int64_t o = it < ITEMS ? place[j & 1][r] : -1;
            if (o >= 0) {
                Eight<float>::load(src + o + c * 32, f[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) f[i][e] = 0.f;
            }
        }
        if (x >= C::kStages) ok = tc_wait(empty + 8 * st, (unsigned)(x / C::kStages - 1) & 1u, failed) && ok;
        x++;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int it = i * C::kProducers + pt, r = it / RC, c = it % RC;
            if (it >= ITEMS) break;
            uint32_t w[3][4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t tt[3];
                split_terms<__nv_bfloat16, 3>(f[i][2 * e], f[i][2 * e + 1], tt);
                w[0][e] = tt[0], w[1][e] = tt[1], w[2][e] = tt[2];
            }
            const unsigned at = ring + st * C::kStage + (unsigned)((c >> 3) * C::kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4));
#pragma unroll
            for (int y = 0; y < 3; y++)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + y * C::kTerm), "r"(w[y][0]), "r"(w[y][1]),
                             "r"(w[y][2]), "r"(w[y][3])
                             : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(full + 8 * st, 1);
    }
    __device__ __forceinline__ void end() {}
};

template <typename KV, int D>
__global__ void __launch_bounds__(ExCfg<KV, D>::kThreads, 1)
    paged_attn_exact_kernel(const __grid_constant__ AttnView a, const __grid_constant__ CUtensorMap mk,
                            const __grid_constant__ CUtensorMap mv) {
    using C = ExCfg<KV, D>;
    constexpr int NH = D / 64, kStages = C::kStages, W = C::kKeys / 2;  // W: keys of a softmax thread
    constexpr uint32_t kIdS = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(C::kKeys >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t kDescVE = (uint32_t)(C::kHalf >> 4) << 16;  // from 64 dims of V to the next
    constexpr uint32_t kIdPV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
    extern __shared__ char smem_raw[];
    __shared__ __align__(8) unsigned long long q_full, kv_full[kStages], kv_empty[kStages], s_full[2], p_full[2],
        pv_full, pv_free;
    __shared__ unsigned tmem_slot;
    __shared__ int failed;
    __shared__ int64_t place[2][128];
    __shared__ float xch[2][2][128];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, wg = t >> 7;
    pdl_wait();
    release_ready(a);
    pdl_trigger();
    clear_hints(a);
    int64_t idx = blockIdx.x;
    const int split = (int)(idx % a.many.splits);
    idx /= a.many.splits;
    const int kvh = (int)(idx % a.p.kv_heads);
    idx /= a.p.kv_heads;
    int b, tile;
    report_one(a);
    find_tile(a, idx, kExRows, lane, b, tile);
    if (b < 0) return;
    const PagedSeq s = paged_seq(a.p, b);
    const int rows = s.n * a.group, r0 = tile * kExRows;
    if (r0 >= rows) return;
    const KeyRange kr = key_range(a, s, r0, a.many);
    if (split >= splits_used(a.many, kr)) return;
    const int k_begin = kr.base + split * a.many.len, k_end = min(k_begin + a.many.len, kr.hi);
    const int n = max(0, (k_end - k_begin + C::kKeys - 1) / C::kKeys);

    const unsigned sb = (smem_addr(smem_raw) + 1023u) & ~1023u;
    if (t == 0) {
        mbar_init(smem_addr(&q_full), 8);
        for (int i = 0; i < kStages; i++) {
            mbar_init(smem_addr(&kv_full[i]), C::kProducers);
            mbar_init(smem_addr(&kv_empty[i]), 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_addr(&s_full[i]), 1);
            mbar_init(smem_addr(&p_full[i]), 8);
        }
        mbar_init(smem_addr(&pv_full), 1);
        mbar_init(smem_addr(&pv_free), 8);
        failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const unsigned tm = tmem_slot;

    if (wg < 2) {
        // ------------------------------------------------------ softmax
        if constexpr (C::kF32)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        else
            asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int hf = wg, row = t & 127, r = r0 + row;  // half of the keys (scores, weights) and of the dims (sums)
        const bool live = r < rows;
        const int pos = live ? s.len - s.n + r / a.group : -1;
        const int rr = min(r, rows - 1);
        const int token = s.start + rr / a.group, head = kvh * a.group + rr % a.group;
        // q's three terms, 16 bytes of each a step
        for (int i = t; i < 128 * (D / 8); i += 256) {
            const int qr = i / (D / 8), c = i % (D / 8), y = min(r0 + qr, rows - 1);
            const char* src = a.q + (int64_t)(s.start + y / a.group) * a.q_row +
                              (int64_t)(kvh * a.group + y % a.group) * a.q_head + c * 32;
            float f[8];
            Eight<float>::load(src, f);
            uint32_t w[3][4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t tt[3];
                split_terms<__nv_bfloat16, 3>(f[2 * e], f[2 * e + 1], tt);
                w[0][e] = tt[0], w[1][e] = tt[1], w[2][e] = tt[2];
            }
            const unsigned at = KvFeed<D, 3>::at(qr, c);
#pragma unroll
            for (int x = 0; x < 3; x++)
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sb + x * C::kQ + at), "r"(w[x][0]),
                             "r"(w[x][1]), "r"(w[x][2]), "r"(w[x][3])
                             : "memory");
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && !(a.stall && blockIdx.x == 0 && t == 0)) mbar_arrive(smem_addr(&q_full), 1);

        const unsigned lanes = (unsigned)(32 * (warp & 3)) << 16;
        const unsigned tPV = tm + C::kPV + (D / 2) * hf + lanes;
        const int pair = 2 + (warp & 3);
        // (two places in turn: the next key tile's scores may be there before the other warp has read)
        auto other = [&](float v, int turn) {
            xch[turn][hf][row] = v;
            asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
            return xch[turn][hf ^ 1][row];
        };
        float m = -INFINITY, l = 0.f, alpha = 0.f;
        float o[D / 2];
#pragma unroll
        for (int d = 0; d < D / 2; d++) o[d] = 0.f;
        bool ok = true;
        // adds key tile j's P.V, which was scaled to the maximum that alpha leads from the sums' to
        auto fold = [&](int j) {
            ok = tc_wait(smem_addr(&pv_full), (unsigned)j & 1u, &failed) && ok;
            __syncwarp();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int d = 0; d < D / 2; d += 16) {
                float v[16];
                tmem_ld16(tPV + d, v);
#pragma unroll
                for (int e = 0; e < 16; e++) o[d + e] = fmaf(o[d + e], alpha, v[e]);
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&pv_free), 1);
        };
        // (no way out of the loop when a wait fails: the other warp of the pair counts on this one)
        for (int j = 0; j < n; j++) {
            const unsigned tS = tm + 128u * (j & 1) + lanes, tL = tm + C::kLow + 64u * (j & 1) + W / 2 * hf + lanes;
            ok = tc_wait(smem_addr(&s_full[j & 1]), (unsigned)(j >> 1) & 1u, &failed) && ok;
            __syncwarp();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float x[W];
            if constexpr (W == 64)
                tmem_ld64(tS + W * hf, x);
            else
                tmem_ld32(tS + W * hf, x);
            const int k0 = k_begin + j * C::kKeys + W * hf;
            const int hi = min(pos, k_end - 1) - k0, lo = a.window > 0 ? pos - a.window + 1 - k0 : 0;
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < W; c++) {
                x[c] = c <= hi && c >= lo ? x[c] * a.scale_log2 : -INFINITY;
                top = fmaxf(top, x[c]);
            }
            const float mn = fmaxf(m, fmaxf(top, other(top, j & 1)));
            const float mb = mn == -INFINITY ? 0.f : mn;
            const float f = ex2_approx(m - mb);
            m = mn;
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < W / 16; h++) {
                uint32_t w[3][8];
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                    const float p0 = ex2_approx(x[16 * h + c] - mb), p1 = ex2_approx(x[16 * h + c + 1] - mb);
                    sum += p0 + p1;
                    uint32_t tt[3];
                    split_terms<__nv_bfloat16, 3>(p0, p1, tt);
                    w[0][c / 2] = tt[0], w[1][c / 2] = tt[1], w[2][c / 2] = tt[2];
                }
                tmem_st8(tS + W / 2 * hf + 8 * h, w[0]);
                tmem_st8(tS + W + W / 2 * hf + 8 * h, w[1]);
                tmem_st8(tL + 8 * h, w[2]);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&p_full[j & 1]), 1);
            l = fmaf(l, f, sum);
            if (j > 0) fold(j - 1);
            alpha = f;
        }
        if (n > 0) fold(n - 1);
        ok = ok && !*(volatile int*)&failed;  // (see the kernel above)
        asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");  // the last maximum has been read
        l += other(ok ? l : nanf(""), 0);
        if (!ok) l = nanf("");
        const bool last = a.many.splits == 1;
        const float inv = last ? 1.f / l : 1.f;
        const int64_t th = (int64_t)token * a.heads + head;
        const int64_t pth = (int64_t)split * a.p.tokens * a.heads + th;
        if (live) {
            float* dst = last ? reinterpret_cast<float*>(a.out + token * a.o_row + head * a.o_head) : a.part + pth * D;
#pragma unroll
            for (int d = 0; d < D / 2; d += 8) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = l == 0.f ? 0.f : o[d + e] * inv;
                Eight<float>::store(dst + (D / 2) * hf + d, y);
            }
            if (hf == 0) {
                if (!last)
                    a.part_ml[pth] = make_float2(m, l);
                else if (a.lse)
                    a.lse[th] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
            }
        }
    } else {
        if constexpr (C::kF32)
            asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        else
            asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 8) {
            // ------------------------------------------------- products (see the kernel above)
            const unsigned leader = elect_one();
            const unsigned utm = __shfl_sync(0xffffffffu, tm, 0);
            const int nk = __shfl_sync(0xffffffffu, n, 0);
            const int k_lo = __shfl_sync(0xffffffffu, kr.lo - k_begin, 0), k_hi = __shfl_sync(0xffffffffu, k_end - k_begin, 0);
            const unsigned q_d = (sb & 0x3FFFFu) >> 4, kv_d = q_d + (C::kOffKV >> 4);
            bool ok = nk > 0 && tc_wait(smem_addr(&q_full), 0u, &failed);
            // K and V come in the order they are used: K0, K1, V0, K2, V1, ...
            auto wait_kv = [&](int push, int j) {
                ok = ok && tc_wait(smem_addr(&kv_full[push % kStages]), (unsigned)(push / kStages) & 1u, &failed);
                // rows that came by cp.async, not TMA (the f32 producers put the fence themselves)
                if (!C::kF32 && (!a.box || j * 128 < k_lo || j * 128 + 128 > k_hi))
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                ok = __all_sync(0xffffffffu, ok);
            };
            int push = 0;
            auto qk = [&](int j) {
                wait_kv(push, j);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (ok) {
                    const unsigned kd = kv_d + (push % kStages) * (C::kStage >> 4);
#pragma unroll
                    for (int x = 0; x < C::kProducts; x++)
#pragma unroll
                        for (int h = 0; h < NH; h++)
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                mma_ss(leader, utm + 128u * (j & 1), q_d + C::left(x) * (C::kQ >> 4) + h * ((128 * 128) >> 4) + 2 * k,
                                       kd + C::right(x) * (C::kTerm >> 4) + h * (C::kHalf >> 4) + 2 * k, kIdS,
                                       x > 0 || h > 0 || k > 0);
                }
                commit_one(leader, smem_addr(&s_full[j & 1]));
                commit_one(leader, smem_addr(&kv_empty[push % kStages]));
                push++;
            };
            if (nk > 0) qk(0);
            for (int j = 0; j < nk; j++) {
                if (j + 1 < nk) qk(j + 1);
                wait_kv(push, j);
                ok = ok && tc_wait(smem_addr(&p_full[j & 1]), (unsigned)(j >> 1) & 1u, &failed);
                if (j > 0) ok = ok && tc_wait(smem_addr(&pv_free), (unsigned)(j - 1) & 1u, &failed);
                ok = __all_sync(0xffffffffu, ok);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (ok) {
                    const unsigned vd = kv_d + (push % kStages) * (C::kStage >> 4);
#pragma unroll
                    for (int x = 0; x < C::kProducts; x++) {
                        const unsigned tp = C::left(x) == 2 ? utm + C::kLow + 64u * (j & 1) : utm + 128u * (j & 1) + W * C::left(x);
#pragma unroll
                        for (int k = 0; k < C::kKeys / 16; k++)
                            mma_ts(leader, utm + C::kPV, tp + 8u * k, vd + C::right(x) * (C::kTerm >> 4) + 128 * k, kDescVE,
                                   kIdPV, x > 0 || k > 0);
                    }
                }
                commit_one(leader, smem_addr(&pv_full));
                commit_one(leader, smem_addr(&kv_empty[push % kStages]));
                push++;
            }
            // every product has landed before the tensor memory goes
            if (nk > 0) tc_wait(smem_addr(&pv_full), (unsigned)(nk - 1) & 1u, nullptr);
        } else {
            // ------------------------------------------------- producers
            const int pt = t - 288;
            auto feed = [&] {
                if constexpr (C::kF32)
                    return SplitFeed<D>{a, place, &failed, sb + C::kOffKV, smem_addr(kv_full), smem_addr(kv_empty),
                                        b, kvh, kr.lo, k_begin, k_end, n, pt};
                else
                    return KvFeed<D, kStages>{a, &mk, &mv, place, &failed, sb + C::kOffKV, smem_addr(kv_full),
                                              smem_addr(kv_empty), b, kvh, kr.lo, k_begin, k_end, n, pt,
                                              a.box ? 128 / a.box : 0};
            }();
            feed.look(0);
            feed.look(1);
            if (n > 0) {
                feed.begin(0);
                feed.push(0, false);
            }
            for (int j = 0; j < n; j++) {
                if (j + 1 < n) {
                    feed.begin(j + 1);
                    feed.push(j + 1, false);
                }
                feed.push(j, true);
                feed.look(j + 2);
            }
            feed.end();
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 8)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512) : "memory");
    if (t == 0 && failed) paged_report(a.p, VB_PAGED_TIMEOUT);
}

// Joins the splits of a row of the many-rows kernels: a warp per (token, head).
template <typename IO, int D>
__global__ void __launch_bounds__(128) paged_attn_merge_kernel(const __grid_constant__ AttnView a) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t th = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (th >= (int64_t)a.p.tokens * a.heads) return;
    const int token = (int)(th / a.heads), head = (int)(th % a.heads);
    const int b = paged_find_seq(a.p.q_start, a.p.batch, token, lane);
    const PagedSeq s = paged_seq(a.p, b);
    if (!s.ok || token < s.start || token >= s.start + s.n) return;
    const int r = (token - s.start) * a.group + head % a.group;
    if (s.n * a.group <= a.few_rows) return;
    const int used = splits_used(a.many, key_range(a, s, r / a.many.rows * a.many.rows, a.many));
    const int64_t step = (int64_t)a.p.tokens * a.heads;
    constexpr int E = D / 32;
    float y[E] = {}, M = -INFINITY, L = 0.f;
    for (int x = lane; x < used; x += 32) M = fmaxf(M, a.part_ml[x * step + th].x);
    M = warp_max(M);
    const float mb = M == -INFINITY ? 0.f : M;
    for (int x = 0; x < used; x++) {
        const float2 p = a.part_ml[x * step + th];
        const float w = ex2_approx(p.x - mb);
        L = fmaf(p.y, w, L);
        const float* src = a.part + (x * step + th) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; e++) y[e] = fmaf(w, src[e], y[e]);
    }
    const float inv = 1.f / L;
    IO* dst = reinterpret_cast<IO*>(a.out + token * a.o_row + head * a.o_head) + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) dst[e] = (IO)(L == 0.f ? 0.f : y[e] * inv);
    if (a.lse && lane == 0) a.lse[th] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945309f;
}

// Joins the pieces of a shared-out tile's rows: grid over (sequence, KV head, group of ROWS
// tile rows), 8 warps, 8 / ROWS of them for a row, taking turns at its pieces.  One row a
// block where there are few blocks (a long sequence has dozens of pieces), eight otherwise
// (every block adds up the batch's lengths).  REDO: looks at the rows (AttnView::redo; the code for it,
// reached or not, cost a mixed batch 2 us).
constexpr int kJoinWarps = 8;
template <typename IO, typename KV, int D, int ROWS, bool REDO>
__global__ void __launch_bounds__(kJoinWarps * 32, 5) paged_attn_join_kernel(const __grid_constant__ AttnView a, int groups) {
    constexpr int W = kJoinWarps / ROWS;  // warps of a row
    __shared__ float sums[kJoinWarps][D];
    __shared__ float2 ml[kJoinWarps];
    __shared__ int done;
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = (int)(blockIdx.x % groups) * ROWS + warp / W, kvh = (int)(blockIdx.x / groups % a.p.kv_heads);
    const int b = (int)(blockIdx.x / groups / a.p.kv_heads);
    int all, u0;
    stream_sums<kJoinWarps>(a, b, all, u0);
    const int n = stream_units(a, b);
    if (n == 0) return;
    const PagedSeq s = paged_seq(a.p, b);
    u0 += kvh * n;
    // the block of unit u: the last c with c W / N <= u, rounded down
    const int blocks = min(a.stream, all);
    const int c0 = (int)(((int64_t)(u0 + 1) * blocks - 1) / all), c1 = (int)(((int64_t)(u0 + n) * blocks - 1) / all);
    const int used = c1 - c0 + 1;
    const bool live = r < s.n * a.group;
    // the block's rows, once they are written: taken again where one has a NaN
    auto look = [&](bool again) {
        if constexpr (REDO) {
            const int first = r - warp / W;
            if (__syncthreads_or(again))
                for (int row = first; row < min(first + ROWS, s.n * a.group); row++)
                    redo_row_apart<IO, KV, D, kJoinWarps>(a, s.start + row / a.group, kvh * a.group + row % a.group, sums, ml,
                                                          &done);
        }
    };
    if (used == 1) {  // written by the kernel itself
        if constexpr (REDO) {
            bool again = false;
            if (live && warp % W == 0) {
                const int token = s.start + r / a.group, head = kvh * a.group + r % a.group;
                const IO* y = reinterpret_cast<const IO*>(a.out + token * a.o_row + head * a.o_head);
#pragma unroll
                for (int e = 0; e < D / 32; e++) again |= isnan((float)y[lane + 32 * e]);
            }
            look(again);
        }
        return;
    }
    // slot 1 of block c0, then slot 0 of the next ones
    auto at = [&](int x) { return ((int64_t)(c0 + x) * 2 + (x == 0)) * a.few.rows + r; };
    float M = -INFINITY, L = 0.f;
    constexpr int E = D / 32;
    float y[E] = {};
    if (live) {
        for (int x = lane; x < used; x += 32) M = fmaxf(M, a.strm_ml[at(x)].x);
        M = warp_max(M);
        const float mb = M == -INFINITY ? 0.f : M;
        for (int x = lane; x < used; x += 32) {
            const float2 p = a.strm_ml[at(x)];
            L = fmaf(p.y, ex2_approx(p.x - mb), L);
        }
        L = warp_sum(L);
#pragma unroll 4
        for (int x = warp % W; x < used; x += W) {
            const float w = ex2_approx(a.strm_ml[at(x)].x - mb);
            const float* src = a.strm + at(x) * D + lane * E;
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = fmaf(w, src[e], y[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) sums[warp][lane * E + e] = y[e];
    __syncthreads();
    bool again = false;
    if (live && warp % W == 0) {
        const int token = s.start + r / a.group, head = kvh * a.group + r % a.group;
        const float inv = 1.f / L;
        IO* dst = reinterpret_cast<IO*>(a.out + token * a.o_row + head * a.o_head);
#pragma unroll
        for (int e = 0; e < E; e++) {
            float z = 0.f;
#pragma unroll
            for (int x = 0; x < W; x++) z += sums[warp + x][lane + 32 * e];
            dst[lane + 32 * e] = (IO)(L == 0.f ? 0.f : z * inv);
            again |= isnan(z * inv) && L != 0.f;
        }
        if (a.lse && lane == 0)
            a.lse[(int64_t)token * a.heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * 0.693147180559945309f;
    }
    look(again);
}

// A tile's rows of several tokens see different keys, and a weight of 0 times an infinity or
// NaN in a v that a row does not see is NaN.  So rows that came out non-finite are looked at
// again (redo_row).  A warp looks at 2 KB of (token, head) rows, 16 bytes a lane and load, and
// where all is finite that is all it does: 6 us after a prompt of 8192 tokens (293 us with it,
// 287 without, in turns), 2 after 256 tokens, so a launch and its wait more than the 33 MB out of
// L2; by 2-byte loads it was 14 us.
constexpr int kCheckLoads = 4;
template <typename IO, int D>
constexpr int check_rows() { return kCheckLoads * 512 / (D * (int)sizeof(IO)); }

// some value of a 16-byte chunk has an exponent of all ones
__device__ __forceinline__ bool any_nonfinite(uint4 c, float) {
    constexpr unsigned e = 0x7f800000u;
    return (c.x & e) == e || (c.y & e) == e || (c.z & e) == e || (c.w & e) == e;
}
__device__ __forceinline__ bool any_nonfinite16(uint4 c, unsigned e) {
    const unsigned hi = e << 16;
    return (c.x & e) == e || (c.x & hi) == hi || (c.y & e) == e || (c.y & hi) == hi || (c.z & e) == e ||
           (c.z & hi) == hi || (c.w & e) == e || (c.w & hi) == hi;
}
__device__ __forceinline__ bool any_nonfinite(uint4 c, __nv_bfloat16) { return any_nonfinite16(c, 0x7f80u); }
__device__ __forceinline__ bool any_nonfinite(uint4 c, __half) { return any_nonfinite16(c, 0x7c00u); }

template <typename IO, typename KV, int D>
__global__ void __launch_bounds__(128, 8) paged_attn_check_kernel(const __grid_constant__ AttnView a) {
    constexpr int kLanes = D * sizeof(IO) / 16, kPass = 32 / kLanes, R = check_rows<IO, D>();  // lanes a row, rows a load
    __shared__ float sums[4][D];
    __shared__ float2 ml[4];
    __shared__ unsigned rows[4];
    __shared__ int done;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned all = (unsigned)(a.p.tokens * (int64_t)a.heads);  // below 2^31
    // A load takes kPass rows; those of a block lie far apart, so that the rows of one bad tile are spread over
    // many blocks.
    auto row_of = [&](int w, int r) {
        return ((unsigned)(r / kPass * 4 + w) * gridDim.x + blockIdx.x) * kPass + r % kPass;
    };
    uint4 y[kCheckLoads];
#pragma unroll
    for (int i = 0; i < kCheckLoads; i++) {
        const unsigned th = min(row_of(warp, i * kPass) + lane / kLanes, all - 1), token = th / a.heads,
                       head = th - token * a.heads;
        y[i] = *reinterpret_cast<const uint4*>(a.out + token * a.o_row + head * a.o_head + lane % kLanes * 16);
    }
    unsigned bad[kCheckLoads], any = 0;
#pragma unroll
    for (int i = 0; i < kCheckLoads; i++) any |= bad[i] = __ballot_sync(0xffffffffu, any_nonfinite(y[i], IO(0.f)));
    if (!__syncthreads_or(any != 0)) return;
    unsigned bits = 0;
#pragma unroll
    for (int r = 0; r < R; r++)
        if (bad[r / kPass] >> (r % kPass * kLanes) & (kLanes == 32 ? ~0u : (1u << kLanes % 32) - 1)) bits |= 1u << r;
    if (lane == 0) rows[warp] = bits;
    __syncthreads();
#pragma unroll 1
    for (int w = 0; w < 4; w++)
#pragma unroll 1
        for (unsigned left = rows[w]; left; left &= left - 1) {
            const unsigned th = row_of(w, __ffs(left) - 1);
            if (th < all) redo_row<IO, KV, D, 4>(a, (int)(th / a.heads), (int)(th % a.heads), sums, ml, &done);
        }
}

// How the work is cut up: from the host's bounds alone, so that a captured
// launch holds for any lengths within them.  A tile's keys are split where the
// tiles alone do not fill the card.
struct Plan {
    int few_rows, stream;
    Cut few, many;
    int max_splits;  // for any window
};
constexpr int kStreamMost = 148 * 3;  // blocks that share out a batch's keys

Plan make_plan(const PagedView& p, int io, int cache, int heads, int D, int window) {
    Plan pl{};
    const int G = heads / p.kv_heads;
    const int64_t most = (int64_t)p.max_new * G, total = (int64_t)p.tokens * G;  // rows of a KV head
    // Batches that may hold more than 16 rows of a KV head a sequence (8 of f32; one decoded token's G
    // in any case) run on the tensor cores' tiles of 256 (128) rows, all but the sequences of a token
    // or few.  Measured with all sequences alike, us, here and there: 64 x 4096 keys, D = 128, 16 rows: bf16
    // 215 and 367, f16 217 and 369, f32 over bf16 338 and 337, f32 (2112 keys) 509 and 529; 32 rows: bf16 364 and
    // 325, f16 372 and 328.  At D = 64 the products weigh less and the crossover lies higher, which the
    // rule leaves alone: 16 rows f32 179 and 348, f32 over bf16 142 and 276; 32 rows bf16 218 and 282.  (All
    // sequences would then run on the wider tiles for the longest one's sake: with 8 rows f32 125 us, with 12
    // 177.)  One sequence alone takes one kernel for all it may hold.
    const int least = G <= 8 ? 8 : G <= 16 || io == VB_F32 ? 16 : 32, many_rows = io == VB_F32 ? kExRows : kTcRows;
    const bool tc = most > (io == VB_F32 ? least : std::max(least, 16));
    pl.few_rows = !tc ? 0x7fffffff : p.batch == 1 ? 0 : least;
    const int64_t all = std::max(p.max_len, 1);
    // keys from a tile's base (its first row's lowest, rounded down) to its last row's
    auto span = [&](int rows, int align) {
        return window > 0 ? std::min<int64_t>(all, (int64_t)window + (rows + G - 1) / G + align - 1) : all;
    };
    // few rows: one tile holds all of a sequence's
    const int64_t few_most = std::min<int64_t>(most, pl.few_rows);
    pl.few = Cut{few_most <= 8 ? 8 : few_most <= 16 ? 16 : 32, 1, 0, 16};
    const int64_t keys = span(pl.few.rows, 16);
    // Clusters where all fit the card at once and a block's share is at most 512 keys: one token of
    // one sequence of 777 keys takes one launch and 7.2 us of its caller instead of two and 9.8.
    // Else as many blocks as the card runs at a time.  37 clusters fit (bf16, 37 tiles of 2000 keys:
    // 8.4 us against 12.2 shared out); of f32 at D = 128, a block an SM, 15 (15 tiles of 2000 keys:
    // 10.1 against 16.7; 16, in two waves: 18.8 against 16.3, of 4000: 31.0 against 21.2).
    if ((int64_t)p.batch * p.kv_heads > (cache == VB_F32 && D == 128 ? 15 : 37) || keys > kCl * 512)
        pl.stream = (int)std::min<int64_t>(cache == VB_F32 && D == 128 ? 148 : kStreamMost,
                                           (int64_t)p.batch * p.kv_heads * ((keys + kUnit - 1) / kUnit));
    // many rows: one CTA for each SM, of at least 512 keys
    const int64_t tiles = std::max<int64_t>(1, (total + many_rows - 1) / many_rows);
    const int64_t want = std::max<int64_t>(1, 148 / (tiles * p.kv_heads));
    const int64_t span_many = span(many_rows, 128);
    const int64_t n = tc ? std::min<int64_t>(want, (span_many + 511) / 512) : 1;
    pl.many = Cut{many_rows, 1, (int)(((span_many + n - 1) / n + 127) / 128 * 128), 128};
    pl.many.splits = (int)((span_many + pl.many.len - 1) / pl.many.len);
    pl.max_splits = tc ? (int)std::min<int64_t>(want, (all + 511) / 512) : 1;
    return pl;
}
// The workspace: first the shared-out tiles' pieces, then the splits', then the hints (many rows: 4 bytes a sequence
// and KV head) and (both kernels) 16 bytes for `ready`.
bool both_kernels(const Plan& pl) { return pl.few_rows && pl.few_rows != 0x7fffffff; }
size_t stream_floats(const Plan& pl, int D) { return pl.few_rows ? (size_t)kStreamMost * 2 * pl.few.rows * (D + 2) : 0; }
size_t split_floats(const Plan& pl, const PagedView& p, int heads, int D) {
    return pl.max_splits > 1 ? (size_t)pl.max_splits * p.tokens * heads * (D + 2) : 0;
}
size_t hint_ints(const Plan& pl, const PagedView& p) {
    return pl.few_rows != 0x7fffffff ? ((size_t)p.batch * p.kv_heads + 3) / 4 * 4 : 0;
}
size_t plan_bytes(const Plan& pl, const PagedView& p, int heads, int D) {
    return 4 * (stream_floats(pl, D) + split_floats(pl, p, heads, D) + hint_ints(pl, p) + (both_kernels(pl) ? 4 : 0));
}

// Tensor map of a pool as [page][kv head][position][dim], boxes of one page's rows (128 at
// most) x 64 dims, 128-byte swizzle.  Returns the rows of a box; 0 where pages are not
// whole groups of 8 rows that tile 128, or the map is refused: the rows are then gathered
// by cp.async.
int page_map(const PagedView& p, const char* base, int D, bool half, CUtensorMap* map) {
    if (p.page_shift < 3) return 0;
    auto fn = tc_encode_fn();
    if (!fn) return 0;
    const int box = std::min(p.page_size, 128);
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)p.page_size, (cuuint64_t)p.kv_heads, (cuuint64_t)p.num_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)p.stride_pos, (cuuint64_t)p.stride_head, (cuuint64_t)p.stride_page};
    const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, es[4] = {1, 1, 1, 1};
    const CUresult r =
        fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<char*>(base),
           dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? box : 0;
}

template <typename IO, typename KV, int D, int NR>
vb_status launch_few(const AttnView& a, cudaStream_t s) {
    using C = FewCfg<KV, D, NR>;
    static std::atomic<unsigned long long> done[2];
    const dim3 block(C::kWarps * 32);
    cudaError_t e;
    if (a.stream) {
        e = smem_attr_once(paged_attn_few_kernel<IO, KV, D, NR, false>, C::kSmem, done[0]);
        if (e == cudaSuccess)
            e = launch_pdl(paged_attn_few_kernel<IO, KV, D, NR, false>, dim3(a.stream), block, C::kSmem, s, a);
    } else {
        e = smem_attr_once(paged_attn_few_kernel<IO, KV, D, NR, true>, C::kSmem, done[1]);
        if (e == cudaSuccess)
            e = launch_pdl_cluster(paged_attn_few_kernel<IO, KV, D, NR, true>, dim3(a.p.batch * a.p.kv_heads * kCl), block,
                                   C::kSmem, dim3(kCl, 1, 1), s, a);
    }
    return e == cudaSuccess ? VB_OK : cuda_fail(e, "paged_attn_few_kernel");
}

template <typename IO, typename KV, int D>
vb_status launch_attn(const AttnView& a, cudaStream_t s) {
    cudaError_t e;
    if (a.few_rows != 0x7fffffff) {
        const int rows = a.many.rows;
        const int64_t tiles = std::min<int64_t>((int64_t)a.p.batch * (((int64_t)a.p.max_new * a.group + rows - 1) / rows),
                                                (int64_t)a.p.tokens * a.group / rows + a.p.batch);
        const int64_t grid = tiles * a.many.splits * a.p.kv_heads;
        if (grid > 0x7fffffffll) return fail(VB_ERR_UNSUPPORTED, "paged_attn: too many rows");
        if (a.ready) {
            e = launch_pdl(paged_attn_clear_kernel, dim3(1), dim3(1), 0, s, a.ready);
            if (e != cudaSuccess) return cuda_fail(e, "paged_attn_clear_kernel");
        }
        AttnView b = a;
        if (fault_armed_for(kFaultPagedQ)) {  // failure-path test: never a launch that is being captured
            cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
            VB_CUDA_TRY(cudaStreamIsCapturing(s, &cs));
            b.stall = cs == cudaStreamCaptureStatusNone && fault_take(kFaultPagedQ);
        }
        CUtensorMap mk{}, mv{};
        if constexpr (sizeof(KV) == 2) {
            b.box = page_map(a.p, a.p.k, D, std::is_same<KV, __half>::value, &mk);
            if (b.box && !page_map(a.p, a.p.v, D, std::is_same<KV, __half>::value, &mv)) b.box = 0;
        }
        static std::atomic<unsigned long long> done{0};
        if constexpr (sizeof(IO) == 4) {
            using C = ExCfg<KV, D>;
            e = smem_attr_once(paged_attn_exact_kernel<KV, D>, C::kSmem, done);
            if (e == cudaSuccess)
                e = launch_pdl(paged_attn_exact_kernel<KV, D>, dim3((unsigned)grid), dim3(C::kThreads), C::kSmem, s, b, mk, mv);
        } else {
            e = smem_attr_once(paged_attn_tc_kernel<IO, D>, TcCfg<D>::kSmem, done);
            if (e == cudaSuccess)
                e = launch_pdl(paged_attn_tc_kernel<IO, D>, dim3((unsigned)grid), dim3(kTcThreads), TcCfg<D>::kSmem, s, b, mk,
                               mv);
        }
        if (e != cudaSuccess) return cuda_fail(e, "paged attention, many rows");
    }
    if (a.few_rows) {
        AttnView f = a;
        f.after_many = a.ready != nullptr;
        vb_status st = VB_OK;
        if (a.few.rows == 8) {
            st = launch_few<IO, KV, D, 1>(f, s);
        } else if (a.few.rows == 16) {
            st = launch_few<IO, KV, D, 2>(f, s);
        } else {
            if constexpr (sizeof(IO) == 2) st = launch_few<IO, KV, D, 4>(f, s);  // (f32: 16 rows at most)
        }
        if (st) return st;
    }
    if (a.few_rows && a.stream) {  // (one sequence alone on the many-rows kernel has nothing shared out)
        const int rows = (int)std::min<int64_t>(a.few.rows, (int64_t)a.p.max_new * a.group);
        const int64_t heads = (int64_t)a.p.batch * a.p.kv_heads;
        const bool one = heads * rows <= 2048;
        const int groups = one ? rows : (rows + 7) / 8;
        if (heads * groups > 0x7fffffffll) return fail(VB_ERR_UNSUPPORTED, "paged_attn: too many rows");
        const dim3 grid((unsigned)(heads * groups)), block(kJoinWarps * 32);
        constexpr bool kRedo = !kAsSeen<IO>;
        if (a.redo && kRedo)
            e = one ? launch_pdl(paged_attn_join_kernel<IO, KV, D, 1, kRedo>, grid, block, 0, s, a, groups)
                    : launch_pdl(paged_attn_join_kernel<IO, KV, D, 8, kRedo>, grid, block, 0, s, a, groups);
        else
            e = one ? launch_pdl(paged_attn_join_kernel<IO, KV, D, 1, false>, grid, block, 0, s, a, groups)
                    : launch_pdl(paged_attn_join_kernel<IO, KV, D, 8, false>, grid, block, 0, s, a, groups);
        if (e != cudaSuccess) return cuda_fail(e, "paged_attn_join_kernel");
    }
    if (a.many.splits > 1) {
        const int64_t grid = ((int64_t)a.p.tokens * a.heads + 3) / 4;
        if (grid > 0x7fffffffll) return fail(VB_ERR_UNSUPPORTED, "paged_attn: too many rows");
        e = launch_pdl(paged_attn_merge_kernel<IO, D>, dim3((unsigned)grid), dim3(128), 0, s, a);
        if (e != cudaSuccess) return cuda_fail(e, "paged_attn_merge_kernel");
    }
    if (a.p.max_new > 1 || (a.few_rows != 0x7fffffff && !kAsSeen<IO>)) {  // (see AttnView::redo)
        constexpr int kBlockRows = 4 * check_rows<IO, D>();
        const int64_t grid = ((int64_t)a.p.tokens * a.heads + kBlockRows - 1) / kBlockRows;
        e = launch_pdl(paged_attn_check_kernel<IO, KV, D>, dim3((unsigned)grid), dim3(128), 0, s, a);
        if (e != cudaSuccess) return cuda_fail(e, "paged_attn_check_kernel");
    }
    VB_LAUNCH_CHECK("paged attention");
    return VB_OK;
}

template <int D>
vb_status launch_attn(const AttnView& a, int io, int cache, cudaStream_t s) {
    if (io == VB_F32 && cache == VB_F32) return launch_attn<float, float, D>(a, s);
    if (io == VB_F32) return launch_attn<float, __nv_bfloat16, D>(a, s);
    if (io == VB_F16) return launch_attn<__half, __half, D>(a, s);
    return launch_attn<__nv_bfloat16, __nv_bfloat16, D>(a, s);
}

}  // namespace
}  // namespace vb

using namespace vb;

extern "C" size_t vb_paged_attn_workspace_bytes(const vb_paged_cache* cache, const vb_paged_batch* batch, int heads) {
    PagedView p{};
    if (!cache || paged_view(cache, batch, cache->dtype, heads, "paged_attn", &p) || !p.batch || !p.tokens) return 0;
    size_t most = 0;  // rows of the cache's type or, over a bf16 cache, f32
    for (const int io : {cache->dtype, (int)VB_F32})
        if (io == cache->dtype || cache->dtype == VB_BF16)
            most = std::max(most, plan_bytes(make_plan(p, io, cache->dtype, heads, cache->head_dim, 0), p, heads, cache->head_dim));
    return most;
}

extern "C" vb_status vb_paged_attn(const vb_paged_cache* cache, const vb_paged_batch* batch, int io, int heads,
                                   const void* q, int64_t q_row, int64_t q_head, void* out, int64_t o_row,
                                   int64_t o_head, float* lse, float scale, int window, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    AttnView a{};
    const vb_status st = paged_view(cache, batch, io, heads, "paged_attn", &a.p);
    if (st) return st;
    if (window < 0) return fail(VB_ERR_ARG, "paged_attn: negative window");
    if (!batch->batch || !batch->tokens || !batch->max_new) return VB_OK;
    if (window >= batch->max_len) window = 0;  // every position is within it
    if (!q || !out) return fail(VB_ERR_ARG, "paged_attn: null pointer");
    const int es = paged_elem_bytes(io), D = cache->head_dim;
    if (!paged_aligned(q, q_row, q_head, es) || !paged_aligned(out, o_row, o_head, es) || !paged_aligned(workspace, 0, 0, 1))
        return fail(VB_ERR_UNSUPPORTED, "paged_attn: 16-byte alignment required");
    if (!paged_words({lse})) return fail(VB_ERR_UNSUPPORTED, "paged_attn: 4-byte alignment required");
    if ((int64_t)batch->tokens * heads > 0x7fffffff) return fail(VB_ERR_UNSUPPORTED, "paged_attn: too many rows");
    const Plan pl = make_plan(a.p, io, cache->dtype, heads, D, window);
    // positions up to a tile past the last one, and the units of shared-out keys, are counted in 32 bits
    if (a.p.max_len > 0x40000000 ||
        (int64_t)a.p.batch * a.p.kv_heads * ((int64_t)a.p.max_len / kUnit + 1) > 0x3fffffff)
        return fail(VB_ERR_UNSUPPORTED, "paged_attn: too many keys");
    const size_t need = plan_bytes(pl, a.p, heads, D);
    if (need > workspace_bytes || (need && !workspace))
        return fail(VB_ERR_ARG, "paged_attn: the workspace is too small");
    // (a row that is taken again reads its q when the output has been written)
    if (q == out) return fail(VB_ERR_ARG, "paged_attn: not in place");
    a.q = static_cast<const char*>(q);
    a.out = static_cast<char*>(out);
    a.q_row = q_row * es, a.q_head = q_head * es, a.o_row = o_row * es, a.o_head = o_head * es;
    a.lse = lse;
    a.heads = heads;
    a.group = heads / cache->kv_heads;
    // a scale of 0 as one that no score outgrows: a masked score stays -inf under it
    a.scale_log2 = (scale == 0.f ? 1.17549435e-38f : scale) * 1.44269504088896341f;
    a.window = window;
    a.few_rows = pl.few_rows;
    a.redo = a.p.max_new == 1 && pl.few_rows == 0x7fffffff;
    a.few = pl.few;
    a.many = pl.many;
    a.stream = pl.stream;
    const size_t parts = (size_t)kStreamMost * 2 * pl.few.rows;
    a.strm = static_cast<float*>(workspace);
    a.strm_ml = reinterpret_cast<float2*>(a.strm + parts * D);
    a.part = a.strm + stream_floats(pl, D);
    a.part_ml = reinterpret_cast<float2*>(a.part + (size_t)pl.max_splits * a.p.tokens * heads * D);
    int* const words = reinterpret_cast<int*>(a.part + split_floats(pl, a.p, heads, D));
    if (hint_ints(pl, a.p)) a.hint = words;
    if (both_kernels(pl)) a.ready = reinterpret_cast<unsigned*>(words + hint_ints(pl, a.p));
    return D == 128 ? launch_attn<128>(a, io, cache->dtype, as_stream(stream))
                    : launch_attn<64>(a, io, cache->dtype, as_stream(stream));
}
