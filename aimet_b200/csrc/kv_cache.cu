// A paged key / value cache in 8-bit codes with one scale per page (a block of tokens) and head:
// writing new tokens into it, reading blocks back as values, and attention over it.
//
//   pages   key, value        int8    [page][head][row][dim]
//           key_scale, ...    float32 [page][head]
//   value of a code = code * scale, codes in [-127, 127]
//   token j of sequence s lives in row j % page_size of page table[s][j / page_size]
//
// A table entry outside [0, num_pages) means "no page here": nothing is written to it, and what lies
// there reads as zeros and is masked in attention.  No other index comes from device memory, so no
// content of the table or of the lengths can lead to an access outside the buffers.
#include <algorithm>

#include "common.cuh"

namespace ab {
namespace {

struct CacheView {
    int8_t *code[2];   // key, value
    float *scale[2];
    int64_t pages;
    int heads, page, dim;
};

__host__ __device__ inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---------------------------------------------------------------------------------------------------
// append
//
// One CTA per (sequence, touched block, head, key or value): largest magnitude of the block's new
// tokens, the block's scale, codes.  A block that starts with a new token takes scale = max * (1 / 127),
// the factor rounded to float32 (what torch computes for max / 127 on a GPU); one that holds tokens
// already keeps its scale while that covers the new tokens and otherwise takes max(that, 1.25 * scale), its codes becoming rint(code * (old / new)).  Growing by a quarter at
// least bounds what repeated rounding can add up to: half a step each time, 2.5 final steps in all.
//
// Bound by reading the new tokens and writing a byte for each element.  x / scale is the correctly rounded
// quotient without the divide unit: r = 1 / s, q0 = x * r, q = q0 + r * (x - q0 * s) with fused
// multiply-adds (Markstein's theorem; scales outside [2^-100, 2^100] are divided by the divide unit).
// ---------------------------------------------------------------------------------------------------
constexpr float kLevels = 127.f;
constexpr float kGrowth = 1.25f;

struct AppendArgs {
    CacheView c;
    const void *x[2];
    int64_t stride_s[2], stride_t[2], stride_h[2];
    const int32_t *table, *context, *lens;
    int64_t table_stride;
    int table_width, seqs, tokens, blocks;  // blocks: most blocks a sequence's new tokens touch
    int vec[2];
};

struct Quantizer {
    float s, r, lim;
    bool plain;
    __device__ __forceinline__ explicit Quantizer(float scale) {
        s = scale;
        plain = !(scale >= 7.8886090522101181e-31f && scale <= 1.2676506002282294e30f);  // 2^-100, 2^100
        r = plain ? 0.f : __frcp_rn(scale);
        lim = __fmul_rn(scale, kLevels);
    }
    // the code in the low byte (two's complement); NaN gives 0, infinities the outermost levels
    __device__ __forceinline__ uint32_t operator()(float x) const {
        x = x == x ? x : 0.f;
        float q;
        if (plain) {
            q = s > 0.f ? __fdiv_rn(x, s) : 0.f;
        } else {
            x = fminf(fmaxf(x, -lim), lim);
            const float q0 = __fmul_rn(x, r);
            q = __fmaf_rn(__fmaf_rn(-q0, s, x), r, q0);
        }
        q = fminf(fmaxf(q, -kLevels), kLevels);
        return __float_as_uint(__fadd_rn(q, 12582912.f)) & 0xffu;  // 1.5 * 2^23: rounds half to even
    }
};

template <typename E, int THREADS> __global__ void __launch_bounds__(THREADS) k_kv_append(AppendArgs a) {
    constexpr int V = 16 / sizeof(E);  // elements per 16-byte vector
    pdl_prologue();
    int64_t at = blockIdx.x;
    const int kv = (int)(at & 1);
    at >>= 1;
    const int h = (int)(at % a.c.heads);
    at /= a.c.heads;
    const int blk = (int)(at % a.blocks), s = (int)(at / a.blocks);
    const int len = a.lens ? min(max(a.lens[s], 0), a.tokens) : a.tokens;
    const int64_t ctx = max(a.context[s], 0);
    const int page = a.c.page, dim = a.c.dim;
    const int64_t b = ctx / page + blk;  // the sequence's block
    const int64_t lo = max(b * page, ctx), hi = min((b + 1) * page, ctx + len);  // positions of its new tokens
    if (lo >= hi || b >= a.table_width) return;
    const int64_t pg = a.table[(int64_t)s * a.table_stride + b];
    if (pg < 0 || pg >= a.c.pages) return;

    const int kept = (int)(lo - b * page), rows = (int)(hi - lo);
    const E *x = static_cast<const E *>(a.x[kv]) + (int64_t)s * a.stride_s[kv] + (int64_t)h * a.stride_h[kv] + (lo - ctx) * a.stride_t[kv];
    const int64_t stride_t = a.stride_t[kv];
    int8_t *code = a.c.code[kv] + ((pg * a.c.heads + h) * page) * (int64_t)dim;
    float *scale_at = a.c.scale[kv] + pg * a.c.heads + h;
    const bool vec = a.vec[kv];
    const int per_row = dim / V, work = rows * per_row;

    float top = 0.f;
    for (int i = threadIdx.x; i < work; i += THREADS) {
        const int r = i / per_row, d = (i - r * per_row) * V;
        const E *p = x + r * stride_t + d;
        Vec16<E> v;
        if (vec)
            v = *reinterpret_cast<const Vec16<E> *>(p);
        else
#pragma unroll
            for (int e = 0; e < V; ++e) v.v[e] = p[e];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float m = fabsf(to_f32(v.v[e]));
            top = fmaxf(top, m <= 3.402823466e38f ? m : 0.f);  // finite values only
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (THREADS > 32) {
        __shared__ float tops[THREADS / 32];
        if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, tops[w]);
    }

    const float old = kept ? *scale_at : 0.f;
    float scale = __fmul_rn(top, 1.f / kLevels);
    if (kept) scale = scale <= old ? old : fmaxf(scale, __fmul_rn(old, kGrowth));
    if (THREADS > 32)
        __syncthreads();  // everyone has read the old scale
    else
        __syncwarp();
    if (threadIdx.x == 0) *scale_at = scale;

    if (kept && scale != old) {  // the codes held so far move onto the coarser grid
        const float ratio = __fdiv_rn(old, scale);
        uint32_t *w = reinterpret_cast<uint32_t *>(code);
        for (int i = threadIdx.x; i < kept * dim / 4; i += THREADS) {
            const uint32_t v = w[i];
            uint32_t o = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float q = __fmul_rn((float)(int8_t)(v >> (8 * e)), ratio);
                o |= (__float_as_uint(__fadd_rn(q, 12582912.f)) & 0xffu) << (8 * e);
            }
            w[i] = o;
        }
    }

    const Quantizer q(scale);
    int8_t *out = code + (int64_t)kept * dim;
    for (int i = threadIdx.x; i < work; i += THREADS) {
        const int r = i / per_row, d = (i - r * per_row) * V;
        const E *p = x + r * stride_t + d;
        Vec16<E> v;
        if (vec)
            v = *reinterpret_cast<const Vec16<E> *>(p);
        else
#pragma unroll
            for (int e = 0; e < V; ++e) v.v[e] = p[e];
        uint32_t o[V / 4];
#pragma unroll
        for (int e = 0; e < V / 4; ++e) {
            o[e] = q(to_f32(v.v[4 * e])) | q(to_f32(v.v[4 * e + 1])) << 8 | q(to_f32(v.v[4 * e + 2])) << 16 |
                   q(to_f32(v.v[4 * e + 3])) << 24;
        }
        int8_t *dst = out + (int64_t)r * dim + d;
        if constexpr (V == 8)
            *reinterpret_cast<uint2 *>(dst) = make_uint2(o[0], o[1]);
        else
            *reinterpret_cast<uint32_t *>(dst) = o[0];
    }
}

// ---------------------------------------------------------------------------------------------------
// gather: codes of a sequence's first `length` positions as values, zeros behind its last token.  One
// CTA per (sequence, block, head, key or value); 16 codes per thread and step.
// ---------------------------------------------------------------------------------------------------
struct GatherArgs {
    CacheView c;
    void *y[2];
    const int32_t *table, *lens;
    int64_t table_stride;
    int table_width, seqs, length, blocks;
};

template <typename E> __global__ void __launch_bounds__(128) k_kv_gather(GatherArgs a) {
    pdl_prologue();
    int64_t at = blockIdx.x;
    const int kv = (int)(at & 1);
    at >>= 1;
    const int h = (int)(at % a.c.heads);
    at /= a.c.heads;
    const int blk = (int)(at % a.blocks), s = (int)(at / a.blocks);
    const int page = a.c.page, dim = a.c.dim;
    const int64_t first = (int64_t)blk * page;
    const int rows = (int)min((int64_t)page, a.length - first);  // rows of the output in this block
    int there = (int)min(max(a.lens[s] - first, (int64_t)0), (int64_t)rows);  // rows that hold tokens
    const int64_t pg = blk < a.table_width ? a.table[(int64_t)s * a.table_stride + blk] : -1;
    if (pg < 0 || pg >= a.c.pages) there = 0;
    const int8_t *code = there ? a.c.code[kv] + ((pg * a.c.heads + h) * page) * (int64_t)dim : nullptr;
    const float scale = there ? a.c.scale[kv][pg * a.c.heads + h] : 0.f;
    E *y = static_cast<E *>(a.y[kv]) + (((int64_t)s * a.length + first) * a.c.heads + h) * dim;
    const int64_t pitch = (int64_t)a.c.heads * dim;
    const int per_row = dim / 16;
    for (int i = threadIdx.x; i < rows * per_row; i += 128) {
        const int r = i / per_row, d = (i - r * per_row) * 16;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < there) v = *reinterpret_cast<const uint4 *>(code + (int64_t)r * dim + d);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        constexpr int V = 16 / sizeof(E);
        Vec16<E> o[16 / V];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float f = r < there ? __fmul_rn((float)(int8_t)(w[e / 4] >> (8 * (e % 4))), scale) : 0.f;
            o[e / V].v[e % V] = Cvt<float, E>::store(f);
        }
        Vec16<E> *dst = reinterpret_cast<Vec16<E> *>(y + r * pitch + d);
#pragma unroll
        for (int e = 0; e < 16 / V; ++e) dst[e] = o[e];
    }
}

int check_cache(const ab_kv_cache *c, CacheView *v) {
    if (!c) return fail(AB_ERR_INVALID, "cache is NULL");
    if (!c->key || !c->value || !c->key_scale || !c->value_scale) return fail(AB_ERR_INVALID, "a buffer of the cache is NULL");
    if (!aligned16(c->key) || !aligned16(c->value)) return fail(AB_ERR_INVALID, "the cache's codes must be 16-byte aligned");
    if (c->num_pages < 1 || c->num_pages > 0x7fffffff) return fail(AB_ERR_INVALID, "num_pages=%lld", (long long)c->num_pages);
    if (c->num_heads < 1 || c->num_heads > 65535) return fail(AB_ERR_INVALID, "num_heads=%d", c->num_heads);
    if (c->page_size < 16 || c->page_size % 16 || c->page_size > 1024)
        return fail(AB_ERR_UNSUPPORTED, "page_size=%d: a multiple of 16 up to 1024", c->page_size);
    if (c->head_dim < 16 || c->head_dim % 16 || c->head_dim > 256)
        return fail(AB_ERR_UNSUPPORTED, "head_dim=%d: a multiple of 16 up to 256", c->head_dim);
    v->code[0] = static_cast<int8_t *>(c->key);
    v->code[1] = static_cast<int8_t *>(c->value);
    v->scale[0] = static_cast<float *>(c->key_scale);
    v->scale[1] = static_cast<float *>(c->value_scale);
    v->pages = c->num_pages;
    v->heads = c->num_heads;
    v->page = c->page_size;
    v->dim = c->head_dim;
    return AB_OK;
}

template <typename E, int THREADS> int launch_append(const AppendArgs &a, int64_t ctas, cudaStream_t st) {
    AB_CUDA_OK(launch_pdl(k_kv_append<E, THREADS>, dim3((unsigned)ctas), dim3(THREADS), 0, st, a));
    AB_LAUNCH_OK();
    return AB_OK;
}
template <typename E> int dispatch_append(const AppendArgs &a, int64_t ctas, cudaStream_t st) {
    // a warp is enough for a few rows and leaves no barriers; whole blocks take 256 threads
    const int rows = std::min(a.tokens, a.c.page);
    if ((int64_t)rows * a.c.dim <= 1024) return launch_append<E, 32>(a, ctas, st);
    return launch_append<E, 256>(a, ctas, st);
}

}  // namespace
}  // namespace ab

using namespace ab;

extern "C" int aimet_b200_kv_append(const ab_kv_cache *cache, const void *key, const void *value, const int64_t *key_strides,
                                    const int64_t *value_strides, int64_t seqs, int64_t tokens, const int32_t *block_table,
                                    int64_t table_stride, int64_t table_width, const int32_t *context_lens, const int32_t *new_lens,
                                    int io_dtype, void *stream) {
    AppendArgs a;
    const int rc = check_cache(cache, &a.c);
    if (rc != AB_OK) return rc;
    if (io_dtype != AB_F32 && io_dtype != AB_F16 && io_dtype != AB_BF16) return fail(AB_ERR_UNSUPPORTED, "io_dtype %d", io_dtype);
    if (seqs < 0 || tokens < 0 || seqs > (1 << 24) || tokens > (1 << 30) || table_width < 0 || table_width > 0x7fffffff)
        return fail(AB_ERR_INVALID, "seqs=%lld tokens=%lld table_width=%lld", (long long)seqs, (long long)tokens, (long long)table_width);
    if (seqs == 0 || tokens == 0 || table_width == 0) return AB_OK;
    if (!key || !value || !key_strides || !value_strides || !block_table || !context_lens) return fail(AB_ERR_INVALID, "a pointer is NULL");
    const int64_t size = dtype_size(io_dtype);
    const void *x[2] = {key, value};
    const int64_t *st[2] = {key_strides, value_strides};
    for (int i = 0; i < 2; ++i) {
        a.x[i] = x[i];
        a.stride_s[i] = st[i][0];
        a.stride_t[i] = st[i][1];
        a.stride_h[i] = st[i][2];
        a.vec[i] = aligned16(x[i]) && (st[i][0] * size) % 16 == 0 && (st[i][1] * size) % 16 == 0 && (st[i][2] * size) % 16 == 0;
    }
    a.table = block_table;
    a.context = context_lens;
    a.lens = new_lens;
    a.table_stride = table_stride;
    a.table_width = (int)table_width;
    a.seqs = (int)seqs;
    a.tokens = (int)tokens;
    a.blocks = (int)std::min(div_up(tokens - 1, a.c.page) + 1, table_width);
    const int64_t ctas = seqs * a.blocks * a.c.heads * 2;
    if (ctas > 0x7fffffff) return fail(AB_ERR_UNSUPPORTED, "%lld blocks in one call", (long long)ctas);
    switch (io_dtype) {
        case AB_F32: return dispatch_append<float>(a, ctas, static_cast<cudaStream_t>(stream));
        case AB_F16: return dispatch_append<__half>(a, ctas, static_cast<cudaStream_t>(stream));
        default: return dispatch_append<__nv_bfloat16>(a, ctas, static_cast<cudaStream_t>(stream));
    }
}

extern "C" int aimet_b200_kv_gather(const ab_kv_cache *cache, void *key, void *value, int64_t seqs, int64_t length,
                                    const int32_t *block_table, int64_t table_stride, int64_t table_width, const int32_t *lens,
                                    int io_dtype, void *stream) {
    GatherArgs a;
    const int rc = check_cache(cache, &a.c);
    if (rc != AB_OK) return rc;
    if (io_dtype != AB_F32 && io_dtype != AB_F16 && io_dtype != AB_BF16) return fail(AB_ERR_UNSUPPORTED, "io_dtype %d", io_dtype);
    if (seqs < 0 || length < 0 || seqs > (1 << 24) || length > 0x7fffffff || table_width < 0 || table_width > 0x7fffffff)
        return fail(AB_ERR_INVALID, "seqs=%lld length=%lld table_width=%lld", (long long)seqs, (long long)length, (long long)table_width);
    if (seqs == 0 || length == 0) return AB_OK;
    if (!key || !value || !lens || (table_width > 0 && !block_table)) return fail(AB_ERR_INVALID, "a pointer is NULL");
    if (!aligned16(key) || !aligned16(value)) return fail(AB_ERR_INVALID, "outputs must be 16-byte aligned");
    a.y[0] = key;
    a.y[1] = value;
    a.table = block_table;
    a.lens = lens;
    a.table_stride = table_stride;
    a.table_width = (int)table_width;
    a.seqs = (int)seqs;
    a.length = (int)length;
    a.blocks = (int)div_up(length, a.c.page);
    const int64_t ctas = seqs * a.blocks * a.c.heads * 2;
    if (ctas > 0x7fffffff) return fail(AB_ERR_UNSUPPORTED, "%lld blocks in one call", (long long)ctas);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (io_dtype) {
        case AB_F32: AB_CUDA_OK(launch_pdl(k_kv_gather<float>, dim3((unsigned)ctas), dim3(128), 0, st, a)); break;
        case AB_F16: AB_CUDA_OK(launch_pdl(k_kv_gather<__half>, dim3((unsigned)ctas), dim3(128), 0, st, a)); break;
        default: AB_CUDA_OK(launch_pdl(k_kv_gather<__nv_bfloat16>, dim3((unsigned)ctas), dim3(128), 0, st, a));
    }
    AB_LAUNCH_OK();
    return AB_OK;
}
