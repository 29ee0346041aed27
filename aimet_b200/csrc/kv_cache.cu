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

// ---------------------------------------------------------------------------------------------------
// append
//
// One CTA per (sequence, touched block, head, key or value): largest magnitude of the block's new
// tokens, the block's scale, codes.  A block that starts with a new token takes scale = max * (1 / 127),
// the factor rounded to float32 (what torch computes for max / 127 on a GPU); one that holds tokens
// already keeps its scale while that covers the new tokens and otherwise takes max(that, 1.25 * scale), its codes becoming rint(code * (old / new)).  Growing by a quarter at
// least bounds what repeated rounding can add up to: half a step each time, 2.5 final steps in all.
//
// Bound by reading the new tokens and writing a byte for each element (4 x up to 2000 tokens, 8 heads of 128, float16: 18 us of
// 7 by itself, most of it the chain lengths - table - page of small blocks).  x / scale is the correctly rounded
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

// The largest magnitude of a piece as the bits of its type (whose order is that of the magnitudes; infinities
// and NaN are the largest), two 16-bit elements at a time.
__device__ __forceinline__ uint32_t max_bits(const Vec16<float> &v, uint32_t top) {
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v.v[e]) & 0x7fffffffu);
    return top;
}
template <typename E> __device__ __forceinline__ uint32_t max_bits(const Vec16<E> &v, uint32_t top) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&v);
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __vmaxu2(top, w[e] & 0x7fff7fffu);
    return top;
}
__device__ __forceinline__ uint32_t fold_bits(uint32_t top, float) { return top; }
template <typename E> __device__ __forceinline__ uint32_t fold_bits(uint32_t top, E) { return max(top & 0xffffu, top >> 16); }
__device__ __forceinline__ float value_of(uint32_t bits, float) { return __uint_as_float(bits); }
__device__ __forceinline__ float value_of(uint32_t bits, __nv_bfloat16) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ float value_of(uint32_t bits, __half) { return __half2float(__ushort_as_half((unsigned short)bits)); }

constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds half to even into the low bits

// The code of a finite x, |x| <= scale * 127 (1 + 2^-22) and scale in [2^-100, 2^100], in the low byte (two's
// complement): the correctly rounded quotient without the divide unit.
__device__ __forceinline__ uint32_t code_fast(float x, float s, float r) {
    const float q0 = __fmul_rn(x, r);
    return __float_as_uint(__fadd_rn(__fmaf_rn(__fmaf_rn(-q0, s, x), r, q0), kRound));
}
// Any x and scale: NaN gives 0, infinities the outermost levels, a zero scale zeros.
__device__ __forceinline__ uint32_t code_any(float x, float s) {
    x = x == x ? x : 0.f;
    const float q = s > 0.f ? __fdiv_rn(x, s) : 0.f;
    return __float_as_uint(__fadd_rn(fminf(fmaxf(q, -kLevels), kLevels), kRound));
}
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// the largest of the CTA's values, for every thread
template <int THREADS> __device__ __forceinline__ uint32_t block_max(uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (THREADS > 32) {
        __shared__ uint32_t of_warp[THREADS / 32];
        __syncthreads();  // a second use may follow the first at once
        if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) v = max(v, of_warp[w]);
    }
    return v;
}

// Walks the 16-byte pieces (per_row of them in a row) of a block, THREADS apart, without a division per piece.
struct Piece {
    int row, piece;
    __device__ __forceinline__ Piece(int first, int per_row) : row(first / per_row), piece(first % per_row) {}
    __device__ __forceinline__ void advance(int rows, int pieces, int per_row) {
        row += rows;
        piece += pieces;
        if (piece >= per_row) piece -= per_row, ++row;
    }
};

// KEEP pieces of a thread stay in registers between the two passes; a block with more is read again (from L1 or L2).
template <typename E, int THREADS, int KEEP> __global__ void __launch_bounds__(THREADS) k_kv_append(AppendArgs a) {
    constexpr int V = 16 / sizeof(E);  // elements per 16-byte piece
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

    const int kept = (int)(lo - b * page), rows = (int)(hi - lo);
    const int64_t stride_t = a.stride_t[kv];
    const E *x = static_cast<const E *>(a.x[kv]) + (int64_t)s * a.stride_s[kv] + (int64_t)h * a.stride_h[kv] + (lo - ctx) * stride_t;
    const bool vec = a.vec[kv];
    const int per_row = dim / V, step_rows = THREADS / per_row, step_pieces = THREADS % per_row;
    auto load = [&](const Piece &p) {
        const E *src = x + p.row * stride_t + p.piece * V;
        Vec16<E> v;
        if (vec) {
            v = *reinterpret_cast<const Vec16<E> *>(src);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v.v[e] = src[e];
        }
        return v;
    };

    // the new tokens are requested before the page is known
    Vec16<E> keep[KEEP];
    uint32_t bits = 0;
    Piece p(threadIdx.x, per_row);
    const Piece first = p;
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        if (p.row < rows) keep[i] = load(p);
        p.advance(step_rows, step_pieces, per_row);
    }
    for (; p.row < rows; p.advance(step_rows, step_pieces, per_row)) bits = max_bits(load(p), bits);
    p = first;
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        if (p.row < rows) bits = max_bits(keep[i], bits);
        p.advance(step_rows, step_pieces, per_row);
    }
    bits = fold_bits(bits, E());
    if (pg < 0 || pg >= a.c.pages) return;  // (the CTA's threads agree)
    int8_t *code = a.c.code[kv] + ((pg * a.c.heads + h) * page) * (int64_t)dim;
    float *scale_at = a.c.scale[kv] + pg * a.c.heads + h;
    const float old = kept ? *scale_at : 0.f;
    bits = block_max<THREADS>(bits);  // (everyone has read the old scale)
    float top = value_of(bits, E());
    const bool finite = top <= 3.402823466e38f;
    if (!finite) {  // the largest of the finite values
        top = 0.f;
        for (p = first; p.row < rows; p.advance(step_rows, step_pieces, per_row)) {
            const Vec16<E> v = load(p);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float m = fabsf(to_f32(v.v[e]));
                top = fmaxf(top, m <= 3.402823466e38f ? m : 0.f);
            }
        }
        top = __uint_as_float(block_max<THREADS>(__float_as_uint(top)));
    }
    float scale = __fmul_rn(top, 1.f / kLevels);
    if (kept) scale = scale <= old ? old : fmaxf(scale, __fmul_rn(old, kGrowth));
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
                o |= (__float_as_uint(__fadd_rn(q, kRound)) & 0xffu) << (8 * e);
            }
            w[i] = o;
        }
    }

    const bool fast = finite && scale >= 7.8886090522101181e-31f && scale <= 1.2676506002282294e30f;  // 2^-100, 2^100
    const float r = fast ? __frcp_rn(scale) : 0.f;
    int8_t *out = code + (int64_t)kept * dim;
    auto store = [&](const Piece &p, const Vec16<E> &v) {
        uint32_t o[V / 4];
#pragma unroll
        for (int e = 0; e < V / 4; ++e) {
            uint32_t c[4];
            if (fast) {
#pragma unroll
                for (int j = 0; j < 4; ++j) c[j] = code_fast(to_f32(v.v[4 * e + j]), scale, r);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) c[j] = code_any(to_f32(v.v[4 * e + j]), scale);
            }
            o[e] = low_bytes(c[0], c[1], c[2], c[3]);
        }
        int8_t *dst = out + p.row * dim + p.piece * V;
        if constexpr (V == 8)
            *reinterpret_cast<uint2 *>(dst) = make_uint2(o[0], o[1]);
        else
            *reinterpret_cast<uint32_t *>(dst) = o[0];
    };
    p = first;
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
        if (p.row < rows) store(p, keep[i]);
        p.advance(step_rows, step_pieces, per_row);
    }
    for (; p.row < rows; p.advance(step_rows, step_pieces, per_row)) store(p, load(p));
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
    // kAhead pieces of a thread requested before the first is stored
    constexpr int V = 16 / sizeof(E), kAhead = 4;
    const int per_row = dim / 16, step_rows = 128 / per_row, step_pieces = 128 % per_row;
    Piece p(threadIdx.x, per_row);
    while (p.row < rows) {
        const Piece first = p;
        uint4 v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            v[i] = make_uint4(0, 0, 0, 0);
            if (p.row < there) v[i] = *reinterpret_cast<const uint4 *>(code + (int64_t)p.row * dim + p.piece * 16);
            p.advance(step_rows, step_pieces, per_row);
        }
        p = first;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (p.row < rows) {
                // code + 128 in the mantissa of 2^23, minus 2^23 + 128: the conversion pipe is the slower way
                const uint32_t w[4] = {v[i].x ^ 0x80808080u, v[i].y ^ 0x80808080u, v[i].z ^ 0x80808080u, v[i].w ^ 0x80808080u};
                const float f = p.row < there ? scale : 0.f;
                Vec16<E> *dst = reinterpret_cast<Vec16<E> *>(y + p.row * pitch + p.piece * 16);
#pragma unroll
                for (int e = 0; e < 16 / V; ++e) {
                    float q[V];
                    Vec16<E> o;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const int c = e * V + j;
                        q[j] = __fmul_rn(__uint_as_float(__byte_perm(w[c / 4], 0x4b000000u, 0x7650 + c % 4)) - 8388736.f, f);
                    }
                    VecCvt<float, E>::pack(q, o);
                    dst[e] = o;
                }
            }
            p.advance(step_rows, step_pieces, per_row);
        }
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

template <typename E, int THREADS, int KEEP> int launch_append(const AppendArgs &a, int64_t ctas, cudaStream_t st) {
    AB_CUDA_OK(launch_pdl(k_kv_append<E, THREADS, KEEP>, dim3((unsigned)ctas), dim3(THREADS), 0, st, a));
    AB_LAUNCH_OK();
    return AB_OK;
}
template <typename E> int dispatch_append(const AppendArgs &a, int64_t ctas, cudaStream_t st) {
    // a warp is enough for a few rows and leaves no barriers; whole blocks take as many threads as hold them in registers
    const int64_t pieces = (int64_t)std::min(a.tokens, a.c.page) * a.c.dim * sizeof(E) / 16;
    if (pieces <= 128) return launch_append<E, 32, 4>(a, ctas, st);
    if (pieces <= 512) return launch_append<E, 128, 4>(a, ctas, st);
    return launch_append<E, 256, 8>(a, ctas, st);
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
