// Attention of a sequence's newest tokens over the paged 8-bit cache (kv_cache.cu):
//
//   o_i = sum_j softmax_j(c q_i . k_j) v_j,   j <= p_i and j > p_i - window,   p_i = context - query_len + i
//
// with k_j, v_j = code * scale of the token's page and head.  One pass over the cache with the running
// maximum and sum of the softmax; the codes go from HBM to the operand registers in 8 bits.
//
// What bounds it is reading the codes: 2 * dim bytes per token and head, for a handful of rows (the
// query heads that share a head of the cache, times the query tokens).  Those rows are one 16-row tile
// of mma.sync (tcgen05 needs 64 rows at least, and here the tensor cores are not the limit): scores =
// Q (16 x dim) . K^T, then O (16 x dim) += P (16 x tokens) . V.  Codes become float16 pairs exactly (a
// byte permute puts code + 128 into the mantissa of 1024, subtracting 1152 leaves the code).  The scales
// never touch an element: a tile of 16 tokens lies in one page, so the key scale multiplies the scores,
// and log2 of the value scale is added to the exponent of the weights that multiply V.
//
// Precision: q is scaled by a power of two per row into float16's range (exact for float16 and
// bfloat16; what a bfloat16 row loses below 2^-39 of its largest element does not reach a float32 sum);
// float32 queries are cut into two float16 terms (22 bits).  Scores, maxima, sums and O are float32.
// The weights are rounded to float16 for the second product (11 bits, at most 2^-11 of a weight, where a
// bfloat16 or float16 output is itself rounded to 2^-8 or 2^-11); float32 outputs take two terms.
//
// Two running maxima: m of the scores (for the sum of weights), mv of score + log2(value scale) (for the
// weighted sum of codes), so a page whose values are large or small against the others' loses nothing.
//
// Split: every warp works alone on tiles of 16 tokens, kStages of them in flight in its own part of
// shared memory (cp.async), and keeps its own maxima, sums and O; a CTA's warps are joined through
// shared memory, and where a sequence is cut into several CTAs a second small kernel joins their parts.
// Every CTA derives the cut from the lengths on the device: pieces of equal size for all sequences of the
// call, so ragged batches and long single sequences both fill the machine, without a host round trip.
#include <algorithm>
#include <math_constants.h>

#include "common.cuh"

namespace ab {
namespace {

constexpr int kWarps = 4;
constexpr int kStages = 4;
constexpr int kTokens = 16;     // per tile
constexpr int kMinPiece = 128;  // tokens a CTA gets at least: two tiles per warp

struct AttnArgs {
    const int8_t *key, *value;
    const float *key_scale, *value_scale;
    int64_t pages;
    int heads, page, dim;
    const void *q;
    int64_t q_seq, q_tok, q_head;
    void *out;
    float *lse;        // or NULL
    float *part;       // partial results of the pieces, or NULL
    const int32_t *table, *context, *qlens;
    int64_t table_stride;
    int table_width, seqs, tokens, group, row_blocks, pieces;
    int causal, window, vec;
    int target;        // CTAs per head and row block that fill the machine
    float scale_log2;  // softmax scale * log2(e)
};

__host__ __device__ inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 floats_of(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2 *>(&h)); }
// 1024 + (code + 128) in both halves -> the codes
__device__ __forceinline__ uint32_t unbias(uint32_t v) {
    const uint32_t bias = 0x64806480u;  // 1152, 1152
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&bias));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// Shared memory of a tile: rows of DP bytes, cut into 16-byte chunks whose place within a 128-byte line is
// permuted so that the operand reads below meet no bank twice.  K is read 16 bytes per lane, eight lanes
// at a time from two neighbouring rows; V four bytes per lane from four rows two apart.
template <int DP> __device__ __forceinline__ uint32_t place_k(int row, int chunk) {
    const uint32_t at = row * DP + chunk * 16;
    return DP == 64 ? at : at ^ ((row & 1) << 6);
}
template <int DP> __device__ __forceinline__ uint32_t place_v(int row, int byte) {
    const uint32_t at = row * DP + byte;
    return at ^ (((row >> 1) & 3) << 5);
}

// 16 consecutive elements of a query row as floats, zeros beyond the row's end
template <typename E> __device__ __forceinline__ void load_row16(const E *p, int left, bool vec, float (&f)[16]) {
    constexpr int V = 16 / sizeof(E);
    if (left <= 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = 0.f;
        return;
    }
    // dim is a multiple of 16, so there are 16 elements or none
#pragma unroll
    for (int j = 0; j < 16 / V; ++j) {
        Vec16<E> v;
        if (vec)
            v = *reinterpret_cast<const Vec16<E> *>(p + j * V);
        else
#pragma unroll
            for (int i = 0; i < V; ++i) v.v[i] = p[j * V + i];
#pragma unroll
        for (int i = 0; i < V; ++i) f[j * V + i] = to_f32(v.v[i]);
    }
}

// What a sequence's row block sees: tokens [lo, hi)
struct Span {
    int lo, hi;
};
__device__ __forceinline__ Span span_of(const AttnArgs &a, int ctx, int len, int first_token, int last_token) {
    Span s;
    const int base = ctx - len;  // position of the first query token; negative if there are more than the context
    s.hi = a.causal ? min(ctx, base + last_token + 1) : ctx;
    s.lo = a.window > 0 ? max(0, base + first_token - a.window + 1) : 0;
    s.hi = max(s.hi, 0);
    s.lo = min(s.lo, s.hi);
    return s;
}

// tokens per piece, the same for every sequence of the call
__device__ __forceinline__ int piece_tokens(const AttnArgs &a, int lane) {
    long long sum = 0;
    int most = 0;
    const int cap = (int)min((long long)a.table_width * a.page, 0x7fffffffll);
    for (int s = lane; s < a.seqs; s += 32) {
        int n = min(max(a.context[s], 0), cap);
        const int len = a.qlens ? min(max(a.qlens[s], 0), a.tokens) : a.tokens;
        // a window's span starts at a multiple of kTokens: up to kTokens - 1 tokens early
        if (a.window > 0) n = min(n, a.window + len + kTokens);
        if (len == 0) n = 0;
        sum += n;
        most = max(most, n);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    long long n = max((sum + a.target - 1) / a.target, ((long long)most + a.pieces - 1) / a.pieces);
    n = max(n, (long long)kMinPiece);
    return (int)((n + 63) / 64 * 64);
}

template <typename E, int DP, int RT> struct Layout {
    static constexpr int kTile = kTokens * DP;             // bytes of K or V of a tile
    static constexpr int kStage = 2 * kTile + 128;          // and the two scales, padded to a swizzle line
    static constexpr int kWarp = kStages * kStage;
    static constexpr int kRows = 16 * RT;
    static constexpr int kJoin = kRows * DP * 4 + kRows * 8;  // a warp's O, maxima and sums
    static constexpr int kPerWarp = kWarp > kJoin ? kWarp : (kJoin + 127) / 128 * 128;
    static constexpr int kSmem = kWarps * kPerWarp;
};

template <typename E, int DP, int RT> __global__ void __launch_bounds__(kWarps * 32) k_kv_attention(AttnArgs a) {
    using L = Layout<E, DP, RT>;
    constexpr bool F32 = sizeof(E) == 4;
    constexpr int NC = DP / 64;       // 64-wide parts of a row
    constexpr int QS = F32 ? 2 : 1;   // float16 terms of q and of the weights
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int piece = blockIdx.x, h = blockIdx.y / a.row_blocks, rb = blockIdx.y % a.row_blocks, s = blockIdx.z;
    pdl_prologue();

    const int cap = (int)min((long long)a.table_width * a.page, 0x7fffffffll);
    const int ctx = min(max(a.context[s], 0), cap);
    const int len = a.qlens ? min(max(a.qlens[s], 0), a.tokens) : a.tokens;
    const int rows = a.tokens * a.group;                    // of the output
    const int row0 = rb * L::kRows;
    const int live = min(max(len * a.group - row0, 0), L::kRows);  // rows of this block with a query
    const int first_token = row0 / a.group, last_token = (row0 + live - 1) / a.group;
    Span span = {0, 0};
    if (live > 0) span = span_of(a, ctx, len, first_token, last_token);
    int from = span.lo, to = span.hi;
    if (a.part) {
        const int n = piece_tokens(a, lane);
        const int start = span.lo & ~(kTokens - 1);
        const long long p0 = (long long)start + (long long)piece * n;
        from = (int)min((long long)to, max((long long)from, p0));
        to = (int)min((long long)to, p0 + n);
        if (piece > 0 && from >= to) return;  // the joining kernel derives the same pieces
    }

    // the queries of this warp's rows as operand fragments
    uint32_t qf[RT][QS][NC][4][4];
    float score_scale[RT][2];
    int lo_row[RT][2], hi_row[RT][2];
    int max_lo = 0, min_hi = 0x7fffffff;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 16 * rt + g + 8 * i;
            const bool alive = r < live;
            const int token = alive ? (row0 + r) / a.group : first_token;
            const int gq = alive ? (row0 + r) % a.group : 0;
            const Span sp = live > 0 ? span_of(a, ctx, len, token, token) : Span{0, 0};
            lo_row[rt][i] = sp.lo;
            hi_row[rt][i] = sp.hi;
            const E *p = static_cast<const E *>(a.q) + (int64_t)s * a.q_seq + (int64_t)token * a.q_tok + (int64_t)(h * a.group + gq) * a.q_head;
            float top = 0.f;
            float f[NC][16];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int d = 64 * c + 16 * t;
                load_row16(p + d, alive ? a.dim - d : 0, a.vec, f[c]);
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(f[c][e]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // top in [2^(e-1), 2^e): times 2^(15-e) it lies in [2^14, 2^15)
            int e = 0;
            float up = 1.f, down = 1.f;
            if (top > 0.f && top <= 3.402823466e38f) {
                frexpf(top, &e);
                e = min(max(15 - e, -120), 120);
                up = ldexpf(1.f, e);
                down = ldexpf(1.f, -e);
            }
            score_scale[rt][i] = down * a.scale_log2;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int st = 0; st < 4; ++st)
#pragma unroll
                    for (int p2 = 0; p2 < 2; ++p2) {
                        const float x0 = f[c][4 * st + 2 * p2] * up, x1 = f[c][4 * st + 2 * p2 + 1] * up;
                        const uint32_t hi = half2_of(x0, x1);
                        qf[rt][0][c][st][i + 2 * p2] = hi;
                        if constexpr (F32) {
                            const float2 b = floats_of(hi);
                            qf[rt][QS - 1][c][st][i + 2 * p2] = half2_of(x0 - b.x, x1 - b.y);
                        }
                    }
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int i = 0; i < 2; ++i) max_lo = max(max_lo, lo_row[rt][i]), min_hi = min(min_hi, hi_row[rt][i]);
    // of all rows of the tile, so that the choice of the masked path is the warp's
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        max_lo = max(max_lo, __shfl_xor_sync(0xffffffffu, max_lo, o));
        min_hi = min(min_hi, __shfl_xor_sync(0xffffffffu, min_hi, o));
    }

    float m[RT][2], mv[RT][2], sum[RT][2];
    float o[RT][DP / 8][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int i = 0; i < 2; ++i) m[rt][i] = mv[rt][i] = -CUDART_INF_F, sum[rt][i] = 0.f;
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[rt][n][i] = 0.f;
    }

    const int tile0 = from / kTokens, tiles = from < to ? (to - 1) / kTokens - tile0 + 1 : 0;
    const int mine = tiles > warp ? (tiles - warp - 1) / kWarps + 1 : 0;  // tiles of this warp
    uint8_t *ring = smem + warp * L::kPerWarp;
    const uint32_t ring_at = smem_u32(ring);
    const int32_t *table = a.table + (int64_t)s * a.table_stride;
    const int chunks = a.dim / 16;

    auto page_of = [&](int i) -> int {  // of this warp's i-th tile; to <= table_width * page
        return i < mine ? table[(int64_t)(tile0 + warp + i * kWarps) * kTokens / a.page] : -1;
    };
    auto request = [&](int i, int pg) {
        if (i < mine) {
            const int token = (tile0 + warp + i * kWarps) * kTokens;
            const bool there = pg >= 0 && pg < a.pages;
            const int64_t ph = there ? (int64_t)pg * a.heads + h : 0;
            const int64_t at = (ph * a.page + token % a.page) * a.dim;
            const uint32_t dst = ring_at + (i % kStages) * L::kStage;
#pragma unroll
            for (int c = lane; c < L::kTile / 16; c += 32) {
                const int r = c / (DP / 16), ch = c % (DP / 16);
                const bool ok = there && ch < chunks;
                const int64_t off = ok ? at + (int64_t)r * a.dim + ch * 16 : 0;
                cp_async16(dst + place_k<DP>(r, ch), a.key + off, ok ? 16 : 0);
                cp_async16(dst + L::kTile + place_v<DP>(r, ch * 16), a.value + off, ok ? 16 : 0);
            }
            // where there is no page, zeros: whatever page 0 holds must not reach the sums
            if (lane == 0) cp_async4(dst + 2 * L::kTile, a.key_scale + ph, there ? 4 : 0);
            if (lane == 1) cp_async4(dst + 2 * L::kTile + 4, a.value_scale + ph, there ? 4 : 0);
        }
        cp_commit();
    };

    int pg_of[kStages];  // pages of the tiles in flight, to know which are not there
#pragma unroll
    for (int i = 0; i < kStages; ++i) pg_of[i] = page_of(i);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) request(i, pg_of[i]);
    int pg_next = pg_of[kStages - 1];
    uint32_t gone = 0;  // bit per stage: its tile has no page
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) gone |= (uint32_t)(pg_of[i] < 0 || pg_of[i] >= a.pages) << i;

    for (int i = 0; i < mine; ++i) {
        cp_wait<kStages - 2>();
        __syncwarp();
        {
            const int nx = i + kStages - 1, slot = nx % kStages;
            const int after = page_of(nx + 1);
            request(nx, pg_next);
            gone = (gone & ~(1u << slot)) | (uint32_t)(pg_next < 0 || pg_next >= a.pages) << slot;
            pg_next = after;
        }
        const int slot = i % kStages;
        const uint8_t *kt = ring + slot * L::kStage, *vt = kt + L::kTile;
        const float2 scales = *reinterpret_cast<const float2 *>(kt + 2 * L::kTile);
        const int token0 = (tile0 + warp + i * kWarps) * kTokens;

        // scores
        float sc[RT][2][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[rt][n][e] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const uint4 w4 = *reinterpret_cast<const uint4 *>(kt + place_k<DP>(8 * n + g, 4 * c + t));
                const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    const uint32_t u = w[st] ^ 0x80808080u;
                    const uint32_t b0 = unbias(__byte_perm(u, 0x64646464u, 0x4140)), b1 = unbias(__byte_perm(u, 0x64646464u, 0x4342));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int q = 0; q < QS; ++q) mma_f16(sc[rt][n], qf[rt][q][c][st], b0, b1);
                }
            }

        const bool masked = token0 < max_lo || token0 + kTokens > min_hi || ((gone >> slot) & 1);
        const float lv = scales.y > 0.f ? log2_fast(scales.y) : -CUDART_INF_F;
        uint32_t pf[RT][QS][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float p[2][2][2];  // [row][n][e]
            bool moved = false;
            float turn[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float f = score_scale[rt][r] * scales.x;
                float top = -CUDART_INF_F;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = sc[rt][n][2 * r + e] * f;
                        if (masked) {
                            const int at = token0 + 8 * n + 2 * t + e;
                            if (at < lo_row[rt][r] || at >= hi_row[rt][r] || ((gone >> slot) & 1)) v = -CUDART_INF_F;
                        }
                        p[r][n][e] = v;
                        top = fmaxf(top, v);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float m1 = fmaxf(m[rt][r], top), ref = m1 == -CUDART_INF_F ? 0.f : m1;
                float add = 0.f;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) add += exp2_fast(p[r][n][e] - ref);
                sum[rt][r] = sum[rt][r] * exp2_fast(m[rt][r] - ref) + add;
                m[rt][r] = m1;
                const float v1 = fmaxf(mv[rt][r], top + lv), vref = v1 == -CUDART_INF_F ? 0.f : v1;
                turn[r] = exp2_fast(mv[rt][r] - vref);
                moved |= v1 != mv[rt][r];
                mv[rt][r] = v1;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) p[r][n][e] = exp2_fast(p[r][n][e] + (lv - vref));
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) {
                    o[rt][n][0] *= turn[0];
                    o[rt][n][1] *= turn[0];
                    o[rt][n][2] *= turn[1];
                    o[rt][n][3] *= turn[1];
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t hi = half2_of(p[r][n][0], p[r][n][1]);
                    pf[rt][0][2 * n + r] = hi;
                    if constexpr (F32) {
                        const float2 b = floats_of(hi);
                        pf[rt][QS - 1][2 * n + r] = half2_of(p[r][n][0] - b.x, p[r][n][1] - b.y);
                    }
                }
        }

        // O += P . V
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                w[r] = *reinterpret_cast<const uint32_t *>(vt + place_v<DP>(2 * t + (r & 1) + 8 * (r >> 1), 32 * c + 4 * g)) ^ 0x80808080u;
            const uint32_t lo0 = __byte_perm(w[0], w[1], 0x5140), hi0 = __byte_perm(w[0], w[1], 0x7362);
            const uint32_t lo1 = __byte_perm(w[2], w[3], 0x5140), hi1 = __byte_perm(w[2], w[3], 0x7362);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t sel = (j & 1) ? 0x4342 : 0x4140;
                const uint32_t b0 = unbias(__byte_perm(j < 2 ? lo0 : hi0, 0x64646464u, sel));
                const uint32_t b1 = unbias(__byte_perm(j < 2 ? lo1 : hi1, 0x64646464u, sel));
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int q = 0; q < QS; ++q) mma_f16(o[rt][4 * c + j], pf[rt][q], b0, b1);
            }
        }
        __syncwarp();
    }
    cp_wait<0>();
    __syncthreads();

    // join the CTA's warps.  A warp's O moves from units of 2^mv to units of 2^m.
    float *mine_o = reinterpret_cast<float *>(ring);
    float *mine_m = mine_o + L::kRows * DP;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float l = sum[rt][r];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            const float unit = mv[rt][r] == -CUDART_INF_F ? 0.f : exp2_fast(mv[rt][r] - m[rt][r]);
            const int row = 16 * rt + g + 8 * r;
            if (t == 0) {
                mine_m[row] = m[rt][r];
                mine_m[L::kRows + row] = l;
            }
            // lane t holds dims 8t .. 8t+7 of every 32: four from column 2t, four from column 2t + 1
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
                float4 x, y;
                x.x = o[rt][4 * c][2 * r] * unit, x.y = o[rt][4 * c + 1][2 * r] * unit;
                x.z = o[rt][4 * c + 2][2 * r] * unit, x.w = o[rt][4 * c + 3][2 * r] * unit;
                y.x = o[rt][4 * c][2 * r + 1] * unit, y.y = o[rt][4 * c + 1][2 * r + 1] * unit;
                y.z = o[rt][4 * c + 2][2 * r + 1] * unit, y.w = o[rt][4 * c + 3][2 * r + 1] * unit;
                float4 *dst = reinterpret_cast<float4 *>(mine_o + row * DP + 32 * c + 8 * t);
                dst[0] = x;
                dst[1] = y;
            }
        }
    __syncthreads();

    const int stored = min(L::kRows, rows - row0);  // rows of the output in this block
    const int per_row = a.dim / 4;
    const int64_t slot_row = (((int64_t)s * a.heads + h) * a.row_blocks + rb) * a.pieces + piece;
    for (int i = threadIdx.x; i < stored * per_row; i += kWarps * 32) {
        const int r = i / per_row, d = (i - r * per_row) * 4;
        float top = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, reinterpret_cast<const float *>(smem + w * L::kPerWarp)[L::kRows * DP + r]);
        const float ref = top == -CUDART_INF_F ? 0.f : top;
        float l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float *b = reinterpret_cast<const float *>(smem + w * L::kPerWarp);
            const float f = exp2_fast(b[L::kRows * DP + r] - ref);
            const float4 x = *reinterpret_cast<const float4 *>(b + r * DP + d);
            l += b[L::kRows * DP + L::kRows + r] * f;
            v.x += x.x * f, v.y += x.y * f, v.z += x.z * f, v.w += x.w * f;
        }
        if (a.part) {
            float *dst = a.part + (slot_row * L::kRows + r) * (int64_t)(a.dim + 4);
            *reinterpret_cast<float4 *>(dst + 4 + d) = v;
            if (d == 0) dst[0] = top, dst[1] = l;
            continue;
        }
        const bool dead = r >= live || !(l > 0.f || l != l);
        const float inv = dead ? 0.f : 1.f / l;
        const int token = (row0 + r) / a.group, hq = h * a.group + (row0 + r) % a.group;
        const int64_t at = ((int64_t)s * a.tokens + token) * (a.heads * a.group) + hq;
        E *dst = static_cast<E *>(a.out) + at * a.dim + d;
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[j] = Cvt<float, E>::store(dead ? 0.f : e[j] * inv);
        if (a.lse && d == 0) a.lse[at] = dead ? -CUDART_INF_F : (top + log2f(l)) * 0.69314718055994531f;
    }
}

// One warp per output row: joins the pieces of its sequence.
template <typename E> __global__ void __launch_bounds__(128) k_kv_join(AttnArgs a, int rows_per_block) {
    const int lane = threadIdx.x & 31;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);  // row of the output
    pdl_prologue();
    const int64_t all_heads = (int64_t)a.heads * a.group;
    if (at >= (int64_t)a.seqs * a.tokens * all_heads) return;
    const int hq = (int)(at % all_heads), token = (int)(at / all_heads % a.tokens), s = (int)(at / all_heads / a.tokens);
    const int h = hq / a.group, row = token * a.group + hq % a.group, rb = row / rows_per_block;
    const int cap = (int)min((long long)a.table_width * a.page, 0x7fffffffll);
    const int ctx = min(max(a.context[s], 0), cap);
    const int len = a.qlens ? min(max(a.qlens[s], 0), a.tokens) : a.tokens;
    const int row0 = rb * rows_per_block;
    const int live = min(max(len * a.group - row0, 0), rows_per_block);
    int pieces = 0;
    if (row - row0 < live) {
        const Span sp = span_of(a, ctx, len, row0 / a.group, (row0 + live - 1) / a.group);
        const int n = piece_tokens(a, lane);
        pieces = sp.hi > sp.lo ? (int)((sp.hi - (sp.lo & ~(kTokens - 1)) + (long long)n - 1) / n) : 0;
    }
    const float *part = a.part + (((((int64_t)s * a.heads + h) * a.row_blocks + rb) * a.pieces) * rows_per_block + (row - row0)) * (int64_t)(a.dim + 4);
    const int64_t step = (int64_t)rows_per_block * (a.dim + 4);
    float top = -CUDART_INF_F;
    for (int p = lane; p < pieces; p += 32) top = fmaxf(top, part[p * step]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float ref = top == -CUDART_INF_F ? 0.f : top;
    float l = 0.f;
    float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
    for (int p = 0; p < pieces; ++p) {
        const float *b = part + p * step;
        const float f = exp2_fast(b[0] - ref);
        l += b[1] * f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int d = 128 * c + 4 * lane;
            if (d < a.dim) {
                const float4 x = *reinterpret_cast<const float4 *>(b + 4 + d);
                v[c].x += x.x * f, v[c].y += x.y * f, v[c].z += x.z * f, v[c].w += x.w * f;
            }
        }
    }
    const bool dead = !(l > 0.f || l != l);
    const float inv = dead ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int d = 128 * c + 4 * lane;
        if (d >= a.dim) continue;
        E *dst = static_cast<E *>(a.out) + at * a.dim + d;
        const float e[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[j] = Cvt<float, E>::store(dead ? 0.f : e[j] * inv);
    }
    if (a.lse && lane == 0) a.lse[at] = dead ? -CUDART_INF_F : (top + log2f(l)) * 0.69314718055994531f;
}

// how a call is cut: row blocks of 16 or 32 rows, pieces along the cache
struct Cut {
    int row_tiles, row_blocks, pieces, target;
};
int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
Cut cut_of(int heads, int dim, int group, int page, int64_t seqs, int64_t tokens, int64_t table_width, int io_dtype) {
    Cut c;
    const int64_t rows = tokens * group;
    // two row tiles per warp read and convert the cache once for 32 rows; O and Q of a second tile do not
    // fit the registers for wider heads, nor for float32's two terms
    c.row_tiles = rows > 16 && padded_dim(dim) <= 128 && io_dtype != AB_F32 ? 2 : 1;
    c.row_blocks = (int)std::min<int64_t>(div_up(rows, 16 * c.row_tiles), 1 << 20);
    const int64_t length = table_width * page;
    const int resident = padded_dim(dim) <= 128 && c.row_tiles == 1 ? 3 : 1;
    const int64_t slots = (int64_t)sm_count() * resident;
    c.target = (int)std::max<int64_t>(1, slots / std::max<int64_t>(1, (int64_t)heads * c.row_blocks));
    const int64_t even = div_up(slots, std::max<int64_t>(1, seqs * heads * c.row_blocks));
    c.pieces = (int)std::max<int64_t>(1, std::min<int64_t>(div_up(length, kMinPiece), even == 1 ? 2 : 4 * even));
    return c;
}

int check_call(const ab_kv_cache *c, int64_t seqs, int64_t tokens, int64_t group, int64_t table_width, int io_dtype) {
    if (!c) return fail(AB_ERR_INVALID, "cache is NULL");
    if (c->num_pages < 1 || c->num_pages > 0x7fffffff) return fail(AB_ERR_INVALID, "num_pages=%lld", (long long)c->num_pages);
    if (c->page_size < 16 || c->page_size % 16 || c->page_size > 1024)
        return fail(AB_ERR_UNSUPPORTED, "page_size=%d: a multiple of 16 up to 1024", c->page_size);
    if (c->head_dim < 16 || c->head_dim % 16 || c->head_dim > 256)
        return fail(AB_ERR_UNSUPPORTED, "head_dim=%d: a multiple of 16 up to 256", c->head_dim);
    if (io_dtype != AB_F32 && io_dtype != AB_F16 && io_dtype != AB_BF16) return fail(AB_ERR_UNSUPPORTED, "io_dtype %d", io_dtype);
    if (seqs < 0 || tokens < 0 || group < 1 || table_width < 0 || seqs > 65535 || tokens > (1 << 20) || group > 1024 ||
        table_width * c->page_size > 0x7fffffffll - 4096)
        return fail(AB_ERR_INVALID, "seqs=%lld tokens=%lld group=%lld table_width=%lld", (long long)seqs, (long long)tokens, (long long)group,
                    (long long)table_width);
    if (c->num_heads < 1 || c->num_heads > 1024) return fail(AB_ERR_INVALID, "num_heads=%d", c->num_heads);
    if ((int64_t)c->num_heads * div_up(tokens * group, 16) > 65535)
        return fail(AB_ERR_UNSUPPORTED, "%lld query rows of %d heads in one call", (long long)(tokens * group), c->num_heads);
    return AB_OK;
}

template <typename E, int DP, int RT> int launch(const AttnArgs &a, cudaStream_t st) {
    using L = Layout<E, DP, RT>;
    const int rc = opt_in_smem<k_kv_attention<E, DP, RT>>(L::kSmem);
    if (rc != AB_OK) return rc;
    AB_CUDA_OK(launch_pdl(k_kv_attention<E, DP, RT>, dim3((unsigned)a.pieces, (unsigned)(a.heads * a.row_blocks), (unsigned)a.seqs),
                          dim3(kWarps * 32), L::kSmem, st, a));
    AB_LAUNCH_OK();
    if (a.part) {
        const int64_t rows = (int64_t)a.seqs * a.tokens * a.heads * a.group;
        AB_CUDA_OK(launch_pdl(k_kv_join<E>, dim3((unsigned)div_up(rows, 4)), dim3(128), 0, st, a, L::kRows));
        AB_LAUNCH_OK();
    }
    return AB_OK;
}
template <typename E> int dispatch(const AttnArgs &a, int row_tiles, cudaStream_t st) {
    const int dp = padded_dim(a.dim);
    if constexpr (sizeof(E) == 2) {
        if (row_tiles == 2) return dp == 64 ? launch<E, 64, 2>(a, st) : launch<E, 128, 2>(a, st);
    }
    return dp == 64 ? launch<E, 64, 1>(a, st) : dp == 128 ? launch<E, 128, 1>(a, st) : launch<E, 256, 1>(a, st);
}

}  // namespace
}  // namespace ab

using namespace ab;

extern "C" int64_t aimet_b200_kv_attention_scratch_bytes(const ab_kv_cache *cache, int64_t seqs, int64_t tokens, int64_t group,
                                                         int64_t table_width, int io_dtype) {
    const int rc = check_call(cache, seqs, tokens, group, table_width, io_dtype);
    if (rc != AB_OK) return rc;
    if (seqs == 0 || tokens == 0) return 0;
    const Cut c = cut_of(cache->num_heads, cache->head_dim, (int)group, cache->page_size, seqs, tokens, table_width, io_dtype);
    if (c.pieces == 1) return 0;
    return seqs * cache->num_heads * c.row_blocks * c.pieces * 16 * c.row_tiles * (int64_t)(cache->head_dim + 4) * 4;
}

extern "C" int aimet_b200_kv_attention(const ab_kv_cache *cache, const void *query, const int64_t *query_strides, void *out, float *lse,
                                       int64_t seqs, int64_t tokens, int64_t group, const int32_t *block_table, int64_t table_stride,
                                       int64_t table_width, const int32_t *context_lens, const int32_t *query_lens, int causal,
                                       int64_t window, double softmax_scale, int io_dtype, void *scratch, int64_t scratch_bytes,
                                       void *stream) {
    const int64_t need = aimet_b200_kv_attention_scratch_bytes(cache, seqs, tokens, group, table_width, io_dtype);
    if (need < 0) return (int)need;
    if (seqs == 0 || tokens == 0) return AB_OK;
    if (!cache->key || !cache->value || !cache->key_scale || !cache->value_scale) return fail(AB_ERR_INVALID, "a buffer of the cache is NULL");
    if (!aligned16(cache->key) || !aligned16(cache->value)) return fail(AB_ERR_INVALID, "the cache's codes must be 16-byte aligned");
    if (!query || !query_strides || !out || !context_lens || (table_width > 0 && !block_table)) return fail(AB_ERR_INVALID, "a pointer is NULL");
    if (window < 0 || window > 0x7fffffff) return fail(AB_ERR_INVALID, "window=%lld", (long long)window);
    if (need > 0 && (!scratch || scratch_bytes < need || !aligned16(scratch)))
        return fail(AB_ERR_SCRATCH, "scratch of %lld bytes, 16-byte aligned, is needed (got %lld)", (long long)need, (long long)scratch_bytes);
    const Cut cut = cut_of(cache->num_heads, cache->head_dim, (int)group, cache->page_size, seqs, tokens, table_width, io_dtype);
    AttnArgs a;
    a.key = static_cast<const int8_t *>(cache->key);
    a.value = static_cast<const int8_t *>(cache->value);
    a.key_scale = static_cast<const float *>(cache->key_scale);
    a.value_scale = static_cast<const float *>(cache->value_scale);
    a.pages = cache->num_pages;
    a.heads = cache->num_heads;
    a.page = cache->page_size;
    a.dim = cache->head_dim;
    a.q = query;
    a.q_seq = query_strides[0];
    a.q_tok = query_strides[1];
    a.q_head = query_strides[2];
    const int64_t size = dtype_size(io_dtype);
    a.vec = aligned16(query) && (a.q_seq * size) % 16 == 0 && (a.q_tok * size) % 16 == 0 && (a.q_head * size) % 16 == 0;
    a.out = out;
    a.lse = lse;
    a.part = need > 0 ? static_cast<float *>(scratch) : nullptr;
    a.table = block_table;
    a.context = context_lens;
    a.qlens = query_lens;
    a.table_stride = table_stride;
    a.table_width = (int)table_width;
    a.seqs = (int)seqs;
    a.tokens = (int)tokens;
    a.group = (int)group;
    a.row_blocks = cut.row_blocks;
    a.pieces = cut.pieces;
    a.target = cut.target;
    a.causal = causal != 0;
    a.window = (int)std::min<int64_t>(window, 1 << 30);
    a.scale_log2 = (float)(softmax_scale * 1.4426950408889634);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (io_dtype) {
        case AB_F32: return dispatch<float>(a, cut.row_tiles, st);
        case AB_F16: return dispatch<__half>(a, cut.row_tiles, st);
        default: return dispatch<__nv_bfloat16>(a, cut.row_tiles, st);
    }
}
