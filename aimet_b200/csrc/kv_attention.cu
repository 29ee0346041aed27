// Attention of a sequence's newest tokens over the paged 8-bit cache (kv_cache.cu):
//
//   o_i = sum_j softmax_j(c q_i . k_j) v_j,   j <= p_i and j > p_i - window,   p_i = context - query_len + i
//
// with k_j, v_j = code * scale of the token's page and head.  One pass over the cache with the running
// maximum and sum of the softmax; the codes go from HBM to the operand registers in 8 bits.
//
// What bounds it is reading the codes: 2 * dim bytes per token and head, for a handful of rows (the
// query heads that share a head of the cache, times the query tokens); at the measured copy rate an SM gets 23
// codes per clock, so what has to be saved is instructions per code.  The codes are the 16-row operand of
// mma.sync and eight query rows the 8 columns (tcgen05 needs 128 rows of converted codes in shared
// memory first): S^T (16 tokens x 8) = K . Q^T, then O^T (dim x 8) += V^T . P^T.  Codes become float16 pairs
// exactly (a byte permute puts code + 128 into the mantissa of 1024, subtracting 1152 leaves the code), P^T
// moves from the first product's result layout to the second's operand layout by an 8 x 8 transpose
// (movmatrix).  More rows are further columns that share the converted codes.  The scales
// never touch an element: a tile of 16 tokens lies in one page, so the key scale multiplies the scores,
// and log2 of the value scale is added to the exponent of the weights that multiply V.
// Measured: 64 contexts of 1000 to 4000 tokens, 8 heads of 128 for 32 query heads, 86 us of 55 (4.1 TB/s; 135 with query
// rows as the 16-row operand), 2 of 131072 tokens 100 us of 71 (4.6 TB/s); issue slots 57 % taken.
//
// Precision: q is scaled by a power of two per row into float16's range (exact for float16 and
// bfloat16; what a bfloat16 row loses below 2^-39 of its largest element does not reach a float32 sum);
// float32 queries are cut into two float16 terms (22 bits).  Scores, maxima, sums and O are float32.
// The weights are rounded to float16 for the second product, scaled by 2^15 so that the largest lies in the
// upper end of its range: at most 2^-11 of a weight is lost (where a bfloat16 or float16 output is itself
// rounded to 2^-8 or 2^-11), 2^-22 where float32 outputs take two terms, and below 2^-29 of the largest weight times
// value scale, where float16 has no more normal numbers, 2^-40 of that largest.
//
// Two running maxima: m of the scores (for the sum of weights), mv of score - m + log2(value scale) (for the
// weighted sum of codes, whose unit is 2^(m + mv - 15)), so a page whose values are large or small against the
// others' loses nothing.  mv is relative to m: both sums take a token's weight from the same difference score - m, and
// stay consistent where scores are so large that m + log2(value scale) would not hold the second term.
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
// Tokens of a piece at least: two tiles per warp where contexts are short (one of 500 tokens: 5.9 us with pieces
// of 128, 7.1 with 256, 8.0 uncut), up to 512 where they are long (one of 32000: 30.1 us with 512 or 192 at most, 32.2
// with 1024; 8000 in a table for 131072: 19.7, 19.2 and 19.7).
constexpr int kMinPiece = 128, kMaxMinPiece = 512;
// Pieces per CTA slot of the machine: one where pieces are all that fills it (two of 131072 tokens: 112 us, 118 with
// two; 8000 in a table for 131072: 19.7 and 25.3); three where sequences and heads do, so that ragged lengths even out
// (64 of 1000 to 4000: 79 us, 82 with one).
constexpr int kWaves = 3;
constexpr int kMostCluster = 8, kClusterPiece = 1024;

constexpr float kWeightExponent = 15.f, kWeightDown = 1.f / 32768.f;  // weights are multiplied as 2^15 times themselves
constexpr float kLeastUnit = -126.f;  // of mv: values that are nothing beside float32's smallest normal number make no unit of their own

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
    uint32_t page_magic;  // tile / (page / kTokens) == umulhi(tile, page_magic) (tiles below 2^26, at most 64 in a page); 0: one tile in a page
    int table_width, seqs, tokens, group, row_blocks, pieces;
    int first_block, blocks;  // row blocks of this launch
    int causal, window, vec;
    int target;        // CTAs per head and row block that fill the machine
    float scale_log2;  // softmax scale * log2(e)
};

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

__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Shared memory of a tile: rows of DP bytes, cut into 16-byte chunks whose place within a 128-byte line is
// permuted so that the operand reads below meet no bank twice.  K is read 16 bytes per lane, eight lanes
// at a time from two neighbouring rows; V eight bytes per lane, sixteen lanes at a time from four rows two apart.
template <int DP> __device__ __forceinline__ uint32_t place_k(int row, int chunk) {
    const uint32_t at = row * DP + chunk * 16;
    return DP == 64 ? at : at ^ ((row & 1) << 6);
}
template <int DP> __device__ __forceinline__ uint32_t place_v(int row, int byte) {
    const uint32_t at = row * DP + byte;
    return at ^ (((row >> 1) & 3) << 5);
}

// 16 consecutive elements of a query row
template <typename E> struct Sixteen {
    Vec16<E> v[sizeof(E)];
};
template <typename E> __device__ __forceinline__ void load_row16(const E *p, bool vec, Sixteen<E> &x) {
    constexpr int V = 16 / sizeof(E);
#pragma unroll
    for (int j = 0; j < (int)sizeof(E); ++j) {
        if (vec) {
            x.v[j] = *reinterpret_cast<const Vec16<E> *>(p + j * V);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) x.v[j].v[i] = p[j * V + i];
        }
    }
}

__device__ __forceinline__ uint32_t in_cluster(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// four neighbouring results, scaled (dims are multiples of 16 and outputs 16-byte aligned)
template <typename E> __device__ __forceinline__ void store4(E *dst, const float4 &v, float inv, bool dead) {
    const float e[4] = {dead ? 0.f : v.x * inv, dead ? 0.f : v.y * inv, dead ? 0.f : v.z * inv, dead ? 0.f : v.w * inv};
    if constexpr (sizeof(E) == 4) {
        *reinterpret_cast<float4 *>(dst) = make_float4(e[0], e[1], e[2], e[3]);
    } else {
        E h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = Cvt<float, E>::store(e[j]);
        *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(h);
    }
}

// What a sequence's row block sees: tokens [lo, hi).  Positions count all of the context, tokens are those that the
// table has room for.
struct Span {
    int lo, hi;
};
__device__ __forceinline__ Span span_of(const AttnArgs &a, int ctx, int cap, int len, int first_token, int last_token) {
    Span s;
    const int base = ctx - len;  // position of the first query token; negative if there are more than the context
    s.hi = a.causal ? min(ctx, base + last_token + 1) : ctx;
    s.lo = a.window > 0 ? max(0, base + first_token - a.window + 1) : 0;
    s.hi = max(min(s.hi, cap), 0);
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
    n = max(n, (long long)min(max(most / 16, kMinPiece), kMaxMinPiece));
    return (int)((n + 63) / 64 * 64);
}

template <typename E, int DP, int NQ> struct Layout {
    static constexpr int kTile = kTokens * DP;              // bytes of K or V of a tile
    static constexpr int kStage = 2 * kTile + 128;           // and the two scales, padded to a swizzle line
    static constexpr int kWarp = kStages * kStage;
    static constexpr int kRows = 8 * NQ;                     // query rows of a CTA
    static constexpr int kJoin = kRows * DP * 4 + kRows * 8;  // a warp's O, maxima and sums
    static constexpr int kPerWarp = kWarp > kJoin ? kWarp : (kJoin + 127) / 128 * 128;
    static constexpr int kSmem = kWarps * kPerWarp + kJoin;  // and a cluster's part
};

// FULL: the head's dim is DP, a constant
template <typename E, int DP, int NQ, bool FULL> __global__ void __launch_bounds__(kWarps * 32) k_kv_attention(AttnArgs a) {
    if (FULL) a.dim = DP;
    using L = Layout<E, DP, NQ>;
    constexpr bool F32 = sizeof(E) == 4;
    constexpr int NC = DP / 64;       // 64-wide parts of a row
    constexpr int QS = F32 ? 2 : 1;   // float16 terms of q and of the weights
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int piece = blockIdx.x, h = blockIdx.y / a.blocks, rb = a.first_block + blockIdx.y % a.blocks, s = blockIdx.z;
    const int rows = a.tokens * a.group;  // of the output
    const int row0 = rb * L::kRows;
    pdl_prologue();

    // this lane's part of query row g of every eight, requested before anything is known of the lengths
    Sixteen<E> raw[NQ][NC];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = row0 + 8 * n + g, token = r / a.group, gq = r - token * a.group;
        const E *p = static_cast<const E *>(a.q) + (int64_t)s * a.q_seq + (int64_t)token * a.q_tok + (int64_t)(h * a.group + gq) * a.q_head;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (r < rows && 64 * c + 16 * t < a.dim) load_row16(p + 64 * c + 16 * t, a.vec, raw[n][c]);
    }

    const int cap = (int)min((long long)a.table_width * a.page, 0x7fffffffll);
    const int ctx = max(a.context[s], 0);
    const int len = a.qlens ? min(max(a.qlens[s], 0), a.tokens) : a.tokens;
    const int live = min(max(len * a.group - row0, 0), L::kRows);  // rows of this block with a query
    const int first_token = row0 / a.group, last_token = (row0 + live - 1) / a.group;
    Span span = {0, 0};
    if (live > 0) span = span_of(a, ctx, cap, len, first_token, last_token);
    int from = span.lo, to = span.hi, count = 1;  // pieces of this row block
    if (a.part) {
        const int n = piece_tokens(a, lane);
        const int start = span.lo & ~(kTokens - 1);
        const long long p0 = (long long)start + (long long)piece * n;
        from = (int)min((long long)to, max((long long)from, p0));
        to = (int)min((long long)to, p0 + n);
        if (piece > 0 && from >= to) return;
        count = max(1, (span.hi - start + n - 1) / n);
    } else if (a.pieces > 1) {  // a cluster: even parts of this sequence
        const int start = span.lo & ~(kTokens - 1);
        const int n = max(((to - start + a.pieces - 1) / a.pieces + 63) / 64 * 64, kMinPiece);
        const long long p0 = (long long)start + (long long)piece * n;
        from = (int)min((long long)to, max((long long)from, p0));
        to = (int)min((long long)to, p0 + n);
    }

    const int tile0 = from / kTokens, tiles = from < to ? (to - 1) / kTokens - tile0 + 1 : 0;
    const int mine = tiles > warp ? (tiles - warp - 1) / kWarps + 1 : 0;  // tiles of this warp
    uint8_t *ring = smem + warp * L::kPerWarp;
    const uint32_t ring_at = smem_u32(ring);
    const int32_t *table = a.table + (int64_t)s * a.table_stride;

    // What a lane copies of every tile: 16-byte chunk lane % CH of rows lane / CH, lane / CH + 32 / CH, ...; chunks
    // beyond the head's dim are filled with zeros.
    constexpr int CH = DP / 16, STEP = 32 / CH, COPIES = kTokens / STEP;
    const int copy_row = lane / CH, copy_chunk = lane % CH;
    const bool copies = copy_chunk * 16 < a.dim;
    const int64_t copy_off = copies ? (int64_t)copy_row * a.dim + copy_chunk * 16 : 0;
    const int copy_step = copies ? STEP * a.dim : 0;
    // page and place in it of this warp's i-th tile; to <= table_width * page, and -1 is no page
    const uint32_t per_page = a.page / kTokens;
    struct Where {
        int page;
        uint32_t in_page;
    };
    auto where = [&](int i) -> Where {
        const uint32_t tile = tile0 + warp + i * kWarps, block = a.page_magic ? __umulhi(tile, a.page_magic) : tile;
        return {i < mine ? table[block] : -1, tile - block * per_page};
    };
    uint32_t gone = 0;  // bit per stage: its tile has no page
    const int64_t page_bytes = (int64_t)a.page * a.dim;
    const int8_t *key = a.key + h * page_bytes + copy_off, *value = a.value + h * page_bytes + copy_off;
    const float *scale = (lane ? a.value_scale : a.key_scale) + h;  // lanes 0 and 1 copy the scales
    const int tile_bytes = kTokens * a.dim;
    auto request = [&](int i, const Where &w) {
        const int slot = i % kStages;
        if (i < mine) {
            const bool there = (uint32_t)w.page < (uint32_t)a.pages;
            const int64_t ph = there ? (int64_t)w.page * a.heads : 0;
            const int64_t at = ph * page_bytes + w.in_page * tile_bytes;
            const int bytes = there && copies ? 16 : 0;  // where there is no page, zeros: what page 0 holds must not reach the sums
            const uint32_t dst = ring_at + slot * L::kStage;
            const int8_t *kp = key + at, *vp = value + at;
            gone = (gone & ~(1u << slot)) | (uint32_t)!there << slot;
#pragma unroll
            for (int j = 0; j < COPIES; ++j) {
                const int r = copy_row + j * STEP;
                cp_async16(dst + place_k<DP>(r, copy_chunk), kp + j * copy_step, bytes);
                cp_async16(dst + L::kTile + place_v<DP>(r, copy_chunk * 16), vp + j * copy_step, bytes);
            }
            if (lane < 2) cp_async4(dst + 2 * L::kTile + 4 * lane, scale + ph, there ? 4 : 0);
            __syncwarp();  // (the products that follow are a warp's lanes together)
        }
        cp_commit();
    };
    Where next;
    {
        Where w[kStages];
#pragma unroll
        for (int i = 0; i < kStages; ++i) w[i] = where(i);
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) request(i, w[i]);
        next = w[kStages - 1];
    }

    // the queries as operand fragments
    uint32_t qf[NQ][QS][NC][4][2];
    float score_scale[NQ][2];             // of rows 2t, 2t + 1 of the eight, as everything below
    int lo_row[NQ][2], hi_row[NQ][2];
    int max_lo = 0, min_hi = 0x7fffffff;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const bool alive = 8 * n + g < live;
        float top = 0.f;
        float f[NC][16];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const bool here = alive && 64 * c + 16 * t < a.dim;  // (dim is a multiple of 16: all sixteen or none)
            constexpr int V = 16 / sizeof(E);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                f[c][e] = here ? to_f32(raw[n][c].v[e / V].v[e % V]) : 0.f;
                top = fmaxf(top, fabsf(f[c][e]));
            }
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
        down *= a.scale_log2;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            score_scale[n][i] = __shfl_sync(0xffffffffu, down, (2 * t + i) * 4);
            const int row = 8 * n + 2 * t + i;
            const int tok = row < live ? (row0 + row) / a.group : first_token;
            const Span sp = live > 0 ? span_of(a, ctx, cap, len, tok, tok) : Span{0, 0};
            lo_row[n][i] = sp.lo;
            hi_row[n][i] = sp.hi;
            max_lo = max(max_lo, sp.lo);
            min_hi = min(min_hi, sp.hi);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int st = 0; st < 4; ++st)
#pragma unroll
                for (int p2 = 0; p2 < 2; ++p2) {
                    const float x0 = f[c][4 * st + 2 * p2] * up, x1 = f[c][4 * st + 2 * p2 + 1] * up;
                    const uint32_t hi = half2_of(x0, x1);
                    qf[n][0][c][st][p2] = hi;
                    if constexpr (F32) {
                        const float2 b = floats_of(hi);
                        qf[n][QS - 1][c][st][p2] = half2_of(x0 - b.x, x1 - b.y);
                    }
                }
    }
    // of all rows, so that the choice of the masked path is the warp's
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        max_lo = max(max_lo, __shfl_xor_sync(0xffffffffu, max_lo, o));
        min_hi = min(min_hi, __shfl_xor_sync(0xffffffffu, min_hi, o));
    }

    float m[NQ][2], mv[NQ][2], sum[NQ][2];
    float o[NQ][DP / 16][4];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) m[n][i] = -CUDART_INF_F, mv[n][i] = kLeastUnit, sum[n][i] = 0.f;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][d][i] = 0.f;
    }

    for (int i = 0; i < mine; ++i) {
        cp_wait<kStages - 2>();
        __syncwarp();
        const int slot = i % kStages;
        const bool hole = (gone >> slot) & 1;
        {
            const Where after = where(i + kStages);
            request(i + kStages - 1, next);
            next = after;
        }
        const uint8_t *kt = ring + slot * L::kStage, *vt = kt + L::kTile;
        const float2 scales = *reinterpret_cast<const float2 *>(kt + 2 * L::kTile);
        const int token0 = (tile0 + warp + i * kWarps) * kTokens;

        // scores: tokens g and g + 8 of the tile, query rows 2t and 2t + 1
        float sc[NQ][4];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const uint4 x4 = *reinterpret_cast<const uint4 *>(kt + place_k<DP>(g, 4 * c + t));
            const uint4 y4 = *reinterpret_cast<const uint4 *>(kt + place_k<DP>(g + 8, 4 * c + t));
            const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                const uint32_t u = x[st] ^ 0x80808080u, v = y[st] ^ 0x80808080u;
                const uint32_t k[4] = {unbias(__byte_perm(u, 0x64646464u, 0x4140)), unbias(__byte_perm(v, 0x64646464u, 0x4140)),
                                       unbias(__byte_perm(u, 0x64646464u, 0x4342)), unbias(__byte_perm(v, 0x64646464u, 0x4342))};
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int q = 0; q < QS; ++q) mma_f16(sc[n], k, qf[n][q][c][st][0], qf[n][q][c][st][1]);
            }
        }

        const bool masked = token0 < max_lo || token0 + kTokens > min_hi || hole;
        const float lv = scales.y > 0.f ? log2_fast(scales.y) : -CUDART_INF_F;
        uint32_t pf[NQ][QS][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            bool moved = false;
            float turn[2], p[2][2];  // [row][token g, g + 8]
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float f = score_scale[n][r] * scales.x;
                float x0 = sc[n][r] * f, x1 = sc[n][2 + r] * f;
                if (masked) {
                    const int at = token0 + g;
                    if (at < lo_row[n][r] || at >= hi_row[n][r] || hole) x0 = -CUDART_INF_F;
                    if (at + 8 < lo_row[n][r] || at + 8 >= hi_row[n][r] || hole) x1 = -CUDART_INF_F;
                }
                float top = fmaxf(x0, x1);
#pragma unroll
                for (int w = 4; w <= 16; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                const float m1 = fmaxf(m[n][r], top), ref = m1 == -CUDART_INF_F ? 0.f : m1;
                const float fall = m[n][r] - ref;
                x0 -= ref, x1 -= ref;
                sum[n][r] = sum[n][r] * exp2_fast(fall) + (exp2_fast(x0) + exp2_fast(x1));
                m[n][r] = m1;
                const float v0 = mv[n][r] + fall, v1 = fmaxf(fmaxf(v0, (top - ref) + lv), kLeastUnit);
                turn[r] = exp2_fast(v0 - v1);
                moved |= v1 != v0;
                mv[n][r] = v1;
                const float up = (lv - v1) + kWeightExponent;
                p[r][0] = exp2_fast(x0 + up);
                p[r][1] = exp2_fast(x1 + up);
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    o[n][d][0] *= turn[0];
                    o[n][d][1] *= turn[1];
                    o[n][d][2] *= turn[0];
                    o[n][d][3] *= turn[1];
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t hi = half2_of(p[0][k], p[1][k]);
                pf[n][0][k] = transpose8(hi);
                if constexpr (F32) {
                    const float2 b = floats_of(hi);
                    pf[n][QS - 1][k] = transpose8(half2_of(p[0][k] - b.x, p[1][k] - b.y));
                }
            }
        }

        // O^T += V^T . P^T: dims 64 c + 8 g + 2 j and + 1 are rows g and g + 8 of product j
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            uint2 w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = *reinterpret_cast<const uint2 *>(vt + place_v<DP>(2 * t + (r & 1) + 8 * (r >> 1), 64 * c + 8 * g));
#pragma unroll
            for (int q4 = 0; q4 < 2; ++q4) {  // four dims at a time
                uint32_t x[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = (q4 ? w[r].y : w[r].x) ^ 0x80808080u;
                const uint32_t a0 = __byte_perm(x[0], x[1], 0x5140), a1 = __byte_perm(x[0], x[1], 0x7362);  // dims 0 1, dims 2 3: tokens in pairs
                const uint32_t b0 = __byte_perm(x[2], x[3], 0x5140), b1 = __byte_perm(x[2], x[3], 0x7362);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t lo = j ? a1 : a0, hi = j ? b1 : b0;
                    const uint32_t v[4] = {unbias(__byte_perm(lo, 0x64646464u, 0x4140)), unbias(__byte_perm(lo, 0x64646464u, 0x4342)),
                                           unbias(__byte_perm(hi, 0x64646464u, 0x4140)), unbias(__byte_perm(hi, 0x64646464u, 0x4342))};
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int q = 0; q < QS; ++q) mma_f16(o[n][4 * c + 2 * q4 + j], v, pf[n][q][0], pf[n][q][1]);
                }
            }
        }
        __syncwarp();
    }
    cp_wait<0>();
    __syncthreads();

    // join the CTA's warps.  A warp's O moves from units of 2^(m + mv - 15) to units of 2^m.
    float *mine_o = reinterpret_cast<float *>(ring);
    float *mine_m = mine_o + L::kRows * DP;
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float l = sum[n][r];
#pragma unroll
            for (int w = 4; w <= 16; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
            const float unit = exp2_fast(mv[n][r]);
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) o[n][d][r] *= kWeightDown, o[n][d][2 + r] *= kWeightDown;
            const int row = 8 * n + 2 * t + r;
            if (g == 0) {
                mine_m[row] = m[n][r];
                mine_m[L::kRows + row] = l;
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float4 *dst = reinterpret_cast<float4 *>(mine_o + row * DP + 64 * c + 8 * g);
                dst[0] = make_float4(o[n][4 * c][r] * unit, o[n][4 * c][2 + r] * unit, o[n][4 * c + 1][r] * unit, o[n][4 * c + 1][2 + r] * unit);
                dst[1] = make_float4(o[n][4 * c + 2][r] * unit, o[n][4 * c + 2][2 + r] * unit, o[n][4 * c + 3][r] * unit, o[n][4 * c + 3][2 + r] * unit);
            }
        }
    __syncthreads();

    const int stored = min(L::kRows, rows - row0);  // rows of the output in this block
    const int per_row = a.dim / 4;
    const int64_t slot_row = (((int64_t)s * a.heads + h) * a.row_blocks + rb) * a.pieces + piece;
    auto emit = [&](int r, int d, const float4 &v, float top, float l) {
        const bool dead = r >= live || !(l > 0.f || l != l);
        const float inv = dead ? 0.f : 1.f / l;
        const int token = (row0 + r) / a.group, hq = h * a.group + (row0 + r) % a.group;
        const int64_t at = ((int64_t)s * a.tokens + token) * (a.heads * a.group) + hq;
        store4(static_cast<E *>(a.out) + at * a.dim + d, v, inv, dead);
        if (a.lse && d == 0) a.lse[at] = dead ? -CUDART_INF_F : (top + log2f(l)) * 0.69314718055994531f;
    };
    float *joined = reinterpret_cast<float *>(smem + kWarps * L::kPerWarp);  // of a cluster's CTA: O, maxima, sums
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
            if (r >= live) v = make_float4(0.f, 0.f, 0.f, 0.f), top = -CUDART_INF_F, l = 0.f;  // no query in this row
            *reinterpret_cast<float4 *>(dst + 4 + d) = v;
            if (d == 0) dst[0] = top, dst[1] = l, dst[2] = __int_as_float(count);
        } else if (a.pieces > 1) {
            *reinterpret_cast<float4 *>(joined + r * DP + d) = v;
            if (d == 0) joined[L::kRows * DP + r] = top, joined[L::kRows * DP + L::kRows + r] = l;
        } else {
            emit(r, d, v, top, l);
        }
    }
    if (a.part || a.pieces == 1) return;
    // join the cluster's CTAs through distributed shared memory, every CTA a share of the output
    cluster_barrier();
    const uint32_t base = smem_u32(joined);
    for (int i = piece * (kWarps * 32) + threadIdx.x; i < stored * per_row; i += a.pieces * (kWarps * 32)) {
        const int r = i / per_row, d = (i - r * per_row) * 4;
        float top = -CUDART_INF_F, l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < a.pieces; ++c) {
            const uint32_t there = in_cluster(base, c);
            const float mc = ld_cluster(there + (L::kRows * DP + r) * 4), lc = ld_cluster(there + (L::kRows * DP + L::kRows + r) * 4);
            const float4 x = ld_cluster4(there + (r * DP + d) * 4);
            const float next_top = fmaxf(top, mc), ref = next_top == -CUDART_INF_F ? 0.f : next_top;
            const float f = exp2_fast(top - ref), g2 = exp2_fast(mc - ref);
            l = l * f + lc * g2;
            v.x = v.x * f + x.x * g2, v.y = v.y * f + x.y * g2, v.z = v.z * f + x.z * g2, v.w = v.w * f + x.w * g2;
            top = next_top;
        }
        emit(r, d, v, top, l);
    }
    cluster_barrier();  // nobody leaves while its part is being read
}

// One CTA per output row joins the pieces of its sequence: the warps take pieces in turn, lanes the dims.
constexpr int kJoinWarps = 4;
template <typename E> __global__ void __launch_bounds__(kJoinWarps * 32) k_kv_join(AttnArgs a, int rows_per_block) {
    __shared__ float tops[kJoinWarps], sums[kJoinWarps];
    __shared__ float4 parts[kJoinWarps][64];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t at = blockIdx.x;  // row of the output
    const int64_t all_heads = (int64_t)a.heads * a.group;
    const int hq = (int)(at % all_heads), token = (int)(at / all_heads % a.tokens), s = (int)(at / all_heads / a.tokens);
    const int h = hq / a.group, row = token * a.group + hq % a.group, rb = row / rows_per_block;
    const float *part = a.part + (((((int64_t)s * a.heads + h) * a.row_blocks + rb) * a.pieces) * rows_per_block + (row - rb * rows_per_block)) * (int64_t)(a.dim + 4);
    const int64_t step = (int64_t)rows_per_block * (a.dim + 4);
    pdl_prologue();
    const int pieces = __float_as_int(part[2]);  // left there by the first piece
    float top = -CUDART_INF_F;
    for (int p = threadIdx.x; p < pieces; p += kJoinWarps * 32) top = fmaxf(top, part[p * step]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, tops[w]);
    const float ref = top == -CUDART_INF_F ? 0.f : top;
    float l = 0.f;
    float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll 4
    for (int p = warp; p < pieces; p += kJoinWarps) {
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
    if (lane == 0) sums[warp] = l;
    parts[warp][lane] = v[0];
    parts[warp][32 + lane] = v[1];
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) l += sums[w];
    const bool dead = !(l > 0.f || l != l);
    const float inv = dead ? 0.f : 1.f / l;
    const int d = 4 * threadIdx.x;
    if (d < a.dim) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) {
            const float4 y = parts[w][threadIdx.x];
            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
        }
        store4(static_cast<E *>(a.out) + at * a.dim + d, x, inv, dead);
    }
    if (a.lse && threadIdx.x == 0) a.lse[at] = dead ? -CUDART_INF_F : (top + log2f(l)) * 0.69314718055994531f;
}

// how a call is cut: row blocks of 8 or 16 rows, pieces along the cache
struct Cut {
    int eights, row_blocks, pieces, target;
    bool cluster;  // the pieces of a row block are a cluster of CTAs; otherwise they leave partial results in scratch
};
int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
Cut cut_of(int heads, int dim, int group, int page, int64_t seqs, int64_t tokens, int64_t table_width) {
    Cut c;
    const int64_t rows = tokens * group;
    // Sixteen rows per CTA share the converted codes.  (Thirty-two leave registers for two CTAs of four warps on an SM
    // and lost: 35 rows of dim 64 over 1500 tokens 27 us against 20, 64 rows of dim 128 over 4000 134 against 100.)
    c.eights = rows <= 8 ? 1 : 2;
    c.row_blocks = (int)std::min<int64_t>(div_up(rows, 8 * c.eights), 1 << 20);
    const int64_t length = table_width * page;
    // CTAs on an SM, by registers and shared memory
    const int wide = padded_dim(dim);
    const int resident = wide == 256 ? 1 : c.eights == 1 ? (wide == 64 ? 5 : 3) : wide == 64 ? 4 : 2;
    const int64_t slots = (int64_t)sm_count() * resident, base = std::max<int64_t>(1, seqs * heads * c.row_blocks);
    const int64_t want = slots * (base >= slots / 2 ? kWaves : 1);
    c.target = (int)std::max<int64_t>(1, want / std::max<int64_t>(1, (int64_t)heads * c.row_blocks));
    // Eight pieces or fewer, or contexts that eight CTAs are not long over, are joined through the cluster's shared
    // memory (one launch, no scratch): one of 500 tokens 5.9 us, 7.9 us as two launches.
    // (where pieces fill the machine, no more than one wave of them: 16 of 1000 tokens 12.3 us; 18.2 against 13.6 with a few more)
    const int64_t wanted = base >= slots / 2 ? div_up(want, base) : std::max<int64_t>(1, want / base), most = std::max<int64_t>(1, div_up(length, kMinPiece));
    c.cluster = std::min(wanted, most) <= kMostCluster || length <= kMostCluster * kClusterPiece;
    // otherwise a sequence may be cut four times finer than evenly long ones would be
    c.pieces = (int)(c.cluster ? std::min<int64_t>(kMostCluster, std::min(wanted, most)) : std::min(most, 4 * wanted));
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
        table_width * c->page_size > (1ll << 30))
        return fail(AB_ERR_INVALID, "seqs=%lld tokens=%lld group=%lld table_width=%lld", (long long)seqs, (long long)tokens, (long long)group,
                    (long long)table_width);
    if (c->num_heads < 1 || c->num_heads > 1024) return fail(AB_ERR_INVALID, "num_heads=%d", c->num_heads);
    if (seqs * tokens * group * c->num_heads > 0x7fffffff || (int64_t)c->num_heads * div_up(tokens * group, 16) >= (1 << 20))
        return fail(AB_ERR_UNSUPPORTED, "%lld query rows of %d heads in one call", (long long)(tokens * group), c->num_heads);
    return AB_OK;
}

template <typename E, int DP, int NQ, bool FULL> int launch_as(AttnArgs a, cudaStream_t st) {
    using L = Layout<E, DP, NQ>;
    const int rc = opt_in_smem<k_kv_attention<E, DP, NQ, FULL>>(L::kSmem);
    if (rc != AB_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = L::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.pieces;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = !a.part && a.pieces > 1 ? 2 : 1;
    // what the grid's second dim does not hold (prompts of many heads) takes further launches
    const int most = 65535 / a.heads;
    for (a.first_block = 0; a.first_block < a.row_blocks; a.first_block += most) {
        a.blocks = std::min(most, a.row_blocks - a.first_block);
        cfg.gridDim = dim3((unsigned)a.pieces, (unsigned)(a.heads * a.blocks), (unsigned)a.seqs);
        AB_CUDA_OK(cudaLaunchKernelEx(&cfg, k_kv_attention<E, DP, NQ, FULL>, a));
        AB_LAUNCH_OK();
    }
    if (a.part) {  // (check_call bounds the rows)
        const int64_t rows = (int64_t)a.seqs * a.tokens * a.heads * a.group;
        AB_CUDA_OK(launch_pdl(k_kv_join<E>, dim3((unsigned)rows), dim3(kJoinWarps * 32), 0, st, a, L::kRows));
        AB_LAUNCH_OK();
    }
    return AB_OK;
}
template <typename E, int DP, int NQ> int launch(const AttnArgs &a, cudaStream_t st) {
    return a.dim == DP ? launch_as<E, DP, NQ, true>(a, st) : launch_as<E, DP, NQ, false>(a, st);
}
template <typename E> int dispatch(const AttnArgs &a, int eights, cudaStream_t st) {
    const int dp = padded_dim(a.dim);
    if (eights == 2) return dp == 64 ? launch<E, 64, 2>(a, st) : dp == 128 ? launch<E, 128, 2>(a, st) : launch<E, 256, 2>(a, st);
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
    const Cut c = cut_of(cache->num_heads, cache->head_dim, (int)group, cache->page_size, seqs, tokens, table_width);
    if (c.cluster) return 0;
    return seqs * cache->num_heads * c.row_blocks * c.pieces * 8 * c.eights * (int64_t)(cache->head_dim + 4) * 4;
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
    if (!aligned16(out)) return fail(AB_ERR_INVALID, "out must be 16-byte aligned");
    if (need > 0 && (!scratch || scratch_bytes < need || !aligned16(scratch)))
        return fail(AB_ERR_SCRATCH, "scratch of %lld bytes, 16-byte aligned, is needed (got %lld)", (long long)need, (long long)scratch_bytes);
    const Cut cut = cut_of(cache->num_heads, cache->head_dim, (int)group, cache->page_size, seqs, tokens, table_width);
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
    const int per_page = cache->page_size / kTokens;
    a.page_magic = per_page == 1 ? 0 : (uint32_t)(((1ull << 32) + per_page - 1) / per_page);
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
        case AB_F32: return dispatch<float>(a, cut.eights, st);
        case AB_F16: return dispatch<__half>(a, cut.eights, st);
        default: return dispatch<__nv_bfloat16>(a, cut.eights, st);
    }
}
