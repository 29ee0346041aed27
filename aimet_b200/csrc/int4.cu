// y[m][n] = sum_k x[m][k] * (u[n][k] - z[n][g]) * s[n][g] + bias[n]   with 4-bit codes u
//
// n output channel, k input channel, g the block of input channels that k lies in, u = code - qmin in
// [0, 15], z = -(qmin + offset).  The weights stay in 4 bits from HBM to registers.
//
// A token or a few (k_matvec).  What bounds it is reading the codes, N * K / 2 bytes; at the measured
// copy rate an SM gets 23 bytes = 46 codes per clock, and converting and multiplying them one by one in
// float32 would take more instructions than it can issue.  So pairs of codes are turned into pairs of
// 16-bit floats (a shift and one three-input logic operation put the code into the mantissa of 128
// (bfloat16) or 1024 (float16); subtracting 128 + z or 1024 + z is exact) and multiplied 16 x 8 x 16
// at a time by mma.sync with the weights as the 16-row operand and up to eight tokens as the 8 columns.
// Products of a 16-bit activation with an integer below 2^8 are exact, sums are float32; every 64
// columns (or smaller blocks) the sums are multiplied by the block's scale and added up in float32.
// A float32 activation is cut into three bfloat16 terms that together hold all its 24 bits, each
// multiplied by the same weights into the same sums.
//
// Layout of the codes: tiles of 16 channels x 64 columns, 512 bytes, one 16-byte load per lane; the
// 32 codes of a lane are the operand fragments of four MMAs.  Columns are permuted within groups of 16
// so that the matching fragment of x is one 8-byte load: lane t of a quad holds columns 4t .. 4t+3.
#include <algorithm>

#include "common.cuh"

namespace ab {
namespace {

constexpr int kTileN = 16;   // output channels per tile
constexpr int kTileK = 64;   // input channels per tile
constexpr int kMvWarps = 8;  // warps of a matvec CTA, each with a share of the columns
constexpr int kMvDepth = 4;  // tiles requested ahead by a warp

__host__ __device__ inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// scales, multipliers and zero points: one entry per channel and block, four, two or one blocks of a
// 64-column tile side by side, [channel tile][tile of columns (or wider block)][16][sub]
struct Int4View {
    const uint4 *codes;
    const void *scales;
    const int8_t *zeros;      // NULL: `zero` for all
    const float *row_scale;   // scale kind 1
    int64_t n, k;
    int kt;                   // tiles along k
    int per;                  // tiles of columns that share a block (1 for blocks of up to 64)
    int entries;              // entries along k: div_up(kt, per)
    float zero;
};

template <typename E> struct Pair16;
template <> struct Pair16<__nv_bfloat16> {
    static constexpr uint32_t kMagic = 0x43004300u;  // 128.0, 128.0
    static constexpr float kBase = 128.f;
    // Codes are multiplied as code / 256, which the same instruction gives: a sum of code * x must not
    // leave float32's range where the sum of w * x, with its far smaller scale, does not.
    static constexpr float kUnit = 1.f / 256.f;
    static __device__ __forceinline__ uint32_t code(uint32_t v, uint32_t zero2) {  // (v - base) / 256 - z / 256
        const uint32_t unit = 0x3b803b80u;
        const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&v), *reinterpret_cast<const __nv_bfloat162 *>(&unit),
                                         *reinterpret_cast<const __nv_bfloat162 *>(&zero2));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    static __device__ __forceinline__ uint32_t both(float v) {
        const __nv_bfloat162 r = __float2bfloat162_rn(v);
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Pair16<__half> {
    static constexpr uint32_t kMagic = 0x64006400u;  // 1024.0, 1024.0
    static constexpr float kBase = 1024.f;
    static constexpr float kUnit = 1.f;
    static __device__ __forceinline__ uint32_t code(uint32_t v, uint32_t zero2) {
        const __half2 r = __hadd2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&zero2));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    static __device__ __forceinline__ uint32_t both(float v) {
        const __half2 r = __float2half2_rn(v);
        return *reinterpret_cast<const uint32_t *>(&r);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <typename E> struct MmaType { using T = E; };
template <> struct MmaType<float> { using T = __nv_bfloat16; };

// what turns a code in the mantissa of kBase into (u - z) * kUnit (all three steps exact)
template <typename H> __device__ __forceinline__ uint32_t zero_pair(float z) {
    return Pair16<H>::both(-(Pair16<H>::kBase + z) * Pair16<H>::kUnit);
}
// the codes of pair p (0..3) of a word as two 16-bit floats, (u - z) * kUnit
template <typename H> __device__ __forceinline__ uint32_t code_pair(uint32_t word, int p, uint32_t zero2) {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(v) : "r"(word >> (4 * p)), "r"(Pair16<H>::kMagic));
    return Pair16<H>::code(v, zero2);
}

// four consecutive activations of one token at column k, zeros beyond the row
template <typename E> struct Quad {
    uint32_t w[sizeof(E)];  // 4 elements: 2 or 4 words
};
template <typename E>
__device__ __forceinline__ Quad<E> load_quad(const E *row, int64_t k, int64_t k_end, bool vec) {
    Quad<E> q;
    if (vec && k + 4 <= k_end) {
        if constexpr (sizeof(E) == 2) {
            const uint2 v = *reinterpret_cast<const uint2 *>(row + k);
            q.w[0] = v.x, q.w[1] = v.y;
        } else {
            const uint4 v = *reinterpret_cast<const uint4 *>(row + k);
            q.w[0] = v.x, q.w[1] = v.y, q.w[2] = v.z, q.w[3] = v.w;
        }
        return q;
    }
    E e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = k + i < k_end ? row[k + i] : E(0.f);
    if constexpr (sizeof(E) == 2) {
        const uint16_t *b = reinterpret_cast<const uint16_t *>(e);
        q.w[0] = b[0] | (uint32_t)b[1] << 16, q.w[1] = b[2] | (uint32_t)b[3] << 16;
    } else {
        const uint32_t *b = reinterpret_cast<const uint32_t *>(e);
        q.w[0] = b[0], q.w[1] = b[1], q.w[2] = b[2], q.w[3] = b[3];
    }
    return q;
}

// x = b[0] + b[1] + b[2] exactly: each bfloat16 term takes eight of the 24 significant bits (terms
// below the smallest bfloat16 are lost, far under the product's float32 rounding).  Infinities and NaN
// stay in the first term alone.
__device__ __forceinline__ void split3(float x, __nv_bfloat16 (&b)[3]) {
    b[0] = __float2bfloat16_rn(x);
    float r = __bfloat162float(b[0]);
    r = (isinf(r) || isnan(r)) ? 0.f : x - r;
    if (isinf(__bfloat162float(b[0])) && !isinf(x)) b[0] = __float2bfloat16_rz(x), r = x - __bfloat162float(b[0]);
    b[1] = __float2bfloat16_rn(r);
    b[2] = __float2bfloat16_rn(r - __bfloat162float(b[1]));
}

template <int SUB> struct SubScales {
    float v[2][SUB];  // rows g and g + 8 of the tile
};

template <typename E, int NT, int SUB, bool ZEROS, bool MULT>
__global__ void __launch_bounds__(kMvWarps * 32) k_matvec(Int4View w, const E *__restrict__ x, int64_t ldx, const E *__restrict__ bias,
                                                          E *__restrict__ y, int64_t ldy, int tokens, int vec) {
    using H = typename MmaType<E>::T;
    constexpr bool F32 = sizeof(E) == 4;
    constexpr int XW = sizeof(E);  // 32-bit words of a Quad
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t tile = blockIdx.x;
    const int m0 = blockIdx.y * 8 * NT;
    const int kt0 = (int)((int64_t)w.kt * warp / kMvWarps), kt1 = (int)((int64_t)w.kt * (warp + 1) / kMvWarps);

    const uint4 *codes = w.codes + (tile * w.kt) * 32 + lane;
    const int64_t entry0 = tile * w.entries;

    uint4 cw[kMvDepth];
    SubScales<SUB> cs[kMvDepth];
    SubScales<SUB> cz[kMvDepth];
    Quad<E> cx[kMvDepth][NT][4];

    auto load_weights = [&](int slot, int kt) {
        cw[slot] = __ldcs(codes + (int64_t)kt * 32);
        const int64_t e = (entry0 + kt / w.per) * kTileN;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int64_t at = (e + g + 8 * r) * SUB;
#pragma unroll
            for (int i = 0; i < SUB; ++i) {
                cs[slot].v[r][i] = MULT ? (float)static_cast<const uint8_t *>(w.scales)[at + i] : static_cast<const float *>(w.scales)[at + i];
                if (ZEROS) cz[slot].v[r][i] = (float)w.zeros[at + i];
            }
        }
    };
    auto load_x = [&](int slot, int kt) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int m = m0 + 8 * j + g;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (m < tokens)
                    cx[slot][j][s] = load_quad(x + (int64_t)m * ldx, (int64_t)kt * kTileK + 16 * s + 4 * t, w.k, vec);
                else
#pragma unroll
                    for (int i = 0; i < XW; ++i) cx[slot][j][s].w[i] = 0;
            }
        }
    };

    float total[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) total[j][i] = 0.f;

    // the weights are written by no kernel that lets its successor start early (aimet_b200_int4_pack
    // does not), so they may be requested before the wait for the predecessor; x may not
    pdl_launch_dependents();
#pragma unroll
    for (int d = 0; d < kMvDepth; ++d)
        if (kt0 + d < kt1) load_weights(d, kt0 + d);
    pdl_wait();
#pragma unroll
    for (int d = 0; d < kMvDepth; ++d)
        if (kt0 + d < kt1) load_x(d, kt0 + d);

    for (int base = kt0; base < kt1; base += kMvDepth) {
#pragma unroll
        for (int d = 0; d < kMvDepth; ++d) {
            const int kt = base + d;
            if (kt >= kt1) break;
            const uint32_t word[4] = {cw[d].x, cw[d].y, cw[d].z, cw[d].w};
            float acc[NT][4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int sub = s * SUB / 4;
                uint32_t z0, z1;
                if (ZEROS) {
                    z0 = zero_pair<H>(cz[d].v[0][sub]);
                    z1 = zero_pair<H>(cz[d].v[1][sub]);
                } else {
                    z0 = z1 = zero_pair<H>(w.zero);
                }
                const int p = 2 * (s & 1), q = 2 * (s >> 1);
                const uint32_t a[4] = {code_pair<H>(word[q], p, z0), code_pair<H>(word[q + 1], p, z1),
                                       code_pair<H>(word[q], p + 1, z0), code_pair<H>(word[q + 1], p + 1, z1)};
                if (s % (4 / SUB) == 0) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const Quad<E> &q4 = cx[d][j][s];
                    if constexpr (F32) {
                        __nv_bfloat16 b[4][3];
#pragma unroll
                        for (int i = 0; i < 4; ++i) split3(__uint_as_float(q4.w[i]), b[i]);
#pragma unroll
                        for (int e = 0; e < 3; ++e) {
                            const __nv_bfloat162 lo = __halves2bfloat162(b[0][e], b[1][e]), hi = __halves2bfloat162(b[2][e], b[3][e]);
                            Pair16<H>::mma(acc[j], a, *reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
                        }
                    } else {
                        Pair16<H>::mma(acc[j], a, q4.w[0], q4.w[1]);
                    }
                }
                if (s % (4 / SUB) == 4 / SUB - 1) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) total[j][i] = fmaf(acc[j][i], cs[d].v[i >> 1][sub] * (1.f / Pair16<H>::kUnit), total[j][i]);
                }
            }
            if (kt + kMvDepth < kt1) {
                load_weights(d, kt + kMvDepth);
                load_x(d, kt + kMvDepth);
            }
        }
    }

    // the warps' sums, added in a fixed order
    __shared__ float part[kMvWarps][NT * 128];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int m = 8 * j + 2 * t + (i & 1), row = g + 8 * (i >> 1);
            part[warp][m * 16 + row] = total[j][i];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 128; i += kMvWarps * 32) {
        const int m = m0 + (i >> 4);
        const int64_t n = tile * kTileN + (i & 15);
        if (m >= tokens || n >= w.n) continue;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < kMvWarps; ++q) v += part[q][i];
        if (MULT) v *= w.row_scale[n];
        if (bias) v += to_f32(bias[n]);
        y[(int64_t)m * ldy + n] = Cvt<float, E>::store(v);
    }
}

// codes [n][k] (one signed byte each, qmin .. qmin + 15) -> the tiled 4-bit layout; what lies outside
// the matrix gets code 0, which meets zeros of x.
__global__ void k_int4_pack(const int8_t *__restrict__ codes, int64_t n, int64_t k, int kt, int qmin, uint4 *__restrict__ out, int64_t total) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= total) return;
    const int lane = (int)(i & 31), g = lane >> 2, t = lane & 3;
    const int64_t tile = (i >> 5) / kt, col = (i >> 5) % kt;
    uint32_t word[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int64_t row = tile * kTileN + g + 8 * (q & 1);
        uint32_t v = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t c = col * kTileK + 16 * (2 * (q >> 1) + (p >> 1)) + 4 * t + 2 * (p & 1) + h;
                const int u = row < n && c < k ? (int)codes[row * k + c] - qmin : 0;
                v |= (uint32_t)(u & 15) << (4 * p + 16 * h);
            }
        }
        word[q] = v;
    }
    out[i] = make_uint4(word[0], word[1], word[2], word[3]);
}

int check_weight(const ab_int4_weight *w, Int4View *v) {
    if (!w) return fail(AB_ERR_INVALID, "weight is NULL");
    if (w->n < 1 || w->k < 1 || w->n > (1ll << 30) || w->k > (1ll << 30))
        return fail(AB_ERR_INVALID, "weight of %lld x %lld", (long long)w->n, (long long)w->k);
    if (w->block != 16 && w->block != 32 && (w->block < 64 || w->block % 64))
        return fail(AB_ERR_UNSUPPORTED, "storage block %d: 16, 32 or a multiple of 64", w->block);
    if (!w->codes || !w->scales) return fail(AB_ERR_INVALID, "codes or scales is NULL");
    if (!aligned16(w->codes)) return fail(AB_ERR_INVALID, "codes must be 16-byte aligned");
    if (w->scale_kind != 0 && w->scale_kind != 1) return fail(AB_ERR_INVALID, "scale_kind %d", w->scale_kind);
    if (w->scale_kind == 1 && !w->row_scale) return fail(AB_ERR_INVALID, "scale_kind 1 needs row_scale");
    if (!w->zeros && (w->zero < -112 || w->zero > 112)) return fail(AB_ERR_INVALID, "zero point %d outside [-112, 112]", w->zero);
    v->codes = static_cast<const uint4 *>(w->codes);
    v->scales = w->scales;
    v->zeros = static_cast<const int8_t *>(w->zeros);
    v->row_scale = static_cast<const float *>(w->row_scale);
    v->n = w->n;
    v->k = w->k;
    v->kt = (int)div_up(w->k, kTileK);
    v->per = w->block <= kTileK ? 1 : w->block / kTileK;
    v->entries = (int)div_up(v->kt, v->per);
    v->zero = (float)w->zero;
    return AB_OK;
}

struct MatvecCall {
    Int4View w;
    const void *x, *bias;
    void *y;
    int64_t ldx, ldy;
    int tokens, vec;
    cudaStream_t stream;
};

template <typename E, int NT, int SUB, bool ZEROS, bool MULT> int launch_matvec(const MatvecCall &c) {
    constexpr int kMost = 65535 * 8 * NT;  // tokens of one launch: the grid's second dim
    for (int64_t m = 0; m < c.tokens; m += kMost) {
        const int tokens = (int)std::min<int64_t>(kMost, c.tokens - m);
        const dim3 grid((unsigned)div_up(c.w.n, kTileN), (unsigned)div_up(tokens, 8 * NT));
        AB_CUDA_OK(launch_pdl(k_matvec<E, NT, SUB, ZEROS, MULT>, grid, dim3(kMvWarps * 32), 0, c.stream, c.w,
                              static_cast<const E *>(c.x) + m * c.ldx, c.ldx, static_cast<const E *>(c.bias),
                              static_cast<E *>(c.y) + m * c.ldy, c.ldy, tokens, c.vec));
        AB_LAUNCH_OK();
    }
    return AB_OK;
}
template <typename E, int NT, int SUB> int dispatch_scales(const MatvecCall &c, bool mult) {
    if (mult) return c.w.zeros ? launch_matvec<E, NT, SUB, true, true>(c) : launch_matvec<E, NT, SUB, false, true>(c);
    return c.w.zeros ? launch_matvec<E, NT, SUB, true, false>(c) : launch_matvec<E, NT, SUB, false, false>(c);
}
template <typename E, int NT> int dispatch_block(const MatvecCall &c, int block, bool mult) {
    if (block == 16) return dispatch_scales<E, NT, 4>(c, mult);
    if (block == 32) return dispatch_scales<E, NT, 2>(c, mult);
    return dispatch_scales<E, NT, 1>(c, mult);
}
template <typename E> int dispatch_tokens(const MatvecCall &c, int block, bool mult) { return dispatch_block<E, 1>(c, block, mult); }

}  // namespace
}  // namespace ab

using namespace ab;

extern "C" int64_t aimet_b200_int4_codes_bytes(int64_t n, int64_t k) {
    if (n < 1 || k < 1 || n > (1ll << 30) || k > (1ll << 30)) return fail(AB_ERR_INVALID, "weight of %lld x %lld", (long long)n, (long long)k);
    return div_up(n, kTileN) * div_up(k, kTileK) * 512;
}

extern "C" int aimet_b200_int4_pack(const void *codes, int64_t n, int64_t k, int qmin, void *out, void *stream) {
    const int64_t bytes = aimet_b200_int4_codes_bytes(n, k);
    if (bytes < 0) return (int)bytes;
    if (!codes || !out) return fail(AB_ERR_INVALID, "codes or out is NULL");
    if (qmin < -128 || qmin > 112) return fail(AB_ERR_INVALID, "qmin=%d: the codes are signed bytes", qmin);
    if (!aligned16(out)) return fail(AB_ERR_INVALID, "out must be 16-byte aligned");
    const int64_t total = bytes / 16;
    const int64_t blocks = div_up(total, 256);
    if (blocks > 0x7fffffff) return fail(AB_ERR_UNSUPPORTED, "weight of %lld x %lld is too large", (long long)n, (long long)k);
    k_int4_pack<<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const int8_t *>(codes), n, k, (int)div_up(k, kTileK), qmin, static_cast<uint4 *>(out), total);
    AB_LAUNCH_OK();
    return AB_OK;
}

extern "C" int aimet_b200_int4_linear(const ab_int4_weight *weight, const void *x, int64_t ldx, const void *bias, void *y, int64_t ldy,
                                      int64_t tokens, int io_dtype, void *stream) {
    MatvecCall c;
    const int rc = check_weight(weight, &c.w);
    if (rc != AB_OK) return rc;
    if (tokens < 0 || tokens > (1 << 24)) return fail(AB_ERR_INVALID, "tokens=%lld out of range [0, 2^24]", (long long)tokens);
    if (tokens == 0) return AB_OK;
    if (!x || !y) return fail(AB_ERR_INVALID, "x or y is NULL");
    if (ldx < weight->k && tokens > 1) return fail(AB_ERR_INVALID, "ldx=%lld is below k=%lld", (long long)ldx, (long long)weight->k);
    if (ldy < weight->n && tokens > 1) return fail(AB_ERR_INVALID, "ldy=%lld is below n=%lld", (long long)ldy, (long long)weight->n);
    if (io_dtype != AB_F32 && io_dtype != AB_F16 && io_dtype != AB_BF16) return fail(AB_ERR_UNSUPPORTED, "io_dtype %d", io_dtype);
    const int size = dtype_size(io_dtype);
    c.x = x;
    c.bias = bias;
    c.y = y;
    c.ldx = ldx;
    c.ldy = ldy;
    c.tokens = (int)tokens;
    c.vec = reinterpret_cast<uintptr_t>(x) % (4 * size) == 0 && (ldx % 4 == 0 || tokens == 1);
    c.stream = static_cast<cudaStream_t>(stream);
    const bool mult = weight->scale_kind == 1;
    switch (io_dtype) {
        case AB_F32: return dispatch_tokens<float>(c, weight->block, mult);
        case AB_F16: return dispatch_tokens<__half>(c, weight->block, mult);
        default: return dispatch_tokens<__nv_bfloat16>(c, weight->block, mult);
    }
}
