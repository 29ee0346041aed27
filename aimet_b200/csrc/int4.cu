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
// at a time by mma.sync with the weights as the 16-row operand and up to eight tokens as the 8 columns
// (tcgen05 has 64 rows at least, and the tensor cores are 16 % busy as it is).  Measured, 1 x 14336 x 4096 with
// blocks of 64: 10.1 us of 4.7 (3.0 TB/s); issue slots 52 % taken while an SM is active, a third of a launch
// by itself is ramp-up and tail, which a neighbouring launch overlaps.
// Products of a 16-bit activation with an integer below 2^8 are exact, sums are float32; every 64
// columns (or smaller blocks) the sums are multiplied by the block's scale and added up in float32.
// A float32 activation is cut into three bfloat16 terms that together hold all its 24 bits, each
// multiplied by the same weights into the same sums.
//
// Layout of the codes: tiles of 16 channels x 64 columns, 512 bytes, one 16-byte load per lane; the
// 32 codes of a lane are the operand fragments of four MMAs.  Columns are permuted within groups of 32
// so that the matching fragment of x is one 16-byte read: lane t of a quad holds eight neighbouring
// columns of every 32 (with blocks of 16 columns, four of every 16).
#include <algorithm>

#include "int4.cuh"

namespace ab {
namespace {

constexpr int kMvWarps = 8;         // warps of a matvec CTA
constexpr int kMvTiles = kMvWarps;  // channel tiles of a CTA: at most as many as warps, so that a warp meets two at most

template <typename E> struct MmaType { using T = E; };
template <> struct MmaType<float> { using T = __nv_bfloat16; };

// x = b0 + b1 + b2 exactly: three bfloat16 terms, cut off rather than rounded, of eight significant bits
// each (terms below the smallest bfloat16 are lost, far under the product's float32 rounding).
// Infinities and NaN stay in the first term alone.  Two values at a time, packed.
__device__ __forceinline__ void split3(uint32_t w0, uint32_t w1, uint32_t (&b)[3]) {
    float x0 = __uint_as_float(w0) + 0.f, x1 = __uint_as_float(w1) + 0.f;  // makes a NaN quiet: its upper half is a NaN too
    b[0] = __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
    x0 -= __uint_as_float(b[0] << 16);
    x1 -= __uint_as_float(b[0] & 0xffff0000u);
    x0 = x0 == x0 ? x0 : 0.f;
    x1 = x1 == x1 ? x1 : 0.f;
    b[1] = __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
    x0 -= __uint_as_float(b[1] << 16);
    x1 -= __uint_as_float(b[1] & 0xffff0000u);
    b[2] = __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
}

// A CTA takes up to kMvTiles tiles of 16 channels (all of their columns), or a cluster of `split` CTAs takes
// one; `pass` tokens, at most eight, whose x lies in shared memory (float32: three bfloat16 planes) before
// the first product.  The warps share the CTA's chunks evenly: a warp streams one contiguous run of codes, two
// chunks requested ahead into registers, and leaves a partial sum for each of the at most two channel tiles
// that it meets.
template <typename E, int SUB, bool ZEROS, bool MULT>
__global__ void __launch_bounds__(kMvWarps * 32, 2) k_matvec(Int4View w, const E *__restrict__ x, int64_t ldx, const E *__restrict__ bias,
                                                             E *__restrict__ y, int64_t ldy, int tokens, int pass, int vec, int split) {
    using H = typename MmaType<E>::T;
    using S = std::conditional_t<MULT, uint8_t, float>;
    using SP = Packed<S, SUB>;
    using ZP = Packed<int8_t, SUB>;
    constexpr bool F32 = sizeof(E) == 4, FINE = SUB == 4;
    constexpr int P = F32 ? 3 : 1;
    constexpr int NB = SUB == 4 && !MULT ? 1 : 2;  // chunks in registers
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float part[kMvWarps][2][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t tiles = (uint32_t)div_up(w.n, kTileN);
    const uint32_t cta = blockIdx.x, ctas = gridDim.x;
    const uint32_t rank = split > 1 ? cta % split : 0;
    // tiles [tile0, tile0 + n_tiles): the first `tiles % ctas` CTAs have one more
    const uint32_t each = tiles / ctas, more = tiles % ctas;
    const uint32_t tile0 = split > 1 ? cta / split : cta * each + min(cta, more), n_tiles = split > 1 ? 1 : each + (cta < more);
    const uint32_t units = n_tiles * w.chunks, parts = kMvWarps * split;
    auto unit_of = [&](uint32_t part) { return units * part / parts; };  // units <= 8 * 2^12, parts <= 64
    const uint32_t u0 = unit_of(rank * kMvWarps + warp), u1 = unit_of(rank * kMvWarps + warp + 1);
    const uint32_t row0 = u0 / w.chunks, turn = (row0 + 1) * w.chunks;  // first unit of the warp's second channel tile
    const int m0 = blockIdx.y * pass;
    tokens = min(tokens - m0, pass);

    struct {
        uint4 code[4];
        typename SP::V scale[4][2];
        typename ZP::V zero[4][2];
    } buf[NB];
    const uint4 *code_at = w.codes + ((uint64_t)tile0 * w.chunks + u0) * 128 + lane;
    const int64_t entry0 = ((int64_t)tile0 * w.chunks + u0) * w.entries * kTileN + g;
    const typename SP::V *scale_at = static_cast<const typename SP::V *>(w.scales) + entry0;
    const typename ZP::V *zero_at = reinterpret_cast<const typename ZP::V *>(w.zeros) + (ZEROS ? entry0 : 0);
    const int step = w.entries * kTileN;
    const int off[4] = {0, w.entries / 4 * kTileN, w.entries / 2 * kTileN, w.entries * 3 / 4 * kTileN};  // of a tile's entry in a chunk
    auto load = [&](int b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) buf[b].code[i] = __ldcs(code_at + 32 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int at = (SUB == 1 ? off[i] : kTileN * i) + 8 * r;
                buf[b].scale[i][r] = scale_at[at];
                if constexpr (ZEROS) buf[b].zero[i][r] = zero_at[at];
            }
        code_at += 128;
        scale_at += step;
        if (ZEROS) zero_at += step;
    };

    // the weights are written by no kernel that lets its successor start early (aimet_b200_int4_pack
    // does not), so they may be requested before the wait for the predecessor; x may not
    pdl_launch_dependents();
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (u0 + b < u1) load(b);
    pdl_wait();

    const uint32_t pitch = w.chunks * (kChunkK * 2) + 64;  // 64 modulo 128: the reads of eight lanes meet no bank twice
    // 16-byte pieces of x: a thread takes two columns of four tokens at once
    constexpr int V = 16 / sizeof(E), MA = 4, CA = 2;
    const int per_row = w.chunks * (kChunkK / V);
    const uint32_t plane = pass * pitch;
    auto put = [&](const Vec16<E> &v, int m, int c) {
        uint8_t *dst = smem + m * pitch + 2 * V * c;
        if constexpr (F32) {
            uint32_t lo[3], hi[3];
            split3(__float_as_uint(v.v[0]), __float_as_uint(v.v[1]), lo);
            split3(__float_as_uint(v.v[2]), __float_as_uint(v.v[3]), hi);
#pragma unroll
            for (int e = 0; e < 3; ++e) *reinterpret_cast<uint2 *>(dst + e * plane) = make_uint2(lo[e], hi[e]);
        } else {
            *reinterpret_cast<Vec16<E> *>(dst) = v;
        }
    };
    if (vec) {  // whole pieces, 16-byte aligned
        const int have = (int)(w.k / V);
        for (int m = 0; m < tokens; m += MA)
            for (int c = threadIdx.x; c < per_row; c += CA * kMvWarps * 32) {
                uint4 v[MA][CA];
#pragma unroll
                for (int i = 0; i < MA; ++i)
#pragma unroll
                    for (int j = 0; j < CA; ++j) {
                        const int cc = c + j * kMvWarps * 32;
                        v[i][j] = make_uint4(0, 0, 0, 0);
                        if (m + i < tokens && cc < have) v[i][j] = *reinterpret_cast<const uint4 *>(x + (int64_t)(m0 + m + i) * ldx + cc * V);
                    }
#pragma unroll
                for (int i = 0; i < MA; ++i)
#pragma unroll
                    for (int j = 0; j < CA; ++j) {
                        const int cc = c + j * kMvWarps * 32;
                        if (m + i < tokens && cc < per_row) put(*reinterpret_cast<const Vec16<E> *>(&v[i][j]), m + i, cc);
                    }
            }
    } else {
        for (int m = 0; m < tokens; ++m)
            for (int c = threadIdx.x; c < per_row; c += kMvWarps * 32) {
                Vec16<E> v;
#pragma unroll
                for (int j = 0; j < V; ++j) v.v[j] = c * V + j < w.k ? x[(int64_t)(m0 + m) * ldx + c * V + j] : E(0.f);
                put(v, m, c);
            }
    }
    __syncthreads();

    // Columns of the product are tokens: a lane whose token does not exist multiplies some other token's x
    // into a column that nobody stores.
    const uint8_t *xs = smem + (size_t)min(g, tokens - 1) * pitch + (FINE ? 8 : 16) * t;
    const uint32_t one_zero = zero_pair<H>(w.zero);
    float total[4] = {0.f, 0.f, 0.f, 0.f};
    auto leave = [&](int segment) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            part[warp][segment][(2 * t + (i & 1)) * 16 + g + 8 * (i >> 1)] = total[i];
            total[i] = 0.f;
        }
    };
    for (uint32_t base = u0; base < u1; base += NB) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint32_t u = base + b;
            if (u >= u1) break;
            if (u == turn) leave(0);
            const uint8_t *xc = xs + (u - (u >= turn ? turn : turn - w.chunks)) * (kChunkK * 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint4 v[2][P];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        const uint8_t *p = xc + e * plane + i * 128 + 64 * h;
                        if constexpr (FINE) {
                            const uint2 lo = *reinterpret_cast<const uint2 *>(p), hi = *reinterpret_cast<const uint2 *>(p + 32);
                            v[h][e] = make_uint4(lo.x, lo.y, hi.x, hi.y);
                        } else {
                            v[h][e] = *reinterpret_cast<const uint4 *>(p);
                        }
                    }
                const uint4 w4 = buf[b].code[i];
                const uint32_t word[4] = {w4.x, w4.y, w4.z, w4.w};
                float acc[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int sub = s * SUB / 4, p = 2 * (s & 1), q = 2 * (s >> 1);
                    const uint32_t z0 = ZEROS ? zero_pair<H>(ZP::get(buf[b].zero[i][0], sub)) : one_zero;
                    const uint32_t z1 = ZEROS ? zero_pair<H>(ZP::get(buf[b].zero[i][1], sub)) : one_zero;
                    const uint32_t a[4] = {code_pair<H>(word[q], p, z0), code_pair<H>(word[q + 1], p, z1),
                                           code_pair<H>(word[q], p + 1, z0), code_pair<H>(word[q + 1], p + 1, z1)};
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        const uint32_t b0 = (s & 1) ? v[s >> 1][e].z : v[s >> 1][e].x, b1 = (s & 1) ? v[s >> 1][e].w : v[s >> 1][e].y;
                        if (s % (4 / SUB) == 0 && e == 0)
                            Pair16<H>::mma_first(acc, a, b0, b1);
                        else
                            Pair16<H>::mma(acc, a, b0, b1);
                    }
                    if (s % (4 / SUB) == 4 / SUB - 1) {
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float f = SP::get(buf[b].scale[i][r], sub);
                            total[2 * r] = fmaf(acc[2 * r], f, total[2 * r]);
                            total[2 * r + 1] = fmaf(acc[2 * r + 1], f, total[2 * r + 1]);
                        }
                    }
                }
            }
            if (u + NB < u1) load(b);
        }
    }
    leave(u1 > turn ? 1 : 0);

    // the warps' sums of every channel tile, added in a fixed order
    if (split > 1)
        cluster_barrier();
    else
        __syncthreads();
    if (rank == 0) {
        for (uint32_t i = threadIdx.x; i < n_tiles * 128; i += kMvWarps * 32) {
            const uint32_t row = i / 128, at = i % 128;
            const int m = (int)(at >> 4);
            const int64_t n = (int64_t)(tile0 + row) * kTileN + (at & 15);
            if (m >= tokens || n >= w.n) continue;
            float v = 0.f;
            if (split > 1) {
                const uint32_t here = (uint32_t)__cvta_generic_to_shared(&part[0][0][at]);
                for (int c = 0; c < split; ++c) {
                    uint32_t there;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(c));
#pragma unroll
                    for (int q = 0; q < kMvWarps; ++q) {
                        float f;
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(there + q * (2 * 128 * 4)) : "memory");
                        v += f;
                    }
                }
            } else {
                const uint32_t lo = row * w.chunks, hi = lo + w.chunks;
#pragma unroll
                for (int q = 0; q < kMvWarps; ++q) {
                    const uint32_t a = unit_of(q), b = unit_of(q + 1);
                    if (a < hi && b > lo && a < b) v += part[q][a < lo ? 1 : 0][at];
                }
            }
            const RowFactor f = row_factor<H>(w.row_scale[n]);
            v = v * f.unit * f.scale;
            if (bias) v += to_f32(bias[n]);
            y[(int64_t)(m0 + m) * ldy + n] = Cvt<float, E>::store(v);
        }
    }
    if (split > 1) cluster_barrier();  // nobody of the cluster leaves while its sums are being read
}

// codes [n][k] (one signed byte each, qmin .. qmin + 15) -> the tiled 4-bit layout; what lies outside
// the matrix gets code 0, which meets zeros of x.
__global__ void k_int4_pack(const int8_t *__restrict__ codes, int64_t n, int64_t k, int kt, int qmin, int fine, uint4 *__restrict__ out, int64_t total) {
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
                const int64_t c = col * kTileK + 32 * (q >> 1) + (fine ? 16 * (p >> 1) + 4 * t : 4 * (p >> 1) + 8 * t) + 2 * (p & 1) + h;
                const int u = row < n && c < k ? (int)codes[row * k + c] - qmin : 0;
                v |= (uint32_t)(u & 15) << (4 * p + 16 * h);
            }
        }
        word[q] = v;
    }
    out[i] = make_uint4(word[0], word[1], word[2], word[3]);
}

bool storable(int block) { return block == 16 || block == 32 || block == 64 || block == 128 || block == 256; }

int check_weight(const ab_int4_weight *w, Int4View *v) {
    if (!w) return fail(AB_ERR_INVALID, "weight is NULL");
    if (w->n < 1 || w->k < 1 || w->n > (1ll << 30) || w->k > kMaxK)
        return fail(AB_ERR_INVALID, "weight of %lld x %lld", (long long)w->n, (long long)w->k);
    if (!storable(w->block)) return fail(AB_ERR_UNSUPPORTED, "storage block %d: 16, 32, 64, 128 or 256", w->block);
    if (!w->codes || !w->scales) return fail(AB_ERR_INVALID, "codes or scales is NULL");
    if (!aligned16(w->codes) || !aligned16(w->scales) || !aligned16(w->zeros))
        return fail(AB_ERR_INVALID, "codes, scales and zeros must be 16-byte aligned");
    if (w->scale_kind != 0 && w->scale_kind != 1) return fail(AB_ERR_INVALID, "scale_kind %d", w->scale_kind);
    if (!w->row_scale) return fail(AB_ERR_INVALID, "row_scale is NULL");
    if (!w->zeros && (w->zero < -112 || w->zero > 112)) return fail(AB_ERR_INVALID, "zero point %d outside [-112, 112]", w->zero);
    v->codes = static_cast<const uint4 *>(w->codes);
    v->scales = w->scales;
    v->zeros = static_cast<const int8_t *>(w->zeros);
    v->row_scale = static_cast<const float *>(w->row_scale);
    v->n = w->n;
    v->k = w->k;
    v->chunks = (int)div_up(w->k, kChunkK);
    v->entries = w->block <= kTileK ? 4 : kChunkK / w->block;
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

constexpr size_t kMvSmem = 218 * 1024, kMvSmemHalf = 104 * 1024;  // one CTA on an SM, two (beside 8 KB of sums each)

// bytes of x of one token in shared memory, and tokens that are multiplied in one pass over the weights (a
// second pass finds them in L2): eight, or what leaves room for a second CTA on the SM
size_t row_bytes(const Int4View &w, int io_dtype) { return (size_t)(io_dtype == AB_F32 ? 3 : 1) * (w.chunks * (kChunkK * 2) + 64); }
int pass_tokens(size_t row) { return (int)std::min<size_t>(8, std::max<size_t>(1, kMvSmemHalf / row)); }

template <typename E, int SUB, bool ZEROS, bool MULT> int launch_matvec(const MatvecCall &c) {
    const auto kernel = k_matvec<E, SUB, ZEROS, MULT>;
    const size_t row = row_bytes(c.w, sizeof(E) == 4 ? AB_F32 : AB_F16);
    if (row > kMvSmem)
        return fail(AB_ERR_UNSUPPORTED, "%lld input channels: x of one token does not fit shared memory", (long long)c.w.k);
    const int rc = opt_in_smem<k_matvec<E, SUB, ZEROS, MULT>>(kMvSmem);
    if (rc != AB_OK) return rc;
    const int64_t tiles = div_up(c.w.n, kTileN);
    const int sms = sm_count();
    int pass = pass_tokens(row);
    pass = (int)div_up(c.tokens, div_up(c.tokens, pass));

    constexpr int kMost = 65535;  // passes of one launch: the grid's second dim
    for (int64_t m = 0; m < c.tokens; m += (int64_t)kMost * pass) {
        const int tokens = (int)std::min<int64_t>((int64_t)kMost * pass, c.tokens - m);
        const int64_t passes = div_up(tokens, pass);
        // Two CTAs per SM and no more than kMvTiles channel tiles for one.  Few channel tiles: a cluster of
        // CTAs per tile, while that leaves a chunk for every warp.
        const int64_t slots = div_up(sms * 2, passes);
        int split = 1;
        while (split < 8 && tiles * split * 2 <= slots && c.w.chunks >= split * 2 * kMvWarps) split *= 2;
        const int64_t ctas = split > 1 ? tiles * split : std::min(tiles, std::max(slots, div_up(tiles, kMvTiles)));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)ctas, (unsigned)passes);
        cfg.blockDim = dim3(kMvWarps * 32);
        cfg.dynamicSmemBytes = row * pass;
        cfg.stream = c.stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = split;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = split > 1 ? 2 : 1;
        AB_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, c.w, static_cast<const E *>(c.x) + m * c.ldx, c.ldx, static_cast<const E *>(c.bias),
                                      static_cast<E *>(c.y) + m * c.ldy, c.ldy, tokens, pass, c.vec, split));
        AB_LAUNCH_OK();
    }
    return AB_OK;
}
template <typename E, int SUB> int dispatch_scales(const MatvecCall &c, bool mult) {
    if (mult) return c.w.zeros ? launch_matvec<E, SUB, true, true>(c) : launch_matvec<E, SUB, false, true>(c);
    return c.w.zeros ? launch_matvec<E, SUB, true, false>(c) : launch_matvec<E, SUB, false, false>(c);
}
template <typename E> int dispatch_matvec(const MatvecCall &c, int block, bool mult) {
    if (block == 16) return dispatch_scales<E, 4>(c, mult);
    if (block == 32) return dispatch_scales<E, 2>(c, mult);
    return dispatch_scales<E, 1>(c, mult);
}

}  // namespace
}  // namespace ab

using namespace ab;

extern "C" int64_t aimet_b200_int4_codes_bytes(int64_t n, int64_t k) {
    if (n < 1 || k < 1 || n > (1ll << 30) || k > kMaxK) return fail(AB_ERR_INVALID, "weight of %lld x %lld", (long long)n, (long long)k);
    return div_up(n, kTileN) * div_up(k, kChunkK) * 2048;
}

extern "C" int aimet_b200_int4_pack(const void *codes, int64_t n, int64_t k, int qmin, int block, void *out, void *stream) {
    if (!storable(block)) return fail(AB_ERR_UNSUPPORTED, "storage block %d: 16, 32, 64, 128 or 256", block);
    const int64_t bytes = aimet_b200_int4_codes_bytes(n, k);
    if (bytes < 0) return (int)bytes;
    if (!codes || !out) return fail(AB_ERR_INVALID, "codes or out is NULL");
    if (qmin < -128 || qmin > 112) return fail(AB_ERR_INVALID, "qmin=%d: the codes are signed bytes", qmin);
    if (!aligned16(out)) return fail(AB_ERR_INVALID, "out must be 16-byte aligned");
    const int64_t total = bytes / 16;
    const int64_t blocks = div_up(total, 256);
    if (blocks > 0x7fffffff) return fail(AB_ERR_UNSUPPORTED, "weight of %lld x %lld is too large", (long long)n, (long long)k);
    k_int4_pack<<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const int8_t *>(codes), n, k, (int)div_up(k, kChunkK) * (kChunkK / kTileK), qmin, block == 16, static_cast<uint4 *>(out), total);
    AB_LAUNCH_OK();
    return AB_OK;
}

extern "C" int aimet_b200_int4_linear(const ab_int4_weight *weight, const void *x, int64_t ldx, const void *bias, void *y, int64_t ldy,
                                      int64_t tokens, int io_dtype, int32_t *status, void *stream) {
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
    c.vec = aligned16(x) && weight->k * size % 16 == 0 && (ldx * size % 16 == 0 || tokens == 1);
    c.stream = static_cast<cudaStream_t>(stream);
    const bool mult = weight->scale_kind == 1;
    // More tokens than two passes over the weights take: the tensor-core kernel, where rows of x start on 16
    // bytes (TMA).  Measured, 14336 x 4096: 16 tokens in two passes 19 us, on the tensor cores 29 us; 24 tokens 36
    // and 29 us; 4096 x 14336, where x of three tokens fits: 16 tokens 67 and 31 us.  float32 stays here:
    // a weight's integer code times three bfloat16 terms is exact, a weight rounded to 16 bits would not be.
    if (tokens > 2 * pass_tokens(row_bytes(c.w, io_dtype)) && io_dtype != AB_F32 && aligned16(x) && ldx * size % 16 == 0) {
        if (!status) return fail(AB_ERR_INVALID, "status is NULL");
        Int4Gemm q;
        q.w = c.w;
        q.x = x;
        q.bias = bias;
        q.y = y;
        q.ldx = ldx;
        q.ldy = ldy;
        q.tokens = (int)tokens;
        q.block = weight->block;
        q.io_dtype = io_dtype;
        q.mult = mult;
        q.status = status;
        q.stream = c.stream;
        return launch_int4_gemm(q);
    }
    switch (io_dtype) {
        case AB_F32: return dispatch_matvec<float>(c, weight->block, mult);
        case AB_F16: return dispatch_matvec<__half>(c, weight->block, mult);
        default: return dispatch_matvec<__nv_bfloat16>(c, weight->block, mult);
    }
}
