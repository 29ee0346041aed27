// Products with 4-bit weights for many tokens, on the 5th-generation tensor cores.
//
//   y[m][n] = row_scale[n] * sum_k x[m][k] * w'[n][k] + bias[n],   w'[n][k] = (u - z) * s'   rounded to x's type
//
// s' = scale / row_scale is at most 1 (or a whole number up to 255), so w' lies well inside the 16-bit types; the one
// rounding of a weight, at most half a step (2^-8 of it in bfloat16, 2^-11 in float16), is the one that the
// simulated weight of a 16-bit model has too, and with whole-number factors up to 16 there is none.  (float16
// weights below 2^-14 of their channel's largest scale keep an absolute error of 2^-25 of it.)  The
// float32 factor s' multiplies in two 16-bit parts, hi + lo, by a product and a fused multiply-add: one
// rounding at the end and no conversions to float32 and back.
//
// Orientation: weights are the M operand (128 output channels = 128 lanes of tensor memory), tokens the N
// operand (`bn` = 32 .. 256 columns).  A stage holds 64 input channels: x comes by TMA, the weights are
// converted, a warp for each 16-channel tile of the packed layout, and stored in
// the 128-byte-swizzled order that tcgen05.mma reads: a lane's eight neighbouring columns are one 16-byte
// store.  What bounds it: a stage of 256 tokens is 524 clocks of MMAs, and about 640 of conversion (1500 x 14336 x
// 4096: 160 us, 1.10 PFLOP/s; 134 us with the conversion's loads taken out).  Tried and not kept: a pair of CTAs that
// each convert half of the channels and store them into both shared memories (304 us: four stages do not cover
// the way of a store, a fence and an arrival to the other SM).
//
// Roles (768 threads): warp 0 TMA, warp 1 TMEM and MMA issue, warps 4-19 conversion (sixteen, in two turns: a
// warp's chain of a stage, from the barrier to the fence, is long), warps 20-23 epilogue.
// Two accumulators in tensor memory, so the epilogue of a tile runs under the MMAs of the next (one CTA per
// SM walks the tiles).  Few tiles: a cluster of `split` CTAs shares the columns of a tile, and
// adds its accumulators up through distributed shared memory in a fixed order.
//
// Every wait is bounded: on a time-out the kernel writes the status word, all roles leave, the producer waits
// (again bounded) for the copies it has in flight, tensor memory is freed.
#include <algorithm>

#include "int4.cuh"
#include "tensor_core.cuh"

namespace ab {
namespace {

constexpr int kConvWarps = 8, kConvTurns = 2;  // a channel tile each; the turns take alternate stages
constexpr int kEpiWarp = 4 + kConvWarps * kConvTurns;  // first epilogue warp
constexpr int kThreads4 = 32 * (kEpiWarp + 4);
constexpr int kChannels = 128;                 // per tile
constexpr uint32_t kWeightBytes = kChannels * 128;  // of a stage
constexpr int kMostStages = 8;
enum { ST4_PRODUCER = 1, ST4_MMA = 2, ST4_CONVERT = 3, ST4_EPILOGUE = 4 };

struct GemmArgs {
    Int4View w;
    const void *bias;
    void *y;
    int64_t ldy;
    int tokens, bn, stages, kt, n_ct, n_tt, split;
    uint32_t idesc, tmem_cols;
    int *status;
    unsigned long long timeout_ns;
};

// pairs of 16-bit floats: a * b rounded, and a * b + c rounded once
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b, __nv_bfloat16) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b, __half) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c, __nv_bfloat16) {
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b),
                                     *reinterpret_cast<const __nv_bfloat162 *>(&c));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c, __half) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b), *reinterpret_cast<const __half2 *>(&c));
    return *reinterpret_cast<const uint32_t *>(&r);
}

template <typename E, int SUB, bool ZEROS, bool MULT>
__global__ void __launch_bounds__(kThreads4, 1) k_int4_gemm(const __grid_constant__ CUtensorMap tm_x, const GemmArgs a) {
    using S = std::conditional_t<MULT, uint8_t, float>;
    using SP = Packed<S, SUB>;
    using ZP = Packed<int8_t, SUB>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *ring = smem_raw + (base - raw);
    const uint32_t x_bytes = a.bn * 128, stage_bytes = kWeightBytes + x_bytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(ring + (size_t)a.stages * stage_bytes);
    const uint32_t bar_full = smem_u32(bars), bar_empty = smem_u32(bars + kMostStages);
    const uint32_t bar_acc_full = smem_u32(bars + 2 * kMostStages), bar_acc_empty = smem_u32(bars + 2 * kMostStages + 2);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kMostStages + 4);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(bar_full + 8 * s, 1 + kConvWarps);  // the TMA's announcement and the converting warps
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(bar_acc_full + 8 * s, 1);
            mbar_init(bar_acc_empty + 8 * s, 4);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(a.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int rank = a.split > 1 ? (int)(blockIdx.x % a.split) : 0;
    const int worker = (int)(blockIdx.x / a.split), workers = (int)(gridDim.x / a.split);
    const int total = a.n_ct * a.n_tt;
    // this CTA's chunks of every tile, and its column tiles of 64 (the last chunk may have fewer than four)
    const int c0 = a.w.chunks * rank / a.split, c1 = a.w.chunks * (rank + 1) / a.split;
    const int kt0 = 4 * c0, kt1 = min(4 * c1, a.kt);

    if (warp == 0) {
        pdl_launch_dependents();
        pdl_wait();
        if (lane == 0) {
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int tile = worker; ok && tile < total; tile += workers) {
                const int row = tile / a.n_ct * a.bn;
                for (int kt = kt0; kt < kt1; ++kt) {
                    ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, a.status, ST4_PRODUCER, a.timeout_ns);
                    if (!ok) break;
                    mbar_expect_tx(bar_full + 8 * stage, x_bytes);
                    tma_load_2d(base + stage * stage_bytes + kWeightBytes, &tm_x, kt * 64, row, bar_full + 8 * stage);
                    ++issued;
                    if (++stage == a.stages) stage = 0, phase ^= 1;
                }
            }
            if (!ok) {
                // The copies in flight write into this CTA's shared memory: give them time to land.  (Their barriers
                // cannot complete any more, the other roles have left.)
                const unsigned long long t0 = global_ns();
                while (issued && global_ns() - t0 < 1000000ull) {
                }
            }
        }
    } else if (warp == 1) {
        // The whole warp walks the loop and one elected lane issues a stage as straight-line code.  The limit of its
        // waits counts from the predecessor's end, before which no stage can be filled.
        pdl_wait();
        int stage = 0;
        uint32_t phase = 0, pass = 0;
        bool ok = true;
        for (int tile = worker; ok && tile < total; tile += workers, ++pass) {
            const uint32_t buf = pass & 1u, use = pass >> 1;
            ok = mbar_wait(bar_acc_empty + 8 * buf, (use & 1u) ^ 1u, abort_flag, a.status, ST4_MMA, a.timeout_ns);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = tmem_base + buf * a.bn;
            for (int kt = kt0; kt < kt1; ++kt) {
                ok = mbar_wait(bar_full + 8 * stage, phase, abort_flag, a.status, ST4_MMA, a.timeout_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint64_t dw = make_smem_desc(base + stage * stage_bytes), dx = make_smem_desc(base + stage * stage_bytes + kWeightBytes);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)  // 16 input channels, 32 bytes inside the swizzled row
                        umma_f16(d, dw + (uint64_t)(k * 2), dx + (uint64_t)(k * 2), a.idesc, (kt > kt0 || k > 0) ? 1u : 0u);
                    umma_commit(bar_empty + 8 * stage);
                }
                __syncwarp();
                if (++stage == a.stages) stage = 0, phase ^= 1;
            }
            if (ok && elect_one()) umma_commit(bar_acc_full + 8 * buf);
            __syncwarp();
        }
    } else if (warp >= 4 && warp < kEpiWarp) {
        const int g = lane >> 2, t = lane & 3, mine = (warp - 4) % kConvWarps, turn = (warp - 4) / kConvWarps;
        const int64_t row_tiles = div_up(a.w.n, kTileN);
        // of a chunk's four column tiles this warp converts `turn` and `turn + 2`
        struct {
            uint4 code[2];
            typename SP::V scale[2][2];
            typename ZP::V zero[2][2];
        } buf[2];
        // the next chunk to request
        int req_tile = worker, req_c = c0;
        bool inside;  // channels behind the matrix: any finite weights, nobody stores their sums
        const uint4 *code_at;
        const typename SP::V *scale_at;
        const typename ZP::V *zero_at;
        auto seek = [&]() {
            const int64_t row = (int64_t)(req_tile % a.n_ct) * (kChannels / kTileN) + mine;
            inside = row < row_tiles && req_tile < total;
            const int64_t chunk = row * a.w.chunks + c0, entry = chunk * a.w.entries * kTileN + g;
            code_at = a.w.codes + chunk * 128 + 32 * turn + lane;
            scale_at = static_cast<const typename SP::V *>(a.w.scales) + entry;
            zero_at = reinterpret_cast<const typename ZP::V *>(a.w.zeros) + (ZEROS ? entry : 0);
        };
        seek();
        const int off[2] = {a.w.entries * turn / 4 * kTileN, a.w.entries * (turn + 2) / 4 * kTileN}, step = a.w.entries * kTileN;
        auto load = [&](int b) {
            if (inside) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    buf[b].code[i] = code_at[64 * i];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        buf[b].scale[i][r] = scale_at[off[i] + 8 * r];
                        if constexpr (ZEROS) buf[b].zero[i][r] = zero_at[off[i] + 8 * r];
                    }
                }
            }
            code_at += 128;
            scale_at += step;
            zero_at += ZEROS ? step : 0;
            if (++req_c == c1) {
                req_c = c0;
                req_tile += workers;
                seek();
            }
        };
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                buf[b].code[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 2; ++r) buf[b].scale[i][r] = typename SP::V{}, buf[b].zero[i][r] = typename ZP::V{};
            }
        const uint32_t one_zero = zero_pair<E>(a.w.zero);
        const uint32_t row_at = (16 * mine + g) * 128;  // and + 1024 for channel g + 8
        int stage = 0, at = 0;  // the stage of column tile `at`, counted over all tiles of this CTA
        uint32_t phase = 0;
        bool ok = true;
        // weights are never written by a kernel that lets its successor start early: before the wait
        load(0);
        pdl_wait();
        int first = -kt0;  // what is added to a column tile's index to count it over all tiles of this CTA
        for (int tile = worker; ok && tile < total; tile += workers, first += kt1 - kt0) {
            for (int c = c0; ok && c < c1; c += 2) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    if (c + b >= c1 || !ok) break;
                    load(b ^ 1);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int kt = 4 * (c + b) + turn + 2 * i;
                        if (kt >= kt1) break;
                        const uint4 w4 = buf[b].code[i];
                        const uint32_t word[4] = {w4.x, w4.y, w4.z, w4.w};
                        uint32_t out[2][2][4];  // [half of the columns][channel g, g + 8][pairs]
#pragma unroll
                        for (int r = 0; r < 2; ++r)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
#pragma unroll
                                for (int p = 0; p < 4; ++p) {
                                    const int q = 2 * e + r;
                                    const int sub = SUB == 1 ? 0 : SUB == 2 ? e : 2 * e + (p >> 1);  // the columns' block within the tile
                                    const float f = SP::get(buf[b].scale[i][r], sub);
                                    const uint32_t z = ZEROS ? zero_pair<E>(ZP::get(buf[b].zero[i][r], sub)) : one_zero;
                                    const uint32_t v = code_pair<E>(word[q], p, z), hi = Pair16<E>::both(f);
                                    if (MULT) {
                                        out[e][r][p] = mul2(v, hi, E());
                                    } else {
                                        const uint32_t lo = Pair16<E>::both(f - to_f32(*reinterpret_cast<const E *>(&hi)));
                                        out[e][r][p] = fma2(v, hi, mul2(v, lo, E()), E());
                                    }
                                }
                        // at most three further (a last chunk with one tile): a warp that skipped more than a ring of stages could
                        // not tell one that is two uses behind from a free one
                        stage += first + kt - at;
                        at = first + kt;
                        if (stage >= a.stages) stage -= a.stages, phase ^= 1;
                        ok = mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, a.status, ST4_CONVERT, a.timeout_ns);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        uint8_t *dst = ring + (size_t)stage * stage_bytes + row_at;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const uint32_t *v = out[e][r];
                                if constexpr (SUB == 4) {  // four columns at 32 h + 4 t and four at 32 h + 16 + 4 t
                                    *reinterpret_cast<uint2 *>(dst + 1024 * r + (((4 * e + (t >> 1)) ^ g) << 4) + 8 * (t & 1)) = make_uint2(v[0], v[1]);
                                    *reinterpret_cast<uint2 *>(dst + 1024 * r + (((4 * e + 2 + (t >> 1)) ^ g) << 4) + 8 * (t & 1)) = make_uint2(v[2], v[3]);
                                } else {
                                    *reinterpret_cast<uint4 *>(dst + 1024 * r + (((4 * e + t) ^ g) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
                                }
                            }
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar_full + 8 * stage);
                    }
                }
            }
            if ((c1 - c0) & 1) buf[0] = buf[1];  // the tile ended on the first buffer: the next one starts there again
        }
    } else if (warp >= kEpiWarp) {
        pdl_wait();
        const int quad = warp & 3;
        uint32_t pass = 0;
        bool ok = true;
        for (int tile = worker; ok && tile < total; tile += workers, ++pass) {
            const uint32_t buf = pass & 1u, use = pass >> 1;
            ok = mbar_wait(bar_acc_full + 8 * buf, use & 1u, abort_flag, a.status, ST4_EPILOGUE, a.timeout_ns);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t t0 = tmem_base + ((uint32_t)(quad * 32) << 16) + buf * a.bn;
            const int64_t n = (int64_t)(tile % a.n_ct) * kChannels + quad * 32 + lane;
            const bool live = n < a.w.n;
            if (a.split > 1) {
                // all products are done: the ring takes the sums, column by column
                float *sums = reinterpret_cast<float *>(ring) + quad * 32 + lane;
                for (int c = 0; c < a.bn; c += 16) {
                    uint32_t r[16];
                    tmem_ld16(t0 + c, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) sums[(c + j) * kChannels] = __uint_as_float(r[j]);
                }
            } else {
                const RowFactor f = row_factor<E>(live ? a.w.row_scale[n] : 0.f);
                const float b = live && a.bias ? to_f32(static_cast<const E *>(a.bias)[n]) : 0.f;
                const int m0 = tile / a.n_ct * a.bn;
                E *y = static_cast<E *>(a.y) + (int64_t)m0 * a.ldy + n;
                const int left = a.tokens - m0;
                uint32_t ra[16], rb[16];
                tmem_ld16(t0, ra);
                for (int c = 0; c < a.bn; c += 32) {
                    tmem_ld_wait();
                    tmem_ld16(t0 + c + 16, rb);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (live && c + j < left) y[(int64_t)(c + j) * a.ldy] = Cvt<float, E>::store(fmaf(__uint_as_float(ra[j]) * f.unit, f.scale, b));
                    __syncwarp();  // (reading tensor memory is a warp's lanes together, after stores that some lanes skip)
                    tmem_ld_wait();
                    if (c + 32 < a.bn) tmem_ld16(t0 + c + 32, ra);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (live && c + 16 + j < left) y[(int64_t)(c + 16 + j) * a.ldy] = Cvt<float, E>::store(fmaf(__uint_as_float(rb[j]) * f.unit, f.scale, b));
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_acc_empty + 8 * buf);
        }
    }

    // every role has left its loop, normally or through the abort flag
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (a.split > 1) {
        cluster_barrier();
        const int tile = worker, m0 = tile / a.n_ct * a.bn;
        const int64_t n0 = (int64_t)(tile % a.n_ct) * kChannels;
        const int share = a.bn / a.split;  // columns that this CTA adds up
        for (int i = threadIdx.x; i < share * kChannels; i += kThreads4) {
            const int col = rank * share + i / kChannels, ch = i % kChannels;
            if (m0 + col >= a.tokens || n0 + ch >= a.w.n) continue;
            const uint32_t here = base + (col * kChannels + ch) * 4;
            float v = 0.f;
            for (int c = 0; c < a.split; ++c) {
                const uint32_t there = map_to_rank(here, c);
                float f;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(there) : "memory");
                v += f;
            }
            const RowFactor f = row_factor<E>(a.w.row_scale[n0 + ch]);
            v = v * f.unit * f.scale;
            if (a.bias) v += to_f32(static_cast<const E *>(a.bias)[n0 + ch]);
            static_cast<E *>(a.y)[(int64_t)(m0 + col) * a.ldy + n0 + ch] = Cvt<float, E>::store(v);
        }
        cluster_barrier();  // nobody leaves while its sums are being read
    }
    tc_fence_after();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(a.tmem_cols) : "memory");
}

template <typename E, int SUB, bool ZEROS, bool MULT> int launch(const Int4Gemm &c) {
    const int sms = sm_count();
    GemmArgs a;
    a.w = c.w;
    a.bias = c.bias;
    a.y = c.y;
    a.ldy = c.ldy;
    a.tokens = c.tokens;
    a.kt = (int)div_up(c.w.k, kTileK);
    a.n_ct = (int)div_up(c.w.n, kChannels);
    // as many tokens per tile as there are, but rather more tiles than idle SMs
    a.bn = c.tokens <= 32 ? 32 : c.tokens <= 64 ? 64 : c.tokens <= 128 || a.n_ct * div_up(c.tokens, 256) < sms ? 128 : 256;
    a.n_tt = (int)div_up(c.tokens, a.bn);
    const int64_t total = (int64_t)a.n_ct * a.n_tt;
    if (total > 0x7fffffff) return fail(AB_ERR_UNSUPPORTED, "%d tokens x %lld channels in one call", c.tokens, (long long)c.w.n);
    a.split = 1;
    while (a.split < 8 && total * a.split * 2 <= sms && c.w.chunks >= a.split * 2) a.split *= 2;
    const uint32_t stage_bytes = kWeightBytes + a.bn * 128;
    a.stages = std::min<int>(kMostStages, 196608 / stage_bytes);
    const size_t smem = (size_t)a.stages * stage_bytes + 1024 /*alignment*/ + 256 /*barriers*/;
    a.tmem_cols = 2 * a.bn;
    const uint32_t fmt = c.io_dtype == AB_BF16 ? 1u : 0u;
    a.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(a.bn >> 3) << 17) | ((kChannels >> 4) << 24);
    a.status = c.status;
    a.timeout_ns = kWaitTimeoutNs;
    CUtensorMap tm;
    int rc = make_map(&tm, c.x, c.tokens, c.w.k, c.ldx, a.bn, c.io_dtype);
    if (rc != AB_OK) return rc;
    if ((rc = opt_in_smem<k_int4_gemm<E, SUB, ZEROS, MULT>>(200 * 1024)) != AB_OK) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.split > 1 ? total * a.split : std::min<int64_t>(total, sms)));
    cfg.blockDim = dim3(kThreads4);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.split;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.split > 1 ? 2 : 1;
    AB_CUDA_OK(cudaLaunchKernelEx(&cfg, k_int4_gemm<E, SUB, ZEROS, MULT>, tm, a));
    AB_LAUNCH_OK();
    return AB_OK;
}
template <typename E, int SUB> int dispatch_scales(const Int4Gemm &c) {
    if (c.mult) return c.w.zeros ? launch<E, SUB, true, true>(c) : launch<E, SUB, false, true>(c);
    return c.w.zeros ? launch<E, SUB, true, false>(c) : launch<E, SUB, false, false>(c);
}
template <typename E> int dispatch_block(const Int4Gemm &c) {
    return c.block == 16 ? dispatch_scales<E, 4>(c) : c.block == 32 ? dispatch_scales<E, 2>(c) : dispatch_scales<E, 1>(c);
}

}  // namespace

int launch_int4_gemm(const Int4Gemm &c) { return c.io_dtype == AB_BF16 ? dispatch_block<__nv_bfloat16>(c) : dispatch_block<__half>(c); }

}  // namespace ab
