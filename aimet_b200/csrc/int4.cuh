// What the products with 4-bit weights share: the packed layout and the conversion of codes to pairs of
// 16-bit floats.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace ab {

constexpr int kTileN = 16;    // output channels per tile
constexpr int kTileK = 64;    // input channels per tile
constexpr int kChunkK = 256;  // input channels per chunk: four tiles, 2 KB that one warp requests at once
constexpr int64_t kMaxK = 1ll << 20;

// Codes [channel tile][tile of columns][lane][16 bytes]; scales (float32, or uint8 factors) and zero points
// (int8) [channel tile][chunk][entry][channel][sub]: one entry per chunk (blocks of 256 columns or more), two
// (128) or four (64 or fewer, with 64 / block neighbouring blocks in an entry).  What lies behind the matrix
// is there and multiplies zeros of x.
struct Int4View {
    const uint4 *codes;
    const void *scales;
    const int8_t *zeros;  // NULL: `zero` for all
    const float *row_scale;
    int64_t n, k;
    int chunks;   // per row: div_up(k, kChunkK)
    int entries;  // per chunk: 1, 2, 4
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
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    }
};
// what turns a code in the mantissa of kBase into (u - z) * kUnit (all three steps exact)
template <typename H> __device__ __forceinline__ uint32_t zero_pair(float z) {
    return Pair16<H>::both(-(Pair16<H>::kBase + z) * Pair16<H>::kUnit);
}
// What a channel's sum of code * kUnit * x is multiplied by: first `unit`, then `scale`; together row_scale / kUnit, which
// by itself may be no float32 number although the result is one.
struct RowFactor {
    float unit, scale;
};
template <typename H> __device__ __forceinline__ RowFactor row_factor(float row_scale) {
    constexpr float kUp = 1.f / Pair16<H>::kUnit;
    if constexpr (kUp == 1.f) return {1.f, row_scale};
    return fabsf(row_scale) < 1.f ? RowFactor{1.f, row_scale * kUp} : RowFactor{kUp, row_scale};
}
// the codes of pair p (0..3) of a word as two 16-bit floats, (u - z) * kUnit
template <typename H> __device__ __forceinline__ uint32_t code_pair(uint32_t word, int p, uint32_t zero2) {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(v) : "r"(word >> (4 * p)), "r"(Pair16<H>::kMagic));
    return Pair16<H>::code(v, zero2);
}

// SUB neighbouring values of type T as one register value (or vector of them)
template <typename T, int SUB> struct Packed;
template <> struct Packed<float, 1> { using V = float; static __device__ __forceinline__ float get(V v, int) { return v; } };
template <> struct Packed<float, 2> { using V = float2; static __device__ __forceinline__ float get(V v, int i) { return i ? v.y : v.x; } };
template <> struct Packed<float, 4> {
    using V = float4;
    static __device__ __forceinline__ float get(V v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
};
template <> struct Packed<uint8_t, 1> { using V = uint8_t; static __device__ __forceinline__ float get(V v, int) { return (float)v; } };
template <> struct Packed<uint8_t, 2> { using V = uint16_t; static __device__ __forceinline__ float get(V v, int i) { return (float)((v >> (8 * i)) & 0xff); } };
template <> struct Packed<uint8_t, 4> { using V = uint32_t; static __device__ __forceinline__ float get(V v, int i) { return (float)((v >> (8 * i)) & 0xff); } };
template <> struct Packed<int8_t, 1> { using V = int8_t; static __device__ __forceinline__ float get(V v, int) { return (float)v; } };
template <> struct Packed<int8_t, 2> { using V = uint16_t; static __device__ __forceinline__ float get(V v, int i) { return (float)(int8_t)(v >> (8 * i)); } };
template <> struct Packed<int8_t, 4> { using V = uint32_t; static __device__ __forceinline__ float get(V v, int i) { return (float)(int8_t)(v >> (8 * i)); } };

// y for many tokens (int4_gemm.cu): 16-bit x, 16-byte aligned rows.  block, mult: as in the descriptor.
struct Int4Gemm {
    Int4View w;
    const void *x, *bias;
    void *y;
    int64_t ldx, ldy;
    int tokens, block, io_dtype;
    bool mult;
    int *status;
    cudaStream_t stream;
};
int launch_int4_gemm(const Int4Gemm &c);

}  // namespace ab
