// Microscaled 4-bit floating point: what the quantizers and the product agree on.
//
// An element is an e2m1 number; two share a byte, element 2j in the low nibble. DUQ4_FP4_MX keeps one e8m0 scale
// (2^(byte - 127), 0xFF = NaN) per 32 neighbours of a row, DUQ4_FP4_NV one e4m3 scale per 16 neighbours and one float
// per row. Block scales are kept in the order in which the tensor cores take them: tiles of 128 rows x 4 blocks, 512
// bytes, row r of a tile at byte 16 * (r % 32) + 4 * (r / 32); tiles of a row block lie one behind the other.
#pragma once
#include <cuda_bf16.h>

#include "duq_common.cuh"

namespace duq4 {
namespace fp4 {

constexpr int kMX = DUQ4_FP4_MX, kNV = DUQ4_FP4_NV;

__host__ __device__ constexpr uint32_t block_of(int format) { return format == kMX ? 32u : 16u; }
// 4-block tiles of a row (columns beyond the row's end have scale bytes too: zero, so that they add nothing)
__host__ __device__ inline uint32_t scale_tiles(int format, uint32_t cols) { return cdiv(cols, 4 * block_of(format)); }
__host__ __device__ inline size_t scale_offset(uint32_t tiles, uint32_t row, uint32_t tile) {
    return ((size_t)(row >> 7) * tiles + tile) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// Eight floats -> eight e2m1 codes, low nibble first (round to nearest, ties to the even code, saturating at 6).
__device__ __forceinline__ uint32_t e2m1x8(const float (&f)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
    return r;
}
// One byte (two codes) -> two halves, exactly.
__device__ __forceinline__ __half2 e2m1x2_to_half2(uint32_t byte) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, z1, z2, z3;\n\tmov.b32 {a, z1, z2, z3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(r) : "r"(byte));
    return *reinterpret_cast<__half2 *>(&r);
}
// A non-negative float -> e4m3 byte (round to nearest even, at most 448), and back.
__device__ __forceinline__ uint32_t e4m3_of(float f) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(f));
    return r & 0xFFu;
}
__device__ __forceinline__ float e4m3_to_float(uint32_t byte) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)byte));
    return __low2float(*reinterpret_cast<__half2 *>(&r));
}
// 2^(byte - 127); 0xFF is NaN.
__device__ __forceinline__ float e8m0_to_float(uint32_t byte) {
    return byte == 0xFFu ? __uint_as_float(0x7FFFFFFFu) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
template <int FMT>
__device__ __forceinline__ float block_scale_to_float(uint32_t byte) {
    return FMT == kMX ? e8m0_to_float(byte) : e4m3_to_float(byte);
}

// The two 16-bit element types as 32-bit words of two.
template <class T>
struct Two;
template <>
struct Two<__half> {
    static constexpr uint32_t kInf = 0x7C00u;
    static __device__ __forceinline__ float2 up(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
    static __device__ __forceinline__ float up1(uint32_t bits) { return __half2float(__ushort_as_half((unsigned short)bits)); }
    // larger magnitudes of two pairs, with signs of no meaning; a NaN wins
    static __device__ __forceinline__ uint32_t abs_max(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <>
struct Two<__nv_bfloat16> {
    static constexpr uint32_t kInf = 0x7F80u;
    static __device__ __forceinline__ float2 up(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
    static __device__ __forceinline__ float up1(uint32_t bits) { return __uint_as_float(bits << 16); }
    static __device__ __forceinline__ uint32_t abs_max(uint32_t a, uint32_t b) {
        uint32_t r;
        asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ uint32_t down(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};

}  // namespace fp4
}  // namespace duq4
