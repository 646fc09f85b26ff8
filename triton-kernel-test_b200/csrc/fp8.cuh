// fp8.cuh -- 8-bit floating point with a power-of-two scale per block of 128, the
// format of include/actcomp.h: sizes, scale positions and conversions.
#pragma once

#include <cuda_fp16.h>
#include <string.h>

#include <type_traits>

#include "common.cuh"

namespace act {
namespace fp8 {

constexpr int BLOCK = 128;
enum Format { E4M3 = 0, E5M2 = 1 };
enum Block { ROWS = 0, COLS = 1, TILES = 2 };

__host__ __device__ __forceinline__ int64_t blocks_of(int64_t n) { return (n + BLOCK - 1) / BLOCK; }
static inline size_t scale_bytes(int64_t rows, int64_t cols, int block) {
    const size_t b = (size_t)blocks_of(rows) * (size_t)blocks_of(cols);
    return block == TILES ? b : b * BLOCK;
}
// Byte of a line's scale (line: a row of blocks 1 x 128, a column of blocks 128 x 1)
// in block b of the other dimension; `groups` = ceil(lines / 128).  A lane of the
// product's scale warps takes the four bytes of lines l, l + 32, l + 64, l + 96 as a word.
__host__ __device__ __forceinline__ int64_t scale_at(int64_t line, int64_t b, int64_t groups) {
    return (b * groups + (line >> 7)) * BLOCK + (line & 31) * 4 + ((line >> 5) & 3);
}

// Scale byte of a block from the bits of its largest magnitude as float32 (as
// integers NaN lies above infinity above every finite value): the smallest exponent
// under which the magnitude is at most 1.75 * 2^top (the format's largest value), so
// that nothing saturates; 255 where the block holds a NaN or an infinity.
__device__ __forceinline__ uint32_t scale_code(uint32_t amax_bits, uint32_t top) {
    const uint32_t e = (amax_bits + 0x1fffffu) >> 23;  // + 1 past a mantissa of 1.75
    return amax_bits >= 0x7f800000u ? 255u : (e > top ? e - top : 0u);
}
__device__ __forceinline__ uint32_t top_of(int format) { return format == E5M2 ? 15u : 8u; }
// 2^(127 - code): the product with it is exact wherever the result is no subnormal of float32.
__device__ __forceinline__ float inv_scale(uint32_t code) {
    return __uint_as_float(code == 255u ? 0x3f800000u : code == 254u ? 0x00400000u : (254u - code) << 23);
}
// 2^(code - 127)
__device__ __forceinline__ float scale_value(uint32_t code) {
    return __uint_as_float(code == 255u ? 0x7fc00000u : (code == 0u ? 0x00400000u : code << 23));
}

// Two scaled values to two codes, `lo` in the low byte (nearest, ties to even).
template <int FORMAT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint16_t r;
    if constexpr (FORMAT == E4M3) asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
    else asm("cvt.rn.satfinite.e5m2x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
    return r;
}
template <int FORMAT>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    return __byte_perm(pack2<FORMAT>(a, b), pack2<FORMAT>(c, d), 0x5410);
}
// Two codes (the low half of `v`) to float32.
template <int FORMAT>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    uint32_t h;
    const uint16_t c = (uint16_t)v;
    if constexpr (FORMAT == E4M3) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
    else asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"(c));
    __half2 t;
    memcpy(&t, &h, 4);
    return __half22float2(t);
}
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

}  // namespace fp8
}  // namespace act
