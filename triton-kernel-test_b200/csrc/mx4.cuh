// mx4.cuh -- the microscaled 4-bit format of include/actcomp.h: sizes, scale
// positions and the conversions of one value group.
#pragma once

#include "common.cuh"

namespace act {
namespace mx4 {

constexpr int BLOCK = 32;      // values that share a scale
constexpr int ATOM_ROWS = 128, ATOM_BLOCKS = 4, ATOM_BYTES = 512;

__host__ __device__ __forceinline__ int64_t blocks_of(int64_t cols) { return (cols + BLOCK - 1) / BLOCK; }
__host__ __device__ __forceinline__ int64_t atoms_of(int64_t cols) { return (cols + 127) / 128; }
__host__ __device__ __forceinline__ int64_t row_bytes(int64_t cols) { return blocks_of(cols) * 16; }
static inline size_t code_bytes(int64_t rows, int64_t cols) { return (size_t)rows * (size_t)row_bytes(cols); }
static inline size_t scale_bytes(int64_t rows, int64_t cols) {
    return (size_t)((rows + 127) / 128) * (size_t)atoms_of(cols) * ATOM_BYTES;
}
// Byte offset of the four scales of row r, blocks 4 ka .. 4 ka + 3.
__device__ __forceinline__ int64_t scale_word(int64_t r, int64_t ka, int64_t nka) {
    return ((r >> 7) * nka + ka) * ATOM_BYTES + (r & 31) * 16 + ((r >> 5) & 3) * 4;
}

// Scale byte of a block from the bits of its largest magnitude as float32
// (integer comparison orders NaN above infinity above every finite value).
__device__ __forceinline__ uint32_t scale_code(uint32_t amax_bits) {
    const uint32_t e = amax_bits >> 23;
    return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 2^(127 - code): multiplying by it is exact wherever the result matters.
__device__ __forceinline__ float inv_scale(uint32_t code) {
    return __uint_as_float(code == 255u ? 0x3f800000u : (254u - code) << 23);
}
__device__ __forceinline__ float scale_value(uint32_t code) {
    return __uint_as_float(code == 255u ? 0x7fc00000u : (code == 0u ? 0x00400000u : code << 23));
}

// Eight scaled values to eight e2m1 codes, value j in nibble j (nearest, ties
// to even, saturating).
__device__ __forceinline__ uint32_t pack8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n .reg .b8 a, b, c, d;\n"
        " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        " mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// Eight codes to four pairs of fp16 (exact).
__device__ __forceinline__ void unpack8(uint32_t codes, uint32_t (&h)[4]) {
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
        " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n cvt.rn.f16x2.e2m1x2 %2, c;\n"
        " cvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
}

}  // namespace mx4
}  // namespace act
