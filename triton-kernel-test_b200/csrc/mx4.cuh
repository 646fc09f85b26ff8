// mx4.cuh -- the microscaled 4-bit format of include/actcomp.h: sizes, scale
// positions and the conversions of one value group.
#pragma once

#include <cuda_fp16.h>
#include <string.h>

#include <type_traits>

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
// to even, saturating).  Each byte leaves its asm block by itself: with four of
// them packed inside one block some kernels wrote zeros.  The cause is not known
// (no reduced case was kept); the tests compare every code with a plain restatement.
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint16_t r;
    asm("{\n .reg .b8 t;\n cvt.rn.satfinite.e2m1x2.f32 t, %2, %1;\n mov.b16 %0, {t, 0};\n}" : "=h"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ uint32_t pack8(const float (&v)[8]) {
    const uint32_t lo = __byte_perm(pack2(v[0], v[1]), pack2(v[2], v[3]), 0x0040);
    const uint32_t hi = __byte_perm(pack2(v[4], v[5]), pack2(v[6], v[7]), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}
// Codes j and j + 4 of a word as a pair of fp16 times 2^-14 (exact): the sign to
// bit 15, exponent and mantissa to bits 11..9.  With fp16's bias of 15 against
// e2m1's 1 that is the value times 2^-14, and e2m1's subnormal (exponent 0) is an
// fp16 subnormal.  (With the conversion instruction from e2m1 pairs, on bytes
// shifted out of the word, some kernels gave wrong values; the cause is not known.)
template <int J>
__device__ __forceinline__ uint32_t tiny_pair(uint32_t codes) {
    const uint32_t m = J < 3 ? codes << (J < 3 ? 9 - 4 * J : 0) : codes >> 3;
    return ((codes << (12 - 4 * J)) & 0x80008000u) | (m & 0x0e000e00u);
}
__device__ __forceinline__ __half2 as_half2(uint32_t v) {
    __half2 h;
    memcpy(&h, &v, 4);
    return h;
}
// The pairs (0, 4), (1, 5), (2, 6), (3, 7) times 2^-14.
__device__ __forceinline__ void tiny8(uint32_t codes, __half2 (&h)[4]) {
    h[0] = as_half2(tiny_pair<0>(codes));
    h[1] = as_half2(tiny_pair<1>(codes));
    h[2] = as_half2(tiny_pair<2>(codes));
    h[3] = as_half2(tiny_pair<3>(codes));
}

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }

// Larger magnitude of each 16-bit half of m (magnitudes) and v; NaN stays.
template <typename T>
__device__ __forceinline__ uint32_t absmax2(uint32_t m, uint32_t v) {
    uint32_t r;
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("{\n .reg .b32 t;\n abs.bf16x2 t, %2;\n max.NaN.bf16x2 %0, %1, t;\n}" : "=r"(r) : "r"(m), "r"(v));
    else
        asm("{\n .reg .b32 t;\n abs.f16x2 t, %2;\n max.NaN.f16x2 %0, %1, t;\n}" : "=r"(r) : "r"(m), "r"(v));
    return r;
}

// Eight values as their words; zero() is eight zeros in every type.
template <typename T>
struct Raw8 {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load_vec(const T *p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const uint4 q = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = q.x, w[4 * i + 1] = q.y, w[4 * i + 2] = q.z, w[4 * i + 3] = q.w;
        }
    }
    // n of them, the others zero
    __device__ __forceinline__ void load(const T *p, int n) {
        zero();
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < n) {
                if constexpr (sizeof(T) == 4) {
                    w[j] = reinterpret_cast<const uint32_t *>(p)[j];
                } else {
                    w[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[j] << (16 * (j & 1));
                }
            }
    }
    __device__ __forceinline__ void floats(float (&f)[8]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    f[2 * j] = __uint_as_float(w[j] << 16);
                    f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
                } else {
                    __half2 h;
                    memcpy(&h, &w[j], 4);
                    const float2 t = __half22float2(h);
                    f[2 * j] = t.x, f[2 * j + 1] = t.y;
                }
            }
        }
    }
    // The largest magnitude's bits: 16-bit types in both halves of the word to
    // be folded by amax_bits, float32 as it is.
    __device__ __forceinline__ uint32_t amax() const {
        if constexpr (sizeof(T) == 4) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, w[j] & 0x7fffffffu);
            return m;
        } else {
            return absmax2<T>(absmax2<T>(absmax2<T>(absmax2<T>(0u, w[0]), w[1]), w[2]), w[3]);
        }
    }
};
template <typename T>
__device__ __forceinline__ uint32_t max_of(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) return max(a, b);
    else return __vmaxu2(a, b);
}
// Magnitude bits as float32 bits (NaN stays above infinity above the finite).
template <typename T>
__device__ __forceinline__ uint32_t amax_bits(uint32_t m) {
    if constexpr (sizeof(T) == 4) {
        return m;
    } else {
        const uint32_t h = max(m & 0xffffu, m >> 16);
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return h << 16;
        else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
    }
}

}  // namespace mx4
}  // namespace act
