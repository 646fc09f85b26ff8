// mx4_quant.cu -- microscaled 4-bit quantisation (by rows, by columns, or both)
// and its inverse; the format is stated in include/actcomp.h.
//
// HBM-bound: by rows 2 bytes in and 17/32 out per bf16 value.  Four lanes share
// a block of 32 values, eight consecutive values each: loads and code stores
// are contiguous over the warp, the block's largest magnitude takes two
// shuffles, and a warp's 256 values fill two whole scale words.
#include <cuda_fp16.h>

#include "mx4.cuh"

namespace act {
namespace mx4 {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

template <typename T>
struct alignas(16) Raw8 {
    T v[8];
};

__device__ __forceinline__ uint32_t abs_bits(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// By rows: one warp per 256 columns of a row, rows rounded up to whole atoms.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    quant_rows_kernel(const T *x, int64_t rows, int64_t cols, int64_t ldx, uint8_t *codes, uint8_t *scales) {
    const int lane = threadIdx.x & 31;
    const int64_t segs = (cols + 255) / 256, nka = atoms_of(cols), rb = row_bytes(cols);
    const int64_t total = (rows + 127) / 128 * 128 * segs;
    const int64_t step = (int64_t)gridDim.x * 8;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < total; i += step) {
        const int64_t r = i / segs, sg = i - r * segs;
        const int64_t c = sg * 256 + 8 * lane;
        float v[8] = {};
        uint32_t m = 0;
        if (r < rows) {
            Raw8<T> raw;
            if (VEC) {
                uint4 *d = reinterpret_cast<uint4 *>(&raw);
                const uint4 *s = reinterpret_cast<const uint4 *>(x + r * ldx + c);
#pragma unroll
                for (int k = 0; k < (int)sizeof(raw) / 16; ++k) d[k] = c < cols ? s[k] : make_uint4(0, 0, 0, 0);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) raw.v[j] = c + j < cols ? x[r * ldx + c + j] : from_f<T>(0.f);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = to_f<T>(raw.v[j]);
                m = max(m, abs_bits(v[j]));
            }
        }
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const uint32_t sc = scale_code(m);
        if (r < rows && c < blocks_of(cols) * BLOCK) {
            const float inv = inv_scale(sc);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= inv;
            *reinterpret_cast<uint32_t *>(codes + r * rb + c / 2) = pack8(v);
        }
        // four blocks' scale bytes to one word (lanes 0 and 16)
        uint32_t w = sc;
        w |= __shfl_down_sync(0xffffffffu, w, 4) << 8;
        w |= __shfl_down_sync(0xffffffffu, w, 8) << 16;
        const int64_t ka = sg * 2 + (lane >> 4);
        if ((lane & 15) == 0 && ka < nka) *reinterpret_cast<uint32_t *>(scales + scale_word(r, ka, nka)) = w;
    }
}

// By columns: a thread takes one column over 32 rows, a row of threads 256
// neighbouring columns.
template <typename T>
__global__ void __launch_bounds__(256)
    quant_cols_kernel(const T *x, int64_t rows, int64_t cols, int64_t ldx, uint8_t *codes, uint8_t *scales) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;  // over cols rounded up to 128
    const int64_t nka = atoms_of(rows), rb = row_bytes(rows), nb = blocks_of(rows);
    if (c >= (cols + 127) / 128 * 128) return;
    for (int64_t b = blockIdx.y; b < nka * ATOM_BLOCKS; b += gridDim.y) {
        uint32_t m = 0;
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const int64_t r = b * 32 + j;
            v[j] = c < cols && r < rows ? to_f<T>(x[r * ldx + c]) : 0.f;
            m = max(m, abs_bits(v[j]));
        }
        const uint32_t sc = scale_code(m);
        if (c < cols && b < nb) {
            const float inv = inv_scale(sc);
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float t[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = v[8 * k + j] * inv;
                w[k] = pack8(t);
            }
            *reinterpret_cast<uint4 *>(codes + c * rb + b * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        scales[scale_word(c, b >> 2, nka) + (b & 3)] = (uint8_t)sc;
    }
}

// One lane per eight values.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    dequant_kernel(const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t cols, T *out, int64_t ldo) {
    const int64_t per_row = (cols + 7) / 8, nka = atoms_of(cols), rb = row_bytes(cols);
    const int64_t total = rows * per_row, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const int64_t r = i / per_row, g = i - r * per_row;
        uint32_t h[4];
        unpack8(*reinterpret_cast<const uint32_t *>(codes + r * rb + g * 4), h);
        const float s = scale_value(scales[scale_word(r, g >> 4, nka) + ((g >> 2) & 3)]);
        Raw8<T> o;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[k]));
            o.v[2 * k] = from_f<T>(f.x * s);
            o.v[2 * k + 1] = from_f<T>(f.y * s);
        }
        T *d = out + r * ldo + g * 8;
        if (VEC) {
            const uint4 *src = reinterpret_cast<const uint4 *>(&o);
#pragma unroll
            for (int k = 0; k < (int)sizeof(o) / 16; ++k) reinterpret_cast<uint4 *>(d)[k] = src[k];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (g * 8 + j < cols) d[j] = o.v[j];
        }
    }
}

template <typename F>
static int with_type(int dtype, F f) {
    if (dtype == 0) return f(float{});
    if (dtype == 1) return f(__nv_bfloat16{});
    return f(__half{});
}

static int check(const actcomp_mx4 *q) {
    ACT_CHECK(q && q->rows > 0 && q->cols > 0, ACT_E_INVALID);
    ACT_CHECK(q->rows <= INT32_MAX - 255 && q->cols <= INT32_MAX - 255, ACT_E_UNSUPPORTED);
    ACT_CHECK(q->codes && q->scales, ACT_E_INVALID);
    ACT_CHECK(aligned(q->codes, 16) && aligned(q->scales, 16), ACT_E_ALIGN);
    return ACT_OK;
}

}  // namespace mx4
int mx4_check(const actcomp_mx4 *q) { return mx4::check(q); }
}  // namespace act

extern "C" size_t actcomp_mx4_code_bytes(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 ? act::mx4::code_bytes(rows, cols) : 0;
}
extern "C" size_t actcomp_mx4_scale_bytes(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 ? act::mx4::scale_bytes(rows, cols) : 0;
}

extern "C" int actcomp_mx4_quantize(const void *x, int64_t rows, int64_t cols, int64_t ldx, int32_t dtype,
                                    const actcomp_mx4 *q, const actcomp_mx4 *qt, void *stream) {
    using namespace act;
    using namespace act::mx4;
    ACT_CHECK(x && (q || qt) && rows > 0 && cols > 0 && ldx >= cols && dtype >= 0 && dtype <= 2, ACT_E_INVALID);
    if (q) {
        ACT_CHECK(q->rows == rows && q->cols == cols, ACT_E_INVALID);
        if (int st = check(q)) return st;
    }
    if (qt) {
        ACT_CHECK(qt->rows == cols && qt->cols == rows, ACT_E_INVALID);
        if (int st = check(qt)) return st;
    }
    const int es = dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(x, es), ACT_E_ALIGN);
    cudaStream_t st = as_stream(stream);
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        const T *xs = static_cast<const T *>(x);
        if (q) {
            const bool vec = cols % 8 == 0 && aligned(x, 16) && (ldx * es) % 16 == 0;
            const int64_t warps = (rows + 127) / 128 * 128 * ((cols + 255) / 256);
            const int64_t cap = (int64_t)num_sms() * 16, ctas = (warps + 7) / 8;
            const int grid = (int)(ctas < cap ? ctas : cap);
            if (vec) quant_rows_kernel<T, true><<<grid, 256, 0, st>>>(xs, rows, cols, ldx, q->codes, q->scales);
            else quant_rows_kernel<T, false><<<grid, 256, 0, st>>>(xs, rows, cols, ldx, q->codes, q->scales);
            if (int rc = launch_status()) return rc;
        }
        if (qt) {
            const int64_t nb = atoms_of(rows) * ATOM_BLOCKS;
            const dim3 grid((unsigned)((cols + 255) / 256), (unsigned)(nb < 65535 ? nb : 65535));
            quant_cols_kernel<T><<<grid, 256, 0, st>>>(xs, rows, cols, ldx, qt->codes, qt->scales);
        }
        return launch_status();
    });
}

extern "C" int actcomp_mx4_dequantize(const actcomp_mx4 *q, void *out, int64_t ldo, int32_t dtype, void *stream) {
    using namespace act;
    using namespace act::mx4;
    if (int st = check(q)) return st;
    ACT_CHECK(out && ldo >= q->cols && dtype >= 0 && dtype <= 2, ACT_E_INVALID);
    const int es = dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(out, es), ACT_E_ALIGN);
    const bool vec = q->cols % 8 == 0 && aligned(out, 16) && (ldo * es) % 16 == 0;
    const int64_t ctas = (q->rows * ((q->cols + 7) / 8) + 255) / 256, cap = (int64_t)num_sms() * 16;
    const int grid = (int)(ctas < cap ? ctas : cap);
    cudaStream_t st = as_stream(stream);
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        T *o = static_cast<T *>(out);
        if (vec) dequant_kernel<T, true><<<grid, 256, 0, st>>>(q->codes, q->scales, q->rows, q->cols, o, ldo);
        else dequant_kernel<T, false><<<grid, 256, 0, st>>>(q->codes, q->scales, q->rows, q->cols, o, ldo);
        return launch_status();
    });
}
