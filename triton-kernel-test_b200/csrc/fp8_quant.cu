// fp8_quant.cu -- 8-bit floating point with a power-of-two scale per block of 128:
// quantisation by rows (1 x 128), by columns (128 x 1), both from one read, or by
// tiles (128 x 128), and the inverse.  The format is stated in include/actcomp.h.
//
// Its floor is HBM: 2 bytes in and 1 (both ways: 2) out per bf16 value.  A CTA takes
// 128 x 128 values into registers, eight rows of eight columns a thread, all loads
// under way at once: a row's block is then 16 lanes (four shuffles for its largest
// magnitude), a column's the CTA (one shuffle, then shared memory), and both forms are
// converted from the same registers.  Codes stay in the matrix's own orientation (the
// tensor cores take either operand with its rows contiguous), so no direction needs a
// transposition, and the scales of a block row or column are 128 bytes in one piece.
//
// 16384 x 11008 on a B200, us and share of the copy rate:
//             rows        columns     tiles       both        inverse
//   bf16      99  83 %    86  96 %    84  98 %    152  73 %   90  92 %
//   float32   150 92 %    138 100 %   134 100 %   192 86 %    180 76 %
// Rows that are not 16-byte aligned go through shared memory, neighbouring lanes
// neighbouring values (2050 x 1338 float32: the inverse 22 us value by value, 8.8 so).
// Three CTAs per SM instead of four: rows 108, columns 95, both 162.
#include "fp8.cuh"
#include "mx4.cuh"
#include "tc_ptx.cuh"

namespace act {
namespace fp8 {

using mx4::Raw8;
constexpr int NR = 8;  // rows of a thread: t / 16 + 16 i

struct Dst {
    uint8_t *codes, *scales;
    int64_t ld;
};
enum Mode { BY_ROWS = 1, BY_COLS = 2, BY_BOTH = 3, BY_TILES = 4 };

// n of eight values times their factors (f(j): of the j-th pair) to codes at p.
template <int FORMAT, typename F>
__device__ __forceinline__ void store_scaled8(uint8_t *p, const float (&v)[8], F f, int n) {
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 t = mul2(make_float2(v[2 * j], v[2 * j + 1]), f(j));
        h[j] = pack2<FORMAT>(t.x, t.y);
    }
    const uint32_t lo = __byte_perm(h[0], h[1], 0x5410), hi = __byte_perm(h[2], h[3], 0x5410);
    if (n == 8) {
        *reinterpret_cast<uint2 *>(p) = make_uint2(lo, hi);
    } else {
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (j < n) p[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
    }
}

template <typename T, bool VEC, int MODE, int FORMAT>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2)
    quant_kernel(const T *x, int64_t rows, int64_t cols, int64_t ldx, Dst a, Dst b) {
    __shared__ __align__(16) uint32_t colmax[8][128];  // of each warp
    __shared__ __align__(16) float colinv[128];
    __shared__ __align__(16) uint8_t line[2][128];  // scales of the rows, of the columns
    tc::launch_dependents();  // the product that follows may set itself up
    const int ctiles = (int)blocks_of(cols), kr = blockIdx.x / ctiles, kc = blockIdx.x - kr * ctiles;
    const int64_t r0 = (int64_t)kr * 128, c0 = (int64_t)kc * 128;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ty = tid >> 4, cl = (tid & 15) * 8;
    const int64_t c = c0 + cl;
    const int n = c >= cols ? 0 : (cols - c < 8 ? (int)(cols - c) : 8);
    constexpr uint32_t TOP = FORMAT == E5M2 ? 15 : 8;
    Raw8<T> raw[NR];
    if constexpr (!VEC) {  // neighbouring lanes neighbouring values, through shared memory
        extern __shared__ __align__(16) uint8_t dyn[];
        T *stage = reinterpret_cast<T *>(dyn);
        const int left = cols - c0 < 128 ? (int)(cols - c0) : 128;
        constexpr int PITCH = 128 + 16 / (int)sizeof(T);
#pragma unroll 4
        for (int i = warp; i < 128; i += 8) {
            T v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = T(0.f);
                if (r0 + i < rows && 32 * j + lane < left) v[j] = x[(r0 + i) * ldx + c0 + 32 * j + lane];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) stage[i * PITCH + 32 * j + lane] = v[j];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NR; ++i) raw[i].load_vec(stage + (ty + 16 * i) * PITCH + cl);
    } else {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int64_t r = r0 + ty + 16 * i;
            if (r < rows && n == 8) raw[i].load_vec(x + r * ldx + c);
            else if (r < rows && n > 0) raw[i].load(x + r * ldx + c, n);
            else raw[i].zero();
        }
    }
    if constexpr ((MODE & BY_COLS) != 0) {
        constexpr int NW = sizeof(T) == 2 ? 4 : 8;  // words of eight columns' magnitudes
        uint32_t m[NW];
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            m[k] = 0;
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                if constexpr (sizeof(T) == 2) m[k] = mx4::absmax2<T>(m[k], raw[i].w[k]);
                else m[k] = max(m[k], raw[i].w[k] & 0x7fffffffu);
            }
            m[k] = mx4::max_of<T>(m[k], __shfl_xor_sync(0xffffffffu, m[k], 16));
        }
        if (lane < 16) {
            uint4 *d = reinterpret_cast<uint4 *>(&colmax[warp][lane * NW]);
#pragma unroll
            for (int k = 0; k < NW / 4; ++k) d[k] = make_uint4(m[4 * k], m[4 * k + 1], m[4 * k + 2], m[4 * k + 3]);
        }
        __syncthreads();
        if (tid < 128) {
            uint32_t v = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (sizeof(T) == 2)
                    v = max(v, (uint32_t) reinterpret_cast<const uint16_t *>(colmax[i])[tid]);
                else
                    v = max(v, colmax[i][tid]);
            }
            const uint32_t sc = scale_code(mx4::amax_bits<T>(v), TOP);
            colinv[tid] = inv_scale(sc);
            line[1][(tid & 31) * 4 + (tid >> 5)] = (uint8_t)sc;
        }
        __syncthreads();
    }
    float tile_inv = 1.f;
    if constexpr (MODE == BY_TILES) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < NR; ++i) m = mx4::max_of<T>(m, raw[i].amax());
        m = __reduce_max_sync(0xffffffffu, mx4::amax_bits<T>(m));
        if (lane == 0) colmax[0][warp] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, colmax[0][i]);
        const uint32_t sc = scale_code(m, TOP);
        tile_inv = inv_scale(sc);
        if (tid == 0) a.scales[blockIdx.x] = (uint8_t)sc;
    }
    float ci[8];
    if constexpr ((MODE & BY_COLS) != 0) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float4 q = reinterpret_cast<const float4 *>(colinv + cl)[k];
            ci[4 * k] = q.x, ci[4 * k + 1] = q.y, ci[4 * k + 2] = q.z, ci[4 * k + 3] = q.w;
        }
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int lr = ty + 16 * i;
        const int64_t r = r0 + lr;
        const bool live = r < rows && n > 0;
        float v[8];
        raw[i].floats(v);
        if constexpr (MODE == BY_TILES || (MODE & BY_ROWS) != 0) {
            float inv = tile_inv;
            if constexpr (MODE != BY_TILES) {
                uint32_t m = raw[i].amax();
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) m = mx4::max_of<T>(m, __shfl_xor_sync(0xffffffffu, m, o));
                const uint32_t sc = scale_code(mx4::amax_bits<T>(m), TOP);
                inv = inv_scale(sc);
                if ((lane & 15) == 0) line[0][(lr & 31) * 4 + (lr >> 5)] = (uint8_t)sc;
            }
            if (live && ACT_DCHECK(c + n <= a.ld))
                store_scaled8<FORMAT>(a.codes + r * a.ld + c, v, [&](int) { return make_float2(inv, inv); }, n);
        }
        if constexpr ((MODE & BY_COLS) != 0) {
            if (live && ACT_DCHECK(c + n <= b.ld))
                store_scaled8<FORMAT>(b.codes + r * b.ld + c, v,
                                      [&](int j) { return make_float2(ci[2 * j], ci[2 * j + 1]); }, n);
        }
    }
    if constexpr (MODE != BY_TILES) {
        __syncthreads();
        if ((MODE & BY_ROWS) != 0 && tid < 32)
            reinterpret_cast<uint32_t *>(a.scales + ((int64_t)kc * blocks_of(rows) + kr) * 128)[tid] =
                reinterpret_cast<const uint32_t *>(line[0])[tid];
        if ((MODE & BY_COLS) != 0 && tid >= 32 && tid < 64)
            reinterpret_cast<uint32_t *>(b.scales + ((int64_t)kr * ctiles + kc) * 128)[tid - 32] =
                reinterpret_cast<const uint32_t *>(line[1])[tid - 32];
    }
}

// The inverse in the same arrangement.
template <typename T, bool VEC, int FORMAT>
__global__ void __launch_bounds__(256)
    dequant_kernel(const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t cols, int64_t ld, int block, T *out,
                   int64_t ldo) {
    __shared__ __align__(16) float value[128];  // of the rows' or the columns' scales
    const int ctiles = (int)blocks_of(cols), kr = blockIdx.x / ctiles, kc = blockIdx.x - kr * ctiles;
    const int64_t r0 = (int64_t)kr * 128, c0 = (int64_t)kc * 128;
    const int tid = threadIdx.x, ty = tid >> 4, cl = (tid & 15) * 8;
    const int64_t c = c0 + cl;
    const int n = c >= cols ? 0 : (cols - c < 8 ? (int)(cols - c) : 8);
    uint2 q[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {  // rows are padded to 16 bytes: eight codes are always there
        const int64_t r = r0 + ty + 16 * i;
        q[i] = r < rows && n > 0 ? *reinterpret_cast<const uint2 *>(codes + r * ld + c) : make_uint2(0, 0);
    }
    if (tid < 128) {
        const int64_t at = block == TILES  ? blockIdx.x
                           : block == ROWS ? ((int64_t)kc * blocks_of(rows) + kr) * 128 + (tid & 31) * 4 + (tid >> 5)
                                           : ((int64_t)kr * ctiles + kc) * 128 + (tid & 31) * 4 + (tid >> 5);
        value[tid] = scale_value(scales[at]);
    }
    __syncthreads();
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = value[block == COLS ? cl + j : 0];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int lr = ty + 16 * i;
        const int64_t r = r0 + lr;
        if (r >= rows || n == 0) continue;
        if (block == ROWS) {
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] = value[lr];
        }
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = unpack2<FORMAT>((j < 2 ? q[i].x : q[i].y) >> (16 * (j & 1)));
            f[2 * j] = t.x * s[2 * j], f[2 * j + 1] = t.y * s[2 * j + 1];
        }
        uint32_t w[2 * sizeof(T)];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (sizeof(T) == 4) {
                w[2 * k] = __float_as_uint(f[2 * k]), w[2 * k + 1] = __float_as_uint(f[2 * k + 1]);
            } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                w[k] = pack_bf16x2(f[2 * k], f[2 * k + 1]);
            } else {
                const __half2 o = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
                memcpy(&w[k], &o, 4);
            }
        }
        T *d = out + r * ldo + c;
        if (!VEC) {
            extern __shared__ __align__(16) uint8_t dyn[];
            constexpr int PITCH = 128 + 16 / (int)sizeof(T);
            T *st = reinterpret_cast<T *>(dyn) + lr * PITCH + cl;
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k)
                reinterpret_cast<uint4 *>(st)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        } else if (n == 8 && ACT_DCHECK(c + 8 <= ldo)) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k)
                reinterpret_cast<uint4 *>(d)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k < n) {
                    if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t *>(d)[k] = w[k];
                    else reinterpret_cast<uint16_t *>(d)[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
                }
        }
    }
    if constexpr (!VEC) {  // neighbouring lanes neighbouring values
        extern __shared__ __align__(16) uint8_t dyn[];
        constexpr int PITCH = 128 + 16 / (int)sizeof(T);
        const T *st = reinterpret_cast<const T *>(dyn);
        const int lane = tid & 31, left = cols - c0 < 128 ? (int)(cols - c0) : 128;
        __syncthreads();
#pragma unroll 4
        for (int i = tid >> 5; i < 128 && r0 + i < rows; i += 8)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (32 * j + lane < left && ACT_DCHECK(c0 + 32 * j + lane < ldo))
                    out[(r0 + i) * ldo + c0 + 32 * j + lane] = st[i * PITCH + 32 * j + lane];
    }
}

// Shared memory of the forms that go through it.
template <typename T>
static constexpr int stage_bytes() {
    return 128 * (128 * (int)sizeof(T) + 16);
}

template <typename F>
static int with_type(int dtype, F f) {
    if (dtype == 0) return f(float{});
    if (dtype == 1) return f(__nv_bfloat16{});
    return f(__half{});
}

int check(const actcomp_fp8 *q) {
    ACT_CHECK(q && q->rows > 0 && q->cols > 0 && q->ld >= q->cols && q->codes && q->scales, ACT_E_INVALID);
    ACT_CHECK(q->format == E4M3 || q->format == E5M2, ACT_E_INVALID);
    ACT_CHECK(q->block >= ROWS && q->block <= TILES && (q->transposed == 0 || q->transposed == 1), ACT_E_INVALID);
    // the contraction of a product runs along the blocks
    ACT_CHECK(q->block != ROWS || !q->transposed, ACT_E_INVALID);
    ACT_CHECK(q->block != COLS || q->transposed, ACT_E_INVALID);
    ACT_CHECK(q->rows <= INT32_MAX - 255 && q->cols <= INT32_MAX - 255, ACT_E_UNSUPPORTED);
    ACT_CHECK(blocks_of(q->rows) * blocks_of(q->cols) <= INT32_MAX, ACT_E_UNSUPPORTED);
    ACT_CHECK(aligned(q->codes, 16) && aligned(q->scales, 16) && q->ld % 16 == 0, ACT_E_ALIGN);
    return ACT_OK;
}

}  // namespace fp8
}  // namespace act

extern "C" size_t actcomp_fp8_scale_bytes(int64_t rows, int64_t cols, int32_t block) {
    return rows > 0 && cols > 0 && block >= 0 && block <= 2 ? act::fp8::scale_bytes(rows, cols, block) : 0;
}

extern "C" int actcomp_fp8_quantize(const void *x, int64_t rows, int64_t cols, int64_t ldx, int32_t dtype,
                                    const actcomp_fp8 *q, const actcomp_fp8 *qt, void *stream) {
    using namespace act;
    using namespace act::fp8;
    ACT_CHECK(x && (q || qt) && rows > 0 && cols > 0 && ldx >= cols && dtype >= 0 && dtype <= 2, ACT_E_INVALID);
    for (const actcomp_fp8 *d : {q, qt}) {
        if (!d) continue;
        if (int st = check(d)) return st;
        ACT_CHECK(d->rows == rows && d->cols == cols, ACT_E_INVALID);
    }
    ACT_CHECK(!q || q->block != COLS, ACT_E_INVALID);
    ACT_CHECK(!qt || qt->block == COLS, ACT_E_INVALID);
    ACT_CHECK(!q || !qt || (q->block == ROWS && q->format == qt->format), ACT_E_INVALID);
    const int es = dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(x, es), ACT_E_ALIGN);
    const bool vec = aligned(x, 16) && (ldx * es) % 16 == 0;
    const int mode = q && qt ? BY_BOTH : qt ? BY_COLS : q->block == TILES ? BY_TILES : BY_ROWS;
    const unsigned grid = (unsigned)(blocks_of(rows) * blocks_of(cols));
    const Dst a = q ? Dst{q->codes, q->scales, q->ld} : Dst{}, b = qt ? Dst{qt->codes, qt->scales, qt->ld} : Dst{};
    cudaStream_t st = as_stream(stream);
    return with_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const int smem = vec ? 0 : stage_bytes<T>();
        auto go = [&](auto k) -> int {
            if (int rc = allow_smem(k, smem + 6 * 1024, stage_bytes<T>())) return rc;
            k<<<grid, 256, smem, st>>>(static_cast<const T *>(x), rows, cols, ldx, a, b);
            return launch_status();
        };
        auto pick = [&](auto fmt) -> int {
            constexpr int F = decltype(fmt)::value;
            if (mode == BY_ROWS) return vec ? go(quant_kernel<T, true, BY_ROWS, F>) : go(quant_kernel<T, false, BY_ROWS, F>);
            if (mode == BY_COLS) return vec ? go(quant_kernel<T, true, BY_COLS, F>) : go(quant_kernel<T, false, BY_COLS, F>);
            if (mode == BY_BOTH) return vec ? go(quant_kernel<T, true, BY_BOTH, F>) : go(quant_kernel<T, false, BY_BOTH, F>);
            return vec ? go(quant_kernel<T, true, BY_TILES, F>) : go(quant_kernel<T, false, BY_TILES, F>);
        };
        return (q ? q : qt)->format == E4M3 ? pick(std::integral_constant<int, E4M3>{})
                                            : pick(std::integral_constant<int, E5M2>{});
    });
}

extern "C" int actcomp_fp8_dequantize(const actcomp_fp8 *q, void *out, int64_t ldo, int32_t dtype, void *stream) {
    using namespace act;
    using namespace act::fp8;
    if (int st = check(q)) return st;
    ACT_CHECK(out && ldo >= q->cols && dtype >= 0 && dtype <= 2, ACT_E_INVALID);
    const int es = dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(out, es), ACT_E_ALIGN);
    const bool vec = aligned(out, 16) && (ldo * es) % 16 == 0;
    const unsigned grid = (unsigned)(blocks_of(q->rows) * blocks_of(q->cols));
    cudaStream_t st = as_stream(stream);
    return with_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const int smem = vec ? 0 : stage_bytes<T>();
        auto go = [&](auto k) -> int {
            if (int rc = allow_smem(k, smem, stage_bytes<T>())) return rc;
            k<<<grid, 256, smem, st>>>(q->codes, q->scales, q->rows, q->cols, q->ld, q->block, static_cast<T *>(out), ldo);
            return launch_status();
        };
        if (q->format == E4M3) return vec ? go(dequant_kernel<T, true, E4M3>) : go(dequant_kernel<T, false, E4M3>);
        return vec ? go(dequant_kernel<T, true, E5M2>) : go(dequant_kernel<T, false, E5M2>);
    });
}
