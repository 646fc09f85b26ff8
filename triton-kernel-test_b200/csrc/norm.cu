// norm.cu -- dropout without a stored mask, layer norm with its backward pass,
// and the two fused across a residual branch (no reference counterpart: the
// reference's low_rank_system_profile_backward.py covers the linear layers
// between them).
//
//   dropout    y = kept ? x * scale : 0                     (mask: philox.cuh)
//   forward    h = residual + dropout(x)                    (fused form only)
//              mean = sum h / n, rstd = 1 / sqrt(sum (h - mean)^2 / n + eps)
//              y = (h - mean) * rstd * w + b
//   backward   g = dy * w, xh = (h - mean) * rstd
//              dr = rstd * (g - sum g / n - xh * sum(g xh) / n) (+ dh)
//              dx = dropout(dr)                             (fused form only)
//              dw = sum over rows of dy * xh, db = sum over rows of dy
//
// All arithmetic is float32 on values rounded once at the end; the fused
// forward normalises the unrounded float32 h.  HBM-bound: each tensor crosses
// memory once.  A row's values stay in registers between the passes over it
// (mean, then squares about the mean, then the output), which also gives the
// variance without the cancellation of a sum of squares.
//
// Work split.  A warp holds a row in segments of 256 values, eight a lane: a
// lane's own eight consecutive values where 16-byte access is possible (VEC),
// else values lane, lane + 32, ... of the segment, so that narrow loads still
// coalesce; the lane then makes the generator call of block `lane` of the
// segment and the keep bits travel by shuffle.  Rows of up to 1024 values take
// a warp each, rows of up to 16384 a CTA each (both persistent: weights and
// the weight-gradient sums stay in registers from row to row); longer rows go
// through kernels that re-read the row.
#include <cuda_fp16.h>

#include "common.cuh"
#include "philox.cuh"

namespace act {
namespace norm {

constexpr int SEG = 256;            // values of a warp's segment
constexpr int MAX_SEGS = 64;        // longest row held in registers: 16384 values
constexpr int LONG_THREADS = 512;

// ---------------------------------------------------------------- types
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

// Eight values as they lie in memory.
template <typename T>
struct alignas(16) Raw8 {
    T v[8];
};

// A lane's eight values of the segment starting at `seg0` of a row of n values.
// VEC: values seg0 + 8 lane + j; else seg0 + 32 j + lane.
template <bool VEC>
__device__ __forceinline__ int64_t col_of(int64_t seg0, int lane, int j) {
    return VEC ? seg0 + 8 * lane + j : seg0 + 32 * j + lane;
}

template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load8(const T *row, int64_t seg0, int64_t n, int lane) {
    Raw8<T> r;
    if constexpr (VEC) {  // n is a multiple of 8
        const int64_t c = seg0 + 8 * lane;
        uint4 *d = reinterpret_cast<uint4 *>(&r);
        if (c < n) {
            const uint4 *s = reinterpret_cast<const uint4 *>(row + c);
#pragma unroll
            for (int i = 0; i < (int)sizeof(r) / 16; ++i) d[i] = s[i];
        } else {
#pragma unroll
            for (int i = 0; i < (int)sizeof(r) / 16; ++i) d[i] = make_uint4(0, 0, 0, 0);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t c = seg0 + 32 * j + lane;
            r.v[j] = c < n ? row[c] : from_f<T>(0.f);
        }
    }
    return r;
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T *row, int64_t seg0, int64_t n, int lane, const float (&f)[8]) {
    if constexpr (VEC) {
        const int64_t c = seg0 + 8 * lane;
        if (c >= n) return;
        Raw8<T> r;
#pragma unroll
        for (int j = 0; j < 8; ++j) r.v[j] = from_f<T>(f[j]);
        const uint4 *s = reinterpret_cast<const uint4 *>(&r);
        uint4 *d = reinterpret_cast<uint4 *>(row + c);
#pragma unroll
        for (int i = 0; i < (int)sizeof(r) / 16; ++i) d[i] = s[i];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t c = seg0 + 32 * j + lane;
            if (c < n) row[c] = from_f<T>(f[j]);
        }
    }
}

// Keep bits of the lane's eight values (bit j: its value j).  All lanes of the warp call it.
template <bool VEC>
__device__ __forceinline__ uint32_t keep_bits(uint64_t row, int64_t seg0, int lane, uint64_t key, uint32_t threshold) {
    const uint32_t mine = drop_keep8(row, (uint32_t)(seg0 >> 3) + lane, key, threshold);
    if constexpr (VEC) return mine;
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // value 32 j + lane belongs to block 4 j + lane / 8
        const uint32_t k = __shfl_sync(0xffffffffu, mine, 4 * j + (lane >> 3));
        bits |= ((k >> (lane & 7)) & 1u) << j;
    }
    return bits;
}

// ---------------------------------------------------------------- dropout
template <typename T>
struct DropArgs {
    const T *x;
    T *y;
    int64_t rows, cols, ldx, ldy;
    DropParams d;
};

// One warp per segment of 256 values, grid-stride over rows x segments.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(DropArgs<T> a) {
    const int lane = threadIdx.x & 31;
    const int64_t segs = (a.cols + SEG - 1) / SEG, total = a.rows * segs;
    const uint64_t key = drop_seed(a.d);
    const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5);
    for (int64_t i = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < total; i += step) {
        const int64_t r = i / segs, seg0 = (i - r * segs) * SEG;
        const Raw8<T> x = load8<T, VEC>(a.x + r * a.ldx, seg0, a.cols, lane);
        const uint32_t keep = keep_bits<VEC>(a.d.row_offset + (uint64_t)r, seg0, lane, key, a.d.threshold);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (keep >> j) & 1u ? to_f<T>(x.v[j]) * a.d.scale : 0.f;
        store8<T, VEC>(a.y + r * a.ldy, seg0, a.cols, lane, f);
    }
}

// ---------------------------------------------------------------- forward
template <typename T, typename W>
struct FwdArgs {
    const T *x, *res;
    const W *w, *b;  // either may be null: 1 and 0
    T *y, *h;
    float *mean, *rstd;
    int64_t rows, cols, ldx, ldr, ldy, ldh;
    float eps;
    DropParams d;
};

// Sum of v over the warps that share a row; every thread gets the same value.
__device__ __forceinline__ float row_sum(float v, float *red, int wpr, int warp, int lane) {
    v = warp_sum(v);
    if (wpr == 1) return v;
    if (lane == 0) red[warp] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < wpr; ++i) s += red[i];
    return s;
}

template <typename T, typename W, int NCH, bool VEC, bool DROP>
__global__ void __launch_bounds__(NCH == 4 ? 512 : 256) ln_fwd_kernel(FwdArgs<T, W> a, int wpr) {
    __shared__ float red[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
    const int rpc = wpr == 1 ? nwarps : 1;  // rows a CTA has in hand at once
    const int w0 = wpr == 1 ? 0 : warp;
    const float inv_n = 1.f / (float)a.cols;
    const uint64_t key = DROP ? drop_seed(a.d) : 0;
    Raw8<W> wv[NCH], bv[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int64_t seg0 = (int64_t)(w0 + i * wpr) * SEG;
        if (a.w) wv[i] = load8<W, VEC>(a.w, seg0, a.cols, lane);
        if (a.b) bv[i] = load8<W, VEC>(a.b, seg0, a.cols, lane);
    }
    for (int64_t r = (int64_t)blockIdx.x * rpc + (wpr == 1 ? warp : 0); r < a.rows; r += (int64_t)gridDim.x * rpc) {
        float v[NCH][8];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int64_t seg0 = (int64_t)(w0 + i * wpr) * SEG;
            const Raw8<T> x = load8<T, VEC>(a.x + r * a.ldx, seg0, a.cols, lane);
            if constexpr (DROP) {
                const Raw8<T> res = load8<T, VEC>(a.res + r * a.ldr, seg0, a.cols, lane);
                const uint32_t keep =
                    keep_bits<VEC>(a.d.row_offset + (uint64_t)r, seg0, lane, key, a.d.threshold);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[i][j] = (keep >> j) & 1u ? __fmaf_rn(to_f<T>(x.v[j]), a.d.scale, to_f<T>(res.v[j]))
                                               : to_f<T>(res.v[j]);
                store8<T, VEC>(a.h + r * a.ldh, seg0, a.cols, lane, v[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = to_f<T>(x.v[j]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[i][j];
        }
        const float mean = row_sum(s, red[0], wpr, warp, lane) * inv_n;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int64_t seg0 = (int64_t)(w0 + i * wpr) * SEG;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[i][j] -= mean;
                if (col_of<VEC>(seg0, lane, j) < a.cols) q = __fmaf_rn(v[i][j], v[i][j], q);
            }
        }
        const float var = row_sum(q, red[1], wpr, warp, lane) * inv_n;
        const float rstd = 1.f / sqrtf(var + a.eps);
        if (lane == 0 && w0 == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int64_t seg0 = (int64_t)(w0 + i * wpr) * SEG;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float xh = v[i][j] * rstd;
                v[i][j] = __fmaf_rn(xh, a.w ? to_f<W>(wv[i].v[j]) : 1.f, a.b ? to_f<W>(bv[i].v[j]) : 0.f);
            }
            store8<T, VEC>(a.y + r * a.ldy, seg0, a.cols, lane, v[i]);
        }
    }
}

// Rows longer than MAX_SEGS segments: one CTA per row, three passes over it
// (the later ones mostly from L2).
template <typename T, typename W, bool VEC, bool DROP>
__global__ void __launch_bounds__(LONG_THREADS) ln_fwd_long_kernel(FwdArgs<T, W> a) {
    __shared__ float red[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = LONG_THREADS / 32;
    const float inv_n = 1.f / (float)a.cols;
    const uint64_t key = DROP ? drop_seed(a.d) : 0;
    const int64_t segs = (a.cols + SEG - 1) / SEG;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        auto fetch = [&](int64_t seg0, float (&v)[8]) {
            const Raw8<T> x = load8<T, VEC>(a.x + r * a.ldx, seg0, a.cols, lane);
            if constexpr (DROP) {
                const Raw8<T> res = load8<T, VEC>(a.res + r * a.ldr, seg0, a.cols, lane);
                const uint32_t keep =
                    keep_bits<VEC>(a.d.row_offset + (uint64_t)r, seg0, lane, key, a.d.threshold);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[j] = (keep >> j) & 1u ? __fmaf_rn(to_f<T>(x.v[j]), a.d.scale, to_f<T>(res.v[j]))
                                            : to_f<T>(res.v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = to_f<T>(x.v[j]);
            }
        };
        float s = 0.f;
        for (int64_t g = warp; g < segs; g += nw) {
            float v[8], t = 0.f;
            fetch(g * SEG, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) t += v[j];
            s += t;
        }
        const float mean = row_sum(s, red[0], nw, warp, lane) * inv_n;
        float q = 0.f;
        for (int64_t g = warp; g < segs; g += nw) {
            float v[8], t = 0.f;
            fetch(g * SEG, v);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (col_of<VEC>(g * SEG, lane, j) < a.cols) t = __fmaf_rn(v[j] - mean, v[j] - mean, t);
            q += t;
        }
        const float var = row_sum(q, red[1], nw, warp, lane) * inv_n;
        const float rstd = 1.f / sqrtf(var + a.eps);
        if (threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        for (int64_t g = warp; g < segs; g += nw) {
            float v[8];
            fetch(g * SEG, v);
            if constexpr (DROP) store8<T, VEC>(a.h + r * a.ldh, g * SEG, a.cols, lane, v);
            Raw8<W> wv, bv;
            if (a.w) wv = load8<W, VEC>(a.w, g * SEG, a.cols, lane);
            if (a.b) bv = load8<W, VEC>(a.b, g * SEG, a.cols, lane);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[j] = __fmaf_rn((v[j] - mean) * rstd, a.w ? to_f<W>(wv.v[j]) : 1.f, a.b ? to_f<W>(bv.v[j]) : 0.f);
            store8<T, VEC>(a.y + r * a.ldy, g * SEG, a.cols, lane, v);
        }
    }
}

// ---------------------------------------------------------------- backward
template <typename T, typename W>
struct BwdArgs {
    const T *dy, *x, *dh;  // x: the normalised input (h in the fused form); dh may be null
    const W *w;            // may be null: 1
    const float *mean, *rstd;
    T *dx, *dr;            // dr: the fused form's residual gradient (dx is then its dropout)
    float *part;           // partial weight gradients, grid x 2 x cols; null if none are wanted
    int64_t rows, cols, lddy, ldx, lddh, lddx, lddr;
    DropParams d;
};

__device__ __forceinline__ float2 row_sum2(float u, float v, float2 *red, int wpr, int warp, int lane) {
    u = warp_sum(u);
    v = warp_sum(v);
    if (wpr == 1) return make_float2(u, v);
    if (lane == 0) red[warp] = make_float2(u, v);
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
    for (int i = 0; i < wpr; ++i) {
        s.x += red[i].x;
        s.y += red[i].y;
    }
    return s;
}

template <typename T, typename W, int NCH, bool VEC, bool DROP>
__global__ void __launch_bounds__(NCH == 4 ? 512 : 256) ln_bwd_kernel(BwdArgs<T, W> a, int wpr) {
    __shared__ float2 red[2][32];
    extern __shared__ float acc_s[];  // wpr == 1: nwarps x 2 x cols, the warps' sums
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
    const int rpc = wpr == 1 ? nwarps : 1;
    const int w0 = wpr == 1 ? 0 : warp;
    const float inv_n = 1.f / (float)a.cols;
    const uint64_t key = DROP ? drop_seed(a.d) : 0;
    Raw8<W> wv[NCH];
    float dw[NCH][8], db[NCH][8];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        if (a.w) wv[i] = load8<W, VEC>(a.w, (int64_t)(w0 + i * wpr) * SEG, a.cols, lane);
#pragma unroll
        for (int j = 0; j < 8; ++j) dw[i][j] = db[i][j] = 0.f;
    }
    int turn = 0;
    for (int64_t r = (int64_t)blockIdx.x * rpc + (wpr == 1 ? warp : 0); r < a.rows; r += (int64_t)gridDim.x * rpc) {
        const float mean = a.mean[r], rstd = a.rstd[r];
        float g[NCH][8], xh[NCH][8];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int64_t seg0 = (int64_t)(w0 + i * wpr) * SEG;
            const Raw8<T> y = load8<T, VEC>(a.dy + r * a.lddy, seg0, a.cols, lane);
            const Raw8<T> x = load8<T, VEC>(a.x + r * a.ldx, seg0, a.cols, lane);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float dy = to_f<T>(y.v[j]);
                const bool in = col_of<VEC>(seg0, lane, j) < a.cols;
                xh[i][j] = in ? (to_f<T>(x.v[j]) - mean) * rstd : 0.f;
                dw[i][j] = __fmaf_rn(dy, xh[i][j], dw[i][j]);
                db[i][j] += dy;
                g[i][j] = a.w ? dy * to_f<W>(wv[i].v[j]) : dy;
                s1 += g[i][j];
                s2 = __fmaf_rn(g[i][j], xh[i][j], s2);
            }
        }
        const float2 s = row_sum2(s1, s2, red[turn], wpr, warp, lane);
        turn ^= 1;
        const float m1 = s.x * inv_n, m2 = s.y * inv_n;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int64_t seg0 = (int64_t)(w0 + i * wpr) * SEG;
#pragma unroll
            for (int j = 0; j < 8; ++j) g[i][j] = rstd * (g[i][j] - __fmaf_rn(xh[i][j], m2, m1));
            if constexpr (DROP) {
                if (a.dh) {
                    const Raw8<T> dh = load8<T, VEC>(a.dh + r * a.lddh, seg0, a.cols, lane);
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[i][j] += to_f<T>(dh.v[j]);
                }
                store8<T, VEC>(a.dr + r * a.lddr, seg0, a.cols, lane, g[i]);
                const uint32_t keep =
                    keep_bits<VEC>(a.d.row_offset + (uint64_t)r, seg0, lane, key, a.d.threshold);
#pragma unroll
                for (int j = 0; j < 8; ++j) g[i][j] = (keep >> j) & 1u ? g[i][j] * a.d.scale : 0.f;
            }
            store8<T, VEC>(a.dx + r * a.lddx, seg0, a.cols, lane, g[i]);
        }
    }
    if (!a.part) return;
    float *part = a.part + (int64_t)blockIdx.x * 2 * a.cols;
    if (wpr != 1) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int64_t seg0 = (int64_t)(w0 + i * wpr) * SEG;
            store8<float, VEC>(part, seg0, a.cols, lane, dw[i]);
            store8<float, VEC>(part + a.cols, seg0, a.cols, lane, db[i]);
        }
        return;
    }
    float *mine = acc_s + (int64_t)warp * 2 * a.cols;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int64_t seg0 = (int64_t)i * SEG;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t c = col_of<VEC>(seg0, lane, j);
            if (c < a.cols) {
                mine[c] = dw[i][j];
                mine[a.cols + c] = db[i][j];
            }
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.cols; c += blockDim.x) {
        float s = 0.f;
        for (int i = 0; i < nwarps; ++i) s += acc_s[(int64_t)i * 2 * a.cols + c];
        part[c] = s;
    }
}

// Rows longer than MAX_SEGS segments, first kernel: the row's two sums.
template <typename T, typename W, bool VEC>
__global__ void __launch_bounds__(LONG_THREADS) ln_bwd_sums_kernel(BwdArgs<T, W> a, float2 *sums) {
    __shared__ float2 red[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = LONG_THREADS / 32;
    const float inv_n = 1.f / (float)a.cols;
    const int64_t segs = (a.cols + SEG - 1) / SEG;
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int64_t sg = warp; sg < segs; sg += nw) {
            const Raw8<T> y = load8<T, VEC>(a.dy + r * a.lddy, sg * SEG, a.cols, lane);
            const Raw8<T> x = load8<T, VEC>(a.x + r * a.ldx, sg * SEG, a.cols, lane);
            Raw8<W> wv;
            if (a.w) wv = load8<W, VEC>(a.w, sg * SEG, a.cols, lane);
            float t1 = 0.f, t2 = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float g = to_f<T>(y.v[j]) * (a.w ? to_f<W>(wv.v[j]) : 1.f);
                if (col_of<VEC>(sg * SEG, lane, j) < a.cols) {
                    t1 += g;
                    t2 = __fmaf_rn(g, (to_f<T>(x.v[j]) - mean) * rstd, t2);
                }
            }
            s1 += t1;
            s2 += t2;
        }
        const float2 s = row_sum2(s1, s2, red[turn], nw, warp, lane);
        turn ^= 1;
        if (threadIdx.x == 0) sums[r] = make_float2(s.x * inv_n, s.y * inv_n);
    }
}

// Second kernel: a warp takes one segment of columns over its share of the
// rows (blockIdx.y of gridDim.y).
template <typename T, typename W, bool VEC, bool DROP>
__global__ void __launch_bounds__(128) ln_bwd_cols_kernel(BwdArgs<T, W> a, const float2 *sums) {
    const int lane = threadIdx.x & 31;
    const int64_t seg0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * SEG;
    if (seg0 >= a.cols) return;
    const uint64_t key = DROP ? drop_seed(a.d) : 0;
    Raw8<W> wv;
    if (a.w) wv = load8<W, VEC>(a.w, seg0, a.cols, lane);
    float dw[8] = {}, db[8] = {};
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float mean = a.mean[r], rstd = a.rstd[r];
        const float2 m = sums[r];
        const Raw8<T> y = load8<T, VEC>(a.dy + r * a.lddy, seg0, a.cols, lane);
        const Raw8<T> x = load8<T, VEC>(a.x + r * a.ldx, seg0, a.cols, lane);
        float g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float dy = to_f<T>(y.v[j]), xh = (to_f<T>(x.v[j]) - mean) * rstd;
            if (col_of<VEC>(seg0, lane, j) < a.cols) dw[j] = __fmaf_rn(dy, xh, dw[j]);
            db[j] += dy;
            g[j] = rstd * ((a.w ? dy * to_f<W>(wv.v[j]) : dy) - __fmaf_rn(xh, m.y, m.x));
        }
        if constexpr (DROP) {
            if (a.dh) {
                const Raw8<T> dh = load8<T, VEC>(a.dh + r * a.lddh, seg0, a.cols, lane);
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] += to_f<T>(dh.v[j]);
            }
            store8<T, VEC>(a.dr + r * a.lddr, seg0, a.cols, lane, g);
            const uint32_t keep = keep_bits<VEC>(a.d.row_offset + (uint64_t)r, seg0, lane, key, a.d.threshold);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = (keep >> j) & 1u ? g[j] * a.d.scale : 0.f;
        }
        store8<T, VEC>(a.dx + r * a.lddx, seg0, a.cols, lane, g);
    }
    if (!a.part) return;
    float *part = a.part + (int64_t)blockIdx.y * 2 * a.cols;
    store8<float, VEC>(part, seg0, a.cols, lane, dw);
    store8<float, VEC>(part + a.cols, seg0, a.cols, lane, db);
}

// dw / db from the `parts` partial sums, in their order: a column's sum does
// not depend on timing.  A warp takes 32 columns, the CTA's eight warps every
// eighth partial.
template <typename W>
__global__ void __launch_bounds__(256) ln_bwd_finish_kernel(const float *part, int parts, int64_t cols, W *dw, W *db) {
    __shared__ float red[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;  // of 2 * cols
    float s = 0.f;
    if (c < 2 * cols)
        for (int i = warp; i < parts; i += 8) s += part[(int64_t)i * 2 * cols + c];
    red[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < 2 * cols) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += red[i][lane];
        if (c < cols) {
            if (dw) dw[c] = from_f<W>(s);
        } else if (db) {
            db[c - cols] = from_f<W>(s);
        }
    }
}

// ---------------------------------------------------------------- launches
struct Shape {
    int nch, wpr, threads, rows_per_cta;
};
// Segments per thread and warps per row.
static Shape shape_of(int64_t cols) {
    const int segs = (int)((cols + SEG - 1) / SEG);
    if (segs <= 4) return {segs <= 1 ? 1 : (segs <= 2 ? 2 : 4), 1, 256, 8};
    const int nch = segs <= 16 ? 2 : 4;
    const int wpr = (segs + nch - 1) / nch;
    return {nch, wpr, 32 * wpr, 1};
}
static int grid_of(const Shape &s, int64_t rows) {
    const int64_t ctas = (rows + s.rows_per_cta - 1) / s.rows_per_cta;
    const int per_sm = 1024 / s.threads < 1 ? 1 : 1024 / s.threads;
    const int64_t cap = (int64_t)num_sms() * per_sm;
    return (int)(ctas < cap ? ctas : cap);
}
static int long_parts(int64_t rows, int64_t cols) {
    const int64_t x = (cols + 4 * SEG - 1) / (4 * SEG);
    int64_t y = ((int64_t)num_sms() * 12 + x - 1) / x;
    if (y > rows) y = rows;
    return (int)(y < 1 ? 1 : (y > 65535 ? 65535 : y));
}
static bool is_long(int64_t cols) { return cols > (int64_t)MAX_SEGS * SEG; }
static size_t up256(size_t b) { return (b + 255) / 256 * 256; }

static size_t bwd_workspace(int64_t rows, int64_t cols) {
    if (is_long(cols)) return up256((size_t)long_parts(rows, cols) * 2 * cols * 4) + up256((size_t)rows * 8);
    return up256((size_t)grid_of(shape_of(cols), rows) * 2 * cols * 4);
}

template <typename T, typename W, bool VEC, bool DROP>
static int fwd_launch(const FwdArgs<T, W> &a, cudaStream_t st) {
    if (is_long(a.cols)) {
        const int64_t cap = (int64_t)num_sms() * 4;
        ln_fwd_long_kernel<T, W, VEC, DROP><<<(int)(a.rows < cap ? a.rows : cap), LONG_THREADS, 0, st>>>(a);
        return launch_status();
    }
    const Shape s = shape_of(a.cols);
    const int grid = grid_of(s, a.rows);
    if (s.nch == 1) ln_fwd_kernel<T, W, 1, VEC, DROP><<<grid, s.threads, 0, st>>>(a, s.wpr);
    else if (s.nch == 2) ln_fwd_kernel<T, W, 2, VEC, DROP><<<grid, s.threads, 0, st>>>(a, s.wpr);
    else ln_fwd_kernel<T, W, 4, VEC, DROP><<<grid, s.threads, 0, st>>>(a, s.wpr);
    return launch_status();
}

template <typename T, typename W, int NCH, bool VEC, bool DROP>
static int bwd_main(const BwdArgs<T, W> &a, const Shape &s, int grid, cudaStream_t st) {
    auto k = ln_bwd_kernel<T, W, NCH, VEC, DROP>;
    const int smem = s.wpr == 1 && a.part ? (int)(s.rows_per_cta * 2 * a.cols * 4) : 0;
    if (smem > 48 * 1024) ACT_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    k<<<grid, s.threads, smem, st>>>(a, s.wpr);
    return launch_status();
}

template <typename T, typename W, bool VEC, bool DROP>
static int bwd_launch(BwdArgs<T, W> a, W *dw, W *db, void *ws, cudaStream_t st) {
    int parts, rc;
    a.part = dw || db ? static_cast<float *>(ws) : nullptr;
    if (is_long(a.cols)) {
        parts = long_parts(a.rows, a.cols);
        float2 *sums = reinterpret_cast<float2 *>(static_cast<uint8_t *>(ws) + up256((size_t)parts * 2 * a.cols * 4));
        const int64_t cap = (int64_t)num_sms() * 4;
        ln_bwd_sums_kernel<T, W, VEC><<<(int)(a.rows < cap ? a.rows : cap), LONG_THREADS, 0, st>>>(a, sums);
        const dim3 grid((unsigned)((a.cols + 4 * SEG - 1) / (4 * SEG)), (unsigned)parts);
        ln_bwd_cols_kernel<T, W, VEC, DROP><<<grid, 128, 0, st>>>(a, sums);
        rc = launch_status();
    } else {
        const Shape s = shape_of(a.cols);
        parts = grid_of(s, a.rows);
        rc = s.nch == 1   ? bwd_main<T, W, 1, VEC, DROP>(a, s, parts, st)
             : s.nch == 2 ? bwd_main<T, W, 2, VEC, DROP>(a, s, parts, st)
                          : bwd_main<T, W, 4, VEC, DROP>(a, s, parts, st);
    }
    if (rc || !a.part) return rc;
    ln_bwd_finish_kernel<W><<<(unsigned)((2 * a.cols + 31) / 32), 256, 0, st>>>(a.part, parts, a.cols, dw, db);
    return launch_status();
}

// f(T tag, W tag) for the run-time types; wide: float32 weights.
template <typename F>
static int with_types(int dtype, int wide, F f) {
    if (dtype == 0) return f(float{}, float{});
    if (dtype == 1) return wide ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
    return wide ? f(__half{}, float{}) : f(__half{}, __half{});
}

static bool drop_params(DropParams &d, uint64_t seed, const uint64_t *seed_ptr, uint64_t row_offset, double p) {
    if (!(p >= 0.0 && p <= 1.0)) return false;
    d.seed = seed;
    d.seed_ptr = seed_ptr;
    d.row_offset = row_offset;
    d.threshold = (uint32_t)__builtin_rint(p * 65536.0);
    d.scale = d.threshold < 65536u ? (float)(65536.0 / (65536.0 - (double)d.threshold)) : 0.f;
    return true;
}

// 16-byte access to every row: base and row stride
static bool vec_ok(const void *p, int64_t ld, int esize) { return !p || (aligned(p, 16) && (ld * esize) % 16 == 0); }

}  // namespace norm
}  // namespace act

extern "C" int actcomp_dropout(const actcomp_drop_args *g, void *stream) {
    using namespace act;
    using namespace act::norm;
    ACT_CHECK(g && g->rows >= 0 && g->cols >= 0, ACT_E_INVALID);
    ACT_CHECK(g->dtype >= 0 && g->dtype <= 2, ACT_E_INVALID);
    DropParams d;
    ACT_CHECK(drop_params(d, g->seed, g->seed_ptr, g->row_offset, g->p), ACT_E_INVALID);
    if (g->rows == 0 || g->cols == 0) return ACT_OK;
    ACT_CHECK(g->x && g->y && g->ldx >= g->cols && g->ldy >= g->cols, ACT_E_INVALID);
    ACT_CHECK(g->cols <= ((int64_t)1 << 34) && g->rows <= ((int64_t)1 << 40), ACT_E_UNSUPPORTED);
    const int es = g->dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(g->x, es) && aligned(g->y, es) && aligned(g->seed_ptr, 8), ACT_E_ALIGN);
    const bool vec = g->cols % 8 == 0 && vec_ok(g->x, g->ldx, es) && vec_ok(g->y, g->ldy, es);
    const int64_t warps = g->rows * ((g->cols + SEG - 1) / SEG);
    const int64_t cap = (int64_t)num_sms() * 16, ctas = (warps + 7) / 8;
    const int grid = (int)(ctas < cap ? ctas : cap);
    cudaStream_t st = as_stream(stream);
    return with_types(g->dtype, 0, [&](auto t, auto) {
        using T = decltype(t);
        DropArgs<T> a{static_cast<const T *>(g->x), static_cast<T *>(g->y), g->rows, g->cols, g->ldx, g->ldy, d};
        if (vec) dropout_kernel<T, true><<<grid, 256, 0, st>>>(a);
        else dropout_kernel<T, false><<<grid, 256, 0, st>>>(a);
        return launch_status();
    });
}

extern "C" int actcomp_layer_norm(const actcomp_ln_args *g, void *stream) {
    using namespace act;
    using namespace act::norm;
    ACT_CHECK(g && g->rows >= 0 && g->cols > 0, ACT_E_INVALID);
    ACT_CHECK(g->dtype >= 0 && g->dtype <= 2 && (g->wdtype == g->dtype || g->wdtype == 0), ACT_E_INVALID);
    const bool drop = g->res != nullptr;
    DropParams d{};
    if (drop) ACT_CHECK(drop_params(d, g->seed, g->seed_ptr, g->row_offset, g->p), ACT_E_INVALID);
    ACT_CHECK(g->eps >= 0.f, ACT_E_INVALID);
    if (g->rows == 0) return ACT_OK;
    ACT_CHECK(g->x && g->y && g->mean && g->rstd, ACT_E_INVALID);
    ACT_CHECK(g->ldx >= g->cols && g->ldy >= g->cols, ACT_E_INVALID);
    ACT_CHECK(!drop || (g->h && g->ldr >= g->cols && g->ldh >= g->cols), ACT_E_INVALID);
    ACT_CHECK(g->cols <= ((int64_t)1 << 30) && g->rows <= ((int64_t)1 << 40), ACT_E_UNSUPPORTED);
    const int es = g->dtype == 0 ? 4 : 2, ws = g->wdtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(g->x, es) && aligned(g->y, es) && aligned(g->res, es) && aligned(g->h, es), ACT_E_ALIGN);
    ACT_CHECK(aligned(g->weight, ws) && aligned(g->bias, ws) && aligned(g->mean, 4) && aligned(g->rstd, 4) &&
                  aligned(g->seed_ptr, 8),
              ACT_E_ALIGN);
    const bool vec = g->cols % 8 == 0 && vec_ok(g->x, g->ldx, es) && vec_ok(g->y, g->ldy, es) &&
                     vec_ok(g->res, g->ldr, es) && vec_ok(g->h, g->ldh, es) && aligned(g->weight, 16) &&
                     aligned(g->bias, 16);
    cudaStream_t st = as_stream(stream);
    return with_types(g->dtype, g->wdtype == 0, [&](auto t, auto w) {
        using T = decltype(t);
        using W = decltype(w);
        FwdArgs<T, W> a{static_cast<const T *>(g->x), static_cast<const T *>(g->res), static_cast<const W *>(g->weight),
                        static_cast<const W *>(g->bias), static_cast<T *>(g->y), static_cast<T *>(g->h), g->mean,
                        g->rstd, g->rows, g->cols, g->ldx, g->ldr, g->ldy, g->ldh, g->eps, d};
        if (drop) return vec ? fwd_launch<T, W, true, true>(a, st) : fwd_launch<T, W, false, true>(a, st);
        return vec ? fwd_launch<T, W, true, false>(a, st) : fwd_launch<T, W, false, false>(a, st);
    });
}

extern "C" size_t actcomp_layer_norm_bwd_workspace(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 ? act::norm::bwd_workspace(rows, cols) : 0;
}

extern "C" int actcomp_layer_norm_bwd(const actcomp_ln_bwd_args *g, void *workspace, size_t workspace_bytes,
                                      void *stream) {
    using namespace act;
    using namespace act::norm;
    ACT_CHECK(g && g->rows >= 0 && g->cols > 0, ACT_E_INVALID);
    ACT_CHECK(g->dtype >= 0 && g->dtype <= 2 && (g->wdtype == g->dtype || g->wdtype == 0), ACT_E_INVALID);
    const bool drop = g->dr != nullptr;
    DropParams d{};
    if (drop) ACT_CHECK(drop_params(d, g->seed, g->seed_ptr, g->row_offset, g->p), ACT_E_INVALID);
    const int es = g->dtype == 0 ? 4 : 2, wsz = g->wdtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(g->dweight, wsz) && aligned(g->dbias, wsz), ACT_E_ALIGN);
    cudaStream_t st = as_stream(stream);
    if (g->rows == 0) {  // the sums over no rows
        if (g->dweight) ACT_CUDA_TRY(cudaMemsetAsync(g->dweight, 0, (size_t)g->cols * wsz, st));
        if (g->dbias) ACT_CUDA_TRY(cudaMemsetAsync(g->dbias, 0, (size_t)g->cols * wsz, st));
        return ACT_OK;
    }
    ACT_CHECK(g->dy && g->x && g->dx && g->mean && g->rstd, ACT_E_INVALID);
    ACT_CHECK(g->lddy >= g->cols && g->ldx >= g->cols && g->lddx >= g->cols, ACT_E_INVALID);
    ACT_CHECK(!drop || g->lddr >= g->cols, ACT_E_INVALID);
    ACT_CHECK(!g->dh || (drop && g->lddh >= g->cols), ACT_E_INVALID);
    ACT_CHECK(g->cols <= ((int64_t)1 << 30) && g->rows <= ((int64_t)1 << 40), ACT_E_UNSUPPORTED);
    ACT_CHECK(aligned(g->dy, es) && aligned(g->x, es) && aligned(g->dx, es) && aligned(g->dr, es) && aligned(g->dh, es),
              ACT_E_ALIGN);
    ACT_CHECK(aligned(g->weight, wsz) && aligned(g->mean, 4) && aligned(g->rstd, 4) && aligned(g->seed_ptr, 8),
              ACT_E_ALIGN);
    ACT_CHECK(workspace && aligned(workspace, 16) && workspace_bytes >= bwd_workspace(g->rows, g->cols),
              ACT_E_WORKSPACE);
    const bool vec = g->cols % 8 == 0 && vec_ok(g->dy, g->lddy, es) && vec_ok(g->x, g->ldx, es) &&
                     vec_ok(g->dh, g->lddh, es) && vec_ok(g->dx, g->lddx, es) && vec_ok(g->dr, g->lddr, es) &&
                     aligned(g->weight, 16);
    return with_types(g->dtype, g->wdtype == 0, [&](auto t, auto w) {
        using T = decltype(t);
        using W = decltype(w);
        BwdArgs<T, W> a{static_cast<const T *>(g->dy), static_cast<const T *>(g->x), static_cast<const T *>(g->dh),
                        static_cast<const W *>(g->weight), g->mean, g->rstd, static_cast<T *>(g->dx),
                        static_cast<T *>(g->dr), nullptr, g->rows, g->cols, g->lddy, g->ldx, g->lddh, g->lddx, g->lddr,
                        d};
        W *dw = static_cast<W *>(g->dweight), *db = static_cast<W *>(g->dbias);
        if (drop)
            return vec ? bwd_launch<T, W, true, true>(a, dw, db, workspace, st)
                       : bwd_launch<T, W, false, true>(a, dw, db, workspace, st);
        return vec ? bwd_launch<T, W, true, false>(a, dw, db, workspace, st)
                   : bwd_launch<T, W, false, false>(a, dw, db, workspace, st);
    });
}
