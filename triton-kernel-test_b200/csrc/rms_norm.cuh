// rms_norm.cuh -- root-mean-square norm of each row with the residual's addition, with
// an 8-bit output, and its backward pass (no reference counterpart: the
// reference's low_rank_system_profile_backward.py covers the linear layers between
// the norms).
//
//   forward    h = x (+ residual)
//              rstd = 1 / sqrt(sum h^2 / n + eps),  y = h * rstd * w
//              y rounded to the activations' type, or to 8 bits with one scale per
//              128 values of the row (fp8.cuh), the next linear layer's operand
//   backward   g = dy * w, xh = h * rstd
//              dx = rstd * (g - xh * sum(g xh) / n) (+ dh)
//              dw = sum over rows of dy * xh
//
// All arithmetic is float32 on values rounded once at the end; with a residual the
// unrounded float32 sum is normalised.  HBM-bound: each tensor crosses memory once.
// The work split is the layer norm's (rows.cuh): a row is held in registers by a warp
// or by a CTA's warps, eight values a lane in segments of 256, and arrives ahead of
// its use by bulk copies; persistent CTAs keep the weight and its gradient's sums in
// registers.  A block of 128 values is then half of a warp's segment, so that its
// largest magnitude takes four shuffles.  Longer rows than registers (16384 values)
// or ring slots hold are read twice.
//
// Measured on a B200, us (floor at the copy rate): 16384 x 4096 bf16
//   forward 42 (41), with the residual 86 (82), 8-bit 57 (31), 8-bit with the residual
//   77 (72), backward 67 (61), 84 with dh (82)
// and float32 94 (82), 188 (164), 66 (51), 142 (133), 128 (123), 140 (164, where dh
// was in L2).  The 8-bit form without a residual is held by its instructions (issue
// slots 61 %, ALU 55 % before its addresses left the loop: 63 us), ragged rows by two-byte
// accesses (16384 x 4097 bf16: 83, 137, 129, 176, 198, 238 us).  8192 x 11008 bf16 57 (55),
// 116 (110), 92 (41), 112 (96), 114 (83), 120 (110); 8192 x 16384 float32 backward 418
// (246): read twice.
#pragma once

#include "fp8.cuh"
#include "rows.cuh"

namespace act {
namespace norm {

// Resident CTAs that the kernels are compiled for, by the launch's threads rounded up.
__host__ __device__ constexpr int rms_ctas(int nch, int maxt) { return maxt > 256 ? 1 : (nch == 1 ? 3 : 2); }
__host__ __device__ constexpr int rms_bwd_ctas(int maxt) { return maxt > 256 ? 1 : 2; }

// ---------------------------------------------------------------- launches
// Segments per thread, warps per row, threads, rows a CTA has in hand, ring slots,
// shared memory and the resident CTAs that the kernel's template allows.
struct RmsShape {
    int nch, wpr, threads, rows_per_cta, depth, smem, per_sm;
};
static RmsShape rms_shape(int64_t cols, int esize, int inputs, bool bwd, bool vec, bool q8 = false) {
    const int segs = (int)((cols + SEG - 1) / SEG);
    RmsShape s{};
    if (bwd) {
        s.nch = segs <= 1 ? 1 : (segs <= 32 ? 2 : 4);
        s.wpr = (segs + s.nch - 1) / s.nch;
        s.rows_per_cta = s.wpr <= 4 ? 8 / s.wpr : 1;  // two or more
        s.threads = 32 * s.wpr * s.rows_per_cta;
        s.per_sm = rms_bwd_ctas(s.threads);
    } else if (segs <= 4) {
        s = {segs <= 1 ? 1 : (segs <= 2 ? 2 : 4), 1, 256, 8, 0, 0, 0};
    } else {
        // fewer, fuller warps spend less on a row's reductions
        const bool full = inputs == 1 && esize == 2 && !q8;
        s.nch = segs <= 8 ? (full ? 2 : 1) : segs <= 16 ? (full ? 4 : 2) : segs <= 24 ? 3 : 4;
        s.wpr = (segs + s.nch - 1) / s.nch;
        s.threads = 32 * s.wpr;
        s.rows_per_cta = 1;
    }
    if (!bwd) s.per_sm = rms_ctas(s.nch, s.threads) * (s.threads <= 128 ? 2 : 1);
    const int64_t slot = (int64_t)row_pitch(cols, esize, vec) * inputs * s.rows_per_cta;
    const int64_t room = SLOT_ROOM / s.per_sm;
    s.depth = (int)(room / slot < MAX_DEPTH ? room / slot : MAX_DEPTH);
    if (s.depth < 2) {  // the longest rows: one CTA per SM
        s.per_sm = 1;
        s.depth = (int)(SLOT_ROOM / slot < MAX_DEPTH ? SLOT_ROOM / slot : MAX_DEPTH);
    }
    s.smem = RING_HEAD + (int)(s.depth * slot);
    if (bwd && s.rows_per_cta > 1) {
        const int acc = RING_HEAD + (int)(s.rows_per_cta * cols * 4);
        if (acc > s.smem) s.smem = acc;
    }
    return s;
}
static int rms_grid(const RmsShape &s, int64_t rows) {
    const int64_t ctas = (rows + s.rows_per_cta - 1) / s.rows_per_cta, cap = (int64_t)num_sms() * s.per_sm;
    return (int)(ctas < cap ? ctas : cap);
}
// Rows that go through the re-reading kernels: more than the registers hold, or
// (backward) than leaves two ring slots in shared memory.
static bool rms_long(int64_t cols, int esize, int inputs, bool bwd) {
    if (cols > (int64_t)MAX_SEGS * SEG) return true;
    return bwd && 2 * (int64_t)row_pitch(cols, esize, false) * inputs > SLOT_ROOM;
}
// f(T tag, W tag) for the run-time types; wide: float32 weights.
template <typename F>
static int rms_types(int dtype, int wide, F f) {
    if (dtype == 0) return f(float{}, float{});
    if (dtype == 1) return wide ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
    return wide ? f(__half{}, float{}) : f(__half{}, __half{});
}
// 16-byte access to every row: base and row stride
static bool rows16(const void *p, int64_t ld, int esize) { return !p || (aligned(p, 16) && (ld * esize) % 16 == 0); }

// 1 / sqrt(v): the hardware's approximation and one Newton step whose correction is
// added in a fused multiply-add, within about half a unit in the last place (an 8-bit
// output changes its code where the values before it move across a tie).
__device__ __forceinline__ float rstd_of(float v) {
    const float r = rsqrtf(v), e = __fmaf_rn(-v * r, r, 1.f), h = __fmaf_rn(0.5f * r, e, r);
    return v > 0.f && v < INFINITY ? h : r;
}

// ---------------------------------------------------------------- forward
template <typename T, typename W>
struct RmsArgs {
    const T *x, *res;  // res may be null
    const W *w;        // may be null: 1
    T *y, *h;          // y: null for the 8-bit output; h: the sum, with res
    uint8_t *codes, *scales;
    float *rstd;
    int64_t rows, cols, ldx, ldr, ldy, ldh, ldc;
    float eps;
};

// The largest magnitude of a, b and m; NaN stays.
__device__ __forceinline__ float absmax3(float m, float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}
// A segment's values to codes (`codes`: the segment's first), and its two blocks' scales
// (`scales`: the first block's, `step` bytes on the second's).
template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t *codes, uint8_t *scales, int64_t step, int n, int lane, const F8 &v,
                                            int64_t left) {
    const float2 *p = v.p;
    if constexpr (VEC) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = absmax3(m, p[j].x, p[j].y);
        uint32_t u = fp8::mag(m);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) u = max(u, __shfl_xor_sync(0xffffffffu, u, o));
        const uint32_t sc = fp8::scale_code(u, 8);
        const float inv = fp8::inv_scale(sc);
        const float2 i2 = make_float2(inv, inv);
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = mul2(p[j], i2);
            h[j] = fp8::pack2<fp8::E4M3>(t.x, t.y);
        }
        if (n && ACT_DCHECK(8 * lane + 8 <= left)) {
            *reinterpret_cast<uint2 *>(codes + 8 * lane) =
                make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
            if ((lane & 15) == 0) scales[lane ? step : 0] = (uint8_t)sc;
        }
    } else {  // value 32 j + lane: block j / 4
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float m = absmax3(absmax3(0.f, p[2 * k].x, p[2 * k].y), p[2 * k + 1].x, p[2 * k + 1].y);
            const uint32_t sc = fp8::scale_code(__reduce_max_sync(0xffffffffu, fp8::mag(m)), 8);
            const float inv = fp8::inv_scale(sc);
#pragma unroll
            for (int j = 2 * k; j < 2 * k + 2; ++j) {
                const uint32_t c = fp8::pack2<fp8::E4M3>(p[j].x * inv, p[j].y * inv);
                if (2 * j < n && ACT_DCHECK(64 * j + lane < left)) codes[64 * j + lane] = (uint8_t)c;
                if (2 * j + 1 < n) codes[64 * j + 32 + lane] = (uint8_t)(c >> 8);
            }
            if (lane == 0 && 4 * k < n) scales[k ? step : 0] = (uint8_t)sc;
        }
    }
}

// NaN over a forward CTA's results (see RowRing); an 8-bit row becomes NaN by its scales.
template <typename T, typename W>
__device__ __noinline__ void rms_nan(const RmsArgs<T, W> &a, int wpr) {
    const Place p(wpr);
    if (a.y) nan_rows(a.y, a.ldy, p.r0, p.step, a.rows, a.cols, p.t, p.nt);
    if (a.res) nan_rows(a.h, a.ldh, p.r0, p.step, a.rows, a.cols, p.t, p.nt);
    nan_rows(a.rstd, 1, p.r0, p.step, a.rows, 1, p.t, p.nt);
    if (a.codes)
        for (int64_t r = p.r0; r < a.rows; r += p.step)
            for (int64_t b = p.t; b < fp8::blocks_of(a.cols); b += p.nt)
                a.scales[fp8::scale_at(r, b, fp8::blocks_of(a.rows))] = 255;
}

// MAXT: the launch's thread count rounded up to 256 or 512.  ONE: a warp per row,
// else a CTA.  Q: 8-bit output.
template <typename T, typename W, int NCH, int MAXT, bool VEC, bool RES, bool Q, bool ONE>
__global__ void __launch_bounds__(MAXT, rms_ctas(NCH, MAXT))
    rms_fwd_kernel(const __grid_constant__ RmsArgs<T, W> a, int warps, int depth) {
    const int wpr = ONE ? 1 : warps;
    extern __shared__ __align__(128) uint8_t dyn[];
    if constexpr (Q) tc::launch_dependents();  // the product that follows may set itself up
    constexpr int NW = MAXT / 32;
    // rows in hand at once: their reductions overlap and share their barriers
    constexpr int R = NCH <= 2 && sizeof(T) == 2 ? 2 : 1;
    __shared__ __align__(16) float red[2][R][NW];
    if (threadIdx.x < 2 * R * NW) red[0][0][threadIdx.x] = 0.f;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
    const int rpc = ONE ? nwarps : 1;
    const int w0 = ONE ? 0 : warp, mine = ONE ? warp : 0;
    const float inv_n = 1.f / (float)a.cols;
    const int64_t groups = fp8::blocks_of(a.rows), step8 = groups * fp8::BLOCK;  // from a block's scales to the next's
    constexpr int IN = RES ? 2 : 1;
    RowRing<T, IN, VEC> ring;
    const bool leader = ONE ? lane == 0 : threadIdx.x == 0;
    const int64_t r0 = (int64_t)blockIdx.x * rpc + mine, step = (int64_t)gridDim.x * rpc;
    auto fill = [&](int s, int64_t row) {
        if (row >= a.rows) return;
        const T *src[IN];
        src[0] = a.x + row * a.ldx;
        if constexpr (RES) src[1] = a.res + row * a.ldr;
        ring.fill(s, src);
    };
    ring.init(dyn, mine, (int)a.cols, depth, leader);
    if (leader)
        for (int i = 0; i < depth; ++i) fill(i, r0 + i * step);
    // the 8-bit form, which its instructions hold, keeps the weight as float32
    constexpr bool WIDE = Q && NCH <= 2;
    Raw8<W> wv[WIDE ? 1 : NCH];
    F8 wf[WIDE ? NCH : 1];
    int n[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int seg0 = (w0 + i * wpr) * SEG;
        n[i] = count_of<VEC>(seg0, a.cols, lane);
        const Raw8<W> raw = load8_or<W, VEC>(a.w, 1.f, seg0, n[i], lane);
        if constexpr (WIDE) wf[i] = unpack<W>(raw);
        else wv[i] = raw;
    }
    int turn = 0;
    for (int64_t r = r0; r < a.rows; r += R * step, ++turn) {
        F8 v[R][NCH];
        float s[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t rk = r + k * step;
            const bool live = k == 0 || rk < a.rows;  // the same for all that share the row
            float2 t = make_float2(0.f, 0.f);
            if (live) ring.wait(dyn, k);
            const RowView<T> xr = ring.view(0, a.x + rk * a.ldx, k);
            const RowView<T> rr = ring.view(IN - 1, RES ? a.res + rk * a.ldr : a.x + rk * a.ldx, k);
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int seg0 = (w0 + i * wpr) * SEG, nk = live ? n[i] : 0;
                v[k][i] = unpack<T>(load8<T, VEC>(xr, seg0, nk, lane));
                if constexpr (RES) {
                    const F8 res = unpack<T>(load8<T, VEC>(rr, seg0, nk, lane));
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[k][i].p[j] = add2(v[k][i].p[j], res.p[j]);
                    store8<T, VEC>(a.h + rk * a.ldh, seg0, nk, lane, v[k][i]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) t = fma2(v[k][i].p[j], v[k][i].p[j], t);  // 0 past the row's end
            }
            s[k] = t.x + t.y;
        }
        const bool go = leader && !*ring.abort_word(dyn);  // no wait has given up
        row_sums<NW, R, ONE>(s, red[turn & 1], warp, lane);
        // every reader of the slots is past its reads
        if (ONE) __syncwarp();
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if (go) fill(ring.slot, r + (depth + k) * step);
            ring.next();
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t rk = r + k * step;
            if (k > 0 && rk >= a.rows) break;
            const float rstd = rstd_of(__fmaf_rn(s[k], inv_n, a.eps));
            if (lane == 0 && w0 == 0) a.rstd[rk] = rstd;
            const float2 rstd2 = make_float2(rstd, rstd);
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int seg0 = (w0 + i * wpr) * SEG;
                F8 w;
                if constexpr (WIDE) {
                    w = wf[i];
                } else {
                    stay_packed(wv[i]);
                    w = unpack<W>(wv[i]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) v[k][i].p[j] = mul2(mul2(v[k][i].p[j], rstd2), w.p[j]);
                if constexpr (Q)
                    store_codes<VEC>(a.codes + rk * a.ldc + seg0, a.scales + fp8::scale_at(rk, 0, groups) + (seg0 >> 7) * step8,
                                     step8, n[i], lane, v[k][i], a.cols - seg0);
                else
                    store8<T, VEC>(a.y + rk * a.ldy, seg0, n[i], lane, v[k][i]);
            }
        }
    }
    if (ring.gave_up(dyn)) rms_nan<T, W>(a, ONE ? 1 : blockDim.x >> 5);
}

// Rows longer than MAX_SEGS segments: one CTA per row, two passes over it.
template <typename T, typename W, bool VEC, bool RES, bool Q>
__global__ void __launch_bounds__(LONG_THREADS) rms_fwd_long_kernel(RmsArgs<T, W> a) {
    constexpr int nw = LONG_THREADS / 32;
    __shared__ __align__(16) float red[2][nw];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inv_n = 1.f / (float)a.cols;
    const int64_t segs = (a.cols + SEG - 1) / SEG, groups = fp8::blocks_of(a.rows);
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
        auto fetch = [&](int64_t seg0, int n) {
            F8 v = unpack<T>(load8<T, VEC>(a.x + r * a.ldx, seg0, n, lane));
            if constexpr (RES) {
                const F8 res = unpack<T>(load8<T, VEC>(a.res + r * a.ldr, seg0, n, lane));
#pragma unroll
                for (int j = 0; j < 4; ++j) v.p[j] = add2(v.p[j], res.p[j]);
            }
            return v;
        };
        float s = 0.f;
        for (int64_t g = warp; g < segs; g += nw) {
            const F8 v = fetch(g * SEG, count_of<VEC>(g * SEG, a.cols, lane));
            float2 t = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 4; ++j) t = fma2(v.p[j], v.p[j], t);
            s += t.x + t.y;
        }
        // two sets of partial sums in turn: one barrier a row
        const float rstd = rstd_of(__fmaf_rn(row_sum<nw>(s, red + turn, warp, lane), inv_n, a.eps));
        if (threadIdx.x == 0) a.rstd[r] = rstd;
        const float2 rstd2 = make_float2(rstd, rstd);
        for (int64_t g = warp; g < segs; g += nw) {
            const int n = count_of<VEC>(g * SEG, a.cols, lane);
            F8 v = fetch(g * SEG, n);
            if constexpr (RES) store8<T, VEC>(a.h + r * a.ldh, g * SEG, n, lane, v);
            const F8 w = unpack<W>(load8_or<W, VEC>(a.w, 1.f, g * SEG, n, lane));
#pragma unroll
            for (int j = 0; j < 4; ++j) v.p[j] = mul2(mul2(v.p[j], rstd2), w.p[j]);
            if constexpr (Q)
                store_codes<VEC>(a.codes + r * a.ldc + g * SEG,
                                              a.scales + fp8::scale_at(r, 2 * g, groups), groups * fp8::BLOCK, n, lane, v,
                                              a.cols - g * SEG);
            else store8<T, VEC>(a.y + r * a.ldy, g * SEG, n, lane, v);
        }
    }
}

template <typename T, typename W>
static RmsArgs<T, W> rms_args(const actcomp_rms_args *g) {
    return {static_cast<const T *>(g->x), static_cast<const T *>(g->res), static_cast<const W *>(g->weight),
            static_cast<T *>(g->y), static_cast<T *>(g->h), g->codes, g->scales, g->rstd, g->rows, g->cols,
            g->ldx, g->ldr, g->ldy, g->ldh, g->ldc, g->eps};
}
// The launch of a forward form.
template <typename T, typename W, bool VEC, bool RES, bool Q>
static int rms_fwd_launch(const RmsArgs<T, W> &a, cudaStream_t st) {
    if (rms_long(a.cols, sizeof(T), RES ? 2 : 1, false)) {
        const int64_t cap = (int64_t)num_sms() * 4;
        rms_fwd_long_kernel<T, W, VEC, RES, Q><<<(int)(a.rows < cap ? a.rows : cap), LONG_THREADS, 0, st>>>(a);
        return launch_status();
    }
    const RmsShape s = rms_shape(a.cols, sizeof(T), RES ? 2 : 1, false, VEC, Q);
    auto go = [&](auto k) -> int {
        if (int rc = allow_smem(k, s.smem, MAX_SMEM)) return rc;
        k<<<rms_grid(s, a.rows), s.threads, s.smem, st>>>(a, s.wpr, s.depth);
        return launch_status();
    };
    if (s.wpr == 1) {
        if (s.nch == 1) return go(rms_fwd_kernel<T, W, 1, 256, VEC, RES, Q, true>);
        return s.nch == 2 ? go(rms_fwd_kernel<T, W, 2, 256, VEC, RES, Q, true>)
                          : go(rms_fwd_kernel<T, W, 4, 256, VEC, RES, Q, true>);
    }
    if constexpr (RES || Q || sizeof(T) == 4) {  // see rms_shape: the others take two segments
        if (s.nch == 1) return go(rms_fwd_kernel<T, W, 1, 256, VEC, RES, Q, false>);
    }
    if (s.nch == 2) return go(rms_fwd_kernel<T, W, 2, 256, VEC, RES, Q, false>);
    if (s.nch == 3) return go(rms_fwd_kernel<T, W, 3, 256, VEC, RES, Q, false>);
    return s.threads <= 256 ? go(rms_fwd_kernel<T, W, 4, 256, VEC, RES, Q, false>)
                            : go(rms_fwd_kernel<T, W, 4, 512, VEC, RES, Q, false>);
}

}  // namespace norm
}  // namespace act
