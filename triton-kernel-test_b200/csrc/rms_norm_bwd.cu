// rms_norm_bwd.cu -- the backward pass of the root-mean-square norm (the mathematics
// and the work split: rms_norm.cuh).
#include "rms_norm.cuh"

namespace act {
namespace norm {

template <typename T, typename W>
struct RmsBwdArgs {
    const T *dy, *x, *dh;  // x: the normalised input (the sum, with a residual); dh may be null
    const W *w;            // may be null: 1
    const float *rstd;
    T *dx;
    float *part;           // partial weight gradients, grid x cols; null if none is wanted
    int64_t rows, cols, lddy, ldx, lddh, lddx;
};

// Sum of v over the warps that share a row (`w0`: this one's place).  red: NW entries,
// zero where there is no warp.  MULTI: several groups of warps share the CTA, each
// with four entries.
template <int NW, bool MULTI>
__device__ __forceinline__ float group_sum(float v, float *red, int wpr, int group, int w0, int lane) {
    v = warp_sum(v);
    if (MULTI && wpr == 1) return v;
    if (MULTI) red += group * 4;
    if (lane == 0) red[w0] = v;
    if (MULTI) tc::named_bar(1 + group, 32 * wpr);
    else __syncthreads();
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < (MULTI ? 1 : NW / 4); ++i) {
        const float4 q = reinterpret_cast<const float4 *>(red)[i];
        s = add2(add2(s, make_float2(q.x, q.y)), make_float2(q.z, q.w));
    }
    return s.x + s.y;
}

template <typename T, typename W>
__device__ __noinline__ void rms_bwd_nan(const RmsBwdArgs<T, W> &a, int wpr) {
    const Place p(wpr);
    nan_rows(a.dx, a.lddx, p.r0, p.step, a.rows, a.cols, p.t, p.nt);
    if (a.part) nan_rows(a.part, a.cols, blockIdx.x, gridDim.x, gridDim.x, a.cols, threadIdx.x, blockDim.x);
}

// MULTI: a CTA has several rows in hand, each a group of `wpr` warps; else one.  DH:
// dh is added.
template <typename T, typename W, int NCH, int MAXT, bool VEC, bool DH, bool MULTI>
__global__ void __launch_bounds__(MAXT, rms_bwd_ctas(MAXT))
    rms_bwd_kernel(const __grid_constant__ RmsBwdArgs<T, W> a, int wpr, int depth) {
    constexpr int NW = MAXT / 32;
    __shared__ __align__(16) float red[2][MULTI ? 4 * NW : NW];
    for (int i = threadIdx.x; i < (int)(sizeof(red) / 4); i += blockDim.x) red[0][i] = 0.f;
    __syncthreads();
    extern __shared__ __align__(128) uint8_t dyn[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
    const int rpc = MULTI ? nwarps / wpr : 1;
    const int mine = MULTI ? warp / wpr : 0, w0 = warp - mine * wpr;
    const float inv_n = 1.f / (float)a.cols;
    constexpr int IN = DH ? 3 : 2;
    RowRing<T, IN, VEC> ring;
    const bool leader = w0 == 0 && lane == 0;
    const int64_t r0 = (int64_t)blockIdx.x * rpc + mine, step = (int64_t)gridDim.x * rpc;
    auto fill = [&](int s, int64_t row) {
        if (row >= a.rows) return;
        const T *src[IN];
        src[0] = a.dy + row * a.lddy;
        src[1] = a.x + row * a.ldx;
        if constexpr (DH) src[2] = a.dh + row * a.lddh;
        ring.fill(s, src);
    };
    ring.init(dyn, mine, (int)a.cols, depth, leader);
    if (leader)
        for (int i = 0; i < depth; ++i) fill(i, r0 + i * step);
    // up to two segments a thread are held from the sums to the output, more are
    // computed again from the slot (registers)
    constexpr bool HOLD = NCH <= 2;
    Raw8<W> wv[HOLD ? NCH : 1];
    F8 dw[NCH];
    int n[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        n[i] = count_of<VEC>((w0 + i * wpr) * SEG, a.cols, lane);
        if constexpr (HOLD) wv[i] = load8_or<W, VEC>(a.w, 1.f, (w0 + i * wpr) * SEG, n[i], lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) dw[i].p[j] = make_float2(0.f, 0.f);
    }
    int turn = 0;
    float rstd = r0 < a.rows ? a.rstd[r0] : 0.f;
    for (int64_t r = r0; r < a.rows; r += step, ++turn) {
        const bool go = leader && turn > 0 && !*ring.abort_word(dyn);
        const float rs = rstd;
        const float2 rstd2 = make_float2(rs, rs);
        if (r + step < a.rows) rstd = a.rstd[r + step];
        const RowView<T> yr = ring.view(0, a.dy + r * a.lddy), xr = ring.view(1, a.x + r * a.ldx);
        float2 s2 = make_float2(0.f, 0.f);
        F8 gh[HOLD ? NCH : 1], xh[HOLD ? NCH : 1];
        ring.wait(dyn);
        auto weights = [&](int i) {
            if constexpr (HOLD) {
                stay_packed(wv[i]);
                return unpack<W>(wv[i]);
            } else {
                return unpack<W>(load8_or<W, VEC>(a.w, 1.f, (w0 + i * wpr) * SEG, n[i], lane));
            }
        };
        auto values = [&](int i, F8 &dy, F8 &x) {  // dy and x-hat, 0 past the row's end
            const int seg0 = (w0 + i * wpr) * SEG;
            dy = unpack<T>(load8<T, VEC>(yr, seg0, n[i], lane));
            x = unpack<T>(load8<T, VEC>(xr, seg0, n[i], lane));
#pragma unroll
            for (int j = 0; j < 4; ++j) x.p[j] = mul2(x.p[j], rstd2);
        };
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            F8 dy, x;
            values(i, dy, x);
            const F8 w = weights(i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 g = mul2(dy.p[j], w.p[j]);
                dw[i].p[j] = fma2(dy.p[j], x.p[j], dw[i].p[j]);
                s2 = fma2(g, x.p[j], s2);
                if constexpr (HOLD) gh[i].p[j] = g, xh[i].p[j] = x.p[j];
            }
        }
        const float s = group_sum<NW, MULTI>(s2.x + s2.y, red[turn & 1], wpr, mine, w0, lane);
        // the row before this one has been read by all
        if (MULTI && wpr == 1) __syncwarp();
        if (go) fill(ring.slot == 0 ? depth - 1 : ring.slot - 1, r + (depth - 1) * step);
        // dx = rstd g - x-hat rstd mean(g x-hat)
        const float c2 = -rs * (s * inv_n);
        const float2 c2_2 = make_float2(c2, c2);
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int seg0 = (w0 + i * wpr) * SEG;
            F8 g, x;
            if constexpr (HOLD) {
                g = gh[i], x = xh[i];
            } else {
                values(i, g, x);
                const F8 w = weights(i);
#pragma unroll
                for (int j = 0; j < 4; ++j) g.p[j] = mul2(g.p[j], w.p[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) g.p[j] = fma2(x.p[j], c2_2, mul2(g.p[j], rstd2));
            if constexpr (DH) {
                const F8 dh = unpack<T>(load8<T, VEC>(ring.view(IN - 1, a.dh + r * a.lddh), seg0, n[i], lane));
#pragma unroll
                for (int j = 0; j < 4; ++j) g.p[j] = add2(g.p[j], dh.p[j]);
            }
            store8<T, VEC>(a.dx + r * a.lddx, seg0, n[i], lane, g);
        }
        ring.next();
    }
    if (a.part) {
        float *part = a.part + (int64_t)blockIdx.x * a.cols;
        if constexpr (MULTI) {
            // the groups' sums, over the rings' space once every warp is done with it
            __syncthreads();
            float *acc = reinterpret_cast<float *>(dyn + RING_HEAD), *own = acc + (int64_t)mine * a.cols;
#pragma unroll
            for (int i = 0; i < NCH; ++i) store8<float, VEC>(own, (w0 + i * wpr) * SEG, n[i], lane, dw[i]);
            __syncthreads();
            for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
                float s = 0.f;
                for (int i = 0; i < rpc; ++i) s += acc[(int64_t)i * a.cols + c];
                part[c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NCH; ++i) store8<float, VEC>(part, (w0 + i * wpr) * SEG, n[i], lane, dw[i]);
        }
    }
    __syncthreads();
    // the same for all: every wait of the CTA lies before this barrier
    if (ring.gave_up(dyn)) rms_bwd_nan<T, W>(a, MULTI ? wpr : blockDim.x >> 5);
}

// Longer rows, first kernel: the row's sum.
template <typename T, typename W, bool VEC>
__global__ void __launch_bounds__(LONG_THREADS) rms_bwd_sums_kernel(RmsBwdArgs<T, W> a, float *sums) {
    constexpr int nw = LONG_THREADS / 32;
    __shared__ __align__(16) float red[2][nw];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inv_n = 1.f / (float)a.cols;
    const int64_t segs = (a.cols + SEG - 1) / SEG;
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
        const float rstd = a.rstd[r];
        float s2 = 0.f;
        for (int64_t sg = warp; sg < segs; sg += nw) {
            const int n = count_of<VEC>(sg * SEG, a.cols, lane);
            const F8 y = unpack<T>(load8<T, VEC>(a.dy + r * a.lddy, sg * SEG, n, lane));
            const F8 x = unpack<T>(load8<T, VEC>(a.x + r * a.ldx, sg * SEG, n, lane));
            const F8 w = unpack<W>(load8_or<W, VEC>(a.w, 1.f, sg * SEG, n, lane));
            float2 t = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 4; ++j) t = fma2(mul2(y.p[j], w.p[j]), mul2(x.p[j], make_float2(rstd, rstd)), t);
            s2 += t.x + t.y;
        }
        const float s = row_sum<nw>(s2, red + turn, warp, lane);
        if (threadIdx.x == 0) sums[r] = s * inv_n;
    }
}

// Second kernel: a warp takes one segment of columns over its share of the rows
// (blockIdx.y of gridDim.y).
template <typename T, typename W, bool VEC, bool DH>
__global__ void __launch_bounds__(128) rms_bwd_cols_kernel(RmsBwdArgs<T, W> a, const float *sums) {
    const int lane = threadIdx.x & 31;
    const int64_t seg0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * SEG;
    if (seg0 >= a.cols) return;
    const int n = count_of<VEC>(seg0, a.cols, lane);
    const F8 w = unpack<W>(load8_or<W, VEC>(a.w, 1.f, seg0, n, lane));
    F8 dw;
#pragma unroll
    for (int j = 0; j < 4; ++j) dw.p[j] = make_float2(0.f, 0.f);
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float rstd = a.rstd[r], c = -rstd * sums[r];
        const float2 rstd2 = make_float2(rstd, rstd), c2 = make_float2(c, c);
        const F8 y = unpack<T>(load8<T, VEC>(a.dy + r * a.lddy, seg0, n, lane));
        const F8 x = unpack<T>(load8<T, VEC>(a.x + r * a.ldx, seg0, n, lane));
        F8 g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 xh = mul2(x.p[j], rstd2);
            dw.p[j] = fma2(y.p[j], xh, dw.p[j]);
            g.p[j] = fma2(xh, c2, mul2(mul2(y.p[j], w.p[j]), rstd2));
        }
        if constexpr (DH) {
            const F8 dh = unpack<T>(load8<T, VEC>(a.dh + r * a.lddh, seg0, n, lane));
#pragma unroll
            for (int j = 0; j < 4; ++j) g.p[j] = add2(g.p[j], dh.p[j]);
        }
        store8<T, VEC>(a.dx + r * a.lddx, seg0, n, lane, g);
    }
    if (a.part) store8<float, VEC>(a.part + (int64_t)blockIdx.y * a.cols, seg0, n, lane, dw);
}

// dw from the `parts` partial sums, in a fixed order: a column's sum does not depend
// on timing.  A warp takes 32 columns, the CTA's eight warps every eighth partial.
// Launched with programmatic dependence on the kernel before it (which gives no
// signal of its own): the CTAs start as that kernel's last ones leave and wait for
// its end before they read.
template <typename W>
__global__ void __launch_bounds__(256) rms_bwd_finish_kernel(const float *part, int parts, int64_t n, W *dw) {
    __shared__ float red[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    float s = 0.f;
    if (c < n) {
        const float *p = part + c;
        int i = warp;
        for (; i + 56 < parts; i += 64) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = __ldcg(p + (int64_t)(i + 8 * k) * n);
#pragma unroll
            for (int k = 0; k < 8; ++k) s += v[k];
        }
        for (; i < parts; i += 8) s += __ldcg(p + (int64_t)i * n);
    }
    red[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < n) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += red[i][lane];
        dw[c] = from_f<W>(s);
    }
}

// ---------------------------------------------------------------- launches
static int rms_long_parts(int64_t rows, int64_t cols) {
    const int64_t x = (cols + 4 * SEG - 1) / (4 * SEG);
    int64_t y = ((int64_t)num_sms() * 12 + x - 1) / x;
    if (y > rows) y = rows;
    return (int)(y < 1 ? 1 : (y > 65535 ? 65535 : y));
}
static size_t rms_up256(size_t b) { return (b + 255) / 256 * 256; }
static size_t rms_bwd_workspace(int64_t rows, int64_t cols) {
    size_t need = 0;
    if (cols <= (int64_t)MAX_SEGS * SEG) {
        const RmsShape s = rms_shape(cols, 2, 2, true, false);  // the largest grid of the forms
        need = rms_up256((size_t)rms_grid(s, rows) * cols * 4);
    }
    if (rms_long(cols, 4, 3, true)) {  // for some type or form
        const size_t l = rms_up256((size_t)rms_long_parts(rows, cols) * cols * 4) + rms_up256((size_t)rows * 4);
        if (l > need) need = l;
    }
    return need;
}

template <typename T, typename W, bool VEC, bool DH>
static int rms_bwd_launch(RmsBwdArgs<T, W> a, W *dw, void *ws, cudaStream_t st) {
    int parts, rc;
    constexpr int IN = DH ? 3 : 2;
    a.part = dw ? static_cast<float *>(ws) : nullptr;
    if (rms_long(a.cols, sizeof(T), IN, true)) {
        parts = rms_long_parts(a.rows, a.cols);
        float *sums = reinterpret_cast<float *>(static_cast<uint8_t *>(ws) + rms_up256((size_t)parts * a.cols * 4));
        const int64_t cap = (int64_t)num_sms() * 4;
        rms_bwd_sums_kernel<T, W, VEC><<<(int)(a.rows < cap ? a.rows : cap), LONG_THREADS, 0, st>>>(a, sums);
        const dim3 grid((unsigned)((a.cols + 4 * SEG - 1) / (4 * SEG)), (unsigned)parts);
        rms_bwd_cols_kernel<T, W, VEC, DH><<<grid, 128, 0, st>>>(a, sums);
        rc = launch_status();
    } else {
        const RmsShape s = rms_shape(a.cols, sizeof(T), IN, true, VEC);
        parts = rms_grid(s, a.rows);
        auto go = [&](auto k) -> int {
            if (int e = allow_smem(k, s.smem, MAX_SMEM)) return e;
            k<<<parts, s.threads, s.smem, st>>>(a, s.wpr, s.depth);
            return launch_status();
        };
        const bool multi = s.rows_per_cta > 1;
        rc = s.nch == 1         ? go(rms_bwd_kernel<T, W, 1, 256, VEC, DH, true>)
             : s.nch == 4       ? go(rms_bwd_kernel<T, W, 4, 512, VEC, DH, false>)
             : multi            ? go(rms_bwd_kernel<T, W, 2, 256, VEC, DH, true>)
             : s.threads <= 256 ? go(rms_bwd_kernel<T, W, 2, 256, VEC, DH, false>)
                                : go(rms_bwd_kernel<T, W, 2, 512, VEC, DH, false>);
    }
    if (rc || !a.part) return rc;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((a.cols + 31) / 32));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    ACT_CUDA_TRY(cudaLaunchKernelEx(&cfg, rms_bwd_finish_kernel<W>, (const float *)a.part, parts, a.cols, dw));
    return ACT_OK;
}

}  // namespace norm
}  // namespace act

extern "C" size_t actcomp_rms_norm_bwd_workspace(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 ? act::norm::rms_bwd_workspace(rows, cols) : 0;
}

extern "C" int actcomp_rms_norm_bwd(const actcomp_rms_bwd_args *g, void *workspace, size_t workspace_bytes,
                                    void *stream) {
    using namespace act;
    using namespace act::norm;
    ACT_CHECK(g && g->rows >= 0 && g->cols > 0, ACT_E_INVALID);
    ACT_CHECK(g->dtype >= 0 && g->dtype <= 2 && (g->wdtype == g->dtype || g->wdtype == 0), ACT_E_INVALID);
    const int es = g->dtype == 0 ? 4 : 2, wsz = g->wdtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(g->dweight, wsz), ACT_E_ALIGN);
    cudaStream_t st = as_stream(stream);
    if (g->rows == 0) {  // the sum over no rows
        if (g->dweight) ACT_CUDA_TRY(cudaMemsetAsync(g->dweight, 0, (size_t)g->cols * wsz, st));
        return ACT_OK;
    }
    ACT_CHECK(g->dy && g->x && g->dx && g->rstd, ACT_E_INVALID);
    ACT_CHECK(g->lddy >= g->cols && g->ldx >= g->cols && g->lddx >= g->cols, ACT_E_INVALID);
    ACT_CHECK(!g->dh || g->lddh >= g->cols, ACT_E_INVALID);
    ACT_CHECK(g->cols <= ((int64_t)1 << 30) && g->rows <= ((int64_t)1 << 40), ACT_E_UNSUPPORTED);
    ACT_CHECK(aligned(g->dy, es) && aligned(g->x, es) && aligned(g->dx, es) && aligned(g->dh, es), ACT_E_ALIGN);
    ACT_CHECK(aligned(g->weight, wsz) && aligned(g->rstd, 4), ACT_E_ALIGN);
    ACT_CHECK(workspace && aligned(workspace, 16) && workspace_bytes >= rms_bwd_workspace(g->rows, g->cols),
              ACT_E_WORKSPACE);
    const bool vec = g->cols % 8 == 0 && rows16(g->dy, g->lddy, es) && rows16(g->x, g->ldx, es) &&
                     rows16(g->dh, g->lddh, es) && rows16(g->dx, g->lddx, es) && aligned(g->weight, 16);
    return rms_types(g->dtype, g->wdtype == 0, [&](auto t, auto w) -> int {
        using T = decltype(t);
        using W = decltype(w);
        RmsBwdArgs<T, W> a{static_cast<const T *>(g->dy), static_cast<const T *>(g->x), static_cast<const T *>(g->dh),
                           static_cast<const W *>(g->weight), g->rstd, static_cast<T *>(g->dx), nullptr, g->rows,
                           g->cols, g->lddy, g->ldx, g->lddh, g->lddx};
        W *dw = static_cast<W *>(g->dweight);
        if (g->dh)
            return vec ? rms_bwd_launch<T, W, true, true>(a, dw, workspace, st)
                       : rms_bwd_launch<T, W, false, true>(a, dw, workspace, st);
        return vec ? rms_bwd_launch<T, W, true, false>(a, dw, workspace, st)
                   : rms_bwd_launch<T, W, false, false>(a, dw, workspace, st);
    });
}
