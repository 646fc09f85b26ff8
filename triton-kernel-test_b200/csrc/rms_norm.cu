// rms_norm.cu -- the root-mean-square norm's forms in the activations' type, and its
// entry point (kernels: rms_norm.cuh).
#include "rms_norm.cuh"

namespace act {
namespace norm {
int rms_fwd_fp8(const actcomp_rms_args *g, bool vec, cudaStream_t st);  // rms_norm_fp8.cu
}
}  // namespace act

extern "C" int actcomp_rms_norm(const actcomp_rms_args *g, void *stream) {
    using namespace act;
    using namespace act::norm;
    ACT_CHECK(g && g->rows >= 0 && g->cols > 0, ACT_E_INVALID);
    ACT_CHECK(g->dtype >= 0 && g->dtype <= 2 && (g->wdtype == g->dtype || g->wdtype == 0), ACT_E_INVALID);
    ACT_CHECK(g->eps >= 0.f, ACT_E_INVALID);
    if (g->rows == 0) return ACT_OK;
    const bool q8 = g->codes != nullptr, add = g->res != nullptr;
    ACT_CHECK(g->x && g->rstd && (q8 ? !g->y && g->scales : g->y != nullptr), ACT_E_INVALID);
    ACT_CHECK(g->ldx >= g->cols && (q8 ? g->ldc >= g->cols : g->ldy >= g->cols), ACT_E_INVALID);
    ACT_CHECK(!add || (g->h && g->ldr >= g->cols && g->ldh >= g->cols), ACT_E_INVALID);
    ACT_CHECK(g->cols <= ((int64_t)1 << 30) && g->rows <= ((int64_t)1 << 40), ACT_E_UNSUPPORTED);
    const int es = g->dtype == 0 ? 4 : 2, ws = g->wdtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(g->x, es) && aligned(g->y, es) && aligned(g->res, es) && aligned(g->h, es), ACT_E_ALIGN);
    ACT_CHECK(aligned(g->weight, ws) && aligned(g->rstd, 4), ACT_E_ALIGN);
    ACT_CHECK(!q8 || (aligned(g->codes, 16) && aligned(g->scales, 16) && g->ldc % 16 == 0), ACT_E_ALIGN);
    const bool vec = g->cols % 8 == 0 && rows16(g->x, g->ldx, es) && rows16(g->y, g->ldy, es) &&
                     rows16(g->res, g->ldr, es) && rows16(g->h, g->ldh, es) && aligned(g->weight, 16);
    cudaStream_t st = as_stream(stream);
    if (q8) return rms_fwd_fp8(g, vec, st);
    return rms_types(g->dtype, g->wdtype == 0, [&](auto t, auto w) -> int {
        const auto a = rms_args<decltype(t), decltype(w)>(g);
        if (add) return vec ? rms_fwd_launch<decltype(t), decltype(w), true, true, false>(a, st)
                            : rms_fwd_launch<decltype(t), decltype(w), false, true, false>(a, st);
        return vec ? rms_fwd_launch<decltype(t), decltype(w), true, false, false>(a, st)
                   : rms_fwd_launch<decltype(t), decltype(w), false, false, false>(a, st);
    });
}
