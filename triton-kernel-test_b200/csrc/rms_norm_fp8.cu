// rms_norm_fp8.cu -- the root-mean-square norm's forms with an 8-bit output (rms_norm.cuh).
#include "rms_norm.cuh"

namespace act {
namespace norm {

int rms_fwd_fp8(const actcomp_rms_args *g, bool vec, cudaStream_t st) {
    return rms_types(g->dtype, g->wdtype == 0, [&](auto t, auto w) -> int {
        const auto a = rms_args<decltype(t), decltype(w)>(g);
        if (a.res) return vec ? rms_fwd_launch<decltype(t), decltype(w), true, true, true>(a, st)
                              : rms_fwd_launch<decltype(t), decltype(w), false, true, true>(a, st);
        return vec ? rms_fwd_launch<decltype(t), decltype(w), true, false, true>(a, st)
                   : rms_fwd_launch<decltype(t), decltype(w), false, false, true>(a, st);
    });
}

}  // namespace norm
}  // namespace act
