// fp8_gemm.cu -- the product of two 8-bit matrices with a power-of-two scale per
// block of 128, C = A . B^T, on the block-scaled tensor cores (tcgen05.mma
// kind::mxf8f6f4; the frame is pair_gemm.cuh).
//
// C[m][n] = sum over blocks of 128 of 2^(ea + eb - 254) sum_j a_j b_j, float32
// accumulation in TMEM.  The scales being powers of two in the hardware's own format, a
// block of 128 is four MMA steps that take the same scale byte: nothing is rescaled
// between the steps, which a product with float scales has to do in registers.  An
// operand whose blocks run down its columns is read with its rows contiguous, so that
// the weight's one copy (tiles of 128 x 128) serves the output and the input gradient.
//
// 16384 x 4096 x 11008, us (2 M N K = 1.48e12): output 550 (2.69 PFLOP/s), input gradient
// 600, weight gradient 575 each by itself; over seconds 663, 696 and 684 (2.1 to 2.2
// PFLOP/s) at 1.5 GHz under the power limit, where bf16 products of the library reach 1.33
// to 1.41.  A stage takes 725 cycles against 512 of MMAs.  200 x 4096 x 11008 has 43
// tiles for 74 pairs: 20 us, of which 12 are its 32 stages and the rest start and end.
#include "pair_gemm.cuh"

namespace act {
namespace fp8 {

int check(const actcomp_fp8 *q);  // fp8_quant.cu
bool few_takes(const actcomp_fp8 *a);  // fp8_few.cu
int few_launch(const actcomp_fp8 *a, const actcomp_fp8 *b, const pair::Scales &sa, const pair::Scales &sb, void *c,
               int64_t ldc, int c_dtype, cudaStream_t st);

template <typename TOut>
struct StoreEpi {
    using P = pair::OutParams;
    const P &o;
    const CUtensorMap *tmC;
    pair::Out<TOut, pair::OUT_BYTES / 4> out;
    int lane, row0 = 0;
    __device__ __forceinline__ StoreEpi(const P &o, uint8_t *stage, const CUtensorMap *tmC, int lane)
        : o(o), tmC(tmC), out{stage}, lane(lane) {}
    __device__ __forceinline__ void begin(const pair::Params &, const pair::Tile &, int r, int) { row0 = r; }
    __device__ __forceinline__ void group(const pair::Params &p, const uint32_t (&r)[32], int col) {
        if (row0 >= p.M || col >= p.N) return;
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        out.put(v, row0, col, p.M, p.N, lane, o, tmC);
    }
    __device__ __forceinline__ void end(const pair::Params &) {}
    __device__ __forceinline__ void lost(const pair::Params &) {}
};

// Lines and contraction of an operand.
struct View {
    int64_t lines, k;
};
static View view_of(const actcomp_fp8 *q) {
    return q->transposed ? View{q->cols, q->rows} : View{q->rows, q->cols};
}
static pair::Scales scales_of(const actcomp_fp8 *q) {
    const int64_t groups = blocks_of(view_of(q).lines), cb = blocks_of(q->cols);
    if (q->block != TILES) return {q->scales, (int)groups, groups * 128, 128, 0};
    return {q->scales, (int)groups, q->transposed ? cb : 1, (int)(q->transposed ? 1 : cb), 1};
}
static int map_of(CUtensorMap *m, const actcomp_fp8 *q) {
    return make_map_3d(m, q->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, q->cols, q->rows, 1, q->ld, 0, 128, 128,
                       CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace fp8
}  // namespace act

extern "C" int actcomp_fp8_gemm(const actcomp_fp8 *a, const actcomp_fp8 *b, void *c, int64_t ldc, int32_t c_dtype,
                                void *stream) {
    using namespace act;
    using namespace act::fp8;
    if (int st = check(a)) return st;
    if (int st = check(b)) return st;
    const View va = view_of(a), vb = view_of(b);
    ACT_CHECK(va.k == vb.k && c && ldc >= vb.lines && c_dtype >= 0 && c_dtype <= 2, ACT_E_INVALID);
    const int es = c_dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(c, es), ACT_E_ALIGN);
    if (few_takes(a)) return few_launch(a, b, scales_of(a), scales_of(b), c, ldc, c_dtype, as_stream(stream));
    pair::Params p{};
    pair::set_tiles(p, (int)va.lines, (int)vb.lines, (int)blocks_of(va.k));
    ACT_CHECK((int64_t)p.m_tiles * p.n_tiles <= INT32_MAX, ACT_E_UNSUPPORTED);
    p.a_mn = a->transposed;
    p.b_mn = b->transposed;
    p.idesc = tc::idesc_mxf8(pair::BM, pair::BN, a->format == E5M2, b->format == E5M2, p.a_mn, p.b_mn);
    p.sa = scales_of(a);
    p.sb = scales_of(b);
    const pair::OutParams o{c, ldc, pair::tma_out(c, ldc, p.N, es)};
    CUtensorMap tmA, tmB;
    if (int st = map_of(&tmA, a)) return st;
    if (int st = map_of(&tmB, b)) return st;
    CUtensorMap tmC = tmA;  // not read without o.tma
    if (o.tma)
        if (int st = make_map_3d(&tmC, c,
                                 c_dtype == 0   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : c_dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                 es, p.N, p.M, 1, ldc, 0, 32, 32,
                                 es == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
            return st;
    cudaStream_t s = as_stream(stream);
    if (c_dtype == 0) return pair::launch<pair::FP8, StoreEpi<float>>(tmA, tmB, tmC, p, o, s);
    if (c_dtype == 1) return pair::launch<pair::FP8, StoreEpi<__nv_bfloat16>>(tmA, tmB, tmC, p, o, s);
    return pair::launch<pair::FP8, StoreEpi<__half>>(tmA, tmB, tmC, p, o, s);
}
