// fp8_few.cu -- x . w^T for a few tokens in 8-bit floating point.
//
// It cannot do without the weight's byte a value, read once: 256-row tiles of the
// tensor cores would be nearly empty and there are too few of them to keep all of
// memory busy.  Here a warp takes 16 rows of the weight and a share of the contraction,
// and multiplies on the warp's own matrix instruction (m16n8k32, float32 accumulation):
// no code is decoded, and eight tokens cost what one does.
//   A lane brings 16 consecutive codes of a row at a time (four lanes 64 bytes); the
// order in which an instruction's steps take them is the same for both operands, and
// of no consequence.  A block of 128 is four instructions from zero, whose sum is
// scaled and added in float32.
//   The warps of a CTA share rows and split their blocks (KS), so that all loads of a
// warp are under way at once; their sums meet in shared memory in a fixed order.
#include <algorithm>

#include "fp8.cuh"

namespace act {
namespace fp8 {

struct FewArgs {
    const uint8_t *x, *w;
    const uint8_t *xs, *ws;
    void *c;
    int64_t ldx, ldw, ldc;
    int tokens, n, k;
    int x_groups;        // of 128 tokens' scales (ROWS)
    int64_t ws_k;        // bytes from a block of the contraction to the next
    int ws_g, ws_lines;  // from 128 rows to the next; whether a scale belongs to a row (else to 128)
    int ks_log;          // log2 of the warps that share rows
};

template <int FX, int FW>
__device__ __forceinline__ void mma_k32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
#define ACT_FP8_MMA(A, B)                                                                                              \
    asm("mma.sync.aligned.m16n8k32.row.col.f32." A "." B                                                               \
        ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"                                         \
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                               \
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
    if constexpr (FW == E4M3 && FX == E4M3) ACT_FP8_MMA("e4m3", "e4m3");
    else if constexpr (FW == E4M3) ACT_FP8_MMA("e4m3", "e5m2");
    else if constexpr (FX == E4M3) ACT_FP8_MMA("e5m2", "e4m3");
    else ACT_FP8_MMA("e5m2", "e5m2");
#undef ACT_FP8_MMA
}

// n of 16 codes at p (16-byte aligned, all there to read where n > 0), the others 0.
__device__ __forceinline__ uint4 load16(const uint8_t *p, int n) {
    if (n <= 0) return make_uint4(0, 0, 0, 0);
    uint4 q = __ldg(reinterpret_cast<const uint4 *>(p));
    if (n < 16) {
        uint32_t *w = reinterpret_cast<uint32_t *>(&q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int left = n - 4 * i;
            w[i] &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
        }
    }
    return q;
}
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

constexpr int FEW_WARPS = 8, THREADS = 32 * FEW_WARPS;
constexpr int X_ROOM = 96 * 1024;  // shared memory for x: two CTAs per SM
// A token's codes in shared memory: whole blocks, and 64 bytes, so that the eight lanes of a quarter warp
// (two tokens, four pieces of 16 bytes) meet all banks.
__host__ __device__ __forceinline__ int x_pitch(int k) { return (k + 127) / 128 * 128 + 64; }

// NT: groups of eight tokens.
template <typename TOut, int NT, int FX, int FW>
__global__ void __launch_bounds__(THREADS, 2) few_kernel(const __grid_constant__ FewArgs a) {
    extern __shared__ __align__(16) uint8_t xs[];  // tokens x pitch codes, then blocks x 8 NT scales
    __shared__ float part[FEW_WARPS][NT][4][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int ks = 1 << a.ks_log, mine = warp & (ks - 1), per = FEW_WARPS >> a.ks_log;
    const int g = lane >> 2, q = lane & 3;
    const int blocks = (a.k + 127) / 128, pitch = x_pitch(a.k);
    float *xf = reinterpret_cast<float *>(xs + a.tokens * pitch);
    const int sets = (a.n + 15) / 16, turns = (sets + per - 1) / per;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    constexpr int UNROLL = NT == 1 ? 4 : 2;  // blocks of a warp on their way together (registers)
    uint4 w[UNROLL][4];  // row, half of the block
    uint32_t sc[UNROLL][2];
    auto fetch = [&](int turn, int b0) {
        const int64_t r0 = ((int64_t)turn * per + (warp >> a.ks_log)) * 16, ra = r0 + g, rb = ra + 8;
        const uint8_t *wa = a.w + ra * a.ldw + 16 * q, *wb = wa + 8 * a.ldw;
        const uint8_t *sa = a.ws + (r0 >> 7) * a.ws_g, *sb = sa;
        if (a.ws_lines) sa += (ra & 31) * 4 + ((ra >> 5) & 3), sb += (rb & 31) * 4 + ((rb >> 5) & 3);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int b = b0 + u * ks;
            if (b < blocks && 128 * b + 128 <= a.k && r0 + 16 <= a.n) {  // a whole block of whole rows
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    w[u][h] = __ldg(reinterpret_cast<const uint4 *>(wa + 128 * b + 64 * h));
                    w[u][2 + h] = __ldg(reinterpret_cast<const uint4 *>(wb + 128 * b + 64 * h));
                }
                sc[u][0] = __ldg(sa + b * a.ws_k);
                sc[u][1] = a.ws_lines ? __ldg(sb + b * a.ws_k) : sc[u][0];
            } else {
                const int left = b < blocks ? a.k - 128 * b - 16 * q : 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    w[u][h] = load16(wa + 128 * b + 64 * h, ra < a.n ? left - 64 * h : 0);
                    w[u][2 + h] = load16(wb + 128 * b + 64 * h, rb < a.n ? left - 64 * h : 0);
                }
                sc[u][0] = b < blocks && ra < a.n ? __ldg(sa + b * a.ws_k) : 0u;
                sc[u][1] = b < blocks && rb < a.n ? __ldg(sb + b * a.ws_k) : 0u;
            }
        }
    };
    int turn = blockIdx.x;
    fetch(turn, mine);
    // x while the first codes of w are on their way
    for (int i = threadIdx.x; i < a.tokens * blocks * 8; i += THREADS) {
        const int tok = i / (blocks * 8), c = i - tok * blocks * 8;
        *reinterpret_cast<uint4 *>(xs + tok * pitch + 16 * c) = load16(a.x + tok * a.ldx + 16 * c, a.k - 16 * c);
    }
    for (int i = threadIdx.x; i < blocks * 8 * NT; i += THREADS) {
        const int b = i / (8 * NT), tok = i - b * 8 * NT;
        xf[i] = scale_value(tok < a.tokens ? __ldg(a.xs + (int64_t)b * a.x_groups * 128 + (tok & 31) * 4 + (tok >> 5)) : 0u);
    }
    __syncthreads();
    for (; turn < turns; turn += gridDim.x) {
        float sum[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[t][i] = 0.f;
        for (int b0 = mine; b0 < blocks; b0 += UNROLL * ks) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int b = b0 + u * ks;
                if (b >= blocks) break;
                const float fa = scale_value(sc[u][0]), fb = scale_value(sc[u][1]);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint8_t *xp = xs + (8 * t + g) * pitch + 128 * b + 16 * q;
                    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 x = 8 * t + g < a.tokens ? *reinterpret_cast<const uint4 *>(xp + 64 * h)
                                                             : make_uint4(0, 0, 0, 0);
                        const uint4 &p = w[u][h], &r = w[u][2 + h];
                        mma_k32<FX, FW>(d, p.x, r.x, p.y, r.y, x.x, x.y);
                        mma_k32<FX, FW>(d, p.z, r.z, p.w, r.w, x.z, x.w);
                    }
                    // columns of the result: tokens 8 t + 2 q and the next
                    const float2 f = *reinterpret_cast<const float2 *>(xf + (b * NT + t) * 8 + 2 * q);
                    sum[t][0] = __fmaf_rn(d[0] * fa, f.x, sum[t][0]);
                    sum[t][1] = __fmaf_rn(d[1] * fa, f.y, sum[t][1]);
                    sum[t][2] = __fmaf_rn(d[2] * fb, f.x, sum[t][2]);
                    sum[t][3] = __fmaf_rn(d[3] * fb, f.y, sum[t][3]);
                }
            }
            if (b0 + UNROLL * ks < blocks) fetch(turn, b0 + UNROLL * ks);
        }
        if (turn + (int)gridDim.x < turns) fetch(turn + gridDim.x, mine);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[warp][t][i][lane] = sum[t][i];
        __syncthreads();
        // the CTA's rows x tokens, neighbouring threads neighbouring rows
        const int rows = 16 * per;
        const int64_t first = (int64_t)turn * rows;
        for (int e = threadIdx.x; e < rows * a.tokens; e += THREADS) {
            const int tok = e / rows, r = e - tok * rows, set = r >> 4, lr = r & 15;
            if (first + r >= a.n) continue;
            // the accumulator's place: row lr & 7 by lane / 4, the upper eight rows two registers on
            const int i = (lr >> 3) * 2 + (tok & 1), l = (lr & 7) * 4 + ((tok & 7) >> 1);
            float s = 0.f;
            for (int j = 0; j < ks; ++j) s += part[(set << a.ks_log) + j][tok >> 3][i][l];
            if (ACT_DCHECK(tok < a.tokens && first + r < a.ldc))
                static_cast<TOut *>(a.c)[tok * a.ldc + first + r] = from_f<TOut>(s);
        }
        __syncthreads();
    }
}

// Whether the product a . b^T goes through the kernel above: few tokens by rows that fit
// shared memory, and a weight whose rows lie along the contraction.
bool few_takes(const actcomp_fp8 *a, const actcomp_fp8 *b) {
    return a->block == ROWS && !b->transposed && a->rows <= ACTCOMP_FP8_FEW_TOKENS && b->cols <= X_ROOM &&
           a->rows * x_pitch((int)b->cols) <= X_ROOM;
}

int few_launch(const actcomp_fp8 *a, const actcomp_fp8 *b, void *c, int64_t ldc, int c_dtype, cudaStream_t st) {
    FewArgs f{a->codes, b->codes, a->scales, b->scales, c, a->ld, b->ld, ldc, (int)a->rows, (int)b->rows, (int)b->cols,
              (int)blocks_of(a->rows), 0, 0, 0, 0};
    f.ws_lines = b->block == ROWS;
    f.ws_k = f.ws_lines ? blocks_of(b->rows) * 128 : 1;
    f.ws_g = f.ws_lines ? 128 : (int)blocks_of(b->cols);
    // Enough warps for the device, as far as there are blocks to share.
    const int64_t sets = (b->rows + 15) / 16, want = (int64_t)num_sms() * 2 * FEW_WARPS, blocks = blocks_of(b->cols);
    while (f.ks_log < 3 && sets << f.ks_log < want && (2 << f.ks_log) <= blocks) ++f.ks_log;
    const int64_t per = FEW_WARPS >> f.ks_log, turns = (sets + per - 1) / per;
    const int nt = a->rows <= 8 ? 1 : a->rows <= 16 ? 2 : 4;
    const int smem = (int)a->rows * x_pitch(f.k) + (int)blocks * nt * 8 * 4;
    const int most = X_ROOM + (X_ROOM / 128 + 1) * 4 * 8 * 4;
    const int64_t cap = (int64_t)num_sms() * 2;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(turns < cap ? turns : cap));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    auto go = [&](auto out, auto n, auto fx, auto fw) -> int {
        auto k = few_kernel<decltype(out), decltype(n)::value, decltype(fx)::value, decltype(fw)::value>;
        ACT_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
        ACT_CUDA_TRY(cudaLaunchKernelEx(&cfg, k, f));
        return ACT_OK;
    };
    auto by_format = [&](auto out, auto n) -> int {
        const std::integral_constant<int, E4M3> e4;
        const std::integral_constant<int, E5M2> e5;
        if (a->format == E4M3) return b->format == E4M3 ? go(out, n, e4, e4) : go(out, n, e4, e5);
        return b->format == E4M3 ? go(out, n, e5, e4) : go(out, n, e5, e5);
    };
    auto by_tokens = [&](auto out) -> int {
        if (nt == 1) return by_format(out, std::integral_constant<int, 1>{});
        if (nt == 2) return by_format(out, std::integral_constant<int, 2>{});
        return by_format(out, std::integral_constant<int, 4>{});
    };
    return c_dtype == 0 ? by_tokens(float{}) : c_dtype == 1 ? by_tokens(__nv_bfloat16{}) : by_tokens(__half{});
}

}  // namespace fp8
}  // namespace act
