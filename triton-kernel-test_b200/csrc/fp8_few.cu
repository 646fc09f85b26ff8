// fp8_few.cu -- the product of two 8-bit matrices of which the first has few rows (a
// batch of tokens being served against a weight): C = X . W^T with the weight's rows as
// the tensor cores' M.
//
// It cannot do without the weight's byte a value, read once.  The tiles of 256 x 256
// (fp8_gemm.cu) would be mostly empty and too few to keep memory busy.  Here a CTA takes
// 128 rows of the weight against all tokens (the MMA's N is their number rounded to 16),
// and the contraction is cut over a cluster of up to eight CTAs, so that the device has
// two to four CTAs per SM; their sums meet in shared memory, each CTA adding some of the
// tokens' columns in the order of the ranks.  Per CTA:
//   warp 0      TMA producer: 128 rows x 128 of W, N x 128 of X a stage;
//   warp 1      TMEM allocation, MMA issue;
//   warps 2..5  scales from memory to TMEM, every lane quadrant the same (as in
//               pair_gemm.cuh), then the sums.
// 4096 x 11008, us with the event's own 2.6: 1 token 17.5, 32 20.5, 128 27 (floor 6.9; the
// same bytes read and dropped take 14.3); 11008 x 4096 18.5, 20.5, 27.6 (in 256 x 256 tiles
// 44); 16384 x 16384 50 (41).  What holds it is the start, 4000 to 9000 cycles until the
// first tile and its scales are there.  Other ways: tokens on the M side with the warps'
// own 8-bit matrix instruction 20.5 (it is made of conversions and 16-bit steps: 242
// instructions for 16 x 128 codes); parts of the tokens for more than 128, the weight read
// again from L2, no better than the tiles.
#include <algorithm>

#include "pair_gemm.cuh"

namespace act {
namespace fp8 {

constexpr int FEW_THREADS = 192;
constexpr int W_BYTES = 128 * 128;  // of a stage
constexpr int FEW_SETS = 8, SET_COLS = 8;  // scale sets in TMEM: 128 rows of W, up to 128 tokens
constexpr int MOST_N = ACTCOMP_FP8_FEW_TOKENS;
// Accumulators that the steps take in turn, so that one waits less for the step before it.
__host__ __device__ constexpr int accumulators(int n) { return n <= 48 ? 4 : n <= 96 ? 2 : 1; }
__host__ __device__ constexpr int columns(int n) { return n * accumulators(n) + FEW_SETS * SET_COLS; }
// TMEM is asked for by CTAs that others of their cluster wait for: it must never be what a resident CTA waits for
// (two launches beside each other could wait for each other's).  So a CTA takes as large a part of the SM's shared
// memory as of its TMEM: 228 KB over 512 columns.
__host__ __device__ constexpr int few_smem(int tmem_cols) { return tmem_cols * (228 * 1024 / 512) - 1024; }

static_assert(columns(16) <= 128 && columns(48) <= 256 && columns(96) <= 256 && columns(MOST_N) <= 256, "TMEM");
static_assert((few_smem(128) - 1536) / (W_BYTES + 16 * 128) >= 3 && (few_smem(256) - 1536) / (W_BYTES + MOST_N * 128) >= 3,
              "stages");

struct FewParams {
    int tokens, n;        // rows of X and of W
    int kblocks, k_split;  // blocks of 128 of the contraction, and of a rank
    int N, accs;           // the MMA's N, and accumulators
    int w_mn;              // whether W lies with its rows contiguous
    uint32_t idesc;
    int stages, tmem_cols;
    pair::Scales sw, sx;
    void *c;
    int64_t ldc;
};

template <typename TOut>
__global__ void __launch_bounds__(FEW_THREADS)
    few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
               const __grid_constant__ FewParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
    const int stage_bytes = W_BYTES + p.N * 128, stages = p.stages;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + stages * stage_bytes);
    uint64_t *empty = full + stages, *set_full = empty + stages, *set_free = set_full + FEW_SETS,
             *acc_full = set_free + FEW_SETS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_full + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    uint32_t ranks, rank;
    asm volatile("mov.u32 %0, %%cluster_nctarank;\n mov.u32 %1, %%cluster_ctarank;" : "=r"(ranks), "=r"(rank));
    const int tile = blockIdx.x / (int)ranks;
    const int k0 = (int)rank * p.k_split, k1 = min(k0 + p.k_split, p.kblocks), steps = k1 > k0 ? k1 - k0 : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        // The scales have barriers of their own: there are more sets than stages, so that their warps may be further
        // ahead than the producer, whose barriers they must not arrive on then.
        for (int s = 0; s < FEW_SETS; ++s) {
            tc::mbar_init(&set_full[s], 4);
            tc::mbar_init(&set_free[s], 1);
        }
        tc::mbar_init(acc_full, 1);
        *abort = 0;
        tc::fence_mbar_init();
        tc::prefetch_tmap(&tmW);
        tc::prefetch_tmap(&tmX);
    }
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, p.tmem_cols);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // launched with programmatic dependence (see pair_gemm.cuh)
    tc::dependence_wait();

    const int sets = p.accs * p.N;  // TMEM column of the scale sets
    bool ok = true;
    if (warp == 0 && lane == 0) {
        int s = 0;
        uint32_t phase = 1;
        for (int i = 0; i < steps; ++i) {
            if (!(ok = tc::mbar_spin(&empty[s], phase, abort))) break;
            uint8_t *w = smem + s * stage_bytes;
            const int k = (k0 + i) * 128;
            tc::mbar_arrive_expect_tx(&full[s], stage_bytes);
            if (p.w_mn) tc::tma_load_3d(w, &tmW, &full[s], tile * 128, k, 0);
            else tc::tma_load_3d(w, &tmW, &full[s], k, tile * 128, 0);
            tc::tma_load_3d(w + W_BYTES, &tmX, &full[s], k, 0, 0);
            if (++s == stages) s = 0, phase ^= 1;
        }
    } else if (warp == 1) {
        // What this loop takes a block when nothing is waited for (300 cycles; with divisions for the stage and
        // sleeping waits 750) is most of a short contraction's time.
        const uint64_t desc_w = tc::smem_desc(smem, p.w_mn ? 8192 : 16, 1024, tc::SW_128B);
        const uint64_t desc_x = tc::smem_desc(smem + W_BYTES, 16, 1024, tc::SW_128B);
        const uint32_t step = p.w_mn ? 32 * 128 / 16 : 2, d1 = tmem + (p.accs > 1 ? p.N : 0),
                       d2 = tmem + (p.accs > 2 ? 2 * p.N : 0), d3 = tmem + (p.accs - 1) * p.N;
        int s = 0, set = 0;
        uint32_t phase = 0, set_phase = 0;
        for (int i = 0; i < steps; ++i) {
            if (!(ok = tc::mbar_spin(&set_full[set], set_phase, abort))) break;
            if (!(ok = tc::mbar_spin(&full[s], phase, abort))) break;
            tc::tc_fence_after();
            const uint64_t da = desc_w + (uint32_t)(s * (stage_bytes / 16)), db = desc_x + (uint32_t)(s * (stage_bytes / 16));
            const uint32_t sf = tmem + sets + set * SET_COLS;
            if (tc::elect_one()) {
                // a step into each accumulator in turn: the first of each starts it
                tc::mma_mxf8(tmem, da, db, p.idesc, sf, sf + 4, i > 0);
                tc::mma_mxf8(d1, da + step, db + 2, p.idesc, sf, sf + 4, i > 0 || p.accs < 2);
                tc::mma_mxf8(d2, da + 2 * step, db + 4, p.idesc, sf, sf + 4, i > 0 || p.accs < 4);
                tc::mma_mxf8(d3, da + 3 * step, db + 6, p.idesc, sf, sf + 4, i > 0 || p.accs < 4);
                if (i + stages < steps) tc::mma_commit(&empty[s]);
                if (i + FEW_SETS < steps) tc::mma_commit(&set_free[set]);
            }
            __syncwarp();
            if (++s == stages) s = 0, phase ^= 1;
            if (++set == FEW_SETS) set = 0, set_phase ^= 1;
        }
        if (tc::elect_one()) tc::mma_commit(acc_full);
        __syncwarp();
    } else if (warp >= 2) {
        const uint32_t quad = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        constexpr int AHEAD = 4;  // blocks whose words are on their way, and written, together
        uint32_t next[AHEAD][2];
        auto fetch = [&](int i0) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int kb = min(k0 + i0 + i, p.kblocks - 1);
                next[i][0] = pair::scale_word(p.sw, kb, tile, lane);
                next[i][1] = pair::scale_word(p.sx, kb, 0, lane);
            }
        };
        if (steps > 0) fetch(0);
        for (int i0 = 0; i0 < steps && ok; i0 += AHEAD) {
            uint32_t w[AHEAD][2];
            memcpy(w, next, sizeof(w));
            if (i0 + AHEAD < steps) fetch(i0 + AHEAD);
            // several blocks' words at once: the stores' latency, not their number, is what a turn here takes
            const int n = min(AHEAD, steps - i0);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int it = i0 + i;
                if (i >= n) break;
                // the set's earlier MMAs are done
                if (it >= FEW_SETS &&
                    !(ok = tc::mbar_spin(&set_free[it % FEW_SETS], (it / FEW_SETS - 1) & 1, abort)))
                    break;
                tc::tc_fence_after();
                uint32_t u[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = w[i][0] >> (8 * j), u[4 + j] = w[i][1] >> (8 * j);
                tc::tmem_st8(quad + sets + it % FEW_SETS * SET_COLS, u);
            }
            tc::tmem_st_wait();
            tc::tc_fence_before();
            __syncwarp();
            if (lane < n && ok) tc::mbar_arrive(&set_full[(i0 + lane) % FEW_SETS]);
            __syncwarp();
        }
        ok = ok && tc::mbar_spin(acc_full, 0, abort);
        tc::tc_fence_after();
    }

    // a thread's row of the weight, sums of N tokens in TMEM
    const int row = (warp & 3) * 32 + lane, out_row = tile * 128 + row;
    TOut *c = static_cast<TOut *>(p.c) + out_row;
    const uint32_t acc = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    auto sums16 = [&](uint32_t acc, int g, uint32_t (&r)[16]) {  // of tokens g .., over the accumulators
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = 0u;
        if (steps == 0) return;
        tc::tmem_ld16(acc + g, r);
        for (int k = 1; k < p.accs; ++k) {
            uint32_t q[16];
            tc::tmem_ld16(acc + k * p.N + g, q);
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(q[i]));
        }
    };
    if (ranks == 1) {
        if (warp >= 2 && ok) {
#pragma unroll 1
            for (int g = 0; g < p.N; g += 16) {
                uint32_t r[16];
                sums16(acc, g, r);
                if (out_row < p.n) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (g + i < p.tokens && ACT_DCHECK(out_row < p.ldc))
                            c[(int64_t)(g + i) * p.ldc] = pair::cvt_out<TOut>(__uint_as_float(r[i]));
                }
            }
        }
    } else {
        // Columns first .. first + each - 1 are this rank's to add.  The sums go to their ranks' shared memory, over
        // the rings once every rank is done with its own: [rank][column][row].
        const int each = p.N / (int)ranks;
        tc::drain_after_abort(abort);  // nothing lands in the rings any more
        __syncwarp();
        tc::cluster_sync();
        if (warp >= 2) {
#pragma unroll 1
            for (int g = 0; g < p.N; g += 16) {
                uint32_t r[16];
                sums16(acc, g, r);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int to = (g + i) / each, col = g + i - to * each;
                    const float v = ok ? __uint_as_float(r[i]) : __uint_as_float(0x7fc00000u);
                    tc::st_cluster_f32(tc::map_cluster(smem, to) + (uint32_t)((((int)rank * each + col) * 128 + row) * 4), v);
                }
            }
        }
        __syncwarp();
        tc::cluster_sync();
        if (warp >= 2 && out_row < p.n) {
            const float *in = reinterpret_cast<const float *>(smem) + row;
            for (int col = 0; col < each; ++col) {
                const int tok = (int)rank * each + col;
                if (tok >= p.tokens) break;
                float s = in[col * 128];
                for (int k = 1; k < (int)ranks; ++k) s += in[(k * each + col) * 128];
                if (ACT_DCHECK(out_row < p.ldc)) c[(int64_t)tok * p.ldc] = pair::cvt_out<TOut>(s);
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::drain_after_abort(abort);
    __syncwarp();
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, p.tmem_cols);
    }
}

// Whether the product a . b^T goes through the kernel above: a's rows are few and lie
// along the contraction.
bool few_takes(const actcomp_fp8 *a) { return !a->transposed && a->rows <= ACTCOMP_FP8_FEW_TOKENS; }

int few_launch(const actcomp_fp8 *a, const actcomp_fp8 *b, const pair::Scales &sa, const pair::Scales &sb, void *c,
               int64_t ldc, int c_dtype, cudaStream_t st) {
    FewParams p{};
    p.tokens = (int)a->rows;
    p.n = (int)(b->transposed ? b->cols : b->rows);
    p.kblocks = (int)blocks_of(a->cols);
    p.N = (p.tokens + 15) / 16 * 16;
    p.accs = accumulators(p.N);
    p.w_mn = b->transposed;
    p.idesc = tc::idesc_mxf8(128, p.N, b->format == E5M2, a->format == E5M2, p.w_mn, false);
    p.sw = sb, p.sx = sa;
    p.c = c, p.ldc = ldc;
    p.tmem_cols = p.N == 16 ? 128 : 256;  // four or two CTAs per SM
    const int stage = W_BYTES + p.N * 128, smem = few_smem(p.tmem_cols), sms = num_sms(), per_sm = 512 / p.tmem_cols;
    p.stages = (smem - 1024 - 512) / stage;
    // Ranks by an estimate in blocks of 0.35 us: an SM's share of the CTAs at a CTA's blocks each, 20 for every wave's
    // start and first loads, and the sums; the most ranks of equal ones (more loads are under way).  us (a weight in
    // memory) at 1 | 2 | 4 | 8 ranks: 11008 x 4096, 1 token 21.3 | 18.5 | 16.4 | 20.5, 64 tokens 22.5 | 24.5 | 30.7 |
    // 36.9; 4096 x 11008, 1 token 38.8 | 26.5 | 20.5 | 18.5.
    const int64_t units = (p.n + 127) / 128;
    int ranks = 1;
    int64_t best = INT64_MAX;
    for (int r = 1; r <= 8 && (r == 1 || p.kblocks >= 2 * r); r *= 2) {
        const int64_t ctas = units * r, blocks = (p.kblocks + r - 1) / r;
        const int64_t cost = (ctas + sms - 1) / sms * blocks + 20 * ((ctas + sms * per_sm - 1) / (sms * per_sm)) +
                             (r > 1 ? p.N / 32 : 0);
        if (cost <= best) best = cost, ranks = r;
    }
    p.k_split = (p.kblocks + ranks - 1) / ranks;
    ACT_CHECK(units * ranks <= INT32_MAX, ACT_E_UNSUPPORTED);
    CUtensorMap tmW, tmX;
    if (int rc = make_map_3d(&tmW, b->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, b->cols, b->rows, 1, b->ld, 0, 128, 128,
                             CU_TENSOR_MAP_SWIZZLE_128B))
        return rc;
    if (int rc = make_map_3d(&tmX, a->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a->cols, a->rows, 1, a->ld, 0, 128, p.N,
                             CU_TENSOR_MAP_SWIZZLE_128B))
        return rc;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = {(unsigned)ranks, 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(units * ranks));
    cfg.blockDim = dim3(FEW_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    auto go = [&](auto out) -> int {
        auto k = few_kernel<decltype(out)>;
        ACT_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, few_smem(256)));
        ACT_CUDA_TRY(cudaLaunchKernelEx(&cfg, k, tmW, tmX, p));
        return ACT_OK;
    };
    return c_dtype == 0 ? go(float{}) : c_dtype == 1 ? go(__nv_bfloat16{}) : go(__half{});
}

}  // namespace fp8
}  // namespace act
