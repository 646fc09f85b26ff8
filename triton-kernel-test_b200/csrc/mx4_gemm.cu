// mx4_gemm.cu -- the product of two microscaled 4-bit matrices, C = A . B^T,
// on the block-scaled tensor cores (tcgen05.mma kind::mxf4).
//
// C[m][n] = sum over blocks of 32 columns of 2^(ea + eb - 254) sum_j a_j b_j.
// Both operands are K-major as stored.  One CTA computes a 128 x 256 tile:
//   warp 0      TMA producer: 256 columns (128 bytes a row) of A and B into a
//               128-byte swizzled ring, and the matching scale atoms (512 bytes
//               per 128 rows x 128 columns) by bulk copy;
//   warp 1      TMEM allocator and MMA issuer: copies the stage's scale atoms
//               to TMEM (tcgen05.cp, each stage its own columns, so that a
//               stage's scales are free again when its tiles are), then four
//               K = 64 MMAs;
//   warps 2..5  epilogue.
// Rows past the end of an operand are zero-filled by the TMA, their scales are
// stored as 0 (2^-127): their products are 0.
#include <cuda_fp16.h>

#include "mx4.cuh"
#include "tc_ptx.cuh"

namespace act {
int mx4_check(const actcomp_mx4 *q);
namespace mx4 {

constexpr int BM = 128, BN = 256, BK = 256, THREADS = 192, STAGES = 4;
constexpr int A_BYTES = BM * BK / 2, B_BYTES = BN * BK / 2;
constexpr int SFA_BYTES = 1024, SFB_BYTES = 2048;  // 2 K atoms x (1 | 2) row atoms
constexpr int STAGE = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
constexpr int SMEM = STAGE * STAGES + 1024 + 256;
constexpr int SF_COLS = 24;  // TMEM columns of a stage's scales: A 8, B 16

struct GemmParams {
    int M, N;
    int kblocks, nka;  // 256-column steps; 128-column scale atoms
    int m_tiles, n_tiles;
    const uint8_t *sfa, *sfb;
    void *C;
    int64_t ldc;
};

template <typename T>
__device__ __forceinline__ T cvt_out(float v);
template <>
__device__ __forceinline__ float cvt_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 cvt_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half cvt_out<__half>(float v) { return __float2half_rn(v); }

template <typename TOut>
__global__ void __launch_bounds__(THREADS, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, GemmParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + STAGE * STAGES);
    uint64_t *empty = full + STAGES;
    uint64_t *acc_full = empty + STAGES;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_full + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int m_t = blockIdx.x % p.m_tiles, n_t = blockIdx.x / p.m_tiles;
    const int m0 = m_t * BM, n0 = n_t * BN;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        tc::mbar_init(acc_full, 1);
        *abort = 0;
        tc::fence_mbar_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, 512);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // row atoms of B in this tile that exist (the last tile may have one)
    const int b_atoms = n0 + 128 < p.N ? 2 : 1;

    if (warp == 0 && lane == 0) {
        tc::prefetch_tmap(&tmA);
        tc::prefetch_tmap(&tmB);
        for (int kb = 0; kb < p.kblocks; ++kb) {
            const int s = kb % STAGES;
            if (!tc::mbar_wait(&empty[s], ((kb / STAGES) & 1) ^ 1, abort)) break;
            uint8_t *a = smem + s * STAGE, *b = a + A_BYTES, *sa = b + B_BYTES, *sb = sa + SFA_BYTES;
            const int ka = p.nka - 2 * kb < 2 ? 1 : 2;
            tc::mbar_arrive_expect_tx(&full[s], A_BYTES + B_BYTES + ka * ATOM_BYTES * (1 + b_atoms));
            tc::tma_load_3d(a, &tmA, &full[s], kb * (BK / 2), m0, 0);
            tc::tma_load_3d(b, &tmB, &full[s], kb * (BK / 2), n0, 0);
            tc::bulk_load(sa, p.sfa + ((int64_t)m_t * p.nka + 2 * kb) * ATOM_BYTES, ka * ATOM_BYTES, &full[s]);
            for (int h = 0; h < b_atoms; ++h)
                tc::bulk_load(sb + h * 1024, p.sfb + ((int64_t)(2 * n_t + h) * p.nka + 2 * kb) * ATOM_BYTES,
                              ka * ATOM_BYTES, &full[s]);
        }
    } else if (warp == 1 && lane == 0) {
        for (int kb = 0; kb < p.kblocks; ++kb) {
            const int s = kb % STAGES;
            if (!tc::mbar_wait(&full[s], (kb / STAGES) & 1, abort)) break;
            tc::tc_fence_after();
            uint8_t *a = smem + s * STAGE, *b = a + A_BYTES, *sa = b + B_BYTES, *sb = sa + SFA_BYTES;
            const uint32_t tsa = tmem + BN + s * SF_COLS, tsb = tsa + 8;
            const int ka = p.nka - 2 * kb < 2 ? 1 : 2;
            for (int k = 0; k < ka; ++k) {
                tc::tmem_cp_scales(tsa + 4 * k, tc::smem_desc(sa + 512 * k, 128, 128, tc::SW_NONE));
                for (int h = 0; h < b_atoms; ++h)
                    tc::tmem_cp_scales(tsb + 8 * k + 4 * h,
                                       tc::smem_desc(sb + 1024 * h + 512 * k, 128, 128, tc::SW_NONE));
            }
            for (int k = 0; k < 2 * ka; ++k) {
                const uint32_t idesc = tc::idesc_mxf4(BM, BN, (k & 1) * 2);
                tc::mma_mxf4(tmem, tc::smem_desc(a + 32 * k, 16, 1024, tc::SW_128B),
                             tc::smem_desc(b + 32 * k, 16, 1024, tc::SW_128B), idesc, tsa + 4 * (k >> 1),
                             tsb + 8 * (k >> 1), (kb | k) != 0);
            }
            tc::mma_commit(&empty[s]);
        }
        tc::mma_commit(acc_full);
    } else if (warp >= 2) {
        const int q = warp & 3;
        const bool ok = tc::mbar_wait(acc_full, 0, abort);
        tc::tc_fence_after();
        if (ok) {
            TOut *C = static_cast<TOut *>(p.C);
            const int row = m0 + q * 32 + lane;
#pragma unroll 1
            for (int c = 0; c < BN / 32; ++c) {
                uint32_t r[32];
                tc::tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + c * 32, r);
                tc::tmem_ld_wait();
                const int col = n0 + c * 32;
                if (row >= p.M) continue;
                TOut *d = C + (int64_t)row * p.ldc + col;
                for (int i = 0; i < 32; ++i)
                    if (col + i < p.N) d[i] = cvt_out<TOut>(__uint_as_float(r[i]));
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, 512);
    }
}

}  // namespace mx4
}  // namespace act

extern "C" int actcomp_mx4_gemm(const actcomp_mx4 *a, const actcomp_mx4 *b, void *c, int64_t ldc, int32_t c_dtype,
                                void *stream) {
    using namespace act;
    using namespace act::mx4;
    if (int st = mx4_check(a)) return st;
    if (int st = mx4_check(b)) return st;
    ACT_CHECK(a->cols == b->cols && c && ldc >= b->rows && c_dtype >= 0 && c_dtype <= 2, ACT_E_INVALID);
    ACT_CHECK(aligned(c, c_dtype == 0 ? 4 : 2), ACT_E_ALIGN);
    const int64_t rb = row_bytes(a->cols);
    CUtensorMap tmA, tmB;
    int st = make_map_3d(&tmA, a->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rb, a->rows, 1, rb, 0, BK / 2, BM,
                         CU_TENSOR_MAP_SWIZZLE_128B);
    if (st) return st;
    st = make_map_3d(&tmB, b->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rb, b->rows, 1, rb, 0, BK / 2, BN,
                     CU_TENSOR_MAP_SWIZZLE_128B);
    if (st) return st;
    GemmParams p{};
    p.M = (int)a->rows;
    p.N = (int)b->rows;
    p.nka = (int)atoms_of(a->cols);
    p.kblocks = (p.nka + 1) / 2;
    p.m_tiles = (p.M + BM - 1) / BM;
    p.n_tiles = (p.N + BN - 1) / BN;
    p.sfa = a->scales;
    p.sfb = b->scales;
    p.C = c;
    p.ldc = ldc;
    ACT_CHECK((int64_t)p.m_tiles * p.n_tiles <= INT32_MAX, ACT_E_UNSUPPORTED);
    auto launch = [&](auto kern) -> int {
        ACT_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        kern<<<p.m_tiles * p.n_tiles, THREADS, SMEM, as_stream(stream)>>>(tmA, tmB, p);
        return launch_status();
    };
    if (c_dtype == 0) return launch(gemm_kernel<float>);
    if (c_dtype == 1) return launch(gemm_kernel<__nv_bfloat16>);
    return launch(gemm_kernel<__half>);
}
