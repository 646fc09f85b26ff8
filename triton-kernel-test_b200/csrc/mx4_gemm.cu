// mx4_gemm.cu -- the product of two microscaled 4-bit matrices, C = A . B^T,
// on the block-scaled tensor cores (tcgen05.mma kind::mxf4).
//
// C[m][n] = sum over blocks of 32 columns of 2^(ea + eb - 254) sum_j a_j b_j,
// both operands K-major as stored, float32 accumulation in TMEM.
//
// A pair of CTAs (cta_group::2) computes 256 x 256 tiles, persistent over the
// tile list; each CTA loads half of A and half of B and holds half of the
// accumulator in its TMEM, so that 64 bytes a cycle and SM of operands come from
// L2 at the MMAs' full rate.  Per CTA:
//   warp 0      TMA producer: 256 columns (128 bytes a row) of 128 rows of A and
//               of B into a 128-byte-swizzled ring, counted on the first CTA's
//               barrier, and the scale atoms (512 bytes per 128 rows x 128
//               columns) of its A rows and of all 256 B rows, counted on its own;
//   warp 1      TMEM allocation; in the first CTA the MMA issuer;
//   warps 2..5  epilogue: TMEM to registers, convert, swizzled shared memory,
//               TMA store (rows or bases that are not 16-byte aligned, or rows that
//               do not end on 16 bytes: plain stores);
//   warps 6..9  scales: shared memory to TMEM, every lane quadrant the same, four
//               sets of 256 columns in turn; a set is written again only after
//               the commit of the MMAs that read it.
// TMEM (512 columns): accumulators at 0 and 160 that share columns 160 to 255,
// scale sets from 416.  The epilogue empties the shared columns first and then
// lets the next tile's MMAs start.
//
// Measured at 16384 x 4096 x 11008, us (operands in L2):
//   240  the MMAs alone (4 per 256 columns, no loads, scales or barriers)
//   249  this kernel: 5.94 PFLOP/s
//   302  256 x 192 tiles, two separate accumulators, five scale sets: an MMA's
//        time grows by 40 cycles less than in proportion to N
//   493  scales by tcgen05.cp: each change between copies and MMAs drains the
//        tensor pipe (about 300 cycles, three copies or six)
// Arrivals and waits at cluster scope (release.cluster 900 cycles, acquire.cluster
// 250) are avoided: the barriers hand over TMEM contents, ordered by the tcgen05
// fences, and tiles that only the async proxy touches.
// Rows and columns past the end of an operand are zero-filled by the TMA (codes
// 0, scale byte 0 = 2^-127): their products are 0.
#include <cuda_fp16.h>

#include "mx4.cuh"
#include "tc_ptx.cuh"

namespace act {
int mx4_check(const actcomp_mx4 *q);
namespace mx4 {

constexpr int BM = 256, BN = 256, BK = 256;  // of a pair; BK in values
constexpr int THREADS = 320, STAGES = 5, SETS = 4;
constexpr int HALF_BYTES = 128 * BK / 2;  // a CTA's half of A or of B
constexpr int SFA_BYTES = 1024, SFB_BYTES = 2048;  // two column atoms x (one | two) row atoms
constexpr int STAGE = 2 * HALF_BYTES + SFA_BYTES + SFB_BYTES;
constexpr int OUT_BYTES = 2 * 4096;  // two staging buffers of 32 rows x up to 128 bytes per epilogue warp
constexpr int RING = STAGE * STAGES;
constexpr int SMEM = 1024 + RING + 4 * OUT_BYTES + 512;
// TMEM columns: second accumulator, shared groups of 32, scale sets (A 2 x 4, B 2 x 8 words)
constexpr int ACC1 = 160, SHARED = (BN - ACC1) / 32, SF0 = ACC1 + BN, SF_STEP = 24;
static_assert(STAGE % 1024 == 0 && SF0 + SETS * SF_STEP <= 512 && SMEM <= 232448 && SETS < STAGES, "placement");

struct GemmParams {
    int M, N;
    int nka;  // atoms of 128 columns
    int m_tiles, n_tiles;
    void *C;
    int64_t ldc;
    int tma_out;
};

template <typename T>
__device__ __forceinline__ T cvt_out(float v);
template <>
__device__ __forceinline__ float cvt_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 cvt_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half cvt_out<__half>(float v) { return __float2half_rn(v); }
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const T a = cvt_out<T>(lo), b = cvt_out<T>(hi);
    return (uint32_t)(*reinterpret_cast<const uint16_t *>(&a)) |
           ((uint32_t)(*reinterpret_cast<const uint16_t *>(&b)) << 16);
}

// Tiles in groups of 8 row tiles, rows fastest inside a group: the tiles that
// run at one time share A rows and B rows in L2.
__device__ __forceinline__ void tile_of(int id, const GemmParams &p, int &m_t, int &n_t) {
    const int gsz = 8 * p.n_tiles, grp = id / gsz, first = grp * 8;
    const int gm = p.m_tiles - first < 8 ? p.m_tiles - first : 8;
    const int in = id - grp * gsz;
    m_t = first + in % gm;
    n_t = in / gm;
}

template <typename TOut>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                     const __grid_constant__ CUtensorMap tmC, GemmParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *out_s = smem + RING;
    uint64_t *full = reinterpret_cast<uint64_t *>(out_s + 4 * OUT_BYTES);  // operands (first CTA's)
    uint64_t *sfull = full + STAGES;                                      // scale atoms (own)
    uint64_t *empty = sfull + STAGES;
    uint64_t *acc_full = empty + STAGES;  // [2]
    uint64_t *acc_free = acc_full + 2;      // the shared columns (first CTA's)
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_free + 1);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;  // in the pair
    const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
    const int tiles = p.m_tiles * p.n_tiles, kblocks = (p.nka + 1) >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(&full[s], 9);  // the producer, and one arrival per scale warp of the pair
            tc::mbar_init(&sfull[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        tc::mbar_init(&acc_full[0], 1);
        tc::mbar_init(&acc_full[1], 1);
        tc::mbar_init(acc_free, 8);  // one arrival per epilogue warp of the pair
        *abort = 0;
        tc::fence_mbar_init();
    }
    if (warp == 1) {
        tc::tmem_alloc_pair(tmem_slot, 512);
        tc::tmem_relinquish_pair();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0 && lane == 0) {
        tc::prefetch_tmap(&tmA);
        tc::prefetch_tmap(&tmB);
        int it = 0;
        bool ok = true;
        for (int t = cluster; t < tiles && ok; t += clusters) {
            int m_t, n_t;
            tile_of(t, p, m_t, n_t);
            const int m0 = m_t * BM + 128 * (int)rank, n0 = n_t * BN;
            for (int kb = 0; kb < kblocks; ++kb, ++it) {
                const int s = it % STAGES;
                if (!(ok = tc::mbar_spin(&empty[s], ((it / STAGES) & 1) ^ 1, abort))) break;
                uint8_t *a = smem + s * STAGE, *b = a + HALF_BYTES, *sa = b + HALF_BYTES, *sb = sa + SFA_BYTES;
                const uint32_t bar = tc::map_cluster(&full[s], 0);
                tc::mbar_arrive_expect_tx(&sfull[s], SFA_BYTES + SFB_BYTES);
                tc::tma_load_3d(sa, &tmSA, &sfull[s], 0, 2 * kb, m0 >> 7);
                tc::tma_load_3d(sb, &tmSB, &sfull[s], 0, 2 * kb, n0 >> 7);
                if (rank == 0) tc::mbar_arrive_expect_tx(&full[s], 4 * HALF_BYTES);
                tc::tma_load_3d_pair(a, &tmA, bar, kb * (BK / 2), m0, 0);
                tc::tma_load_3d_pair(b, &tmB, bar, kb * (BK / 2), n0 + BN / 2 * (int)rank, 0);
            }
        }
    } else if (warp == 1 && rank == 0) {
        // Descriptors of the first stage; a stage further is STAGE / 16 and a K step of 32 bytes 2 in their
        // address field.  One thread issues every MMA of two SMs: the warp stays converged around it, so that
        // the addresses are held in uniform registers.
        const uint64_t desc_a = tc::smem_desc(smem, 16, 1024, tc::SW_128B);
        const uint64_t desc_b = tc::smem_desc(smem + HALF_BYTES, 16, 1024, tc::SW_128B);
        constexpr uint32_t ID0 = tc::idesc_mxf4(BM, BN, 0), ID1 = tc::idesc_mxf4(BM, BN, 2);
        int s = 0, set = 0, turn = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = cluster; t < tiles && ok; t += clusters, ++turn) {
            const uint32_t acc = tmem + (turn & 1) * ACC1;
            // the epilogues have emptied the columns shared with the tile before
            if (turn > 0 && !tc::mbar_spin(acc_free, (turn - 1) & 1, abort)) break;
            for (int kb = 0; kb < kblocks; ++kb) {
                if (!(ok = tc::mbar_spin(&full[s], phase, abort))) break;
                tc::tc_fence_after();
                const uint64_t da = desc_a + (uint32_t)(s * (STAGE / 16)), db = desc_b + (uint32_t)(s * (STAGE / 16));
                const uint32_t tsa = tmem + SF0 + set * SF_STEP, tsb = tsa + 8;
                if (tc::elect_one()) {
                    tc::mma_mxf4_pair(acc, da, db, ID0, tsa, tsb, kb != 0);
                    tc::mma_mxf4_pair(acc, da + 2, db + 2, ID1, tsa, tsb, 1);
                    if (2 * kb + 1 < p.nka) {
                        tc::mma_mxf4_pair(acc, da + 4, db + 4, ID0, tsa + 4, tsb + 8, 1);
                        tc::mma_mxf4_pair(acc, da + 6, db + 6, ID1, tsa + 4, tsb + 8, 1);
                    }
                    tc::mma_commit_pair(&empty[s]);
                }
                __syncwarp();
                if (++s == STAGES) s = 0, phase ^= 1;
                if (++set == SETS) set = 0;
            }
            if (tc::elect_one()) tc::mma_commit_pair(&acc_full[turn & 1]);
            __syncwarp();
        }
    } else if (warp >= 2 && warp < 6) {
        const int q = warp & 3;  // TMEM lane quadrant this warp may access
        uint8_t *stage = out_s + q * OUT_BYTES;
        const uint32_t free_bar = tc::map_cluster(acc_free, 0);
        constexpr int ES = (int)sizeof(TOut);
        int turn = 0, buf = 0;
        for (int t = cluster; t < tiles; t += clusters, ++turn) {
            int m_t, n_t;
            tile_of(t, p, m_t, n_t);
            const int row0 = m_t * BM + 128 * (int)rank + 32 * q, n0 = n_t * BN;
            if (!tc::mbar_spin(&acc_full[turn & 1], (turn >> 1) & 1, abort)) break;
            tc::tc_fence_after();
            const uint32_t acc = tmem + (turn & 1) * ACC1 + ((uint32_t)(q * 32) << 16);
            auto put = [&](int g, const uint32_t (&r)[32]) {
                const int col = n0 + g * 32;
                if (row0 >= p.M || col >= p.N) return;
                uint8_t *dst = stage + buf * 4096;
                tc::bulk_wait_read<1>();  // lane 0's store before the last has left this buffer
                __syncwarp();
#pragma unroll
                for (int c = 0; c < 2 * ES; ++c) {  // 16-byte chunks of a row
                    uint4 v;
                    if constexpr (ES == 4) {
                        v = make_uint4(r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]);
                    } else {
                        const auto F = [&](int j) { return __uint_as_float(r[8 * c + j]); };
                        v = make_uint4(pack2<TOut>(F(0), F(1)), pack2<TOut>(F(2), F(3)), pack2<TOut>(F(4), F(5)),
                                       pack2<TOut>(F(6), F(7)));
                    }
                    *reinterpret_cast<uint4 *>(dst + kmajor_swz<32 * ES>(lane, c)) = v;
                }
                if (p.tma_out) {
                    tc::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0 && ACT_DCHECK(row0 < p.M && col < p.N)) {
                        tc::tma_store_3d(&tmC, dst, col, row0, 0);
                        tc::bulk_commit();
                    }
                    buf ^= 1;
                } else {  // a row at a time, neighbouring lanes neighbouring columns
                    __syncwarp();
                    constexpr int PER = 16 / ES;
                    const int rows = p.M - row0 < 32 ? p.M - row0 : 32;
                    TOut *d = static_cast<TOut *>(p.C) + (int64_t)row0 * p.ldc + col + lane;
                    if (col + lane < p.N && ACT_DCHECK(col + lane < p.ldc && row0 + rows <= p.M))
                        for (int i = 0; i < rows; ++i, d += p.ldc)
                            *d = *reinterpret_cast<const TOut *>(dst + kmajor_swz<32 * ES>(i, lane / PER) +
                                                                 lane % PER * ES);
                    __syncwarp();
                }
            };
            // the shared columns: the first accumulator's last, the second's first
            const int g0 = (turn & 1) ? 0 : BN / 32 - SHARED;
            {
                uint32_t r[SHARED][32];
#pragma unroll
                for (int i = 0; i < SHARED; ++i) tc::tmem_ld32(acc + (g0 + i) * 32, r[i]);
                tc::tmem_ld_wait();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive_remote_tmem(free_bar);
#pragma unroll
                for (int i = 0; i < SHARED; ++i) put(g0 + i, r[i]);
            }
            const int g1 = (turn & 1) ? SHARED : 0;
#pragma unroll 1
            for (int g = g1; g < g1 + BN / 32 - SHARED; ++g) {
                uint32_t r[32];
                tc::tmem_ld32(acc + g * 32, r);
                tc::tmem_ld_wait();
                put(g, r);
            }
        }
        tc::bulk_wait<0>();
    } else if (warp >= 6) {
        const uint32_t quad = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        int it = 0;
        bool ok = true;
        for (int t = cluster; t < tiles && ok; t += clusters) {
            for (int kb = 0; kb < kblocks; ++kb, ++it) {
                const int s = it % STAGES;
                if (!(ok = tc::mbar_wait(&sfull[s], (it / STAGES) & 1, abort))) break;
                const uint8_t *sa = smem + s * STAGE + 2 * HALF_BYTES, *sb = sa + SFA_BYTES;
                // a lane's words: rows lane, lane + 32, ... of each atom
                uint32_t u[8], v[16];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(sa + 512 * h + 16 * lane);
                    u[4 * h] = x.x, u[4 * h + 1] = x.y, u[4 * h + 2] = x.z, u[4 * h + 3] = x.w;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint4 y = *reinterpret_cast<const uint4 *>(sb + 1024 * i + 512 * h + 16 * lane);
                        uint32_t *w = v + 8 * h + 4 * i;
                        w[0] = y.x, w[1] = y.y, w[2] = y.z, w[3] = y.w;
                    }
                }
                // the set's earlier MMAs are done
                if (it >= SETS &&
                    !(ok = tc::mbar_spin(&empty[(it - SETS) % STAGES], ((it - SETS) / STAGES) & 1, abort)))
                    break;
                tc::tc_fence_after();
                const uint32_t d = quad + SF0 + it % SETS * SF_STEP;
                tc::tmem_st8(d, u);
                tc::tmem_st16(d + 8, v);
                tc::tmem_st_wait();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive_remote_tmem(tc::map_cluster(&full[s], 0));
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();  // neither CTA leaves while the other may still read its shared memory or signal it
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc_pair(tmem, 512);
    }
}

// Resident pairs on the device (its SM count, less what cluster placement leaves over).
template <typename K>
static int max_pairs(K kern) {
    static int cache[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    if (!cache[dev]) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(num_sms() & ~1);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = SMEM;
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim = {2, 1, 1};
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
            cudaGetLastError();
            n = num_sms() / 2;
        }
        cache[dev] = n;
    }
    return cache[dev];
}

template <typename TOut>
static int launch_pair(const CUtensorMap &tmA, const CUtensorMap &tmB, const CUtensorMap &tmSA, const CUtensorMap &tmSB,
                       const CUtensorMap &tmC, const GemmParams &p, cudaStream_t st) {
    auto kern = gemm_pair_kernel<TOut>;
    ACT_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    const int tiles = p.m_tiles * p.n_tiles, pairs = max_pairs(kern);
    kern<<<2 * (tiles < pairs ? tiles : pairs), THREADS, SMEM, st>>>(tmA, tmB, tmSA, tmSB, tmC, p);
    return launch_status();
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
    const int es = c_dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(c, es), ACT_E_ALIGN);
    GemmParams p{};
    p.M = (int)a->rows;
    p.N = (int)b->rows;
    p.nka = (int)atoms_of(a->cols);
    p.m_tiles = (p.M + BM - 1) / BM;
    p.n_tiles = (p.N + BN - 1) / BN;
    p.C = c;
    p.ldc = ldc;
    // rows of whole 16 bytes: a tile store that is clipped inside 16 bytes writes zeros to their end
    p.tma_out = aligned(c, 16) && (ldc * es) % 16 == 0 && ((int64_t)p.N * es) % 16 == 0;
    ACT_CHECK((int64_t)p.m_tiles * p.n_tiles <= INT32_MAX, ACT_E_UNSUPPORTED);
    const int64_t rb = row_bytes(a->cols);
    CUtensorMap tmA, tmB, tmSA, tmSB, tmC;
    int st = make_map_3d(&tmA, a->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rb, p.M, 1, rb, 0, BK / 2, 128,
                         CU_TENSOR_MAP_SWIZZLE_128B);
    if (!st)
        st = make_map_3d(&tmB, b->codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rb, p.N, 1, rb, 0, BK / 2, BN / 2,
                         CU_TENSOR_MAP_SWIZZLE_128B);
    // scale atoms as 128 words: (row atom, column atom, word)
    auto scale_map = [&](CUtensorMap *m, const actcomp_mx4 *q, uint32_t row_atoms) {
        return make_map_3d_box(m, q->scales, CU_TENSOR_MAP_DATA_TYPE_INT32, 4, 128, p.nka, (q->rows + 127) / 128, 128,
                               (uint64_t)p.nka * 128, 128, 2, row_atoms, CU_TENSOR_MAP_SWIZZLE_NONE);
    };
    if (!st) st = scale_map(&tmSA, a, 1);
    if (!st) st = scale_map(&tmSB, b, 2);
    tmC = tmA;  // not read when tma_out is 0
    if (!st && p.tma_out)
        st = make_map_3d(&tmC, c,
                         c_dtype == 0   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                         : c_dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                        : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         es, p.N, p.M, 1, ldc, 0, 32, 32, es == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
    if (st) return st;
    cudaStream_t s = as_stream(stream);
    if (c_dtype == 0) return launch_pair<float>(tmA, tmB, tmSA, tmSB, tmC, p, s);
    if (c_dtype == 1) return launch_pair<__nv_bfloat16>(tmA, tmB, tmSA, tmSB, tmC, p, s);
    return launch_pair<__half>(tmA, tmB, tmSA, tmSB, tmC, p, s);
}
