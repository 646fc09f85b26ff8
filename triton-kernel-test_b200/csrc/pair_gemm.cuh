// pair_gemm.cuh -- C = A . B^T on CTA pairs (tcgen05 cta_group::2), the frame of the
// 8-bit product (fp8_gemm.cu) and of the cross entropy's products (xent.cu).
//
// A pair computes 256 x 256 tiles, persistent over the tile list; each CTA loads half
// of A and half of B (128 rows x 128 bytes of the contraction a stage) and holds half
// of the accumulator in its TMEM.  Either operand may be stored with the contraction
// contiguous (K-major) or its rows (MN-major).  Per CTA:
//   warp 0      TMA producer into a 128-byte-swizzled ring, counted on the first
//               CTA's barrier;
//   warp 1      TMEM allocation; in the first CTA the MMA issuer;
//   warps 2..5  epilogue, one accumulator row a thread (class Epi);
//   warps 6..9  16-bit operands: epilogue too, the other 128 columns;
//               8-bit operands: scales from memory to TMEM, every lane quadrant the
//               same, eight sets of 12 columns in turn; a set is written again only
//               after the commit of the MMAs that read it.
// TMEM (512 columns): two accumulators, so that a tile's epilogue runs beside the
// next tile's MMAs.  With scales they lie at 0 and 160 and share columns 160 to 255,
// which the epilogue empties first; then the next tile's MMAs start.
// Arrivals and waits at cluster scope (release.cluster 900 cycles, acquire.cluster
// 250) are avoided: the barriers hand over TMEM contents, ordered by the tcgen05
// fences, and tiles that only the async proxy touches.
// Rows, columns and contraction steps past the end of an operand are zero-filled by
// the TMA; what a scale byte past the end holds reaches only results past the end.
#pragma once

#include "fp8.cuh"
#include "tc_ptx.cuh"

namespace act {
namespace pair {

constexpr int BM = 256, BN = 256;  // of a pair
constexpr int THREADS = 320, STAGES = 6, SETS = 8;
constexpr int HALF_BYTES = 128 * 128;  // a CTA's half of A or of B: 128 rows x 128 bytes
constexpr int STAGE = 2 * HALF_BYTES;
constexpr int OUT_BYTES = 32 * 1024;  // staging of the output, over the epilogue warps
constexpr int RING = STAGE * STAGES;
constexpr int SMEM = 1024 + RING + OUT_BYTES + 512;
constexpr int SF_STEP = 12;  // TMEM columns of a scale set: A 4 words, B 2 x 4
static_assert(SMEM <= 232448, "placement");

enum Kind { F16 = 0, FP8 = 1 };
template <int KIND>
struct Tmem {
    static constexpr int ACC1 = KIND == FP8 ? 160 : 256;
    static constexpr int SHARED = KIND == FP8 ? (BN - ACC1) / 32 : 0;  // groups of 32 shared columns
    static constexpr int SF0 = ACC1 + BN;
    static constexpr int EPI_WARPS = KIND == FP8 ? 4 : 8;
    static constexpr int GROUPS = BN / 32 / (EPI_WARPS / 4);  // of 32 columns a warp takes
    static_assert(KIND == F16 || SF0 + SETS * SF_STEP <= 512, "TMEM");
};

// Scales of an operand: per line of 128 contraction steps in groups of 128 lines
// (fp8.cuh), or one per 128 x 128.
struct Scales {
    const uint8_t *p;
    int groups;       // of 128 lines
    int64_t step_k;   // bytes from one block of the contraction to the next
    int step_g;       // bytes from one group to the next; 128: a byte a line, else one byte for all
    int tiles;
};

struct Params {
    int M, N;
    int kblocks;  // stages of the contraction
    int m_tiles, n_tiles;
    int splits, k_split;  // parts that the contraction is cut into, and stages of one: every part has a tile list
    int a_mn, b_mn;
    uint32_t idesc;
    Scales sa, sb;
};

// Tiles in groups of 8 row tiles, rows fastest inside a group: the tiles that
// run at one time share A rows and B rows in L2.
struct Tile {
    int m, n, k0, k1, split;  // stages k0 .. k1 - 1
};
__device__ __forceinline__ Tile tile_of(int id, const Params &p) {
    const int per = p.m_tiles * p.n_tiles, split = id / per;
    id -= split * per;
    const int gsz = 8 * p.n_tiles, grp = id / gsz, first = grp * 8;
    const int gm = p.m_tiles - first < 8 ? p.m_tiles - first : 8;
    const int in = id - grp * gsz, k0 = split * p.k_split, k1 = k0 + p.k_split;
    return {first + in % gm, in / gm, k0, k1 < p.kblocks ? k1 : p.kblocks, split};
}
// Host: the tiles of an M x N result, its contraction in one part.
static inline void set_tiles(Params &p, int M, int N, int kblocks) {
    p.M = M, p.N = N, p.kblocks = p.k_split = kblocks, p.splits = 1;
    p.m_tiles = (M + BM - 1) / BM, p.n_tiles = (N + BN - 1) / BN;
}

// A lane's scale bytes of lines l, l + 32, l + 64, l + 96 of a group, as a word.
__device__ __forceinline__ uint32_t scale_word(const Scales &s, int kb, int g, int lane) {
    if (g >= s.groups) return 0u;
    const uint8_t *p = s.p + kb * s.step_k + (int64_t)g * s.step_g;
    return s.tiles ? __ldg(p) * 0x01010101u : __ldg(reinterpret_cast<const uint32_t *>(p) + lane);
}

template <typename T>
__device__ __forceinline__ T cvt_out(float v);
template <>
__device__ __forceinline__ float cvt_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 cvt_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half cvt_out<__half>(float v) { return __float2half_rn(v); }
template <typename T>
__device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
    const T a = cvt_out<T>(lo), b = cvt_out<T>(hi);
    return (uint32_t)(*reinterpret_cast<const uint16_t *>(&a)) |
           ((uint32_t)(*reinterpret_cast<const uint16_t *>(&b)) << 16);
}

struct OutParams {
    void *C;
    int64_t ldc;
    int tma;  // through a tensor map (tma_out)
};
// Host: whether a tensor map can take the output: 16-byte aligned base and rows, and
// rows of whole 16 bytes, since a store clipped inside 16 bytes writes zeros to their end.
static inline bool tma_out(const void *c, int64_t ldc, int64_t n, int es) {
    return aligned(c, 16) && (ldc * es) % 16 == 0 && (n * es) % 16 == 0;
}
// A warp's store of 32 rows x 32 columns (a row a lane) through swizzled shared memory.
// BYTES: the warp's staging space.
template <typename TOut, int BYTES>
struct Out {
    static constexpr int ES = (int)sizeof(TOut), TILE = 32 * 32 * ES, BUFS = BYTES / TILE;
    static_assert(BUFS >= 1, "staging");
    uint8_t *stage;
    int buf = 0;

    __device__ __forceinline__ void put(const float (&v)[32], int row0, int col, int M, int N, int lane,
                                        const OutParams &o, const CUtensorMap *tmC, int z = 0) {
        uint8_t *dst = stage + buf * TILE;
        tc::bulk_wait_read<(BUFS > 1 ? 1 : 0)>();  // the store that read this buffer has left it
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 2 * ES; ++c) {  // 16-byte chunks of a row
            uint4 q;
            if constexpr (ES == 4) {
                q = make_uint4(__float_as_uint(v[4 * c]), __float_as_uint(v[4 * c + 1]), __float_as_uint(v[4 * c + 2]),
                               __float_as_uint(v[4 * c + 3]));
            } else {
                q = make_uint4(pack_out<TOut>(v[8 * c], v[8 * c + 1]), pack_out<TOut>(v[8 * c + 2], v[8 * c + 3]),
                               pack_out<TOut>(v[8 * c + 4], v[8 * c + 5]), pack_out<TOut>(v[8 * c + 6], v[8 * c + 7]));
            }
            *reinterpret_cast<uint4 *>(dst + kmajor_swz<32 * ES>(lane, c)) = q;
        }
        if (o.tma) {
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0 && ACT_DCHECK(row0 < M && col < N)) {
                tc::tma_store_3d(tmC, dst, col, row0, z);
                tc::bulk_commit();
            }
            if (++buf == BUFS) buf = 0;
        } else {  // a row at a time, neighbouring lanes neighbouring columns
            __syncwarp();
            constexpr int PER = 16 / ES;
            const int rows = M - row0 < 32 ? M - row0 : 32;
            TOut *d = static_cast<TOut *>(o.C) + (int64_t)row0 * o.ldc + col + lane;
            if (col + lane < N && ACT_DCHECK(col + lane < o.ldc && row0 + rows <= M))
                for (int i = 0; i < rows; ++i, d += o.ldc)
                    *d = *reinterpret_cast<const TOut *>(dst + kmajor_swz<32 * ES>(i, lane / PER) + lane % PER * ES);
            __syncwarp();
        }
    }
};

// Epi: constructed once a thread with its parameters, the warp's staging space, the
// output's tensor map and the lane; per tile begin(p, tile, first of the warp's 32 rows,
// which half of the columns), then group(p, values, first column) per 32 columns (the same calls in every lane
// of a warp), then end(p); or lost(p) where a bounded wait gave up.
template <int KIND, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmC, const __grid_constant__ Params p,
                const __grid_constant__ typename Epi::P ep) {
    using L = Tmem<KIND>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *out_s = smem + RING;
    uint64_t *full = reinterpret_cast<uint64_t *>(out_s + OUT_BYTES);  // operands (first CTA's)
    uint64_t *empty = full + STAGES;
    uint64_t *acc_full = empty + STAGES;  // [2]
    uint64_t *acc_free = acc_full + 2;    // [2], first CTA's
    uint64_t *set_full = acc_free + 2;    // scale sets (first CTA's)
    uint64_t *set_free = set_full + SETS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(set_free + SETS);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x & 1;  // in the pair
    const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
    const int tiles = p.m_tiles * p.n_tiles * p.splits;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(&full[s], 1);
            tc::mbar_init(&empty[s], 1);
        }
        // The scales have barriers of their own: there are more sets than stages, so that their warps may be further
        // ahead than the producer, whose barriers they must not arrive on then.
        for (int i = 0; i < SETS; ++i) {
            tc::mbar_init(&set_full[i], 8);  // the pair's scale warps
            tc::mbar_init(&set_free[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&acc_full[i], 1);
            tc::mbar_init(&acc_free[i], 2 * L::EPI_WARPS);  // the pair's epilogue warps
        }
        *abort = 0;
        tc::fence_mbar_init();
    }
    if (threadIdx.x == 32) {
        tc::prefetch_tmap(&tmA);
        tc::prefetch_tmap(&tmB);
    }
    if (warp == 1) {
        __syncwarp();
        tc::tmem_alloc_pair(tmem_slot, 512);
        tc::tmem_relinquish_pair();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Launched with programmatic dependence: what is above runs beside the end of the
    // kernel before, nothing in memory is touched before it has ended.
    tc::dependence_wait();

    if (warp == 0 && lane == 0) {
        constexpr int BK = KIND == FP8 ? 128 : 64;  // values of a stage
        int s = 0;
        uint32_t phase = 1;
        bool ok = true;
        for (int t = cluster; t < tiles && ok; t += clusters) {
            const Tile tl = tile_of(t, p);
            const int m0 = tl.m * BM + 128 * (int)rank, n0 = tl.n * BN + 128 * (int)rank;
            for (int kb = tl.k0; kb < tl.k1; ++kb) {
                if (!(ok = tc::mbar_spin(&empty[s], phase, abort))) break;
                uint8_t *a = smem + s * STAGE, *b = a + HALF_BYTES;
                const uint32_t bar = tc::map_cluster(&full[s], 0);
                if (rank == 0) tc::mbar_arrive_expect_tx(&full[s], 2 * STAGE);
                const int k = kb * BK;
                if (!p.a_mn) {
                    tc::tma_load_3d_pair(a, &tmA, bar, k, m0, 0);
                } else {
                    tc::tma_load_3d_pair(a, &tmA, bar, m0, k, 0);
                    if constexpr (KIND == F16) tc::tma_load_3d_pair(a + 8192, &tmA, bar, m0 + 64, k, 0);
                }
                if (!p.b_mn) {
                    tc::tma_load_3d_pair(b, &tmB, bar, k, n0, 0);
                } else {
                    tc::tma_load_3d_pair(b, &tmB, bar, n0, k, 0);
                    if constexpr (KIND == F16) tc::tma_load_3d_pair(b + 8192, &tmB, bar, n0 + 64, k, 0);
                }
                if (++s == STAGES) s = 0, phase ^= 1;
            }
        }
    } else if (warp == 1 && rank == 0) {
        // Descriptors of the first stage; a stage further is STAGE / 16 in their address field, a step of the
        // contraction (32 bytes of it) 2, or MN-major 16 or 32 rows of 128 bytes.  One thread issues every MMA of
        // two SMs: the warp stays converged around it, so that the addresses are held in uniform registers.
        constexpr uint32_t MN_STEP = (KIND == FP8 ? 32 : 16) * 128 / 16;
        const uint64_t desc_a = p.a_mn ? tc::smem_desc(smem, 8192, 1024, tc::SW_128B)
                                       : tc::smem_desc(smem, 16, 1024, tc::SW_128B);
        const uint64_t desc_b = p.b_mn ? tc::smem_desc(smem + HALF_BYTES, 8192, 1024, tc::SW_128B)
                                       : tc::smem_desc(smem + HALF_BYTES, 16, 1024, tc::SW_128B);
        const uint32_t ka = p.a_mn ? MN_STEP : 2, kb_ = p.b_mn ? MN_STEP : 2, idesc = p.idesc;
        int s = 0, set = 0, turn = 0;
        uint32_t phase = 0, set_phase = 0;
        bool ok = true;
        for (int t = cluster; t < tiles && ok; t += clusters, ++turn) {
            const uint32_t acc = tmem + (turn & 1) * L::ACC1;
            if constexpr (KIND == FP8) {  // the columns shared with the tile before have been emptied
                if (turn > 0 && !tc::mbar_spin(&acc_free[(turn - 1) & 1], ((turn - 1) >> 1) & 1, abort)) break;
            } else {  // the accumulator has been emptied
                if (turn > 1 && !tc::mbar_spin(&acc_free[turn & 1], ((turn >> 1) - 1) & 1, abort)) break;
            }
            tc::tc_fence_after();
            const Tile tl = tile_of(t, p);
            const int steps = tl.k1 - tl.k0;
            for (int kb = 0; kb < steps; ++kb) {
                if constexpr (KIND == FP8)
                    if (!(ok = tc::mbar_spin(&set_full[set], set_phase, abort))) break;
                if (!(ok = tc::mbar_spin(&full[s], phase, abort))) break;
                tc::tc_fence_after();
                const uint64_t da = desc_a + (uint32_t)(s * (STAGE / 16)), db = desc_b + (uint32_t)(s * (STAGE / 16));
                if (tc::elect_one()) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (KIND == FP8) {
                            const uint32_t tsa = tmem + L::SF0 + set * SF_STEP;
                            tc::mma_mxf8_pair(acc, da + i * ka, db + i * kb_, idesc, tsa, tsa + 4, (kb | i) != 0);
                        } else {
                            tc::mma_f16_pair(acc, da + i * ka, db + i * kb_, idesc, (kb | i) != 0);
                        }
                    }
                    tc::mma_commit_pair(&empty[s]);
                    if constexpr (KIND == FP8) tc::mma_commit_pair(&set_free[set]);
                }
                __syncwarp();
                if (++s == STAGES) s = 0, phase ^= 1;
                if (++set == SETS) set = 0, set_phase ^= 1;
            }
            if (tc::elect_one()) tc::mma_commit_pair(&acc_full[turn & 1]);
            __syncwarp();
        }
    } else if (warp >= 2 && warp < 2 + L::EPI_WARPS) {
        const int q = warp & 3;  // TMEM lane quadrant this warp may access
        const int half = (warp - 2) >> 2, first = half * L::GROUPS;
        constexpr int ROOM = OUT_BYTES / L::EPI_WARPS;
        Epi epi(ep, out_s + (warp - 2) * ROOM, &tmC, lane);
        int turn = 0;
        for (int t = cluster; t < tiles; t += clusters, ++turn) {
            const Tile tl = tile_of(t, p);
            const int n0 = tl.n * BN;
            epi.begin(p, tl, tl.m * BM + 128 * (int)rank + 32 * q, half);
            if (!tc::mbar_spin(&acc_full[turn & 1], (turn >> 1) & 1, abort)) {
                epi.lost(p);  // the abort word is set: the later tiles' waits end at once
                continue;
            }
            tc::tc_fence_after();
            const uint32_t acc = tmem + (turn & 1) * L::ACC1 + ((uint32_t)(q * 32) << 16);
            const uint32_t free_bar = tc::map_cluster(&acc_free[turn & 1], 0);
            auto release = [&] {
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive_remote_tmem(free_bar);
            };
            if constexpr (KIND == FP8) {
                // the shared columns: the first accumulator's last, the second's first
                const int g0 = (turn & 1) ? 0 : BN / 32 - L::SHARED;
                {
                    uint32_t r[L::SHARED][32];
#pragma unroll
                    for (int i = 0; i < L::SHARED; ++i) tc::tmem_ld32(acc + (g0 + i) * 32, r[i]);
#pragma unroll
                    for (int i = 0; i < L::SHARED; ++i) tc::tmem_ld_wait(r[i]);
                    release();
#pragma unroll
                    for (int i = 0; i < L::SHARED; ++i) epi.group(p, r[i], n0 + (g0 + i) * 32);
                }
                const int g1 = (turn & 1) ? L::SHARED : 0;
#pragma unroll 1
                for (int g = g1; g < g1 + BN / 32 - L::SHARED; ++g) {
                    uint32_t r[32];
                    tc::tmem_ld32(acc + g * 32, r);
                    tc::tmem_ld_wait(r);
                    epi.group(p, r, n0 + g * 32);
                }
            } else {
                // two groups in hand: the second's load beside the first's arithmetic
                uint32_t r[2][32];
                tc::tmem_ld32(acc + first * 32, r[0]);
                tc::tmem_ld_wait(r[0]);
#pragma unroll
                for (int g = 0; g < L::GROUPS; ++g) {
                    if (g + 1 < L::GROUPS) tc::tmem_ld32(acc + (first + g + 1) * 32, r[(g + 1) & 1]);
                    epi.group(p, r[g & 1], n0 + (first + g) * 32);
                    if (g + 1 < L::GROUPS) tc::tmem_ld_wait(r[(g + 1) & 1]);
                    if (g + 2 == L::GROUPS) release();
                }
            }
            epi.end(p);
        }
        tc::bulk_wait<0>();
    } else if (KIND == FP8 && warp >= 6) {
        const uint32_t quad = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        constexpr int AHEAD = 4;  // stages whose words are on their way, and written, together
        // the words of stages k0 .. of tile t, past its last one those of the last
        auto fetch = [&](uint32_t (&w)[AHEAD][3], const Tile &tl, int k0) {
            const int ga = tl.m * 2 + (int)rank, gb = tl.n * 2;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int kb = k0 + i < tl.k1 ? k0 + i : tl.k1 - 1;
                w[i][0] = scale_word(p.sa, kb, ga, lane);
                w[i][1] = scale_word(p.sb, kb, gb, lane);
                w[i][2] = scale_word(p.sb, kb, gb + 1, lane);
            }
        };
        int it = 0, t = cluster;
        bool ok = t < tiles;
        Tile tl = tile_of(ok ? t : 0, p);
        int k0 = tl.k0;
        uint32_t next[AHEAD][3];
        if (ok) fetch(next, tl, k0);
        while (ok) {
            uint32_t w[AHEAD][3];
            memcpy(w, next, sizeof(w));
            const int n = tl.k1 - k0 < AHEAD ? tl.k1 - k0 : AHEAD;
            // the words after these are asked for before these are needed
            bool more = true;
            if ((k0 += AHEAD) >= tl.k1) {
                if ((more = (t += clusters) < tiles)) tl = tile_of(t, p), k0 = tl.k0;
            }
            if (more) fetch(next, tl, k0);
            // several stages' words at once: the stores' latency, not their number, is what a turn here takes
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (i >= n) break;
                // the set's earlier MMAs are done
                const int set = (it + i) % SETS;
                if (it + i >= SETS && !(ok = tc::mbar_spin(&set_free[set], ((it + i) / SETS - 1) & 1, abort))) break;
                tc::tc_fence_after();
                uint32_t u[8];
                const uint32_t d = quad + L::SF0 + set * SF_STEP;
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = w[i][0] >> (8 * j), u[4 + j] = w[i][1] >> (8 * j);
                tc::tmem_st8(d, u);
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = w[i][2] >> (8 * j);
                tc::tmem_st4(d + 8, u);
            }
            tc::tmem_st_wait();
            tc::tc_fence_before();
            __syncwarp();
            if (lane < n && ok) tc::mbar_arrive_remote_tmem(tc::map_cluster(&set_full[(it + lane) % SETS], 0));
            __syncwarp();
            it += n;
            if (!more) break;
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::drain_after_abort(abort);
    __syncwarp();
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

template <int KIND, class Epi>
static int launch(const CUtensorMap &tmA, const CUtensorMap &tmB, const CUtensorMap &tmC, const Params &p,
                  const typename Epi::P &ep, cudaStream_t st) {
    auto kern = pair_kernel<KIND, Epi>;
    ACT_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    const int tiles = p.m_tiles * p.n_tiles * p.splits, pairs = max_pairs(kern);
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(2 * (tiles < pairs ? tiles : pairs)));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    ACT_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmC, p, ep));
    return ACT_OK;
}

}  // namespace pair
}  // namespace act
