// norm.cu -- dropout without a stored mask, layer norm with its backward pass,
// and the two fused across a residual branch (no reference counterpart: the
// reference's low_rank_system_profile_backward.py covers the linear layers
// between them).
//
//   dropout    y = kept ? x * scale : 0                     (mask: philox.cuh)
//   forward    h = residual + dropout(x)                    (fused form only)
//              mean = sum h / n, rstd = 1 / sqrt(sum (h - mean)^2 / n + eps)
//              y = (h - mean) * rstd * w + b
//   backward   g = dy * w, xh = (h - mean) * rstd
//              dr = rstd * (g - sum g / n - xh * sum(g xh) / n) (+ dh)
//              dx = dropout(dr)                             (fused form only)
//              dw = sum over rows of dy * xh, db = sum over rows of dy
//
// All arithmetic is float32 on values rounded once at the end; the fused
// forward normalises the unrounded float32 h.  HBM-bound: each tensor crosses
// memory once.  A row's values stay in registers between the passes over it
// (mean, then squares about the mean, then the output), which also gives the
// variance without the cancellation of a sum of squares.
//
// Work split.  A warp holds a row in segments of 256 values, eight a lane: a
// lane's own eight consecutive values where 16-byte access is possible (VEC),
// else values lane, lane + 32, ... of the segment, so that narrow accesses still
// coalesce; the lane then makes the generator call of block `lane` of the
// segment and the keep bits travel by shuffle.  Rows arrive ahead of their use
// by bulk copies into shared memory (RowRing).  Persistent CTAs: weights and the
// weight-gradient sums stay in registers from row to row.  Short rows take a warp
// or a group of warps each, rows of up to 16384 values a CTA; longer ones go
// through kernels that re-read the row, and so do float32 rows of the backward pass
// that leave no two ring slots in shared memory: past 13952 values, with dropout
// (three inputs) past 9300.
//
// Measured on a B200, 16384 x 4096 bf16 (share of the copy rate, 6.47 TB/s):
//   dropout                 60 us  4.5 TB/s  70 %  (float32 87 us, 95 %)
//   forward                 47 us  5.7 TB/s  88 %
//   backward                70 us  5.7 TB/s  89 %
//   branch forward          97 us  5.5 TB/s  86 %
//   branch backward        122 us  5.5 TB/s  85 %
// The bf16 dropout saturates no pipe (issue slots 58 %, FMA 67 %); ten generator
// rounds instead of one are 10 of its 60 us.  p = 0 draws its masks all the same.
// Before the ring (loads in the row's own time) forward took 123 us and backward
// 245; value by value instead of in pairs 90 and 112.  Ragged rows (16384 x 4097)
// take 92 and 212 us, with dropout 224 and 346: two-byte accesses, four times the
// instructions, and spilled registers (59 of the ragged forms, up to 260 bytes).
// Longer rows at 8192 rows bf16 (floor; backward and branch backward): 6144 values 64
// (47) and 104 (78) us, 8192 76 (62) and 123 (104), 9216 134 (70) and 217 (117), 11008
// 141 (84) and 221 (139), 16384 182 (125) and 288 (208): one CTA per SM there.
#include <cuda_fp16.h>
#include <string.h>

#include <type_traits>

#include "philox.cuh"
#include "tc_ptx.cuh"

namespace act {
namespace norm {

constexpr int SEG = 256;            // values of a warp's segment
constexpr int MAX_SEGS = 64;        // longest row held in registers: 16384 values
constexpr int LONG_THREADS = 512;
constexpr int SLOT_ROOM = 218 * 1024;  // shared memory for row slots

// ---------------------------------------------------------------- types
template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Eight values as they lie in memory.
template <typename T>
struct alignas(16) Raw8 {
    T v[8];
};
// Their float32 values in pairs (packed f32x2 arithmetic takes two at a time).
struct F8 {
    float2 p[4];
};

template <typename T>
__device__ __forceinline__ F8 unpack(const Raw8<T> &r) {
    F8 f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
            f.p[j] = make_float2(to_f<T>(r.v[2 * j]), to_f<T>(r.v[2 * j + 1]));
        } else {
            uint32_t w;
            memcpy(&w, &r.v[2 * j], 4);
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                f.p[j] = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
            } else {
                __half2 h;
                memcpy(&h, &w, 4);
                f.p[j] = __half22float2(h);
            }
        }
    }
    return f;
}
template <typename T>
__device__ __forceinline__ Raw8<T> pack(const F8 &f) {
    Raw8<T> r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
            r.v[2 * j] = f.p[j].x, r.v[2 * j + 1] = f.p[j].y;
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 h = __float22bfloat162_rn(f.p[j]);
            memcpy(&r.v[2 * j], &h, 4);
        } else {
            const __half2 h = __float22half2_rn(f.p[j]);
            memcpy(&r.v[2 * j], &h, 4);
        }
    }
    return r;
}

// Keeps loop-invariant 16-bit values packed: without it their unpacked form is
// carried through the loop in twice the registers.
template <typename T>
__device__ __forceinline__ void stay_packed(Raw8<T> &r) {
    if constexpr (sizeof(T) == 2) {
        uint32_t q[4];
        memcpy(q, &r, 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("" : "+r"(q[i]));
        memcpy(&r, q, 16);
    }
}

// Number of the lane's eight values of the segment at `seg0` that lie in a row
// of n values (VEC: 8 or 0, the row length is a multiple of 8).
// A lane's values: VEC seg0 + 8 lane + j; else seg0 + 32 j + lane.
template <bool VEC>
__device__ __forceinline__ int count_of(int64_t seg0, int64_t n, int lane) {
    const int64_t left = n - seg0 - (VEC ? 8 * lane : lane);
    const int count = VEC ? (left > 0 ? 8 : 0) : left <= 0 ? 0 : (left > 224 ? 8 : (int)((left + 31) >> 5));
    return ACT_DCHECK(count == 0 || (VEC ? 8 : 32 * (count - 1) + 1) <= left) ? count : 0;
}

// Values outside the row read as `fill`.
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load8(const T *row, int64_t seg0, int count, int lane, float fill = 0.f) {
    Raw8<T> r;
    if constexpr (VEC) {
        if (count) {
            const uint4 *s = reinterpret_cast<const uint4 *>(row + seg0 + 8 * lane);
            uint4 q[sizeof(r) / 16];
#pragma unroll
            for (int i = 0; i < (int)sizeof(r) / 16; ++i) q[i] = s[i];
            memcpy(&r, q, sizeof(r));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) r.v[j] = from_f<T>(fill);
        }
    } else {
        const T *s = row + seg0 + lane;
#pragma unroll
        for (int j = 0; j < 8; ++j) r.v[j] = j < count ? s[32 * j] : from_f<T>(fill);
    }
    return r;
}
// The same of a weight vector that may be absent.
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load8_or(const T *row, float absent, int64_t seg0, int count, int lane) {
    return load8<T, VEC>(row, seg0, row ? count : 0, lane, absent);
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T *row, int64_t seg0, int count, int lane, const F8 &f) {
    const Raw8<T> r = pack<T>(f);
    if constexpr (VEC) {
        if (!count) return;
        uint4 q[sizeof(r) / 16];
        memcpy(q, &r, sizeof(r));
        uint4 *d = reinterpret_cast<uint4 *>(row + seg0 + 8 * lane);
#pragma unroll
        for (int i = 0; i < (int)sizeof(r) / 16; ++i) d[i] = q[i];
    } else {
        T *d = row + seg0 + lane;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) d[32 * j] = r.v[j];
    }
}

// x * scale where kept, else 0 (whatever x holds).  All lanes of the warp call it.
template <bool VEC>
__device__ __forceinline__ F8 drop8(const F8 &x, uint64_t row, int64_t seg0, int lane, uint64_t key,
                                    const DropParams &d) {
    F8 y;
    const float2 sc = make_float2(d.scale, d.scale);
    const uint32_t block = (uint32_t)(seg0 >> 3) + lane;
    if constexpr (VEC) {
        const uint4 r = philox4x32_10(block, (uint32_t)row, (uint32_t)(row >> 32), key);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = mul2(x.p[j], sc);
            y.p[j] = make_float2((w[j] & 0xffffu) >= d.threshold ? t.x : 0.f, (w[j] >> 16) >= d.threshold ? t.y : 0.f);
        }
    } else {
        const uint32_t mine = drop_keep8(row, block, key, d.threshold);
        // value 32 j + lane belongs to block 4 j + lane / 8
        const uint32_t bit = 1u << (lane & 7);
        uint32_t k[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) k[j] = __shfl_sync(0xffffffffu, mine, 4 * j + (lane >> 3)) & bit;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = mul2(x.p[j], sc);
            y.p[j] = make_float2(k[2 * j] ? t.x : 0.f, k[2 * j + 1] ? t.y : 0.f);
        }
    }
    return y;
}

// ---------------------------------------------------------------- dropout
template <typename T>
struct DropArgs {
    const T *x;
    T *y;
    int64_t cols, ldx, ldy;
    DropParams d;
};

// One warp per segment of 256 values, grid-stride over `units` = rows x segs
// segments (32-bit: longer tensors take several launches); row = unit / segs by
// a multiplication (`mul`, `shift`: exact for 32-bit dividends, or mul 0 for
// segs == 1).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(DropArgs<T> a, uint32_t units, uint32_t segs, uint32_t mul,
                                                      uint32_t shift) {
    const int lane = threadIdx.x & 31;
    const uint64_t key = drop_seed(a.d);
    const uint32_t step = gridDim.x * 8u;
    constexpr int UNROLL = 2;
    for (uint32_t u0 = blockIdx.x * 8u + (threadIdx.x >> 5); u0 < units; u0 += UNROLL * step) {
        Raw8<T> x[UNROLL];
        uint32_t row[UNROLL];
        int64_t seg0[UNROLL];
        int n[UNROLL];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
            const uint32_t u = u0 + k * step;
            const uint32_t hi = __umulhi(u, mul);
            row[k] = mul ? (((u - hi) >> 1) + hi) >> shift : u;
            seg0[k] = (int64_t)(u - row[k] * segs) * SEG;
            n[k] = u < units && u >= u0 ? count_of<VEC>(seg0[k], a.cols, lane) : 0;
            x[k] = load8<T, VEC>(a.x + row[k] * a.ldx, seg0[k], n[k], lane);
        }
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
            const F8 y = drop8<VEC>(unpack<T>(x[k]), a.d.row_offset + row[k], seg0[k], lane, key, a.d);
            store8<T, VEC>(a.y + row[k] * a.ldy, seg0[k], n[k], lane, y);
        }
        if (u0 + UNROLL * step < u0) break;
    }
}

// ---------------------------------------------------------------- forward
template <typename T, typename W>
struct FwdArgs {
    const T *x, *res;
    const W *w, *b;  // either may be null: 1 and 0
    T *y, *h;
    float *mean, *rstd;
    int64_t rows, cols, ldx, ldr, ldy, ldh;
    float eps;
    DropParams d;
};

// Sums over the warps that share a row (ONE: one warp), for R rows; every thread
// gets the same values.  red: NW entries a row, zero where there is no warp.
template <int NW, int R, bool ONE>
__device__ __forceinline__ void row_sums(float (&v)[R], float (*red)[NW], int warp, int lane) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = warp_sum(v[i]);
    if (ONE) return;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) red[i][warp] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < R; ++k) {
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NW / 4; ++i) {
            const float4 q = reinterpret_cast<const float4 *>(red[k])[i];
            s = add2(add2(s, make_float2(q.x, q.y)), make_float2(q.z, q.w));
        }
        v[k] = s.x + s.y;
    }
}
template <int NW>
__device__ __forceinline__ float row_sum(float v, float (*red)[NW], int warp, int lane) {
    float a[1] = {v};
    row_sums<NW, 1, false>(a, red, warp, lane);
    return a[0];
}
// 1 / sqrt(v): the hardware's approximation and one Newton step (the IEEE square
// root and division cost 40 instructions a row and warp).
__device__ __forceinline__ float inv_sqrt(float v) {
    const float r = rsqrtf(v), h = r * __fmaf_rn(-0.5f * v * r, r, 1.5f);
    return v > 0.f && v < INFINITY ? h : r;
}

// Resident CTAs for launches of up to 256, 320 or 512 threads (register use).
__host__ __device__ constexpr int fwd_ctas(int nch, int maxt) { return maxt > 256 ? 1 : (nch == 1 ? 3 : 2); }
__host__ __device__ constexpr int bwd_ctas(int maxt) { return maxt > 320 ? 1 : 2; }
constexpr int MAX_DEPTH = 4;
constexpr int RING_HEAD = 8 * MAX_DEPTH * 8 + 16;  // barriers of up to eight warps' rings, the abort word
constexpr int MAX_SMEM = RING_HEAD + SLOT_ROOM;
static_assert(MAX_SMEM + STATIC_ROOM <= 227 * 1024, "shared memory");  // the reductions' arrays: 256 bytes at most
// NaN in rows r0, r0 + step, ... of p, by the `nt` threads of which this is `t`.
template <typename T>
__device__ __forceinline__ void nan_rows(T *p, int64_t ld, int64_t r0, int64_t step, int64_t rows, int64_t cols, int t,
                                         int nt) {
#pragma unroll 1
    for (int64_t r = r0; r < rows; r += step)
#pragma unroll 1
        for (int64_t c = t; c < cols; c += nt) p[r * ld + c] = from_f<T>(__uint_as_float(0x7fc00000u));
}
// Bytes of a row in a slot.
__host__ __device__ __forceinline__ uint32_t row_pitch(int64_t cols, int esize, bool vec) {
    return (uint32_t)(vec ? cols * esize : (cols * esize + 15) / 16 * 16);
}

// One input's current row: values lo <= c < hi lie at s[c] in shared memory,
// the others (a ragged row's ends) at g[c] in global memory.
template <typename T>
struct RowView {
    const T *s, *g;
    int lo, hi;
};

// The rows a CTA (or, with one warp per row, a warp) works through, brought to
// shared memory ahead of their use: `depth` slots, one bulk copy per input and
// row, issued by one thread.  A slot is filled again once every reader has
// passed the barrier that follows its last read.  A bulk copy takes whole
// 16-byte pieces: of a row that is not aligned so (VEC false) the pieces inside
// it, which leaves up to seven 16-bit values at either end to plain loads.
// Waits are bounded.  One that gives up sets the device error word and the CTA's
// abort word: no slot is filled again, and after its last row a CTA that sees the
// word writes NaN over all its results (fwd_nan, bwd_nan: calls at the kernels' ends,
// so that the rows' own registers stay as they were; a test of each wait's outcome in
// the rows' code cost up to 17 %, this 0 to 5, on one ragged form 6).
template <typename T, int INPUTS, bool VEC>
struct RowRing {
    uint8_t *slots;
    uint64_t *bars;
    uint32_t pitch;  // of one input's row in a slot
    int cols, depth, slot;
    uint32_t phase;

    // dyn: barriers of up to eight rings, the abort word, then the slots.
    __device__ __forceinline__ void init(uint8_t *dyn, int which, int n, int d, bool leader) {
        cols = n, depth = d, slot = 0, phase = 0;
        pitch = row_pitch(n, sizeof(T), VEC);
        bars = reinterpret_cast<uint64_t *>(dyn) + which * MAX_DEPTH;
        slots = dyn + RING_HEAD + (size_t)which * d * INPUTS * pitch;
        if (threadIdx.x == 0) *abort_word(dyn) = 0;
        if (leader) {
            for (int i = 0; i < d; ++i) tc::mbar_init(&bars[i], 1);
            tc::fence_mbar_init();
        }
        __syncthreads();
    }
    __device__ __forceinline__ static volatile int *abort_word(uint8_t *dyn) {
        return reinterpret_cast<volatile int *>(dyn + RING_HEAD - 16);
    }
    // Values before the row's first whole 16-byte piece, and up to the end of its last.
    __device__ __forceinline__ void inside(const T *row, int &lo, int &hi) const {
        const uint32_t a = (uint32_t)reinterpret_cast<uintptr_t>(row);
        lo = (int)((0u - a) & 15u) / (int)sizeof(T);
        hi = cols - (int)((a + (uint32_t)cols * (uint32_t)sizeof(T)) & 15u) / (int)sizeof(T);
        if (hi <= lo) lo = hi = 0;
    }
    __device__ __forceinline__ void fill(int s, const T *const (&row)[INPUTS]) {
        if constexpr (VEC) {
            tc::mbar_arrive_expect_tx(&bars[s], pitch * INPUTS);
#pragma unroll
            for (int k = 0; k < INPUTS; ++k)
                tc::bulk_load(slots + (s * INPUTS + k) * pitch, row[k], pitch, &bars[s]);
        } else {
            int lo[INPUTS], hi[INPUTS];
            uint32_t bytes = 0;
#pragma unroll
            for (int k = 0; k < INPUTS; ++k) {
                inside(row[k], lo[k], hi[k]);
                bytes += (uint32_t)(hi[k] - lo[k]) * (uint32_t)sizeof(T);
            }
            tc::mbar_arrive_expect_tx(&bars[s], bytes);
#pragma unroll
            for (int k = 0; k < INPUTS; ++k)
                if (hi[k] > lo[k])
                    tc::bulk_load(slots + (s * INPUTS + k) * pitch, row[k] + lo[k],
                                  (uint32_t)(hi[k] - lo[k]) * (uint32_t)sizeof(T), &bars[s]);
        }
    }
    // `ahead` (0 or 1): the row after the current one
    __device__ __forceinline__ bool wait(uint8_t *dyn, int ahead = 0, uint32_t polls = 1u << 24) {
        const bool wrap = slot + ahead >= depth;
        return tc::mbar_wait(&bars[wrap ? 0 : slot + ahead], phase ^ (wrap ? 1u : 0u), abort_word(dyn), polls);
    }
    // After the last row, past a barrier of the warps that share it: whether a wait
    // has given up.  Copies still under way are then waited for, again with a limit
    // (a barrier's older phase reads as complete, so both parities are asked for).
    __device__ __forceinline__ bool gave_up(uint8_t *dyn) const {
        if (!*abort_word(dyn)) return false;
        for (int i = 0; i < 2 * depth; ++i)
            for (uint32_t k = 0; k < (1u << 12) && !tc::mbar_try_wait(&bars[i >> 1], i & 1); ++k) {
            }
        return true;
    }
    __device__ __forceinline__ RowView<T> view(int k, const T *row, int ahead = 0) const {
        const int s = slot + ahead >= depth ? 0 : slot + ahead;
        RowView<T> v{reinterpret_cast<const T *>(slots + (s * INPUTS + k) * pitch), row, 0, cols};
        if constexpr (!VEC) {
            inside(row, v.lo, v.hi);
            v.s -= v.lo;
        }
        return v;
    }
    __device__ __forceinline__ void next() {
        if (++slot == depth) slot = 0, phase ^= 1;
    }
};

// A group's rows and this thread's place in it, found again from the launch (opaque
// to the compiler: carried along the row loop they cost its registers).
struct Place {
    int64_t r0, step;
    int t, nt;
    __device__ __forceinline__ explicit Place(int wpr) {
        int tid, cta;
        asm volatile("mov.u32 %0, %%tid.x;\n mov.u32 %1, %%ctaid.x;" : "=r"(tid), "=r"(cta));
        nt = 32 * wpr;
        const int groups = (int)blockDim.x / nt, mine = tid / nt;
        t = tid - mine * nt;
        r0 = (int64_t)cta * groups + mine;
        step = (int64_t)gridDim.x * groups;
    }
};

// A lane's values of a segment of the row.
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load8(const RowView<T> &row, int seg0, int count, int lane) {
    if constexpr (VEC) {
        return load8<T, true>(row.s, seg0, count, lane);
    } else {
        Raw8<T> r;
        if (seg0 >= row.lo && seg0 + SEG <= row.hi) {
#pragma unroll
            for (int j = 0; j < 8; ++j) r.v[j] = row.s[seg0 + 32 * j + lane];
        } else {
            // one generic load each, no branch between them: their latencies overlap
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = seg0 + 32 * j + lane;
                const T *p = c >= row.lo && c < row.hi ? row.s + c : row.g + c;
                r.v[j] = j < count ? *p : from_f<T>(0.f);
            }
        }
        return r;
    }
}

// NaN over a forward CTA's results (see RowRing).
template <typename T, typename W>
__device__ __noinline__ void fwd_nan(const FwdArgs<T, W> &a, int wpr) {
    const Place p(wpr);
    nan_rows(a.y, a.ldy, p.r0, p.step, a.rows, a.cols, p.t, p.nt);
    if (a.res) nan_rows(a.h, a.ldh, p.r0, p.step, a.rows, a.cols, p.t, p.nt);
    nan_rows(a.mean, 1, p.r0, p.step, a.rows, 1, p.t, p.nt);
    nan_rows(a.rstd, 1, p.r0, p.step, a.rows, 1, p.t, p.nt);
}

// MAXT: the launch's thread count rounded up to 256, 320 or 512.
// ONE: a warp per row, else a CTA.
template <typename T, typename W, int NCH, int MAXT, bool VEC, bool DROP, bool ONE>
__global__ void __launch_bounds__(MAXT, fwd_ctas(NCH, MAXT))
    ln_fwd_kernel(const __grid_constant__ FwdArgs<T, W> a, int warps, int depth) {
    const int wpr = ONE ? 1 : warps;  // warps per row
    extern __shared__ __align__(128) uint8_t dyn[];
    constexpr int NW = MAXT / 32;
    // rows in hand at once: the reductions of two rows overlap and share their barriers
    constexpr int R = NCH <= 2 && sizeof(T) == 2 ? 2 : 1;
    __shared__ __align__(16) float red[2][R][NW];
    if (threadIdx.x < 2 * R * NW) red[0][0][threadIdx.x] = 0.f;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
    const int rpc = ONE ? nwarps : 1;  // rows a CTA has in hand at once
    const int w0 = ONE ? 0 : warp, mine = ONE ? warp : 0;
    const float inv_n = 1.f / (float)a.cols;
    const uint64_t key = DROP ? drop_seed(a.d) : 0;
    constexpr int IN = DROP ? 2 : 1;
    RowRing<T, IN, VEC> ring;
    const bool leader = ONE ? lane == 0 : threadIdx.x == 0;
    const int64_t r0 = (int64_t)blockIdx.x * rpc + mine, step = (int64_t)gridDim.x * rpc;
    auto fill = [&](int s, int64_t row) {
        if (row >= a.rows) return;
        const T *src[IN];
        src[0] = a.x + row * a.ldx;
        if constexpr (DROP) src[1] = a.res + row * a.ldr;
        ring.fill(s, src);
    };
    ring.init(dyn, mine, (int)a.cols, depth, leader);
    if (leader)
        for (int i = 0; i < depth; ++i) fill(i, r0 + i * step);
    Raw8<W> wv[NCH], bv[NCH];
    int n[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int seg0 = (w0 + i * wpr) * SEG;
        n[i] = count_of<VEC>(seg0, a.cols, lane);
        wv[i] = load8_or<W, VEC>(a.w, 1.f, seg0, n[i], lane);
        bv[i] = load8_or<W, VEC>(a.b, 0.f, seg0, n[i], lane);
    }
    for (int64_t r = r0; r < a.rows; r += R * step) {
        F8 v[R][NCH];
        float s[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t rk = r + k * step;
            const bool live = k == 0 || rk < a.rows;  // the same for all that share the row
            float2 t = make_float2(0.f, 0.f);
            if (live) ring.wait(dyn, k);
            const RowView<T> xr = ring.view(0, a.x + rk * a.ldx, k);
            const RowView<T> rr = ring.view(IN - 1, DROP ? a.res + rk * a.ldr : a.x + rk * a.ldx, k);
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int seg0 = (w0 + i * wpr) * SEG, nk = live ? n[i] : 0;
                v[k][i] = unpack<T>(load8<T, VEC>(xr, seg0, nk, lane));
                if constexpr (DROP) {
                    const F8 res = unpack<T>(load8<T, VEC>(rr, seg0, nk, lane));
                    const F8 d = drop8<VEC>(v[k][i], a.d.row_offset + (uint64_t)rk, seg0, lane, key, a.d);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[k][i].p[j] = add2(d.p[j], res.p[j]);
                    store8<T, VEC>(a.h + rk * a.ldh, seg0, nk, lane, v[k][i]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) t = add2(t, v[k][i].p[j]);
            }
            s[k] = t.x + t.y;
        }
        const bool go = leader && !*ring.abort_word(dyn);  // no wait has given up
        row_sums<NW, R, ONE>(s, red[0], warp, lane);
        // every reader of the slots is past its reads
        if (ONE) __syncwarp();
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if (go) fill(ring.slot, r + (depth + k) * step);
            ring.next();
        }
        float mean[R], q[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            mean[k] = s[k] * inv_n;
            const float2 mean2 = make_float2(mean[k], mean[k]);
            float2 t = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float2 &p = v[k][i].p[j];
                    p = sub2(p, mean2);
                    if constexpr (!VEC) {
                        if (2 * j >= n[i]) p.x = 0.f;
                        if (2 * j + 1 >= n[i]) p.y = 0.f;
                    }
                    if (!VEC || n[i]) t = fma2(p, p, t);
                }
            }
            q[k] = t.x + t.y;
        }
        row_sums<NW, R, ONE>(q, red[1], warp, lane);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int64_t rk = r + k * step;
            if (k > 0 && rk >= a.rows) break;
            const float rstd = inv_sqrt(__fmaf_rn(q[k], inv_n, a.eps));
            if (lane == 0 && w0 == 0) {
                a.mean[rk] = mean[k];
                a.rstd[rk] = rstd;
            }
            const float2 rstd2 = make_float2(rstd, rstd);
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                stay_packed(wv[i]);
                stay_packed(bv[i]);
                const F8 w = unpack<W>(wv[i]), b = unpack<W>(bv[i]);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[k][i].p[j] = fma2(mul2(v[k][i].p[j], rstd2), w.p[j], b.p[j]);
                store8<T, VEC>(a.y + rk * a.ldy, (w0 + i * wpr) * SEG, n[i], lane, v[k][i]);
            }
        }
    }
    if (ring.gave_up(dyn)) fwd_nan<T, W>(a, ONE ? 1 : blockDim.x >> 5);
}

// Rows longer than MAX_SEGS segments: one CTA per row, three passes over it
// (the later ones mostly from L2).
template <typename T, typename W, bool VEC, bool DROP>
__global__ void __launch_bounds__(LONG_THREADS) ln_fwd_long_kernel(FwdArgs<T, W> a) {
    constexpr int nw = LONG_THREADS / 32;
    __shared__ __align__(16) float red[2][nw];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inv_n = 1.f / (float)a.cols;
    const uint64_t key = DROP ? drop_seed(a.d) : 0;
    const int64_t segs = (a.cols + SEG - 1) / SEG;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        auto fetch = [&](int64_t seg0, int n) {
            F8 v = unpack<T>(load8<T, VEC>(a.x + r * a.ldx, seg0, n, lane));
            if constexpr (DROP) {
                const F8 res = unpack<T>(load8<T, VEC>(a.res + r * a.ldr, seg0, n, lane));
                const F8 d = drop8<VEC>(v, a.d.row_offset + (uint64_t)r, seg0, lane, key, a.d);
#pragma unroll
                for (int j = 0; j < 4; ++j) v.p[j] = add2(d.p[j], res.p[j]);
            }
            return v;
        };
        float s = 0.f;
        for (int64_t g = warp; g < segs; g += nw) {
            const F8 v = fetch(g * SEG, count_of<VEC>(g * SEG, a.cols, lane));
            const float2 t = add2(add2(v.p[0], v.p[1]), add2(v.p[2], v.p[3]));
            s += t.x + t.y;
        }
        const float mean = row_sum<nw>(s, red, warp, lane) * inv_n;
        const float2 mean2 = make_float2(mean, mean);
        float q = 0.f;
        for (int64_t g = warp; g < segs; g += nw) {
            const int n = count_of<VEC>(g * SEG, a.cols, lane);
            const F8 v = fetch(g * SEG, n);
            float2 t = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 c = sub2(v.p[j], mean2);
                if (2 * j >= n) c.x = 0.f;
                if (2 * j + 1 >= n) c.y = 0.f;
                t = fma2(c, c, t);
            }
            q += t.x + t.y;
        }
        const float var = row_sum<nw>(q, red + 1, warp, lane) * inv_n;
        const float rstd = inv_sqrt(var + a.eps);
        if (threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        const float2 rstd2 = make_float2(rstd, rstd);
        for (int64_t g = warp; g < segs; g += nw) {
            const int n = count_of<VEC>(g * SEG, a.cols, lane);
            F8 v = fetch(g * SEG, n);
            if constexpr (DROP) store8<T, VEC>(a.h + r * a.ldh, g * SEG, n, lane, v);
            const F8 w = unpack<W>(load8_or<W, VEC>(a.w, 1.f, g * SEG, n, lane));
            const F8 b = unpack<W>(load8_or<W, VEC>(a.b, 0.f, g * SEG, n, lane));
#pragma unroll
            for (int j = 0; j < 4; ++j) v.p[j] = fma2(mul2(sub2(v.p[j], mean2), rstd2), w.p[j], b.p[j]);
            store8<T, VEC>(a.y + r * a.ldy, g * SEG, n, lane, v);
        }
    }
}

// ---------------------------------------------------------------- backward
template <typename T, typename W>
struct BwdArgs {
    const T *dy, *x, *dh;  // x: the normalised input (h in the fused form); dh may be null
    const W *w;            // may be null: 1
    const float *mean, *rstd;
    T *dx, *dr;            // dr: the fused form's residual gradient (dx is then its dropout)
    float *part;           // partial weight gradients, grid x 2 x cols; null if none are wanted
    int64_t rows, cols, lddy, ldx, lddh, lddx, lddr;
    DropParams d;
};

// Sums of u and v over the warps that share a row (`w0`: this one's place).  red:
// NW entries, zero where there is no warp.  MULTI: several groups of warps share the
// CTA, each with two or four entries.
template <int NW, bool MULTI>
__device__ __forceinline__ float2 row_sum2(float u, float v, float2 *red, int wpr, int group, int w0, int lane) {
    u = warp_sum(u);
    v = warp_sum(v);
    if (MULTI && wpr == 1) return make_float2(u, v);
    const int room = wpr <= 2 ? 2 : 4;
    if (MULTI) red += group * room;
    if (lane == 0) red[w0] = make_float2(u, v);
    if (MULTI) tc::named_bar(1 + group, 32 * wpr);
    else __syncthreads();
    float2 s = make_float2(0.f, 0.f);
    const float4 *p = reinterpret_cast<const float4 *>(red);
    if constexpr (!MULTI) {
#pragma unroll
        for (int i = 0; i < NW / 2; ++i) s = add2(add2(s, make_float2(p[i].x, p[i].y)), make_float2(p[i].z, p[i].w));
    } else {
        for (int i = 0; i < room / 2; ++i) s = add2(add2(s, make_float2(p[i].x, p[i].y)), make_float2(p[i].z, p[i].w));
    }
    return s;
}

// NaN over a backward CTA's results, its part of the weight gradients' sums among them.
template <typename T, typename W>
__device__ __noinline__ void bwd_nan(const BwdArgs<T, W> &a, int wpr) {
    const Place p(wpr);
    nan_rows(a.dx, a.lddx, p.r0, p.step, a.rows, a.cols, p.t, p.nt);
    if (a.dr) nan_rows(a.dr, a.lddr, p.r0, p.step, a.rows, a.cols, p.t, p.nt);
    if (a.part)
        nan_rows(a.part, 2 * a.cols, blockIdx.x, gridDim.x, gridDim.x, 2 * a.cols, threadIdx.x, blockDim.x);
}

// MULTI: a CTA has several rows in hand, each a group of `wpr` warps; else one.
template <typename T, typename W, int NCH, int MAXT, bool VEC, bool DROP, bool MULTI>
__global__ void __launch_bounds__(MAXT, bwd_ctas(MAXT))
    ln_bwd_kernel(const __grid_constant__ BwdArgs<T, W> a, int wpr, int depth) {
    constexpr int NW = MAXT / 32;
    __shared__ __align__(16) float2 red[2][NW];
    if (threadIdx.x < 2 * NW) red[0][threadIdx.x] = make_float2(0.f, 0.f);
    __syncthreads();
    extern __shared__ __align__(128) uint8_t dyn[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
    const int rpc = MULTI ? nwarps / wpr : 1;  // rows a CTA has in hand at once
    const int mine = MULTI ? warp / wpr : 0, w0 = warp - mine * wpr;
    const float inv_n = 1.f / (float)a.cols;
    const uint64_t key = DROP ? drop_seed(a.d) : 0;
    constexpr int IN = DROP ? 3 : 2;
    RowRing<T, IN, VEC> ring;
    bool leader = w0 == 0 && lane == 0;
    const int64_t r0 = (int64_t)blockIdx.x * rpc + mine, step = (int64_t)gridDim.x * rpc;
    auto fill = [&](int s, int64_t row) {
        if (row >= a.rows) return;
        const T *src[IN];
        src[0] = a.dy + row * a.lddy;
        src[1] = a.x + row * a.ldx;
        // without dh its slot holds dy again and is not read
        if constexpr (DROP) src[2] = a.dh ? a.dh + row * a.lddh : src[0];
        ring.fill(s, src);
    };
    ring.init(dyn, mine, (int)a.cols, depth, leader);
    if (leader)
        for (int i = 0; i < depth; ++i) fill(i, r0 + i * step);
    // Up to two segments a thread the row's g and x-hat are held from the sums to
    // the output, past that they are computed again from the slot (registers); so
    // too at 320 threads, where that fits two CTAs (8192 x 5120 bf16 with dropout
    // 89 us; held, in one CTA, 99 us).  Past 320 threads two CTAs do not fit, and
    // float32 holds in one CTA from there on (8192 x 5120 without dropout 82 us,
    // computed again in two CTAs 89 us).
    constexpr bool HOLD = NCH <= 2 && MAXT != 320;
    // four segments: their sums fill the registers, the weights are read again too
    constexpr bool WREG = NCH <= 2;
    Raw8<W> wv[WREG ? NCH : 1];
    F8 dw[NCH], db[NCH];
    int n[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        n[i] = count_of<VEC>((w0 + i * wpr) * SEG, a.cols, lane);
        if constexpr (WREG) wv[i] = load8_or<W, VEC>(a.w, 1.f, (w0 + i * wpr) * SEG, n[i], lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) dw[i].p[j] = db[i].p[j] = make_float2(0.f, 0.f);
    }
    // How the leader knows that a slot must not be filled again: by its own waits or by
    // the abort word.  8192 rows bf16, us: 9216 values 132 and 147, 5120 61 and 58.
    constexpr bool OWN_WAIT = NCH == 4 && VEC;
    int turn = 0;
    float mean = r0 < a.rows ? a.mean[r0] : 0.f, rstd = r0 < a.rows ? a.rstd[r0] : 0.f;
    for (int64_t r = r0; r < a.rows; r += step, ++turn) {
        const bool go = leader && turn > 0 && (OWN_WAIT || !*ring.abort_word(dyn));
        const float2 mean2 = make_float2(mean, mean), rstd2 = make_float2(rstd, rstd);
        const float rs = rstd;
        if (r + step < a.rows) mean = a.mean[r + step], rstd = a.rstd[r + step];
        const RowView<T> yr = ring.view(0, a.dy + r * a.lddy), xr = ring.view(1, a.x + r * a.ldx);
        float2 s1 = make_float2(0.f, 0.f), s2 = s1;
        F8 gh[HOLD ? NCH : 1], xh[HOLD ? NCH : 1];
        if (!ring.wait(dyn) && OWN_WAIT) leader = false;
        auto weights = [&](int i) {
            if constexpr (WREG) {
                stay_packed(wv[i]);
                return unpack<W>(wv[i]);
            } else {
                return unpack<W>(load8_or<W, VEC>(a.w, 1.f, (w0 + i * wpr) * SEG, n[i], lane));
            }
        };
        auto values = [&](int i, F8 &dy, F8 &x) {  // dy and x-hat
            const int seg0 = (w0 + i * wpr) * SEG;
            dy = unpack<T>(load8<T, VEC>(yr, seg0, n[i], lane));
            x = unpack<T>(load8<T, VEC>(xr, seg0, n[i], lane));
#pragma unroll
            for (int j = 0; j < 4; ++j) x.p[j] = mul2(sub2(x.p[j], mean2), rstd2);
        };
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            F8 dy, x;
            values(i, dy, x);
            const F8 w = weights(i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // dy is 0 past the row's end
                const float2 g = mul2(dy.p[j], w.p[j]);
                dw[i].p[j] = fma2(dy.p[j], x.p[j], dw[i].p[j]);
                db[i].p[j] = add2(db[i].p[j], dy.p[j]);
                s1 = add2(s1, g);
                s2 = fma2(g, x.p[j], s2);
                if constexpr (HOLD) gh[i].p[j] = g, xh[i].p[j] = x.p[j];
            }
        }
        const float2 s = row_sum2<NW, MULTI>(s1.x + s1.y, s2.x + s2.y, red[turn & 1], wpr, mine, w0, lane);
        // the row before this one has been read by all
        if (MULTI && wpr == 1) __syncwarp();
        if (OWN_WAIT ? leader && turn > 0 : go)
            fill(ring.slot == 0 ? depth - 1 : ring.slot - 1, r + (depth - 1) * step);
        // dx = rstd g - rstd mean(g) - x-hat rstd mean(g x-hat)
        const float c1 = -rs * (s.x * inv_n), c2 = -rs * (s.y * inv_n);
        const float2 c1_2 = make_float2(c1, c1), c2_2 = make_float2(c2, c2);
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
            for (int j = 0; j < 4; ++j) g.p[j] = fma2(x.p[j], c2_2, fma2(g.p[j], rstd2, c1_2));
            if constexpr (DROP) {
                if (a.dh) {
                    const F8 dh = unpack<T>(
                        load8<T, VEC>(ring.view(IN - 1, a.dh + r * a.lddh), seg0, n[i], lane));
#pragma unroll
                    for (int j = 0; j < 4; ++j) g.p[j] = add2(g.p[j], dh.p[j]);
                }
                store8<T, VEC>(a.dr + r * a.lddr, seg0, n[i], lane, g);
                g = drop8<VEC>(g, a.d.row_offset + (uint64_t)r, seg0, lane, key, a.d);
            }
            store8<T, VEC>(a.dx + r * a.lddx, seg0, n[i], lane, g);
        }
        ring.next();
    }
    if (a.part) {
        float *part = a.part + (int64_t)blockIdx.x * 2 * a.cols;
        if constexpr (MULTI) {
            // the groups' sums, over the rings' space once every warp is done with it
            __syncthreads();
            float *acc = reinterpret_cast<float *>(dyn + RING_HEAD), *own = acc + (int64_t)mine * 2 * a.cols;
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                store8<float, VEC>(own, (w0 + i * wpr) * SEG, n[i], lane, dw[i]);
                store8<float, VEC>(own + a.cols, (w0 + i * wpr) * SEG, n[i], lane, db[i]);
            }
            __syncthreads();
            for (int c = threadIdx.x; c < 2 * a.cols; c += blockDim.x) {
                float s = 0.f;
                for (int i = 0; i < rpc; ++i) s += acc[(int64_t)i * 2 * a.cols + c];
                part[c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int seg0 = (w0 + i * wpr) * SEG;
                store8<float, VEC>(part, seg0, n[i], lane, dw[i]);
                store8<float, VEC>(part + a.cols, seg0, n[i], lane, db[i]);
            }
        }
    }
    __syncthreads();
    // the same for all: every wait of the CTA lies before this barrier
    if (ring.gave_up(dyn)) bwd_nan<T, W>(a, MULTI ? wpr : blockDim.x >> 5);
}

// Rows longer than MAX_SEGS segments, first kernel: the row's two sums.
template <typename T, typename W, bool VEC>
__global__ void __launch_bounds__(LONG_THREADS) ln_bwd_sums_kernel(BwdArgs<T, W> a, float2 *sums) {
    constexpr int nw = LONG_THREADS / 32;
    __shared__ __align__(16) float2 red[2][nw];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inv_n = 1.f / (float)a.cols;
    const int64_t segs = (a.cols + SEG - 1) / SEG;
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.f, s2 = 0.f;
        const float2 mean2 = make_float2(mean, mean), rstd2 = make_float2(rstd, rstd);
        for (int64_t sg = warp; sg < segs; sg += nw) {
            const int n = count_of<VEC>(sg * SEG, a.cols, lane);
            const F8 y = unpack<T>(load8<T, VEC>(a.dy + r * a.lddy, sg * SEG, n, lane));
            const F8 x = unpack<T>(load8<T, VEC>(a.x + r * a.ldx, sg * SEG, n, lane));
            const F8 w = unpack<W>(load8_or<W, VEC>(a.w, 1.f, sg * SEG, n, lane));
            float2 t1 = make_float2(0.f, 0.f), t2 = t1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // dy is 0 past the row's end
                const float2 g = mul2(y.p[j], w.p[j]);
                t1 = add2(t1, g);
                t2 = fma2(g, mul2(sub2(x.p[j], mean2), rstd2), t2);
            }
            s1 += t1.x + t1.y;
            s2 += t2.x + t2.y;
        }
        const float2 s = row_sum2<nw, false>(s1, s2, red[turn], nw, 0, warp, lane);
        turn ^= 1;
        if (threadIdx.x == 0) sums[r] = make_float2(s.x * inv_n, s.y * inv_n);
    }
}

// Second kernel: a warp takes one segment of columns over its share of the
// rows (blockIdx.y of gridDim.y).
template <typename T, typename W, bool VEC, bool DROP>
__global__ void __launch_bounds__(128) ln_bwd_cols_kernel(BwdArgs<T, W> a, const float2 *sums) {
    const int lane = threadIdx.x & 31;
    const int64_t seg0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * SEG;
    if (seg0 >= a.cols) return;
    const uint64_t key = DROP ? drop_seed(a.d) : 0;
    const int n = count_of<VEC>(seg0, a.cols, lane);
    const F8 w = unpack<W>(load8_or<W, VEC>(a.w, 1.f, seg0, n, lane));
    F8 dw, db;
#pragma unroll
    for (int j = 0; j < 4; ++j) dw.p[j] = db.p[j] = make_float2(0.f, 0.f);
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float rstd = a.rstd[r];
        const float2 mean2 = make_float2(a.mean[r], a.mean[r]), rstd2 = make_float2(rstd, rstd), m = sums[r];
        const float2 c1 = make_float2(-rstd * m.x, -rstd * m.x), c2 = make_float2(-rstd * m.y, -rstd * m.y);
        const F8 y = unpack<T>(load8<T, VEC>(a.dy + r * a.lddy, seg0, n, lane));
        const F8 x = unpack<T>(load8<T, VEC>(a.x + r * a.ldx, seg0, n, lane));
        F8 g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 xh = mul2(sub2(x.p[j], mean2), rstd2);
            dw.p[j] = fma2(y.p[j], xh, dw.p[j]);
            db.p[j] = add2(db.p[j], y.p[j]);
            g.p[j] = fma2(xh, c2, fma2(mul2(y.p[j], w.p[j]), rstd2, c1));
        }
        if constexpr (DROP) {
            if (a.dh) {
                const F8 dh = unpack<T>(load8<T, VEC>(a.dh + r * a.lddh, seg0, n, lane));
#pragma unroll
                for (int j = 0; j < 4; ++j) g.p[j] = add2(g.p[j], dh.p[j]);
            }
            store8<T, VEC>(a.dr + r * a.lddr, seg0, n, lane, g);
            g = drop8<VEC>(g, a.d.row_offset + (uint64_t)r, seg0, lane, key, a.d);
        }
        store8<T, VEC>(a.dx + r * a.lddx, seg0, n, lane, g);
    }
    if (!a.part) return;
    float *part = a.part + (int64_t)blockIdx.y * 2 * a.cols;
    store8<float, VEC>(part, seg0, n, lane, dw);
    store8<float, VEC>(part + a.cols, seg0, n, lane, db);
}

// dw / db from the `parts` partial sums, in a fixed order: a column's sum does
// not depend on timing.  A warp takes 32 columns, the CTA's eight warps every
// eighth partial, eight loads in flight.  Launched with programmatic dependence on
// the kernel before it, which gives no signal of its own: the CTAs start as that
// kernel's last ones leave, which hides the launch, and wait for its end (and its
// writes) before they read.
template <typename W>
__global__ void __launch_bounds__(256) ln_bwd_finish_kernel(const float *part, int parts, int64_t cols, W *dw, W *db) {
    __shared__ float red[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t n = 2 * cols, c = (int64_t)blockIdx.x * 32 + lane;
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
        if (c < cols) {
            if (dw) dw[c] = from_f<W>(s);
        } else if (db) {
            db[c - cols] = from_f<W>(s);
        }
    }
}

// Self-test of the ring's waits: a warp takes `rows` rows of 4 * 32 values of which
// only the first `brought` are copied, with waits cut to `polls` polls, and writes
// their sums as the kernels above write their results.
__global__ void __launch_bounds__(32) selftest_ring_kernel(const float *x, int rows, int brought, uint32_t polls,
                                                           float *out) {
    __shared__ __align__(128) uint8_t dyn[RING_HEAD + 2 * 128 * 4];
    RowRing<float, 1, true> ring;
    const int lane = threadIdx.x & 31;
    auto fill = [&](int s, int row) {
        if (row >= brought || *ring.abort_word(dyn)) return;
        const float *src[1] = {x + row * 128};
        ring.fill(s, src);
    };
    ring.init(dyn, 0, 128, 2, lane == 0);
    if (lane == 0)
        for (int i = 0; i < 2; ++i) fill(i, i);
    for (int r = 0; r < rows; ++r) {
        ring.wait(dyn, 0, polls);
        const float4 v = reinterpret_cast<const float4 *>(ring.view(0, x + r * 128).s)[lane];
        const float s = warp_sum(v.x + v.y + v.z + v.w);
        __syncwarp();
        if (lane == 0) {
            out[r] = s;
            fill(ring.slot, r + 2);
        }
        ring.next();
    }
    __syncwarp();
    if (ring.gave_up(dyn))
        for (int r = lane; r < rows; r += 32) out[r] = __uint_as_float(0x7fc00000u);
}

// ---------------------------------------------------------------- launches
// Segments per thread, warps per row, the template's thread bound (backward), ring
// slots, the kernel's shared memory and the resident CTAs that its template allows.
struct Shape {
    int nch, wpr, threads, maxt, rows_per_cta, depth, smem, per_sm;
};
static Shape shape_of(int64_t cols, int esize, bool drop, bool bwd, bool vec) {
    const int segs = (int)((cols + SEG - 1) / SEG);
    Shape s{};
    if (bwd) {
        // two segments a thread (its sums' registers); short rows several to a CTA
        s.nch = segs <= 1 ? 1 : (segs <= 32 ? 2 : 4);
        s.wpr = (segs + s.nch - 1) / s.nch;
        s.rows_per_cta = s.wpr <= 4 ? 8 / s.wpr : 1;  // two or more
        s.threads = 32 * s.wpr * s.rows_per_cta;
        s.maxt = s.nch == 4 ? 512 : s.threads <= 256 ? 256 : s.threads <= 320 && esize == 2 ? 320 : 512;
    } else if (segs <= 4) {
        s = {segs <= 1 ? 1 : (segs <= 2 ? 2 : 4), 1, 256, 0, 8, 0, 0, 0};
    } else {
        // Fewer, fuller warps spend less on a row's reductions: 16384 x 4096 bf16
        // in 52 us with four segments a thread, 56 with two, 86 with one; the
        // dropout's and float32's registers allow two.
        const bool full = !drop && esize == 2;
        s.nch = segs <= 8 ? (full ? 2 : 1) : segs <= 16 ? (full ? 4 : 2) : segs <= 24 ? 3 : 4;
        s.wpr = (segs + s.nch - 1) / s.nch;
        s.threads = 32 * s.wpr;
        s.rows_per_cta = 1;
    }
    const int inputs = (bwd ? 2 : 1) + (drop ? 1 : 0);
    const int64_t slot = (int64_t)row_pitch(cols, esize, vec) * inputs * s.rows_per_cta;
    s.per_sm = bwd ? bwd_ctas(s.maxt) : fwd_ctas(s.nch, s.threads) * (s.threads <= 128 ? 2 : 1);
    const int64_t room = SLOT_ROOM / s.per_sm;
    s.depth = (int)(room / slot < MAX_DEPTH ? room / slot : MAX_DEPTH);
    if (s.depth < 2) {  // the longest rows: one CTA per SM
        s.per_sm = 1;
        s.depth = (int)(SLOT_ROOM / slot < MAX_DEPTH ? SLOT_ROOM / slot : MAX_DEPTH);
    }
    // Four segments a thread read the weights again from L1, and the slots take L1's
    // room: 8192 rows, us with four (what fits) | three | two slots: bf16 9216 137 |
    // 133 | 140, with dropout 245 | 221 | 219; float32 9216 228 (three fit) | 228 |
    // 188; bf16 ragged 8705 326 | 327 | 315.
    if (bwd && s.nch == 4) {
        const int most = vec && esize == 2 && !drop ? 3 : 2;
        if (s.depth > most) s.depth = most;
    }
    s.smem = RING_HEAD + (int)(s.depth * slot);
    if (bwd && s.rows_per_cta > 1) {
        const int acc = RING_HEAD + (int)(s.rows_per_cta * 2 * cols * 4);
        if (acc > s.smem) s.smem = acc;
    }
    return s;
}
static int grid_of(const Shape &s, int64_t rows) {
    const int64_t ctas = (rows + s.rows_per_cta - 1) / s.rows_per_cta;
    const int64_t cap = (int64_t)num_sms() * s.per_sm;
    return (int)(ctas < cap ? ctas : cap);
}
static int long_parts(int64_t rows, int64_t cols) {
    const int64_t x = (cols + 4 * SEG - 1) / (4 * SEG);
    int64_t y = ((int64_t)num_sms() * 12 + x - 1) / x;
    if (y > rows) y = rows;
    return (int)(y < 1 ? 1 : (y > 65535 ? 65535 : y));
}
// Rows that go through the re-reading kernels: more than the registers hold, or
// (backward) than leaves two ring slots in shared memory.
static bool is_long(int64_t cols, int esize, bool drop, bool bwd) {
    if (cols > (int64_t)MAX_SEGS * SEG) return true;
    return bwd && 2 * (int64_t)row_pitch(cols, esize, false) * (drop ? 3 : 2) > SLOT_ROOM;
}
static size_t up256(size_t b) { return (b + 255) / 256 * 256; }

static size_t bwd_workspace(int64_t rows, int64_t cols) {
    size_t need = 0;
    if (cols <= (int64_t)MAX_SEGS * SEG) {
        const Shape s = shape_of(cols, 2, false, true, false);  // the largest grid of the forms
        need = up256((size_t)grid_of(s, rows) * 2 * cols * 4);
    }
    if (is_long(cols, 4, true, true)) {  // for some type or form
        const size_t l = up256((size_t)long_parts(rows, cols) * 2 * cols * 4) + up256((size_t)rows * 8);
        if (l > need) need = l;
    }
    return need;
}

template <typename T, typename W, bool VEC, bool DROP>
static int fwd_launch(const FwdArgs<T, W> &a, cudaStream_t st) {
    if (is_long(a.cols, sizeof(T), DROP, false)) {
        const int64_t cap = (int64_t)num_sms() * 4;
        ln_fwd_long_kernel<T, W, VEC, DROP><<<(int)(a.rows < cap ? a.rows : cap), LONG_THREADS, 0, st>>>(a);
        return launch_status();
    }
    const Shape s = shape_of(a.cols, sizeof(T), DROP, false, VEC);
    const int grid = grid_of(s, a.rows);
    auto go = [&](auto k) -> int {
        if (int rc = allow_smem(k, s.smem, MAX_SMEM)) return rc;
        k<<<grid, s.threads, s.smem, st>>>(a, s.wpr, s.depth);
        return launch_status();
    };
    if (s.wpr == 1) {
        if (s.nch == 1) return go(ln_fwd_kernel<T, W, 1, 256, VEC, DROP, true>);
        return s.nch == 2 ? go(ln_fwd_kernel<T, W, 2, 256, VEC, DROP, true>) : go(ln_fwd_kernel<T, W, 4, 256, VEC, DROP, true>);
    }
    if constexpr (DROP || sizeof(T) == 4) {  // see shape_of: the others take two segments
        if (s.nch == 1) return go(ln_fwd_kernel<T, W, 1, 256, VEC, DROP, false>);
    }
    if (s.nch == 2) return go(ln_fwd_kernel<T, W, 2, 256, VEC, DROP, false>);
    if (s.nch == 3) return go(ln_fwd_kernel<T, W, 3, 256, VEC, DROP, false>);
    return s.threads <= 256 ? go(ln_fwd_kernel<T, W, 4, 256, VEC, DROP, false>)
                            : go(ln_fwd_kernel<T, W, 4, 512, VEC, DROP, false>);
}

template <typename T, typename W, int NCH, int MAXT, bool VEC, bool DROP, bool MULTI>
static int bwd_main(const BwdArgs<T, W> &a, const Shape &s, int grid, cudaStream_t st) {
    auto k = ln_bwd_kernel<T, W, NCH, MAXT, VEC, DROP, MULTI>;
    if (int rc = allow_smem(k, s.smem, MAX_SMEM)) return rc;
    k<<<grid, s.threads, s.smem, st>>>(a, s.wpr, s.depth);
    return launch_status();
}

template <typename T, typename W, bool VEC, bool DROP>
static int bwd_launch(BwdArgs<T, W> a, W *dw, W *db, void *ws, cudaStream_t st) {
    int parts, rc;
    a.part = dw || db ? static_cast<float *>(ws) : nullptr;
    if (is_long(a.cols, sizeof(T), DROP, true)) {
        parts = long_parts(a.rows, a.cols);
        float2 *sums = reinterpret_cast<float2 *>(static_cast<uint8_t *>(ws) + up256((size_t)parts * 2 * a.cols * 4));
        const int64_t cap = (int64_t)num_sms() * 4;
        ln_bwd_sums_kernel<T, W, VEC><<<(int)(a.rows < cap ? a.rows : cap), LONG_THREADS, 0, st>>>(a, sums);
        const dim3 grid((unsigned)((a.cols + 4 * SEG - 1) / (4 * SEG)), (unsigned)parts);
        ln_bwd_cols_kernel<T, W, VEC, DROP><<<grid, 128, 0, st>>>(a, sums);
        rc = launch_status();
    } else {
        const Shape s = shape_of(a.cols, sizeof(T), DROP, true, VEC);
        parts = grid_of(s, a.rows);
        const bool multi = s.rows_per_cta > 1;
        constexpr int MID = sizeof(T) == 2 ? 320 : 512;  // float32 has no form of 320 threads (shape_of)
        rc = s.nch == 1           ? bwd_main<T, W, 1, 256, VEC, DROP, true>(a, s, parts, st)
             : s.nch == 4         ? bwd_main<T, W, 4, 512, VEC, DROP, false>(a, s, parts, st)
             : multi              ? bwd_main<T, W, 2, 256, VEC, DROP, true>(a, s, parts, st)
             : s.maxt == 256      ? bwd_main<T, W, 2, 256, VEC, DROP, false>(a, s, parts, st)
             : s.maxt == MID      ? bwd_main<T, W, 2, MID, VEC, DROP, false>(a, s, parts, st)
                                  : bwd_main<T, W, 2, 512, VEC, DROP, false>(a, s, parts, st);
    }
    if (rc || !a.part) return rc;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((2 * a.cols + 31) / 32));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    ACT_CUDA_TRY(cudaLaunchKernelEx(&cfg, ln_bwd_finish_kernel<W>, (const float *)a.part, parts, a.cols, dw, db));
    return ACT_OK;
}

// f(T tag, W tag) for the run-time types; wide: float32 weights.
template <typename F>
static int with_types(int dtype, int wide, F f) {
    if (dtype == 0) return f(float{}, float{});
    if (dtype == 1) return wide ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
    return wide ? f(__half{}, float{}) : f(__half{}, __half{});
}

static bool drop_params(DropParams &d, uint64_t seed, const uint64_t *seed_ptr, uint64_t row_offset, double p) {
    if (!(p >= 0.0 && p <= 1.0)) return false;
    d.seed = seed;
    d.seed_ptr = seed_ptr;
    d.row_offset = row_offset;
    d.threshold = (uint32_t)__builtin_rint(p * 65536.0);
    d.scale = d.threshold < 65536u ? (float)(65536.0 / (65536.0 - (double)d.threshold)) : 0.f;
    return true;
}

// 16-byte access to every row: base and row stride
static bool vec_ok(const void *p, int64_t ld, int esize) { return !p || (aligned(p, 16) && (ld * esize) % 16 == 0); }

}  // namespace norm
}  // namespace act

extern "C" int actcomp_dropout(const actcomp_drop_args *g, void *stream) {
    using namespace act;
    using namespace act::norm;
    ACT_CHECK(g && g->rows >= 0 && g->cols >= 0, ACT_E_INVALID);
    ACT_CHECK(g->dtype >= 0 && g->dtype <= 2, ACT_E_INVALID);
    DropParams d;
    ACT_CHECK(drop_params(d, g->seed, g->seed_ptr, g->row_offset, g->p), ACT_E_INVALID);
    if (g->rows == 0 || g->cols == 0) return ACT_OK;
    ACT_CHECK(g->x && g->y && g->ldx >= g->cols && g->ldy >= g->cols, ACT_E_INVALID);
    ACT_CHECK(g->cols <= ((int64_t)1 << 34) && g->rows <= ((int64_t)1 << 40), ACT_E_UNSUPPORTED);
    const int es = g->dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(g->x, es) && aligned(g->y, es) && aligned(g->seed_ptr, 8), ACT_E_ALIGN);
    const bool vec = g->cols % 8 == 0 && vec_ok(g->x, g->ldx, es) && vec_ok(g->y, g->ldy, es);
    // division by segs: quotient of a 32-bit u = (((u - h) >> 1) + h) >> (l - 1), h = umulhi(u, mul),
    // l = ceil(log2 segs), mul = floor(2^32 (2^l - segs) / segs) + 1
    const uint32_t segs = (uint32_t)((g->cols + SEG - 1) / SEG);
    uint32_t l = 0;
    while (((uint64_t)1 << l) < segs) ++l;
    const uint32_t mul = segs > 1 ? (uint32_t)((((((uint64_t)1 << l) - segs) << 32) / segs) + 1) : 0;
    const int64_t most = 0x7fffffff / segs;  // rows a launch
    cudaStream_t st = as_stream(stream);
    return with_types(g->dtype, 0, [&](auto t, auto) {
        using T = decltype(t);
        for (int64_t r = 0; r < g->rows; r += most) {
            const int64_t rows = g->rows - r < most ? g->rows - r : most;
            DropArgs<T> a{static_cast<const T *>(g->x) + r * g->ldx, static_cast<T *>(g->y) + r * g->ldy, g->cols,
                          g->ldx, g->ldy, d};
            a.d.row_offset += (uint64_t)r;
            const uint32_t units = (uint32_t)(rows * segs);
            const int64_t cap = (int64_t)num_sms() * 8, ctas = ((int64_t)units + 7) / 8;
            const int grid = (int)(ctas < cap ? ctas : cap);
            if (vec) dropout_kernel<T, true><<<grid, 256, 0, st>>>(a, units, segs, mul, l - 1);
            else dropout_kernel<T, false><<<grid, 256, 0, st>>>(a, units, segs, mul, l - 1);
            if (int rc = launch_status()) return rc;
        }
        return (int)ACT_OK;
    });
}

extern "C" int actcomp_layer_norm(const actcomp_ln_args *g, void *stream) {
    using namespace act;
    using namespace act::norm;
    ACT_CHECK(g && g->rows >= 0 && g->cols > 0, ACT_E_INVALID);
    ACT_CHECK(g->dtype >= 0 && g->dtype <= 2 && (g->wdtype == g->dtype || g->wdtype == 0), ACT_E_INVALID);
    const bool drop = g->res != nullptr;
    DropParams d{};
    if (drop) ACT_CHECK(drop_params(d, g->seed, g->seed_ptr, g->row_offset, g->p), ACT_E_INVALID);
    ACT_CHECK(g->eps >= 0.f, ACT_E_INVALID);
    if (g->rows == 0) return ACT_OK;
    ACT_CHECK(g->x && g->y && g->mean && g->rstd, ACT_E_INVALID);
    ACT_CHECK(g->ldx >= g->cols && g->ldy >= g->cols, ACT_E_INVALID);
    ACT_CHECK(!drop || (g->h && g->ldr >= g->cols && g->ldh >= g->cols), ACT_E_INVALID);
    ACT_CHECK(g->cols <= ((int64_t)1 << 30) && g->rows <= ((int64_t)1 << 40), ACT_E_UNSUPPORTED);
    const int es = g->dtype == 0 ? 4 : 2, ws = g->wdtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(g->x, es) && aligned(g->y, es) && aligned(g->res, es) && aligned(g->h, es), ACT_E_ALIGN);
    ACT_CHECK(aligned(g->weight, ws) && aligned(g->bias, ws) && aligned(g->mean, 4) && aligned(g->rstd, 4) &&
                  aligned(g->seed_ptr, 8),
              ACT_E_ALIGN);
    const bool vec = g->cols % 8 == 0 && vec_ok(g->x, g->ldx, es) && vec_ok(g->y, g->ldy, es) &&
                     vec_ok(g->res, g->ldr, es) && vec_ok(g->h, g->ldh, es) && aligned(g->weight, 16) &&
                     aligned(g->bias, 16);
    cudaStream_t st = as_stream(stream);
    return with_types(g->dtype, g->wdtype == 0, [&](auto t, auto w) {
        using T = decltype(t);
        using W = decltype(w);
        FwdArgs<T, W> a{static_cast<const T *>(g->x), static_cast<const T *>(g->res), static_cast<const W *>(g->weight),
                        static_cast<const W *>(g->bias), static_cast<T *>(g->y), static_cast<T *>(g->h), g->mean,
                        g->rstd, g->rows, g->cols, g->ldx, g->ldr, g->ldy, g->ldh, g->eps, d};
        if (drop) return vec ? fwd_launch<T, W, true, true>(a, st) : fwd_launch<T, W, false, true>(a, st);
        return vec ? fwd_launch<T, W, true, false>(a, st) : fwd_launch<T, W, false, false>(a, st);
    });
}

extern "C" size_t actcomp_layer_norm_bwd_workspace(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 ? act::norm::bwd_workspace(rows, cols) : 0;
}

extern "C" int actcomp_layer_norm_bwd(const actcomp_ln_bwd_args *g, void *workspace, size_t workspace_bytes,
                                      void *stream) {
    using namespace act;
    using namespace act::norm;
    ACT_CHECK(g && g->rows >= 0 && g->cols > 0, ACT_E_INVALID);
    ACT_CHECK(g->dtype >= 0 && g->dtype <= 2 && (g->wdtype == g->dtype || g->wdtype == 0), ACT_E_INVALID);
    const bool drop = g->dr != nullptr;
    DropParams d{};
    if (drop) ACT_CHECK(drop_params(d, g->seed, g->seed_ptr, g->row_offset, g->p), ACT_E_INVALID);
    const int es = g->dtype == 0 ? 4 : 2, wsz = g->wdtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(g->dweight, wsz) && aligned(g->dbias, wsz), ACT_E_ALIGN);
    cudaStream_t st = as_stream(stream);
    if (g->rows == 0) {  // the sums over no rows
        if (g->dweight) ACT_CUDA_TRY(cudaMemsetAsync(g->dweight, 0, (size_t)g->cols * wsz, st));
        if (g->dbias) ACT_CUDA_TRY(cudaMemsetAsync(g->dbias, 0, (size_t)g->cols * wsz, st));
        return ACT_OK;
    }
    ACT_CHECK(g->dy && g->x && g->dx && g->mean && g->rstd, ACT_E_INVALID);
    ACT_CHECK(g->lddy >= g->cols && g->ldx >= g->cols && g->lddx >= g->cols, ACT_E_INVALID);
    ACT_CHECK(!drop || g->lddr >= g->cols, ACT_E_INVALID);
    ACT_CHECK(!g->dh || (drop && g->lddh >= g->cols), ACT_E_INVALID);
    ACT_CHECK(g->cols <= ((int64_t)1 << 30) && g->rows <= ((int64_t)1 << 40), ACT_E_UNSUPPORTED);
    ACT_CHECK(aligned(g->dy, es) && aligned(g->x, es) && aligned(g->dx, es) && aligned(g->dr, es) && aligned(g->dh, es),
              ACT_E_ALIGN);
    ACT_CHECK(aligned(g->weight, wsz) && aligned(g->mean, 4) && aligned(g->rstd, 4) && aligned(g->seed_ptr, 8),
              ACT_E_ALIGN);
    ACT_CHECK(workspace && aligned(workspace, 16) && workspace_bytes >= bwd_workspace(g->rows, g->cols),
              ACT_E_WORKSPACE);
    const bool vec = g->cols % 8 == 0 && vec_ok(g->dy, g->lddy, es) && vec_ok(g->x, g->ldx, es) &&
                     vec_ok(g->dh, g->lddh, es) && vec_ok(g->dx, g->lddx, es) && vec_ok(g->dr, g->lddr, es) &&
                     aligned(g->weight, 16);
    return with_types(g->dtype, g->wdtype == 0, [&](auto t, auto w) {
        using T = decltype(t);
        using W = decltype(w);
        BwdArgs<T, W> a{static_cast<const T *>(g->dy), static_cast<const T *>(g->x), static_cast<const T *>(g->dh),
                        static_cast<const W *>(g->weight), g->mean, g->rstd, static_cast<T *>(g->dx),
                        static_cast<T *>(g->dr), nullptr, g->rows, g->cols, g->lddy, g->ldx, g->lddh, g->lddx, g->lddr,
                        d};
        W *dw = static_cast<W *>(g->dweight), *db = static_cast<W *>(g->dbias);
        if (drop)
            return vec ? bwd_launch<T, W, true, true>(a, dw, db, workspace, st)
                       : bwd_launch<T, W, false, true>(a, dw, db, workspace, st);
        return vec ? bwd_launch<T, W, true, false>(a, dw, db, workspace, st)
                   : bwd_launch<T, W, false, false>(a, dw, db, workspace, st);
    });
}

extern "C" int actcomp_selftest_row_waits(const float *x, int32_t rows, int32_t brought, uint32_t polls, float *out,
                                          void *stream) {
    using namespace act;
    using namespace act::norm;
    ACT_CHECK(x && out && rows >= 1 && rows <= 1024 && brought >= 0 && brought <= rows, ACT_E_INVALID);
    ACT_CHECK(polls >= 1 && polls <= (1u << 24), ACT_E_INVALID);
    ACT_CHECK(aligned(x, 16) && aligned(out, 4), ACT_E_ALIGN);
    selftest_ring_kernel<<<1, 32, 0, as_stream(stream)>>>(x, rows, brought, polls, out);
    return launch_status();
}
