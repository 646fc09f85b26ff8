// rows.cuh -- what the kernels that work on whole rows share (layer norm, root-mean-square
// norm): a warp's segments of a row and their types, the reductions over the warps
// of a row, and the ring that brings rows to shared memory ahead of their use.
#pragma once

#include <cuda_fp16.h>
#include <string.h>

#include <type_traits>

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

// ---------------------------------------------------------------- reductions
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

// ---------------------------------------------------------------- rows ahead of their use
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

}  // namespace norm
}  // namespace act
