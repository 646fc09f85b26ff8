// xent.cu -- softmax cross entropy of a linear layer over a large vocabulary, with its
// gradients; the logits are never in memory (no reference counterpart: the
// reference's low_rank_system_profile_backward.py ends at the linear layers).
//
//   z = x . W^T,  lse = log sum_v exp z_v,  loss = lse - z_target
//   g = exp(z - lse) (dloss + dlse) - [v = target] dloss
//   dx = g . W,   dW = g^T . x
//
// Four products of 2 T V H operations on CTA pairs (pair_gemm.cuh), one forward and
// three backward: the logits are computed again there, since what the forward pass
// keeps is lse, four bytes a token.
//   forward   a tile's epilogue holds a token's 128 logits of a thread's half row as
//             they leave TMEM: running maximum and sum of exponentials, written as
//             one pair per token and half tile, joined by a second small kernel; the
//             target's logit is written by the thread that meets it.
//   backward  the vocabulary in pieces: a piece's g (tokens x piece, 16 bits) is
//             written by the epilogue of its logits, and both gradients' products read
//             it.  dx is summed over the pieces in float32.
// Exponentials are base 2 of values scaled by log2 e in one fused multiply-add; sums
// and maxima are float32, the last step from them to lse and loss is double.
//
// g enters the tensor cores in the activations' type, rounded once.  So that fp16 holds
// it whatever the size of dloss, each token's g is divided by the power of two s_t
// below max(|dloss|, |dloss + dlse|), dx is multiplied by it again in float32, and
// for dW, which sums over tokens, x's rows are multiplied by s_t / max s (exact but for
// subnormals) and the result by max s.  The same copy of x has zeros in the rows of
// tokens that have no gradient, so that nothing they hold reaches dW.
//
// Bound by the tensor pipe under the power limit: forward of 8192 x 4096 x 64000 2.67 ms
// (1.61 PFLOP/s), over seconds 1.38 to 1.40 PFLOP/s (the library's product alone 1.33 to
// 1.36); backward 2.85 (g), 3.0 (dx) and 3.2 ms (dW).  Small ones by start and end of
// their five launches: 511 x 1024 x 32000 33, 34, 31 and 37 us of 20.5 at the burst rate,
// and 5 each for the factors and the sum of dx's parts (18, 14 and 13 us for the join,
// the factors and the sum with less parallelism and a launch more).  The tensor cores'
// sums truncate: lse is within 1.6e-6 of the exact one at 4096 channels (4e-7 at 1024),
// float32 sums on the CUDA cores within 1.4e-7.  g in panels of 64
// columns, a tile of it one piece of memory, was 1.5 to 2 % slower.
#include "pair_gemm.cuh"

namespace act {
namespace xent {

using pair::Params;
using pair::Tile;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int BK = 64;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---------------------------------------------------------------- epilogues
// Per token and half tile: the scaled maximum and the sum of exponentials about it.
struct FwdP {
    float2 *part;  // [2 n_tiles][M]
    float *at;     // the target's logit
    const int64_t *target;
};
struct FwdEpi {
    using P = FwdP;
    const P &o;
    int lane, row = 0, half_tile = 0;
    int64_t target = -1;
    float m = 0.f, s = 0.f;
    __device__ __forceinline__ FwdEpi(const P &o, uint8_t *, const CUtensorMap *, int lane) : o(o), lane(lane) {}
    __device__ __forceinline__ void begin(const Params &p, const Tile &t, int row0, int half) {
        row = row0 + lane;
        half_tile = 2 * t.n + half;
        target = row < p.M ? o.target[row] : -1;
        m = -INFINITY, s = 0.f;
    }
    __device__ __forceinline__ void group(const Params &p, const uint32_t (&r)[32], int col) {
        if (col >= p.N) return;
        const int n = p.N - col;  // 32 or more but for the last group
        float v[32], top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            v[i] = i < n ? __uint_as_float(r[i]) : -INFINITY;
            top[i & 3] = fmaxf(top[i & 3], v[i]);
        }
        const float t = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * LOG2E;
        const float now = fmaxf(m, t);
        if (now > -INFINITY) {  // of -inf alone nothing is summed
            const float2 l = make_float2(LOG2E, LOG2E), c = make_float2(-now, -now);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 e = fma2(make_float2(v[2 * i], v[2 * i + 1]), l, c);
                sum = add2(sum, make_float2(ex2(e.x), ex2(e.y)));
            }
            s = __fmaf_rn(s, ex2(m - now), sum.x + sum.y);
            m = now;
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (v[i] != v[i]) s = v[i];  // the maximum passes NaN over
        }
        const int64_t j = target - col;
        if (__any_sync(0xffffffffu, j >= 0 && j < 32 && j < n)) {
            float z = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) z = j == i ? v[i] : z;
            if (j >= 0 && j < 32 && j < n && row < p.M) o.at[row] = z;
        }
    }
    __device__ __forceinline__ void end(const Params &p) {
        if (row < p.M && ACT_DCHECK(half_tile < 2 * p.n_tiles)) o.part[(int64_t)half_tile * p.M + row] = make_float2(m, s);
    }
    __device__ __forceinline__ void lost(const Params &p) {
        m = 0.f, s = __uint_as_float(0x7fc00000u);
        end(p);
    }
};

// What the gradient's epilogue needs of a token.
struct alignas(16) Row {
    float lse2, a, d, scale;  // lse log2 e; (dloss + dlse) / scale, dloss / scale; s_t
};
struct GradP {
    pair::OutParams o;
    const Row *rows;
    const int64_t *target;
    int64_t v0;  // first column of the piece
};
template <typename T>
struct GradEpi {
    using P = GradP;
    const P &o;
    const CUtensorMap *tmC;
    pair::Out<T, pair::OUT_BYTES / 8> out;
    int lane, row0 = 0;
    int64_t target = -1;
    Row r{};
    __device__ __forceinline__ GradEpi(const P &o, uint8_t *stage, const CUtensorMap *tmC, int lane)
        : o(o), tmC(tmC), out{stage}, lane(lane) {}
    __device__ __forceinline__ void begin(const Params &p, const Tile &, int first, int) {
        row0 = first;
        const int row = first + lane;
        r = Row{0.f, 0.f, 0.f, 0.f};
        target = -1;
        if (row < p.M) {
            const float4 q = __ldg(reinterpret_cast<const float4 *>(o.rows) + row);
            r = Row{q.x, q.y, q.z, q.w};
            target = r.d != 0.f ? o.target[row] - o.v0 : -1;
        }
    }
    __device__ __forceinline__ void group(const Params &p, const uint32_t (&z)[32], int col) {
        if (row0 >= p.M || col >= p.N) return;
        const bool live = !(r.a == 0.f && r.d == 0.f);
        const float2 l = make_float2(LOG2E, LOG2E), c = make_float2(-r.lse2, -r.lse2), a2 = make_float2(r.a, r.a);
        float v[32];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 e = fma2(make_float2(__uint_as_float(z[2 * i]), __uint_as_float(z[2 * i + 1])), l, c);
            const float2 g = mul2(make_float2(ex2(e.x), ex2(e.y)), a2);
            v[2 * i] = live ? g.x : 0.f;
            v[2 * i + 1] = live ? g.y : 0.f;
        }
        const int64_t j = target - col;
        if (__any_sync(0xffffffffu, j >= 0 && j < 32)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = j == i ? v[i] - r.d : v[i];
        }
        out.put(v, row0, col, p.M, p.N, lane, o.o, tmC);
    }
    __device__ __forceinline__ void end(const Params &) {}
    // g unwritten would be read as it lies: NaN in its place
    __device__ __forceinline__ void lost(const Params &p) {
        const int row = row0 + lane;
        if (row >= p.M) return;
        T *d = static_cast<T *>(o.o.C) + (int64_t)row * o.o.ldc;
        for (int c = 0; c < p.N; ++c) d[c] = pair::cvt_out<T>(__uint_as_float(0x7fc00000u));
    }
};

// A gradient's tile: (acc + what is there already) * scale of the row * scale of all.
struct SumP {
    pair::OutParams o;
    const float *add;        // float32, row stride ld_add; null: 0
    int64_t ld_add, part;    // part: floats from one split's buffer to the next (of o.C too)
    const Row *rows;         // null: 1
    const float *scale;      // null: 1
};
template <typename T>
struct SumEpi {
    using P = SumP;
    const P &o;
    const CUtensorMap *tmC;
    pair::Out<T, pair::OUT_BYTES / 8> out;
    pair::OutParams to;
    int lane, row0 = 0, split = 0;
    const float *add = nullptr;
    float f = 1.f, all;
    __device__ __forceinline__ SumEpi(const P &o, uint8_t *stage, const CUtensorMap *tmC, int lane)
        : o(o), tmC(tmC), out{stage}, to(o.o), lane(lane), all(o.scale ? __ldg(o.scale) : 1.f) {}
    __device__ __forceinline__ void begin(const Params &p, const Tile &t, int first, int) {
        row0 = first;
        const int row = first + lane;
        f = all;
        if (o.rows && row < p.M) f *= o.rows[row].scale;
        split = t.split;
        to.C = static_cast<T *>(o.o.C) + split * o.part;
        add = o.add && row < p.M ? o.add + split * o.part + (int64_t)row * o.ld_add : nullptr;
    }
    __device__ __forceinline__ void group(const Params &p, const uint32_t (&r)[32], int col) {
        if (row0 >= p.M || col >= p.N) return;
        float v[32];
        if (add) {
            const int n = p.N - col;
            if (n >= 32) {  // rows of part are 16-byte aligned
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 q = __ldcg(reinterpret_cast<const float4 *>(add + col) + i);
                    v[4 * i] = q.x, v[4 * i + 1] = q.y, v[4 * i + 2] = q.z, v[4 * i + 3] = q.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = i < n ? __ldcg(add + col + i) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = (__uint_as_float(r[i]) + v[i]) * f;
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]) * f;
        }
        out.put(v, row0, col, p.M, p.N, lane, to, tmC, split);
    }
    __device__ __forceinline__ void end(const Params &) {}
    __device__ __forceinline__ void lost(const Params &) {}
};

// ---------------------------------------------------------------- small kernels
// A token's partial maxima and sums joined: 32 tokens a CTA, a lane each, 32 warps over
// the partials, eight on their way at a time.
constexpr int JOIN_WARPS = 32;
__global__ void __launch_bounds__(32 * JOIN_WARPS)
    join_kernel(const float2 *part, int parts, int tokens, int64_t vocab, const int64_t *target, int64_t ignore,
                float *loss, float *lse) {
    __shared__ float2 red[JOIN_WARPS][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x * 32 + lane;
    float m = -INFINITY, s = 0.f;
    // N pairs into (m, s): one scale to the new maximum; without one (all -inf) the sums, 0 or the NaN of a tile
    // that had nothing else, are added as they are
    auto join = [&](auto &q) {
        constexpr int N = sizeof(q) / sizeof(float2);
        float now = m;
#pragma unroll
        for (int i = 0; i < N; ++i) now = fmaxf(now, q[i].x);
        if (now > -INFINITY) {
            s *= ex2(m - now);
#pragma unroll
            for (int i = 0; i < N; ++i) s = __fmaf_rn(q[i].y, ex2(q[i].x - now), s);
            m = now;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) s += q[i].y;
        }
    };
    tc::dependence_wait();
    if (row < tokens) {
        const float2 *p = part + row;
        int i = warp;
        for (; i + 7 * JOIN_WARPS < parts; i += 8 * JOIN_WARPS) {
            float2 q[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) q[k] = p[(int64_t)(i + k * JOIN_WARPS) * tokens];
            join(q);
        }
        float2 q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            q[k] = i + k * JOIN_WARPS < parts ? p[(int64_t)(i + k * JOIN_WARPS) * tokens] : make_float2(-INFINITY, 0.f);
        join(q);
    }
    red[warp][lane] = make_float2(m, s);
    __syncthreads();
    if (warp != 0 || row >= tokens) return;
    for (int i = 1; i < JOIN_WARPS; ++i) {
        float2 q[1] = {red[i][lane]};
        join(q);
    }
    const double l = (double)m * 0.69314718055994530942 + (double)logf(s);
    lse[row] = (float)l;
    const int64_t t = target[row];
    loss[row] = t == ignore              ? 0.f
                : t >= 0 && t < vocab ? (float)(l - (double)loss[row])
                                         : __uint_as_float(0x7fc00000u);
}

struct GradArgs {
    const int64_t *target;
    const float *lse, *dloss, *dlse;  // dlse may be null
    int64_t ignore, vocab, tokens;
};
// The token's factors of exp(z - lse) and of the target's one.
__device__ __forceinline__ void factors(const GradArgs &g, int64_t row, float &a, float &d) {
    const int64_t t = g.target[row];
    const bool out = t < 0 || t >= g.vocab;
    d = t == g.ignore ? 0.f : out ? __uint_as_float(0x7fc00000u) : g.dloss[row];
    a = g.dlse ? d + g.dlse[row] : d;
}
// The power of two at or below |v| (1 for 0, the smallest normal for less; NaN gives 2^127).
__device__ __forceinline__ float pow2_below(float v) {
    const uint32_t e = __float_as_uint(v) & 0x7f800000u;
    return v == 0.f ? 1.f : __uint_as_float(e == 0x7f800000u ? 0x7f000000u : e == 0u ? 0x00800000u : e);
}
// The tokens' factors, and x's rows scaled for dW (null: not wanted).  A warp a token;
// every CTA finds the largest factor for itself (a pass over 12 bytes a token from L2,
// on at most one CTA per SM, where a kernel of its own took 5 us).
template <typename T>
__global__ void __launch_bounds__(1024)
    rows_kernel(GradArgs g, float *scale, Row *rows, const T *x, int64_t ldx, int64_t cols, T *xs, int64_t lds) {
    __shared__ float red[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    tc::dependence_wait();
    float m = 0.f;
    for (int64_t r = threadIdx.x; r < g.tokens; r += 1024) {
        float a, d;
        factors(g, r, a, d);
        m = fmaxf(m, fmaxf(fabsf(a), fabsf(d)));  // passes NaN over
    }
    m = warp_max(m);
    if (lane == 0) red[warp] = m;
    __syncthreads();
    const float top = pow2_below(warp_max(red[lane]));
    if (blockIdx.x == 0 && threadIdx.x == 0) *scale = top;
    for (int64_t r = (int64_t)blockIdx.x * 32 + warp; r < g.tokens; r += (int64_t)gridDim.x * 32) {
        float a, d;
        factors(g, r, a, d);
        const bool live = !(a == 0.f && d == 0.f);
        const float s = pow2_below(fmaxf(fabsf(a), fabsf(d)));
        if (lane == 0) rows[r] = Row{live ? g.lse[r] * LOG2E : 0.f, a / s, d / s, live ? s : 1.f};
        if (!xs) continue;
        const float f = live ? s / top : 0.f;
        const T *src = x + r * ldx;
        T *dst = xs + r * lds;
        const int64_t whole = cols & ~(int64_t)7;  // rows are 16-byte aligned
        auto scaled = [&](T v) { return live ? pair::cvt_out<T>((float)v * f) : pair::cvt_out<T>(0.f); };
        for (int64_t c0 = 8 * lane; c0 < whole; c0 += 4 * 256) {
            uint4 q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (c0 + 256 * k < whole) q[k] = *reinterpret_cast<const uint4 *>(src + c0 + 256 * k);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (c0 + 256 * k >= whole) break;
                T v[8];
                memcpy(v, &q[k], 16);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = scaled(v[j]);
                memcpy(&q[k], v, 16);
                *reinterpret_cast<uint4 *>(dst + c0 + 256 * k) = q[k];
            }
        }
        for (int64_t c = whole + lane; c < cols; c += 32) dst[c] = scaled(src[c]);
    }
}
// dx from the splits' sums, in a fixed order: four values a thread, blockIdx.y over the
// tokens.
template <typename T>
__global__ void __launch_bounds__(256)
    sum_kernel(const float *part, int splits, int tokens, int cols, int64_t ld, const Row *rows, T *dx, int64_t lddx) {
    const int c = (blockIdx.x * 256 + threadIdx.x) * 4;
    tc::dependence_wait();
    if (c >= cols) return;
    for (int r = blockIdx.y; r < tokens; r += gridDim.y) {
        const float *p = part + (int64_t)r * ld + c;
        const int64_t step = (int64_t)tokens * ld;
        float4 s = *reinterpret_cast<const float4 *>(p);  // ld is a multiple of 4: whole pieces are there
        for (int k = 1; k < splits; ++k) {
            const float4 q = *reinterpret_cast<const float4 *>(p + k * step);
            s.x += q.x, s.y += q.y, s.z += q.z, s.w += q.w;
        }
        const float f = rows[r].scale, v[4] = {s.x * f, s.y * f, s.z * f, s.w * f};
        T *d = dx + (int64_t)r * lddx + c;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < cols && ACT_DCHECK(c + i < lddx)) d[i] = pair::cvt_out<T>(v[i]);
    }
}
// A launch with programmatic dependence on the kernel before it.
template <typename... P, typename... A>
static int launch_after(void (*k)(P...), dim3 grid, int threads, cudaStream_t st, A... args) {
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    ACT_CUDA_TRY(cudaLaunchKernelEx(&cfg, k, P(args)...));
    return ACT_OK;
}

// ---------------------------------------------------------------- host
static size_t up256(size_t b) { return (b + 255) / 256 * 256; }
static int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }
static int map_k(CUtensorMap *m, CUtensorMapDataType dt, const void *p, int64_t k, int64_t lines, int64_t ld) {
    return make_map_3d(m, p, dt, 2, k, lines, 1, ld, 0, BK, 128, CU_TENSOR_MAP_SWIZZLE_128B);
}
static int map_mn(CUtensorMap *m, CUtensorMapDataType dt, const void *p, int64_t lines, int64_t k, int64_t ld) {
    return make_map_3d(m, p, dt, 2, lines, k, 1, ld, 0, 64, BK, CU_TENSOR_MAP_SWIZZLE_128B);
}
static int map_out(CUtensorMap *m, CUtensorMapDataType dt, int es, void *p, int64_t cols, int64_t rows, int64_t ld) {
    return make_map_3d(m, p, dt, es, cols, rows, 1, ld, 0, 32, 32,
                       es == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}
static bool tma_rows(const void *p, int64_t ld, int es) { return aligned(p, 16) && (ld * es) % 16 == 0; }

// Columns of the vocabulary in a piece: what is asked for, or g in at most 1 GiB, but 4096
// at least (every piece reads and writes dx's sums, 8 bytes a value, against 2 operations
// a value and column); pieces of about one size, whole tiles.
static int64_t piece_of(int64_t tokens, int64_t vocab, int64_t asked) {
    int64_t most = asked > 0 ? asked : ((int64_t)1 << 29) / (tokens > 0 ? tokens : 1);
    if (!asked && most < 4096) most = 4096;
    const int64_t whole = (vocab + pair::BN - 1) / pair::BN * pair::BN;
    most = most < whole ? most / pair::BN * pair::BN : whole;  // any number above the vocabulary is all of it
    if (most < pair::BN) most = pair::BN;
    const int64_t pieces = (vocab + most - 1) / most;
    return ((vocab + pieces - 1) / pieces + pair::BN - 1) / pair::BN * pair::BN;
}
// Parts of dx's contraction (a piece of the vocabulary): as many as fill the device
// when its tiles do not, at least sixteen stages each.
static int splits_of(int64_t tokens, int64_t channels, int64_t piece) {
    const int64_t tiles = ((tokens + 255) / 256) * ((channels + 255) / 256), pairs = num_sms() / 2;
    int64_t s = pairs / tiles;
    const int64_t most = (piece / BK) / 16;
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}
struct Plan {
    int64_t piece, ldg, ldx, ldd;
    int pieces, splits;
    size_t rows, scale, g, xs, part, total;  // offsets
};
static Plan plan_of(int64_t tokens, int64_t channels, int64_t vocab, int64_t asked) {
    Plan q{};
    q.piece = piece_of(tokens, vocab, asked);
    q.pieces = (int)((vocab + q.piece - 1) / q.piece);
    q.splits = splits_of(tokens, channels, q.piece < vocab ? q.piece : (vocab + 255) / 256 * 256);
    q.ldg = q.piece;
    q.ldx = up8(channels);
    q.ldd = (channels + 3) / 4 * 4;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += up256(bytes);
        return o;
    };
    q.rows = take((size_t)tokens * sizeof(Row));
    q.scale = take(4);
    q.g = take((size_t)tokens * q.ldg * 2);
    q.xs = take((size_t)tokens * q.ldx * 2);
    q.part = take(q.splits > 1 || q.pieces > 1 ? (size_t)q.splits * tokens * q.ldd * 4 : 0);
    q.total = at;
    return q;
}

static int check(const actcomp_xent_args *g) {
    ACT_CHECK(g && g->tokens >= 0 && g->channels > 0 && g->vocab > 0, ACT_E_INVALID);
    ACT_CHECK(g->dtype == 1 || g->dtype == 2, ACT_E_INVALID);
    if (g->tokens == 0) return ACT_OK;
    ACT_CHECK(g->x && g->weight && g->target && g->lse && g->ldx >= g->channels && g->ldw >= g->channels,
              ACT_E_INVALID);
    const int64_t most = INT32_MAX - 511;
    ACT_CHECK(g->tokens <= most && g->channels <= most && g->vocab <= most, ACT_E_UNSUPPORTED);
    ACT_CHECK(((g->tokens + 255) / 256) * ((g->vocab + 255) / 256) <= most &&
                  ((g->vocab + 255) / 256) * ((g->channels + 255) / 256) <= most &&
                  ((g->tokens + 255) / 256) * ((g->channels + 255) / 256) * 64 <= most,
              ACT_E_UNSUPPORTED);
    ACT_CHECK(tma_rows(g->x, g->ldx, 2) && tma_rows(g->weight, g->ldw, 2), ACT_E_ALIGN);
    ACT_CHECK(aligned(g->target, 8) && aligned(g->lse, 4) && aligned(g->loss, 4), ACT_E_ALIGN);
    return ACT_OK;
}
static CUtensorMapDataType map_type(int dtype) {
    return dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

template <typename T>
static int backward(const actcomp_xent_args *g, const actcomp_xent_grads *o, const Plan &q, uint8_t *ws,
                    cudaStream_t st) {
    const CUtensorMapDataType dt = map_type(g->dtype);
    const bool bf = g->dtype == 1;
    const int T_ = (int)g->tokens, H = (int)g->channels;
    Row *rows = reinterpret_cast<Row *>(ws + q.rows);
    float *scale = reinterpret_cast<float *>(ws + q.scale), *part = reinterpret_cast<float *>(ws + q.part);
    T *gs = reinterpret_cast<T *>(ws + q.g), *xs = reinterpret_cast<T *>(ws + q.xs);
    const GradArgs ga{g->target, g->lse, o->dloss, o->dlse, g->ignore_index, g->vocab, g->tokens};
    const int64_t cap = num_sms(), need = (g->tokens + 31) / 32;
    if (int rc = launch_after(rows_kernel<T>, dim3((unsigned)(need < cap ? need : cap)), 1024, st, ga, scale, rows,
                              static_cast<const T *>(g->x), g->ldx, g->channels, o->dweight ? xs : nullptr, q.ldx))
        return rc;
    const int k_first = (int)(((g->vocab < q.piece ? g->vocab : q.piece) + BK - 1) / BK);
    const int k_split = (k_first + q.splits - 1) / q.splits, splits = (k_first + k_split - 1) / k_split;
    for (int i = 0; i < q.pieces; ++i) {
        const int64_t v0 = i * q.piece;
        const int n = (int)(g->vocab - v0 < q.piece ? g->vocab - v0 : q.piece);
        const T *w = static_cast<const T *>(g->weight) + v0 * g->ldw;
        CUtensorMap tmA, tmB, tmC;
        Params p{};
        // g of the piece
        pair::set_tiles(p, T_, n, (H + BK - 1) / BK);
        p.idesc = tc::idesc_f16(pair::BM, pair::BN, bf, false, false);
        int rc = map_k(&tmA, dt, g->x, H, T_, g->ldx);
        if (!rc) rc = map_k(&tmB, dt, w, H, n, g->ldw);
        if (!rc) rc = map_out(&tmC, dt, 2, gs, n, T_, q.ldg);
        if (!rc)
            rc = pair::launch<pair::F16, GradEpi<T>>(tmA, tmB, tmC, p, GradP{{gs, q.ldg, 1}, rows, g->target, v0}, st);
        if (rc) return rc;
        if (o->dx) {  // dx (+)= g . W
            pair::set_tiles(p, T_, H, (n + BK - 1) / BK);
            p.a_mn = 0, p.b_mn = 1;
            p.idesc = tc::idesc_f16(pair::BM, pair::BN, bf, false, true);
            rc = map_k(&tmA, dt, gs, n, T_, q.ldg);
            if (!rc) rc = map_mn(&tmB, dt, w, H, n, g->ldw);
            if (rc) return rc;
            const bool last = i + 1 == q.pieces;
            SumP s{};
            s.add = i > 0 ? part : nullptr;
            s.ld_add = q.ldd;
            s.part = (int64_t)T_ * q.ldd;
            // every piece is cut by the first's share; a shorter last one leaves the last splits' sums as they are
            p.k_split = k_split;
            p.splits = (p.kblocks + k_split - 1) / k_split;
            if (last && splits == 1) {
                s.rows = rows;
                s.o = {o->dx, o->lddx, pair::tma_out(o->dx, o->lddx, H, 2)};
                tmC = tmA;
                if (s.o.tma) rc = map_out(&tmC, dt, 2, o->dx, H, T_, o->lddx);
                if (!rc) rc = pair::launch<pair::F16, SumEpi<T>>(tmA, tmB, tmC, p, s, st);
            } else {
                s.o = {part, q.ldd, 1};
                rc = make_map_3d(&tmC, part, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, H, T_, splits, q.ldd, s.part, 32, 32,
                                 CU_TENSOR_MAP_SWIZZLE_128B);
                if (!rc) rc = pair::launch<pair::F16, SumEpi<float>>(tmA, tmB, tmC, p, s, st);
            }
            if (rc) return rc;
            if (last && splits > 1) {
                const dim3 grid((unsigned)((H + 1023) / 1024), (unsigned)(T_ < 65535 ? T_ : 65535));
                if ((rc = launch_after(sum_kernel<T>, grid, 256, st, part, splits, T_, H, q.ldd, rows,
                                       static_cast<T *>(o->dx), o->lddx)))
                    return rc;
            }
        }
        if (o->dweight) {  // dW = g^T . x
            pair::set_tiles(p, n, H, (T_ + BK - 1) / BK);
            p.a_mn = 1, p.b_mn = 1;
            p.idesc = tc::idesc_f16(pair::BM, pair::BN, bf, true, true);
            T *dw = static_cast<T *>(o->dweight) + v0 * o->lddw;
            SumP s{};
            s.scale = scale;
            s.o = {dw, o->lddw, pair::tma_out(dw, o->lddw, H, 2)};
            rc = map_mn(&tmA, dt, gs, n, T_, q.ldg);
            if (!rc) rc = map_mn(&tmB, dt, xs, H, T_, q.ldx);
            tmC = tmA;
            if (!rc && s.o.tma) rc = map_out(&tmC, dt, 2, dw, H, n, o->lddw);
            if (!rc) rc = pair::launch<pair::F16, SumEpi<T>>(tmA, tmB, tmC, p, s, st);
            if (rc) return rc;
        }
    }
    return ACT_OK;
}

}  // namespace xent
}  // namespace act

extern "C" size_t actcomp_xent_workspace(int64_t tokens, int64_t vocab) {
    return tokens > 0 && vocab > 0 ? (size_t)tokens * (size_t)((vocab + 255) / 256) * 2 * sizeof(float2) : 0;
}

extern "C" int actcomp_xent(const actcomp_xent_args *g, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace act;
    using namespace act::xent;
    if (int st = xent::check(g)) return st;
    if (g->tokens == 0) return ACT_OK;
    ACT_CHECK(g->loss, ACT_E_INVALID);
    ACT_CHECK(workspace && aligned(workspace, 16) && workspace_bytes >= actcomp_xent_workspace(g->tokens, g->vocab),
              ACT_E_WORKSPACE);
    const CUtensorMapDataType dt = map_type(g->dtype);
    CUtensorMap tmA, tmB;
    if (int st = map_k(&tmA, dt, g->x, g->channels, g->tokens, g->ldx)) return st;
    if (int st = map_k(&tmB, dt, g->weight, g->channels, g->vocab, g->ldw)) return st;
    pair::Params p{};
    pair::set_tiles(p, (int)g->tokens, (int)g->vocab, (int)((g->channels + BK - 1) / BK));
    p.idesc = tc::idesc_f16(pair::BM, pair::BN, g->dtype == 1, false, false);
    float2 *part = static_cast<float2 *>(workspace);
    cudaStream_t st = as_stream(stream);
    if (int rc = pair::launch<pair::F16, FwdEpi>(tmA, tmB, tmA, p, FwdP{part, g->loss, g->target}, st)) return rc;
    return launch_after(join_kernel, dim3((unsigned)((g->tokens + 31) / 32)), 32 * JOIN_WARPS, st, part, 2 * p.n_tiles,
                        (int)g->tokens, g->vocab, g->target, g->ignore_index, g->loss, g->lse);
}

extern "C" size_t actcomp_xent_bwd_workspace(int64_t tokens, int64_t channels, int64_t vocab, int64_t piece) {
    return tokens > 0 && channels > 0 && vocab > 0 ? act::xent::plan_of(tokens, channels, vocab, piece).total : 0;
}

extern "C" int actcomp_xent_bwd(const actcomp_xent_args *g, const actcomp_xent_grads *o, int64_t piece, void *workspace,
                                size_t workspace_bytes, void *stream) {
    using namespace act;
    using namespace act::xent;
    if (int st = xent::check(g)) return st;
    ACT_CHECK(o && piece >= 0 && (o->dx || o->dweight), ACT_E_INVALID);
    ACT_CHECK((!o->dx || o->lddx >= g->channels) && (!o->dweight || o->lddw >= g->channels), ACT_E_INVALID);
    ACT_CHECK(aligned(o->dx, 2) && aligned(o->dweight, 2) && aligned(o->dloss, 4) && aligned(o->dlse, 4), ACT_E_ALIGN);
    cudaStream_t st = as_stream(stream);
    if (g->tokens == 0) {  // the sum over no tokens
        if (o->dweight)
            ACT_CUDA_TRY(cudaMemset2DAsync(o->dweight, (size_t)o->lddw * 2, 0, (size_t)g->channels * 2, (size_t)g->vocab, st));
        return ACT_OK;
    }
    ACT_CHECK(o->dloss, ACT_E_INVALID);
    const Plan q = plan_of(g->tokens, g->channels, g->vocab, piece);
    ACT_CHECK(workspace && aligned(workspace, 256) && workspace_bytes >= q.total, ACT_E_WORKSPACE);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    return g->dtype == 1 ? backward<__nv_bfloat16>(g, o, q, ws, st) : backward<__half>(g, o, q, ws, st);
}
