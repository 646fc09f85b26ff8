// mx4_linear.cu -- x . w^T for a few tokens: x is quantised by rows on the way,
// w is a microscaled 4-bit matrix.
//
// It cannot do without the weight's 17/32 byte a value, read once, and one launch;
// the tensor cores' 128-row tiles would be nearly empty and the quantisation a
// launch of its own (1 x 4096 x 11008, weight in L2: 16.0 us for both, 8.9 us here; in
// memory 17.4 and 9.9).  Every CTA quantises all of x (it is small) into shared
// memory as 8-bit integers (twice the e2m1 value: 0, 1, 2, 3, 4, 6, 8, 12 and their
// negatives), one scale per block.
//   warp  the four rows r0, r0 + 32, r0 + 64, r0 + 96 of a scale atom, whose
//         scale words lie in one 16-byte piece; its pieces arrive by cp.async;
//   lane  whole blocks of 32 values (16 bytes), every 32nd; a block's dot product
//         is an exact integer (__dp4a), scaled and added in float32.
// A code's magnitude comes from a byte permutation: three bits of a code select
// one of eight table bytes, the fourth (the sign) replaces it by its sign bit,
// 0; the codes with their signs flipped give the negative ones' magnitudes.
// Few rows: a CTA's warps share rows and split their blocks (KS).
// Not the weight's bytes (24 MB, 3.7 us) but the work per code holds it: each
// further token adds 3 us, so that three tokens or four on a large weight are
// better off with the product (host.cpp has the rule and both sides' figures).  No
// pipe is saturated (integer 55 %, issue slots 61 % at one token): the rest is
// latency.  fp16 pairs and HFMA2 instead took 10.8 us.
#include "mx4.cuh"

namespace act {
int mx4_check(const actcomp_mx4 *q);
namespace mx4 {

constexpr int MAX_TOKENS = ACTCOMP_MX4_LINEAR_TOKENS;
constexpr int MAX_X_BYTES = ACTCOMP_MX4_LINEAR_BYTES;  // shared memory for x
constexpr int DEPTH = 2, STAGE = 5 * 512;  // a warp's stages: four rows' pieces of 512 bytes and the scale words
constexpr int MAX_SMEM = MAX_X_BYTES + 8 * DEPTH * STAGE;
static_assert(MAX_X_BYTES % 16 == 0 && 8 * 4 * MAX_TOKENS * sizeof(float) <= STATIC_ROOM &&
                  MAX_SMEM + STATIC_ROOM <= 227 * 1024,
              "shared memory");

struct LinArgs {
    const void *x;
    int64_t ldx;
    const uint8_t *codes, *scales;
    void *c;
    int64_t ldc;
    int n, k;       // rows and columns of w
    int nb, nka;    // its blocks and atoms
    int ks_log;     // log2 of the warps that share rows
};

__device__ __forceinline__ void cp_async16(uint8_t *dst, const uint8_t *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
                 : "memory");
}
constexpr uint32_t MAG_LO = 0x03020100u, MAG_HI = 0x0c080604u;
// Table bytes selected by the four low nibbles of `sel` (three bits each; the
// fourth bit gives the byte's sign bit in all places instead).
__device__ __forceinline__ uint32_t magnitudes(uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(MAG_LO), "r"(MAG_HI), "r"(sel));
    return r;
}
// min and max that keep a NaN
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

template <typename T, typename TOut, int M, bool VEC>
__global__ void __launch_bounds__(256, M == 1 ? 4 : (M == 2 ? 3 : 2)) linear_kernel(LinArgs a) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ float red[8][4 * M];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nb = a.nb, nka = a.nka;
    float *xsc = reinterpret_cast<float *>(dyn + (size_t)M * nb * 32);
    // this warp's rows
    const int ks = 1 << a.ks_log, part = warp & (ks - 1);
    const int unit = blockIdx.x * (8 >> a.ks_log) + (warp >> a.ks_log), atom = unit >> 5, r0 = unit & 31;
    const int row = atom * 128 + r0;
    const int64_t rb = (int64_t)nb * 16;
    const uint8_t *cw = a.codes + row * rb;
    const uint8_t *sw = a.scales + ((int64_t)atom * nka) * ATOM_BYTES + r0 * 16;
    // its first blocks, on their way while x is quantised (a lane reads only what it copied)
    uint8_t *ring = dyn + (((size_t)M * nb * 36 + 15) & ~(size_t)15) + warp * (DEPTH * STAGE) + lane * 16;
    auto fetch = [&](int t) {
        const int b = (t * ks + part) * 32 + lane;
        uint8_t *d = ring + t % DEPTH * STAGE;
        if (b < nb && row < a.n) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (row + 32 * j < a.n && ACT_DCHECK(16 * (int64_t)b + 16 <= rb)) cp_async16(d + 512 * j, cw + 32 * j * rb + 16 * (int64_t)b);
            cp_async16(d + 2048, sw + (int64_t)(b >> 2) * ATOM_BYTES);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int t = 0; t < DEPTH - 1; ++t) fetch(t);
    // x: four lanes a block
    for (int i0 = tid; i0 - tid < nb * 4; i0 += 512) {
        Raw8<T> raw[2][M];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int c = (i0 + 256 * u) * 8;
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const T *x = static_cast<const T *>(a.x) + m * a.ldx + c;
                if (VEC && c + 8 <= a.k) raw[u][m].load_vec(x);
                else raw[u][m].load(x, a.k - c);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = i0 + 256 * u, blk = i >> 2;
#pragma unroll
            for (int m = 0; m < M; ++m) {
                uint32_t amax = raw[u][m].amax();
                amax = max_of<T>(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = max_of<T>(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                if (blk < nb) {
                    const uint32_t sc = scale_code(amax_bits<T>(amax));
                    const float inv = inv_scale(sc);
                    float v[8];
                    raw[u][m].floats(v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] *= inv;
                    const uint32_t q = pack8(v), f = q ^ 0x88888888u;
                    uint2 o;
                    o.x = __vsub4(magnitudes(q), magnitudes(f));
                    o.y = __vsub4(magnitudes(q >> 16), magnitudes(f >> 16));
                    // halves of 16 values apart: a warp's 16-byte reads are contiguous
                    *reinterpret_cast<uint2 *>(dyn + ((size_t)(2 * m + ((i >> 1) & 1)) * nb + blk) * 16 + (i & 1) * 8) =
                        o;
                    if ((i & 3) == 0) xsc[m * nb + blk] = 0.25f * scale_value(sc);  // both operands are twice their values
                }
            }
        }
    }
    __syncthreads();
    float acc[4][M] = {};
    for (int t = 0;; ++t) {
        const int b = (t * ks + part) * 32 + lane;
        if ((t * ks + part) * 32 >= nb) break;
        fetch(t + DEPTH - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
        if (b >= nb) continue;
        const uint8_t *d0 = ring + t % DEPTH * STAGE;
        const uint4 s4 = *reinterpret_cast<const uint4 *>(d0 + 2048);
        const int sh = 8 * (b & 3);
        const float sa[4] = {scale_value((s4.x >> sh) & 255u), scale_value((s4.y >> sh) & 255u),
                             scale_value((s4.z >> sh) & 255u), scale_value((s4.w >> sh) & 255u)};
        int xv[M][8];
        float sb[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const int4 lo = *reinterpret_cast<const int4 *>(dyn + ((size_t)(2 * m) * nb + b) * 16);
            const int4 hi = *reinterpret_cast<const int4 *>(dyn + ((size_t)(2 * m + 1) * nb + b) * 16);
            xv[m][0] = lo.x, xv[m][1] = lo.y, xv[m][2] = lo.z, xv[m][3] = lo.w;
            xv[m][4] = hi.x, xv[m][5] = hi.y, xv[m][6] = hi.z, xv[m][7] = hi.w;
            sb[m] = xsc[m * nb + b];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            int pos[M] = {}, neg[M] = {};
            const uint4 w = *reinterpret_cast<const uint4 *>(d0 + 512 * j);
            const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t f = q[k] ^ 0x88888888u;
                const int p0 = magnitudes(q[k]), p1 = magnitudes(q[k] >> 16);
                const int n0 = magnitudes(f), n1 = magnitudes(f >> 16);
#pragma unroll
                for (int m = 0; m < M; ++m) {
                    pos[m] = __dp4a(p1, xv[m][2 * k + 1], __dp4a(p0, xv[m][2 * k], pos[m]));
                    neg[m] = __dp4a(n1, xv[m][2 * k + 1], __dp4a(n0, xv[m][2 * k], neg[m]));
                }
            }
#pragma unroll
            for (int m = 0; m < M; ++m) {
                // a whole number times a power of two: exact even as a subnormal; the smaller
                // scale first, so that only a result out of range overflows
                const float t = i2f_exact(pos[m] - neg[m]) * min_nan(sa[j], sb[m]);
                acc[j][m] = __fmaf_rn(t, max_nan(sa[j], sb[m]), acc[j][m]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int m = 0; m < M; ++m) {
            acc[j][m] = warp_sum(acc[j][m]);
            if (lane == 0) red[warp][j * M + m] = acc[j][m];
        }
    __syncthreads();
    if (part == 0 && lane < 4 * M) {
        float t = 0.f;
        for (int i = 0; i < ks; ++i) t += red[warp + i][lane];
        const int j = lane / M, m = lane - j * M, r = row + 32 * j;
        if (r < a.n && ACT_DCHECK(r < a.ldc)) static_cast<TOut *>(a.c)[m * a.ldc + r] = from_f<TOut>(t);
    }
}

template <typename F>
static int by_type(int dtype, F f) {
    if (dtype == 0) return f(float{});
    if (dtype == 1) return f(__nv_bfloat16{});
    return f(__half{});
}

}  // namespace mx4
}  // namespace act

extern "C" int actcomp_mx4_linear(const void *x, int64_t tokens, int64_t cols, int64_t ldx, int32_t dtype,
                                  const actcomp_mx4 *w, void *c, int64_t ldc, int32_t c_dtype, void *stream) {
    using namespace act;
    using namespace act::mx4;
    if (int st = mx4_check(w)) return st;
    ACT_CHECK(x && c && tokens > 0 && cols == w->cols && ldx >= cols && ldc >= w->rows, ACT_E_INVALID);
    ACT_CHECK(dtype >= 0 && dtype <= 2 && (c_dtype == dtype || c_dtype == 0), ACT_E_INVALID);
    ACT_CHECK(tokens <= MAX_TOKENS, ACT_E_UNSUPPORTED);
    const int es = dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(x, es) && aligned(c, c_dtype == 0 ? 4 : 2), ACT_E_ALIGN);
    LinArgs a{x, ldx, w->codes, w->scales, c, ldc, (int)w->rows, (int)w->cols, (int)blocks_of(w->cols),
              (int)atoms_of(w->cols), 0};
    ACT_CHECK(tokens * a.nb * 36 <= MAX_X_BYTES, ACT_E_UNSUPPORTED);
    const int64_t smem = ((tokens * a.nb * 36 + 15) & ~(int64_t)15) + 8 * DEPTH * STAGE;
    const bool vec = aligned(x, 16) && (ldx * es) % 16 == 0;
    // a warp per four rows; split K while that leaves SMs short of sixteen warps
    const int64_t units = (w->rows + 127) / 128 * 32;
    while (a.ks_log < 3 && (units << a.ks_log) < (int64_t)num_sms() * 16 && a.nb > (32 << a.ks_log)) ++a.ks_log;
    const int grid = (int)(((units << a.ks_log) + 7) / 8);
    cudaStream_t st = as_stream(stream);
    return by_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        auto go = [&](auto kern) -> int {
            if (int rc = allow_smem(kern, (size_t)smem, MAX_SMEM)) return rc;
            kern<<<grid, 256, (int)smem, st>>>(a);
            return launch_status();
        };
        auto out = [&](auto o) -> int {
            using TOut = decltype(o);
            switch (tokens) {
                case 1: return vec ? go(linear_kernel<T, TOut, 1, true>) : go(linear_kernel<T, TOut, 1, false>);
                case 2: return vec ? go(linear_kernel<T, TOut, 2, true>) : go(linear_kernel<T, TOut, 2, false>);
                case 3: return vec ? go(linear_kernel<T, TOut, 3, true>) : go(linear_kernel<T, TOut, 3, false>);
                default: return vec ? go(linear_kernel<T, TOut, 4, true>) : go(linear_kernel<T, TOut, 4, false>);
            }
        };
        return c_dtype == 0 ? out(float{}) : out(t);
    });
}
