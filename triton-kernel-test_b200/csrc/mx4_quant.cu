// mx4_quant.cu -- microscaled 4-bit quantisation (by rows, by columns, or both)
// and its inverse; the format is stated in include/actcomp.h.
//
// Its floor is HBM: 2 bytes in and 17/32 out per bf16 value and direction; instruction
// issue and the integer pipe (65 to 72 % busy) hold it.  16384 x 11008 on a B200, us
// and share of the copy rate:
//             rows       columns    both       inverse
//   bf16      86  82 %   93  76 %   144  59 %  90  78 %
//   float32   132 96 %   206 61 %   259 55 %   190 66 %   (tile forms spill 60 to 88 bytes)
//   rows   a lane takes eight consecutive values, four lanes a block of 32: loads
//          and code stores are contiguous over the warp, the block's largest
//          magnitude takes two shuffles; four rows of a scale atom together, so
//          that their scale words are one 16-byte store (106 us two rows at a
//          time, a word each).
//   tiles  by columns, or both ways from one read: a CTA takes 128 x 128 values
//          through shared memory; the column direction needs 32 rows of a column
//          in one thread, and whole 64-byte pieces of the output's rows (one K
//          atom) leave together (a thread per column straight from memory: 377 us).
#include "mx4.cuh"

namespace act {
namespace mx4 {

// The 4 x 4 bytes of a, b, c, d (rows) transposed.
__device__ __forceinline__ uint4 transpose_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);  // a0 b0 a1 b1 | a2 b2 a3 b3
    const uint32_t cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
    return make_uint4(__byte_perm(ab0, cd0, 0x5410), __byte_perm(ab0, cd0, 0x7632), __byte_perm(ab1, cd1, 0x5410),
                      __byte_perm(ab1, cd1, 0x7632));
}

// By rows: a warp takes 256 columns of the four rows r0, r0 + 32, r0 + 64,
// r0 + 96 of a scale atom, whose four scale words lie in one 16-byte piece;
// blockIdx.y covers the columns, blockIdx.x strides over the rows' groups.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    quant_rows_kernel(const T *x, int rows, int cols, int64_t ldx, uint8_t *codes, uint8_t *scales) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sg = blockIdx.y, c = sg * 256 + 8 * lane;
    const int nka = (int)atoms_of(cols);
    const int64_t rb = row_bytes(cols);
    const int groups = (rows + 127) / 128 * 32, step = gridDim.x * 8;
    const int n = c >= cols ? 0 : (cols - c < 8 ? cols - c : 8);
    const bool code = c < (int)blocks_of(cols) * BLOCK;
    const int ka = sg * 2 + (lane >> 4);
    const bool word = (lane & 15) == 0 && ka < nka;
    for (int g = blockIdx.x * 8 + warp; g < groups; g += step) {
        const int r0 = (g >> 5) * 128 + (g & 31);
        const T *src = x + r0 * ldx + c;
        Raw8<T> raw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool live = r0 + 32 * j < rows;
            if (VEC && live && n == 8) raw[j].load_vec(src + 32 * j * ldx);
            else raw[j].load(src + 32 * j * ldx, live ? n : 0);
        }
        uint8_t *dst = codes + r0 * rb + c / 2;
        uint32_t sc4 = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t m = raw[j].amax();
            m = max_of<T>(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = max_of<T>(m, __shfl_xor_sync(0xffffffffu, m, 2));
            const uint32_t sc = scale_code(amax_bits<T>(m));
            sc4 |= sc << (8 * j);
            if (code && r0 + 32 * j < rows && ACT_DCHECK(c / 2 + 4 <= rb)) {
                const float inv = inv_scale(sc);
                float v[8];
                raw[j].floats(v);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] *= inv;
                *reinterpret_cast<uint32_t *>(dst + 32 * j * rb) = pack8(v);
            }
        }
        // four blocks x four rows of scale bytes (lanes 0 and 16)
        const uint32_t b1 = __shfl_down_sync(0xffffffffu, sc4, 4), b2 = __shfl_down_sync(0xffffffffu, sc4, 8),
                       b3 = __shfl_down_sync(0xffffffffu, sc4, 12);
        if (word && ACT_DCHECK(g < groups && ka < nka))
            *reinterpret_cast<uint4 *>(scales + ((int64_t)(g >> 5) * nka + ka) * ATOM_BYTES + (g & 31) * 16) =
                transpose_bytes(sc4, b1, b2, b3);
    }
}

// A CTA's 128 x 128 tile: x rows r0.., columns c0... Shared memory holds it as
// rows of PITCH values; every thread then takes one column of 32 rows at a time
// (two neighbouring columns of a 16-bit type: one word a row).
//   BY_ROWS: the tile's rows are quantised too, from the same read.
template <typename T, bool VEC, bool BY_ROWS>
__global__ void __launch_bounds__(256, 4)
    quant_tile_kernel(const T *x, int64_t rows, int64_t cols, int64_t ldx, uint8_t *codes, uint8_t *scales,
                      uint8_t *codes_t, uint8_t *scales_t) {
    constexpr int PITCH = 128 + 16 / (int)sizeof(T);  // 16-byte rows, a shift of four banks from row to row
    extern __shared__ __align__(16) uint8_t dyn[];
    T *tile = reinterpret_cast<T *>(dyn);
    uint32_t *words = reinterpret_cast<uint32_t *>(dyn + 128 * PITCH * sizeof(T));  // 128 columns x 4 scale bytes
    const int ctiles = (int)((cols + 127) / 128), kr = blockIdx.x / ctiles, kc = blockIdx.x - kr * ctiles;
    const int64_t r0 = (int64_t)kr * 128, c0 = (int64_t)kc * 128;
    const int tid = threadIdx.x, lane = tid & 31;
    // in: sixteen lanes a row, eight values a lane
    const int64_t nka = atoms_of(cols), rb = row_bytes(cols);
    const int64_t c = c0 + (tid & 15) * 8;
    const int n = c >= cols ? 0 : (cols - c < 8 ? (int)(cols - c) : 8);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        Raw8<T> raw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = r0 + 64 * h + 16 * i + (tid >> 4);
            if (r < rows && n == 8 && VEC) raw[i].load_vec(x + r * ldx + c);
            else if (r < rows && n > 0) raw[i].load(x + r * ldx + c, n);
            else raw[i].zero();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int lr = 64 * h + 16 * i + (tid >> 4);
            const int64_t r = r0 + lr;
            uint4 *d = reinterpret_cast<uint4 *>(tile + lr * PITCH + (tid & 15) * 8);
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k)
                d[k] = make_uint4(raw[i].w[4 * k], raw[i].w[4 * k + 1], raw[i].w[4 * k + 2], raw[i].w[4 * k + 3]);
            if constexpr (BY_ROWS) {
                uint32_t m = raw[i].amax();
                m = max_of<T>(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = max_of<T>(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const uint32_t sc = scale_code(amax_bits<T>(m));
                if (r < rows && c < blocks_of(cols) * BLOCK && ACT_DCHECK(c / 2 + 4 <= rb)) {
                    const float inv = inv_scale(sc);
                    float v[8];
                    raw[i].floats(v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] *= inv;
                    *reinterpret_cast<uint32_t *>(codes + r * rb + c / 2) = pack8(v);
                }
                uint32_t w = sc;
                w |= __shfl_down_sync(0xffffffffu, w, 4) << 8;
                w |= __shfl_down_sync(0xffffffffu, w, 8) << 16;
                if ((lane & 15) == 0 && ACT_DCHECK(kc < nka && r < (rows + 127) / 128 * 128))
                    *reinterpret_cast<uint32_t *>(scales + scale_word(r, kc, nka)) = w;
            }
        }
    }
    __syncthreads();
    // by columns: warp = (block of 32 rows, half of the columns), two columns a lane
    const int64_t nka_t = atoms_of(rows), rb_t = row_bytes(rows);
    const int b = tid >> 6, pair = tid & 63;  // columns 2 pair, 2 pair + 1
    const bool live = r0 + 32 * b < rows;     // the block exists
    uint32_t sc2[2];
    uint32_t code[2][4];
    if constexpr (sizeof(T) == 2) {
        uint32_t w[32], m = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            w[j] = *reinterpret_cast<const uint32_t *>(tile + (32 * b + j) * PITCH + 2 * pair);
            m = absmax2<T>(m, w[j]);
        }
        sc2[0] = scale_code(amax_bits<T>(m & 0xffffu));
        sc2[1] = scale_code(amax_bits<T>(m >> 16));
        const float inv[2] = {inv_scale(sc2[0]), inv_scale(sc2[1])};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float lo[8], hi[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t u = w[8 * k + j];
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    lo[j] = __uint_as_float(u << 16) * inv[0];
                    hi[j] = __uint_as_float(u & 0xffff0000u) * inv[1];
                } else {
                    __half2 h;
                    memcpy(&h, &u, 4);
                    const float2 t = __half22float2(h);
                    lo[j] = t.x * inv[0], hi[j] = t.y * inv[1];
                }
            }
            code[0][k] = pack8(lo);
            code[1][k] = pack8(hi);
        }
    } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            float v[32];
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                v[j] = to_f<T>(tile[(32 * b + j) * PITCH + 2 * pair + s]);
                m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
            }
            sc2[s] = scale_code(m);
            const float inv = inv_scale(sc2[s]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float t[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = v[8 * k + j] * inv;
                code[s][k] = pack8(t);
            }
        }
    }
    __syncthreads();  // the tile has been read: its space takes the codes, 128 columns x 64 bytes (and a pad of 16)
    uint8_t *out = dyn;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int col = 2 * pair + s;
        *reinterpret_cast<uint4 *>(out + col * 80 + 16 * b) =
            make_uint4(code[s][0], code[s][1], code[s][2], code[s][3]);
        reinterpret_cast<uint8_t *>(words)[col * 4 + b] = live ? (uint8_t)sc2[s] : 0;
    }
    __syncthreads();
    // out: four lanes a column's 64 bytes
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int col = 64 * i + (tid >> 2), q = tid & 3;
        if (c0 + col < cols && r0 + 32 * q < rows && ACT_DCHECK(r0 / 2 + 16 * q + 16 <= rb_t))
            *reinterpret_cast<uint4 *>(codes_t + (c0 + col) * rb_t + r0 / 2 + 16 * q) =
                *reinterpret_cast<const uint4 *>(out + col * 80 + 16 * q);
    }
    if (tid < 128 && ACT_DCHECK(kr < nka_t && c0 + tid < (cols + 127) / 128 * 128))
        *reinterpret_cast<uint32_t *>(scales_t + scale_word(c0 + tid, kr, nka_t)) = words[tid];
}

// Rows and columns as in quant_rows_kernel: one 16-byte load brings a lane the
// scales of its four rows.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
    dequant_kernel(const uint8_t *codes, const uint8_t *scales, int rows, int cols, T *out, int64_t ldo) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __shared__ __align__(16) uint8_t turn[VEC ? 1 : 8][VEC ? 16 : 256 * sizeof(T)];
    const int c0 = blockIdx.y * 256, c = c0 + 8 * lane;
    const int nka = (int)atoms_of(cols), groups = (rows + 127) / 128 * 32, step = gridDim.x * 8;
    const int64_t rb = row_bytes(cols);
    const int n = c >= cols ? 0 : (cols - c < 8 ? cols - c : 8);
    const int sh = 8 * ((c >> 5) & 3);
    for (int g = blockIdx.x * 8 + warp; g < groups; g += step) {
        const int r0 = (g >> 5) * 128 + (g & 31);
        if (r0 >= rows) continue;  // the same for the warp
        const uint8_t *src = codes + r0 * rb + c / 2;
        uint32_t q[4] = {};
        uint4 s4 = make_uint4(0, 0, 0, 0);
        if (n > 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r0 + 32 * j < rows) q[j] = *reinterpret_cast<const uint32_t *>(src + 32 * j * rb);
            s4 = *reinterpret_cast<const uint4 *>(scales + ((int64_t)(g >> 5) * nka + (c >> 7)) * ATOM_BYTES +
                                                  (g & 31) * 16);
        }
        const uint32_t sc[4] = {(s4.x >> sh) & 255u, (s4.y >> sh) & 255u, (s4.z >> sh) & 255u, (s4.w >> sh) & 255u};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (r0 + 32 * j >= rows) break;
            __half2 h[4];
            tiny8(q[j], h);
            const float s = scale_value(sc[j]);
            float f[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 t = mul2(__half22float2(__hmul2(h[k], __float2half2_rn(16384.f))), make_float2(s, s));
                f[k] = t.x, f[k + 4] = t.y;
            }
            uint32_t w[2 * sizeof(T)];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(T) == 4) {
                    w[2 * k] = __float_as_uint(f[2 * k]), w[2 * k + 1] = __float_as_uint(f[2 * k + 1]);
                } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    w[k] = pack_bf16x2(f[2 * k], f[2 * k + 1]);
                } else {
                    const __half2 o = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
                    memcpy(&w[k], &o, 4);
                }
            }
            T *row = out + (r0 + 32 * j) * ldo + c0;
            if (VEC && n == 8 && ACT_DCHECK(c + 8 <= cols && r0 + 32 * j < rows)) {
#pragma unroll
                for (int k = 0; k < (int)sizeof(T) / 2; ++k)
                    reinterpret_cast<uint4 *>(row + 8 * lane)[k] =
                        make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
            } else if (VEC) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k < n) {
                        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t *>(row)[8 * lane + k] = w[k];
                        else reinterpret_cast<uint16_t *>(row)[8 * lane + k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
                    }
            } else {  // through shared memory, so that neighbouring lanes store neighbouring values
                uint4 *mine = reinterpret_cast<uint4 *>(turn[warp]) + lane * (sizeof(T) / 2);
#pragma unroll
                for (int k = 0; k < (int)sizeof(T) / 2; ++k)
                    mine[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                __syncwarp();
                const int left = cols - c0 < 256 ? cols - c0 : 256;
                const T *v = reinterpret_cast<const T *>(turn[warp]);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (32 * k + lane < left && ACT_DCHECK(c0 + 32 * k + lane < cols && r0 + 32 * j < rows))
                        row[32 * k + lane] = v[32 * k + lane];
                __syncwarp();
            }
        }
    }
}

template <typename F>
static int with_type(int dtype, F f) {
    if (dtype == 0) return f(float{});
    if (dtype == 1) return f(__nv_bfloat16{});
    return f(__half{});
}

static int check(const actcomp_mx4 *q) {
    ACT_CHECK(q && q->rows > 0 && q->cols > 0, ACT_E_INVALID);
    ACT_CHECK(q->rows <= INT32_MAX - 255 && q->cols <= INT32_MAX - 255, ACT_E_UNSUPPORTED);
    ACT_CHECK(q->codes && q->scales, ACT_E_INVALID);
    ACT_CHECK(aligned(q->codes, 16) && aligned(q->scales, 16), ACT_E_ALIGN);
    return ACT_OK;
}

// Grid of the row kernels: y covers the columns, x the rows with enough CTAs to
// fill the device `waves` times over.
static bool row_grid(dim3 &g, int64_t rows, int64_t cols, int waves) {
    const int64_t segs = (cols + 255) / 256, need = (rows + 127) / 128 * 4;  // eight warps a CTA, four rows a warp
    if (segs > 65535) return false;
    int64_t x = ((int64_t)num_sms() * waves + segs - 1) / segs;
    g = dim3((unsigned)(x < need ? x : need), (unsigned)segs);
    return true;
}

}  // namespace mx4
int mx4_check(const actcomp_mx4 *q) { return mx4::check(q); }
}  // namespace act

extern "C" size_t actcomp_mx4_code_bytes(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 ? act::mx4::code_bytes(rows, cols) : 0;
}
extern "C" size_t actcomp_mx4_scale_bytes(int64_t rows, int64_t cols) {
    return rows > 0 && cols > 0 ? act::mx4::scale_bytes(rows, cols) : 0;
}

extern "C" int actcomp_mx4_quantize(const void *x, int64_t rows, int64_t cols, int64_t ldx, int32_t dtype,
                                    const actcomp_mx4 *q, const actcomp_mx4 *qt, void *stream) {
    using namespace act;
    using namespace act::mx4;
    ACT_CHECK(x && (q || qt) && rows > 0 && cols > 0 && ldx >= cols && dtype >= 0 && dtype <= 2, ACT_E_INVALID);
    const int64_t tiles = ((cols + 127) / 128) * ((rows + 127) / 128);
    if (q) {
        ACT_CHECK(q->rows == rows && q->cols == cols, ACT_E_INVALID);
        if (int st = check(q)) return st;
    }
    if (qt) {
        ACT_CHECK(qt->rows == cols && qt->cols == rows, ACT_E_INVALID);
        if (int st = check(qt)) return st;
        ACT_CHECK(tiles <= INT32_MAX, ACT_E_UNSUPPORTED);
    }
    const int es = dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(x, es), ACT_E_ALIGN);
    const bool vec = aligned(x, 16) && (ldx * es) % 16 == 0;
    dim3 grid;
    if (!qt) ACT_CHECK(row_grid(grid, rows, cols, 16), ACT_E_UNSUPPORTED);
    cudaStream_t st = as_stream(stream);
    return with_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        const T *xs = static_cast<const T *>(x);
        if (!qt) {
            if (vec) quant_rows_kernel<T, true><<<grid, 256, 0, st>>>(xs, (int)rows, (int)cols, ldx, q->codes, q->scales);
            else quant_rows_kernel<T, false><<<grid, 256, 0, st>>>(xs, (int)rows, (int)cols, ldx, q->codes, q->scales);
            return launch_status();
        }
        const int smem = 128 * (128 + 16 / (int)sizeof(T)) * (int)sizeof(T) + 512;
        auto go = [&](auto k) -> int {
            if (smem > 48 * 1024) ACT_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            k<<<(unsigned)tiles, 256, smem, st>>>(xs, rows, cols, ldx, q ? q->codes : nullptr, q ? q->scales : nullptr, qt->codes,
                                    qt->scales);
            return launch_status();
        };
        if (q) return vec ? go(quant_tile_kernel<T, true, true>) : go(quant_tile_kernel<T, false, true>);
        return vec ? go(quant_tile_kernel<T, true, false>) : go(quant_tile_kernel<T, false, false>);
    });
}

extern "C" int actcomp_mx4_dequantize(const actcomp_mx4 *q, void *out, int64_t ldo, int32_t dtype, void *stream) {
    using namespace act;
    using namespace act::mx4;
    if (int st = check(q)) return st;
    ACT_CHECK(out && ldo >= q->cols && dtype >= 0 && dtype <= 2, ACT_E_INVALID);
    const int es = dtype == 0 ? 4 : 2;
    ACT_CHECK(aligned(out, es), ACT_E_ALIGN);
    const bool vec = aligned(out, 16) && (ldo * es) % 16 == 0;
    dim3 grid;
    ACT_CHECK(row_grid(grid, q->rows, q->cols, 16), ACT_E_UNSUPPORTED);
    cudaStream_t st = as_stream(stream);
    return with_type(dtype, [&](auto t) {
        using T = decltype(t);
        T *o = static_cast<T *>(out);
        if (vec) dequant_kernel<T, true><<<grid, 256, 0, st>>>(q->codes, q->scales, (int)q->rows, (int)q->cols, o, ldo);
        else dequant_kernel<T, false><<<grid, 256, 0, st>>>(q->codes, q->scales, (int)q->rows, (int)q->cols, o, ldo);
        return launch_status();
    });
}
