// host.cpp -- the host side of actcomp.norm, mx4, fp8 and loss: argument checks,
// output allocation and the call of the C ABI, as a Python extension module
// (built and named by actcomp/build.py).  It computes nothing.  A call's host time
// is what a user waits for at small sizes: layer norm of 8 x 4096 is 3 us on the
// device, and its Python path (three tensors, a dozen attribute reads, ctypes) took
// 13 us where this takes 8.
//
// The entry points' addresses come from the library that the package has loaded
// (bind), so another build of it serves here as well.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <tuple>

#include "../../include/actcomp.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct Api {
    decltype(&actcomp_dropout) dropout;
    decltype(&actcomp_layer_norm) layer_norm;
    decltype(&actcomp_layer_norm_bwd) layer_norm_bwd;
    decltype(&actcomp_layer_norm_bwd_workspace) layer_norm_bwd_workspace;
    decltype(&actcomp_mx4_quantize) mx4_quantize;
    decltype(&actcomp_mx4_dequantize) mx4_dequantize;
    decltype(&actcomp_mx4_gemm) mx4_gemm;
    decltype(&actcomp_mx4_linear) mx4_linear;
    decltype(&actcomp_rms_norm) rms_norm;
    decltype(&actcomp_rms_norm_bwd) rms_norm_bwd;
    decltype(&actcomp_rms_norm_bwd_workspace) rms_norm_bwd_workspace;
    decltype(&actcomp_fp8_quantize) fp8_quantize;
    decltype(&actcomp_fp8_dequantize) fp8_dequantize;
    decltype(&actcomp_fp8_gemm) fp8_gemm;
    decltype(&actcomp_xent_workspace) xent_workspace;
    decltype(&actcomp_xent) xent;
    decltype(&actcomp_xent_bwd_workspace) xent_bwd_workspace;
    decltype(&actcomp_xent_bwd) xent_bwd;
} api{};

template <typename F>
void bind_one(const py::dict &addresses, const char *name, F &f) {
    f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}
// An entry point that an earlier build of the library lacks stays null; its callers ask need().
template <typename F>
void bind_later(const py::dict &addresses, const char *name, F &f) {
    if (addresses.contains(name)) bind_one(addresses, name, f);
}
template <typename F>
F need(F f, const char *name) {
    if (!f) {
        PyErr_SetString(PyExc_ImportError, (std::string("the loaded library lacks ") + name).c_str());
        throw py::error_already_set();
    }
    return f;
}
void bind(const py::dict &d) {
    bind_one(d, "actcomp_dropout", api.dropout);
    bind_one(d, "actcomp_layer_norm", api.layer_norm);
    bind_one(d, "actcomp_layer_norm_bwd", api.layer_norm_bwd);
    bind_one(d, "actcomp_layer_norm_bwd_workspace", api.layer_norm_bwd_workspace);
    bind_one(d, "actcomp_mx4_quantize", api.mx4_quantize);
    bind_one(d, "actcomp_mx4_dequantize", api.mx4_dequantize);
    bind_one(d, "actcomp_mx4_gemm", api.mx4_gemm);
    bind_one(d, "actcomp_mx4_linear", api.mx4_linear);
    bind_later(d, "actcomp_rms_norm", api.rms_norm);
    bind_later(d, "actcomp_rms_norm_bwd", api.rms_norm_bwd);
    bind_later(d, "actcomp_rms_norm_bwd_workspace", api.rms_norm_bwd_workspace);
    bind_later(d, "actcomp_fp8_quantize", api.fp8_quantize);
    bind_later(d, "actcomp_fp8_dequantize", api.fp8_dequantize);
    bind_later(d, "actcomp_fp8_gemm", api.fp8_gemm);
    bind_later(d, "actcomp_xent_workspace", api.xent_workspace);
    bind_later(d, "actcomp_xent", api.xent);
    bind_later(d, "actcomp_xent_bwd_workspace", api.xent_bwd_workspace);
    bind_later(d, "actcomp_xent_bwd", api.xent_bwd);
}

// Raises the package's ActcompError for a non-zero status.
void check(const char *name, int status) {
    if (status) py::module_::import("actcomp._lib").attr("check")(name, status);
}
[[noreturn]] void bad_value(const std::string &msg) { throw py::value_error(msg); }
[[noreturn]] void bad_type(const std::string &msg) { throw py::type_error(msg); }

std::string str(const Tensor &t) {
    std::ostringstream s;
    s << t.sizes() << " " << t.scalar_type() << " on " << t.device();
    return s.str();
}

int dtype_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return 0;
        case at::kBFloat16: return 1;
        case at::kHalf: return 2;
        default: bad_type(std::string("float32, bfloat16 or float16 expected, got ") + at::toString(t));
    }
}
void need_cuda(const Tensor &t) {
    if (!t.is_cuda()) bad_value("actcomp kernels run on CUDA tensors only (no CPU fallback)");
}
void need_cuda(const OptTensor &t) {
    if (t) need_cuda(*t);
}

// Uninitialised tensors on x's device, by torch's own allocation without its dispatcher
// (a call's outputs are up to four: 0.3 us each).
Tensor empty_on(const Tensor &x, at::IntArrayRef sizes, at::ScalarType type) {
    return Tensor(at::detail::empty_cuda(sizes, type, x.device(), std::nullopt));
}
Tensor fresh(const Tensor &x) { return empty_on(x, x.sizes(), x.scalar_type()); }
void *ptr(const Tensor &t) { return t.data_ptr(); }
void *ptr(const OptTensor &t) { return t ? t->data_ptr() : nullptr; }
void *stream_of(const Tensor &x) { return c10::cuda::getCurrentCUDAStream(x.device().index()).stream(); }

// x as rows of `cols` with unit column stride; copied only if the leading
// dimensions have no common stride.  A row stride smaller than a row (an
// expanded tensor) is copied too.
struct Rows {
    Tensor t;
    int64_t ld;
};
Rows rows_of(const Tensor &x, int64_t cols) {
    if (x.is_contiguous() || x.numel() == 0) return {x, cols};
    Tensor t = x.dim() == 2 ? x : x.reshape({-1, cols});
    if ((cols != 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < cols)) t = t.contiguous();
    return {t, std::max(t.stride(0), cols)};
}

struct Geometry {
    int64_t rows, cols;
};
Geometry geometry(const Tensor &x) {
    if (x.dim() == 0) bad_value("a tensor of at least one dimension is expected");
    const int64_t cols = x.size(-1);
    return {cols ? x.numel() / cols : 0, cols};
}

void same(const Tensor &x, const Tensor &t, const char *name) {
    if (t.sizes() != x.sizes() || t.scalar_type() != x.scalar_type() || t.device() != x.device())
        bad_value(std::string(name) + " must have the shape, dtype and device of the activation (" + str(x) + "), got " +
                  str(t));
}

// Checks weight and bias; returns their dtype code.
int affine(const Tensor &x, int64_t cols, const OptTensor &w, const OptTensor &b) {
    for (const OptTensor *t : {&w, &b}) {
        if (!*t) continue;
        const Tensor &v = **t;
        if (v.dim() != 1 || v.numel() != cols || v.device() != x.device())
            bad_value("weight and bias must be vectors of " + std::to_string(cols) + " values on the activation's device");
        if (v.scalar_type() != x.scalar_type() && v.scalar_type() != at::kFloat)
            bad_type(std::string("weight and bias must be ") + at::toString(x.scalar_type()) + " or float32, got " +
                     at::toString(v.scalar_type()));
    }
    if (w && b && w->scalar_type() != b->scalar_type()) bad_type("weight and bias must have one dtype");
    return dtype_of(w ? w->scalar_type() : b ? b->scalar_type() : x.scalar_type());
}
OptTensor packed(const OptTensor &t) { return t && !t->is_contiguous() ? OptTensor(t->contiguous()) : t; }

Tensor stats(const Tensor &t, int64_t rows, const Tensor &x, const char *name) {
    if (t.scalar_type() != at::kFloat || t.numel() != rows || t.device() != x.device())
        bad_value(std::string(name) + " must hold " + std::to_string(rows) + " float32 values on the activation's device");
    return t.contiguous();
}

struct Draw {
    double p;
    uint64_t seed, row_offset;
    const uint64_t *seed_ptr;
    Tensor seed_tensor;
};
Draw draw(const Tensor &x, double p, const py::object &seed, const py::object &row_offset) {
    if (!(p >= 0.0 && p <= 1.0)) bad_value("dropout probability must be in [0, 1], got " + std::to_string(p));
    Draw d{p, 0, 0, nullptr, {}};
    int overflow = 0;
    const long long off = PyLong_AsLongLongAndOverflow(row_offset.ptr(), &overflow);
    if (PyErr_Occurred()) throw py::error_already_set();
    if (overflow || off < 0) bad_value("row_offset must be a non-negative 64-bit integer");
    d.row_offset = (uint64_t)off;
    if (THPVariable_Check(seed.ptr())) {
        d.seed_tensor = THPVariable_Unpack(seed.ptr());
        const Tensor &t = d.seed_tensor;
        if (t.scalar_type() != at::kLong || t.numel() != 1 || t.device() != x.device())
            bad_value("a seed tensor holds one int64 on the activation's device");
        d.seed_ptr = reinterpret_cast<const uint64_t *>(t.data_ptr());
        return d;
    }
    if (!PyLong_Check(seed.ptr())) bad_type("seed must be an int or an int64 tensor");
    d.seed = PyLong_AsUnsignedLongLong(seed.ptr());
    if (PyErr_Occurred()) {
        PyErr_Clear();
        bad_value("seed must be in [0, 2^64)");
    }
    return d;
}

Tensor dropout(const Tensor &x, double p, const py::object &seed, const py::object &row_offset, const OptTensor &out) {
    need_cuda(x);
    const int dt = dtype_of(x.scalar_type());
    const Geometry g = geometry(x);
    const Draw d = draw(x, p, seed, row_offset);
    if (out) {
        same(x, *out, "out");
        if (!out->is_contiguous()) bad_value("out must be contiguous");
    }
    const Tensor y = out ? *out : fresh(x);
    Rows r = rows_of(x, g.cols);
    // out lies over part of x, elsewhere than x's own values: rows would be
    // overwritten before they are read
    if (out && x.numel() > 0 && (ptr(r.t) != ptr(y) || r.ld != g.cols)) {
        const auto xa = reinterpret_cast<uintptr_t>(ptr(r.t)), ya = reinterpret_cast<uintptr_t>(ptr(y));
        const size_t es = x.element_size(), xn = ((g.rows - 1) * r.ld + g.cols) * es, yn = x.numel() * es;
        if (xa < ya + yn && ya < xa + xn) r = {x.clone(at::MemoryFormat::Contiguous), g.cols};
    }
    const actcomp_drop_args a{g.rows, g.cols, ptr(r.t), r.ld, ptr(y), g.cols, dt, 0, d.p, d.seed, d.seed_ptr, d.row_offset};
    const c10::cuda::CUDAGuard guard(x.device());
    check("actcomp_dropout", api.dropout(&a, stream_of(x)));
    return y;
}

std::tuple<Tensor, OptTensor, Tensor, Tensor> forward(const Tensor &x, const OptTensor &res, const OptTensor &weight,
                                                      const OptTensor &bias, double eps, const Draw &d) {
    const int dt = dtype_of(x.scalar_type());
    const Geometry g = geometry(x);
    const int wdt = affine(x, g.cols, weight, bias);
    if (g.cols == 0) bad_value("layer norm over an empty last dimension");
    if (!(eps >= 0.0)) bad_value("eps must not be negative");
    const Rows r = rows_of(x, g.cols), rr = res ? rows_of(*res, g.cols) : Rows{};
    const OptTensor w = packed(weight), b = packed(bias);
    const Tensor y = fresh(x);
    const OptTensor h = res ? OptTensor(fresh(x)) : OptTensor();
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    const Tensor mean = at::empty(lead, x.options().dtype(at::kFloat)), rstd = at::empty(lead, mean.options());
    const actcomp_ln_args a{g.rows, g.cols, ptr(r.t), r.ld, res ? ptr(rr.t) : nullptr, res ? rr.ld : 0,
                            ptr(w), ptr(b), ptr(y), g.cols, ptr(h), g.cols, static_cast<float *>(ptr(mean)),
                            static_cast<float *>(ptr(rstd)), dt, wdt, (float)eps, 0, d.p, d.seed, d.seed_ptr,
                            d.row_offset};
    const c10::cuda::CUDAGuard guard(x.device());
    check("actcomp_layer_norm", api.layer_norm(&a, stream_of(x)));
    return {y, h, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm(const Tensor &x, const OptTensor &weight, const OptTensor &bias,
                                              double eps) {
    need_cuda(x);
    auto [y, h, mean, rstd] = forward(x, {}, weight, bias, eps, Draw{});
    return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> branch(const Tensor &x, const Tensor &residual, const OptTensor &weight,
                                                  const OptTensor &bias, double p, const py::object &seed,
                                                  const py::object &row_offset, double eps) {
    need_cuda(x);
    same(x, residual, "residual");
    auto [y, h, mean, rstd] = forward(x, residual, weight, bias, eps, draw(x, p, seed, row_offset));
    return {y, *h, mean, rstd};
}

std::tuple<Tensor, OptTensor, OptTensor, OptTensor> backward(const Tensor &dy, const Tensor &x, const OptTensor &weight,
                                                             const Tensor &mean, const Tensor &rstd, const OptTensor &dh,
                                                             bool fused, bool bias_grad,
                                                             std::optional<at::ScalarType> bias_dtype, const Draw &d) {
    const int dt = dtype_of(x.scalar_type());
    const Geometry g = geometry(x);
    // what the weight gradients are in: the weight's dtype, without one the bias's
    const at::ScalarType wtype = weight ? weight->scalar_type() : bias_dtype.value_or(x.scalar_type());
    affine(x, g.cols, weight, {});
    if (wtype != x.scalar_type() && wtype != at::kFloat)
        bad_type(std::string("bias_dtype must be ") + at::toString(x.scalar_type()) + " or float32, got " +
                 at::toString(wtype));
    if (bias_dtype && *bias_dtype != wtype) bad_type("weight and bias must have one dtype");
    const int wdt = dtype_of(wtype);
    if (g.cols == 0) bad_value("layer norm over an empty last dimension");
    const Tensor m = stats(mean, g.rows, x, "mean"), s = stats(rstd, g.rows, x, "rstd");
    const Rows ry = rows_of(dy, g.cols), rx = rows_of(x, g.cols), rh = dh ? rows_of(*dh, g.cols) : Rows{};
    const OptTensor w = packed(weight);
    const Tensor dx = fresh(x);
    const OptTensor dr = fused ? OptTensor(fresh(x)) : OptTensor();
    const auto wopt = x.options().dtype(wtype);
    const OptTensor dw = weight ? OptTensor(at::empty({g.cols}, wopt)) : OptTensor();
    const OptTensor db = bias_grad ? OptTensor(at::empty({g.cols}, wopt)) : OptTensor();
    const c10::cuda::CUDAGuard guard(x.device());
    const size_t need = api.layer_norm_bwd_workspace(g.rows, g.cols);
    const Tensor ws = at::empty({(int64_t)std::max<size_t>(need, 1)}, x.options().dtype(at::kByte));
    const actcomp_ln_bwd_args a{g.rows, g.cols, ptr(ry.t), ry.ld, ptr(rx.t), rx.ld, dh ? ptr(rh.t) : nullptr,
                                dh ? rh.ld : 0, ptr(w), static_cast<const float *>(ptr(m)),
                                static_cast<const float *>(ptr(s)), ptr(dx), g.cols, ptr(dr), g.cols, ptr(dw), ptr(db),
                                dt, wdt, d.p, d.seed, d.seed_ptr, d.row_offset};
    check("actcomp_layer_norm_bwd", api.layer_norm_bwd(&a, ptr(ws), need, stream_of(x)));
    return {dx, dr, dw, db};
}

std::tuple<Tensor, OptTensor, OptTensor> layer_norm_backward(const Tensor &dy, const Tensor &x, const OptTensor &weight,
                                                             const Tensor &mean, const Tensor &rstd, bool bias_grad,
                                                             std::optional<at::ScalarType> bias_dtype) {
    need_cuda(x);
    same(x, dy, "dy");
    auto [dx, dr, dw, db] = backward(dy, x, weight, mean, rstd, {}, false, bias_grad, bias_dtype, Draw{});
    return {dx, dw, db};
}

std::tuple<Tensor, Tensor, OptTensor, OptTensor> branch_backward(const Tensor &dy, const Tensor &h,
                                                                 const OptTensor &weight, const Tensor &mean,
                                                                 const Tensor &rstd, double p, const py::object &seed,
                                                                 const py::object &row_offset, const OptTensor &dh,
                                                                 bool bias_grad,
                                                                 std::optional<at::ScalarType> bias_dtype) {
    need_cuda(h);
    same(h, dy, "dy");
    if (dh) same(h, *dh, "dh");
    auto [dx, dr, dw, db] = backward(dy, h, weight, mean, rstd, dh, true, bias_grad, bias_dtype,
                                     draw(h, p, seed, row_offset));
    return {dx, *dr, dw, db};
}

// ---------------------------------------------------------------- microscaled 4-bit
// x with its leading dimensions joined to rows.
Rows matrix(const Tensor &x) {
    if (x.dim() < 1 || x.numel() == 0) bad_value("a non-empty tensor is expected, got shape " + str(x));
    return rows_of(x, x.size(-1));
}

struct Quantised {
    Tensor codes, scales;
    actcomp_mx4 desc;
};
Quantised empty_mx4(const Tensor &x, int64_t rows, int64_t cols) {
    const auto opt = x.options().dtype(at::kByte);
    Quantised q{at::empty({rows, (cols + 31) / 32 * 16}, opt), at::empty({(rows + 127) / 128 * ((cols + 127) / 128) * 512}, opt),
                {}};
    q.desc = {rows, cols, static_cast<uint8_t *>(ptr(q.codes)), static_cast<uint8_t *>(ptr(q.scales))};
    return q;
}
actcomp_mx4 desc_of(int64_t rows, int64_t cols, const Tensor &codes, const Tensor &scales) {
    need_cuda(codes);
    if (codes.numel() != rows * ((cols + 31) / 32 * 16) ||
        scales.numel() != (rows + 127) / 128 * ((cols + 127) / 128) * 512 || !codes.is_contiguous() ||
        !scales.is_contiguous() || codes.scalar_type() != at::kByte || scales.scalar_type() != at::kByte ||
        scales.device() != codes.device())
        bad_value("codes and scales do not belong to a matrix of " + std::to_string(rows) + " x " + std::to_string(cols));
    return {rows, cols, static_cast<uint8_t *>(ptr(codes)), static_cast<uint8_t *>(ptr(scales))};
}

// (rows, cols, codes, scales of x, codes, scales of x^T); what is not asked for is None
std::tuple<int64_t, int64_t, OptTensor, OptTensor, OptTensor, OptTensor> quantize(const Tensor &x, bool by_rows,
                                                                                 bool by_cols) {
    need_cuda(x);
    const int dt = dtype_of(x.scalar_type());
    const Rows r = matrix(x);
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    std::optional<Quantised> q, qt;
    if (by_rows) q = empty_mx4(x, rows, cols);
    if (by_cols) qt = empty_mx4(x, cols, rows);
    const c10::cuda::CUDAGuard guard(x.device());
    check("actcomp_mx4_quantize", api.mx4_quantize(ptr(r.t), rows, cols, r.ld, dt, q ? &q->desc : nullptr,
                                                   qt ? &qt->desc : nullptr, stream_of(x)));
    const auto c = [](const std::optional<Quantised> &v) { return v ? OptTensor(v->codes) : OptTensor(); };
    const auto s = [](const std::optional<Quantised> &v) { return v ? OptTensor(v->scales) : OptTensor(); };
    return {rows, cols, c(q), s(q), c(qt), s(qt)};
}

Tensor dequantize(int64_t rows, int64_t cols, const Tensor &codes, const Tensor &scales, at::ScalarType dtype) {
    const int dt = dtype_of(dtype);
    const actcomp_mx4 d = desc_of(rows, cols, codes, scales);
    const Tensor out = at::empty({rows, cols}, codes.options().dtype(dtype));
    const c10::cuda::CUDAGuard guard(codes.device());
    check("actcomp_mx4_dequantize", api.mx4_dequantize(&d, ptr(out), cols, dt, stream_of(codes)));
    return out;
}

Tensor product(const actcomp_mx4 &a, const actcomp_mx4 &b, const Tensor &like, at::IntArrayRef shape,
               at::ScalarType dtype) {
    const int dt = dtype_of(dtype);
    const Tensor out = at::empty(shape, like.options().dtype(dtype));
    const c10::cuda::CUDAGuard guard(like.device());
    check("actcomp_mx4_gemm", api.mx4_gemm(&a, &b, ptr(out), b.rows, dt, stream_of(like)));
    return out;
}

Tensor matmul(int64_t m, int64_t n, int64_t k, const Tensor &a_codes, const Tensor &a_scales, const Tensor &b_codes,
              const Tensor &b_scales, at::ScalarType dtype) {
    if (a_codes.device() != b_codes.device()) bad_value("operands on different devices");
    return product(desc_of(m, k, a_codes, a_scales), desc_of(n, k, b_codes, b_scales), a_codes, {m, n}, dtype);
}

// Whether x . w^T goes through the one-kernel form (actcomp_mx4_linear) or through
// quantisation and product.  The one kernel decodes the weight again for every token,
// the product does not (a weight in memory, us, one kernel / two):
//   n x k           1 token      2            3            4
//   4096 x 4096     6.2 / 14.4   8.4 / 14.4   10.8 / 14.4  13.0 / 14.3
//   11008 x 4096    9.9 / 17.4   12.6 / 17.2  16.0 / 15.4  19.0 / 15.4
//   4096 x 11008    12.1 / 23.3  18.1 / 23.4  23.7 / 23.2  29.3 / 23.1
//   8192 x 8192     13.3 / 22.9  18.4 / 20.2  23.6 / 23.8  28.6 / 20.2
//   16384 x 16384   38.8 / 42.2  53.8 / 43.4  66.3 / 40.2  81.0 / 40.0
// They cross near 2^27 multiplications; one token stays below at every size.
bool one_kernel(int64_t tokens, int64_t n, int64_t k) {
    return tokens <= ACTCOMP_MX4_LINEAR_TOKENS && tokens * ((k + 31) / 32) * 36 <= ACTCOMP_MX4_LINEAR_BYTES &&
           (tokens == 1 || (double)tokens * (double)n * (double)k <= (double)(1 << 27));
}

// x . w^T
Tensor linear(const Tensor &x, int64_t n, int64_t k, const Tensor &codes, const Tensor &scales,
              std::optional<at::ScalarType> out_dtype) {
    need_cuda(x);
    const int dt = dtype_of(x.scalar_type());
    if (x.dim() < 1 || x.size(-1) != k)
        bad_value("x is " + str(x) + ", the weight has " + std::to_string(k) + " columns");
    if (x.device() != codes.device()) bad_value("operands on different devices");
    const actcomp_mx4 w = desc_of(n, k, codes, scales);
    const Rows r = matrix(x);
    const at::ScalarType dtype = out_dtype.value_or(x.scalar_type());
    const int odt = dtype_of(dtype);
    const int64_t tokens = x.numel() / k;
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    if (one_kernel(tokens, n, k) && (odt == dt || odt == 0)) {
        const Tensor out = at::empty(shape, x.options().dtype(dtype));
        const c10::cuda::CUDAGuard guard(x.device());
        check("actcomp_mx4_linear",
              api.mx4_linear(ptr(r.t), tokens, k, r.ld, dt, &w, ptr(out), n, odt, stream_of(x)));
        return out;
    }
    const Quantised q = empty_mx4(x, tokens, k);
    {
        const c10::cuda::CUDAGuard guard(x.device());
        check("actcomp_mx4_quantize",
              api.mx4_quantize(ptr(r.t), tokens, k, r.ld, dt, &q.desc, nullptr, stream_of(x)));
    }
    return product(q.desc, w, x, shape, dtype);
}

// ---------------------------------------------------------------- root-mean-square norm
// (y or codes, scales, h, rstd)
struct RmsOut {
    Tensor y, scales, rstd;
    OptTensor h;
};
RmsOut rms_forward(const Tensor &x, const OptTensor &residual, const OptTensor &weight, double eps, bool codes) {
    need_cuda(x);
    const auto fn = need(api.rms_norm, "actcomp_rms_norm");
    const int dt = dtype_of(x.scalar_type());
    const Geometry g = geometry(x);
    if (residual) same(x, *residual, "residual");
    const int wdt = affine(x, g.cols, weight, {});
    if (g.cols == 0) bad_value("norm over an empty last dimension");
    if (codes && g.rows == 0) bad_value("a non-empty tensor is expected, got shape " + str(x));
    if (!(eps >= 0.0)) bad_value("eps must not be negative");
    const Rows r = rows_of(x, g.cols), rr = residual ? rows_of(*residual, g.cols) : Rows{};
    const OptTensor w = packed(weight);
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    RmsOut o;
    const int64_t ldc = (g.cols + 15) / 16 * 16;
    if (codes) {
        o.y = empty_on(x, {g.rows, ldc}, at::kByte);
        o.scales = empty_on(x, {(g.cols + 127) / 128 * ((g.rows + 127) / 128) * 128}, at::kByte);
    } else {
        o.y = fresh(x);
    }
    if (residual) o.h = fresh(x);
    o.rstd = empty_on(x, lead, at::kFloat);
    const actcomp_rms_args a{g.rows, g.cols, ptr(r.t), r.ld, residual ? ptr(rr.t) : nullptr, residual ? rr.ld : 0, ptr(w),
                             codes ? nullptr : ptr(o.y), g.cols, ptr(o.h), g.cols,
                             codes ? static_cast<uint8_t *>(ptr(o.y)) : nullptr, ldc,
                             codes ? static_cast<uint8_t *>(ptr(o.scales)) : nullptr,
                             static_cast<float *>(ptr(o.rstd)), dt, wdt, (float)eps, 0};
    const c10::cuda::CUDAGuard guard(x.device());
    check("actcomp_rms_norm", fn(&a, stream_of(x)));
    return o;
}
std::tuple<Tensor, Tensor> rms_norm(const Tensor &x, const OptTensor &weight, double eps) {
    const RmsOut o = rms_forward(x, {}, weight, eps, false);
    return {o.y, o.rstd};
}
std::tuple<Tensor, Tensor, Tensor> add_rms_norm(const Tensor &x, const Tensor &residual, const OptTensor &weight,
                                                double eps) {
    const RmsOut o = rms_forward(x, residual, weight, eps, false);
    return {o.y, *o.h, o.rstd};
}
std::tuple<int64_t, int64_t, Tensor, Tensor, OptTensor, Tensor> rms_norm_fp8(const Tensor &x, const OptTensor &residual,
                                                                            const OptTensor &weight, double eps) {
    const RmsOut o = rms_forward(x, residual, weight, eps, true);
    return {o.y.size(0), x.size(-1), o.y, o.scales, o.h, o.rstd};
}

std::tuple<Tensor, OptTensor> rms_norm_backward(const Tensor &dy, const Tensor &x, const OptTensor &weight,
                                                const Tensor &rstd, const OptTensor &dh) {
    need_cuda(x);
    const auto fn = need(api.rms_norm_bwd, "actcomp_rms_norm_bwd");
    const int dt = dtype_of(x.scalar_type());
    const Geometry g = geometry(x);
    same(x, dy, "dy");
    if (dh) same(x, *dh, "dh");
    const int wdt = affine(x, g.cols, weight, {});
    if (g.cols == 0) bad_value("norm over an empty last dimension");
    const Tensor s = stats(rstd, g.rows, x, "rstd");
    const Rows ry = rows_of(dy, g.cols), rx = rows_of(x, g.cols), rh = dh ? rows_of(*dh, g.cols) : Rows{};
    const OptTensor w = packed(weight);
    const Tensor dx = fresh(x);
    const OptTensor dw = weight ? OptTensor(empty_on(x, {g.cols}, weight->scalar_type())) : OptTensor();
    const c10::cuda::CUDAGuard guard(x.device());
    const size_t bytes = need(api.rms_norm_bwd_workspace, "actcomp_rms_norm_bwd_workspace")(g.rows, g.cols);
    const Tensor ws = empty_on(x, {(int64_t)std::max<size_t>(bytes, 1)}, at::kByte);
    const actcomp_rms_bwd_args a{g.rows, g.cols, ptr(ry.t), ry.ld, ptr(rx.t), rx.ld, dh ? ptr(rh.t) : nullptr,
                                 dh ? rh.ld : 0, ptr(w), static_cast<const float *>(ptr(s)), ptr(dx), g.cols, ptr(dw),
                                 dt, wdt};
    check("actcomp_rms_norm_bwd", fn(&a, ptr(ws), bytes, stream_of(x)));
    return {dx, dw};
}

// ---------------------------------------------------------------- 8-bit floating point
// The stored matrix of a descriptor (rows, cols as stored).
actcomp_fp8 fp8_desc(int64_t rows, int64_t cols, const Tensor &codes, const Tensor &scales, int format, int block,
                     bool transposed) {
    need_cuda(codes);
    if (format < 0 || format > 1 || block < 0 || block > 2) bad_value("unknown 8-bit format or block form");
    const int64_t b = ((rows + 127) / 128) * ((cols + 127) / 128) * (block == ACTCOMP_FP8_TILES ? 1 : 128);
    if (rows < 1 || cols < 1 || codes.dim() != 2 || codes.size(0) != rows || codes.size(1) != (cols + 15) / 16 * 16 ||
        scales.numel() != b || !codes.is_contiguous() || !scales.is_contiguous() || codes.scalar_type() != at::kByte ||
        scales.scalar_type() != at::kByte || scales.device() != codes.device())
        bad_value("codes and scales do not belong to a matrix of " + std::to_string(rows) + " x " + std::to_string(cols));
    return {rows, cols, codes.size(1), static_cast<uint8_t *>(ptr(codes)), static_cast<uint8_t *>(ptr(scales)), format,
            block, transposed, 0};
}
struct Fp8Buffers {
    Tensor codes, scales;
    actcomp_fp8 desc;
};
Fp8Buffers empty_fp8(const Tensor &x, int64_t rows, int64_t cols, int format, int block) {
    const int64_t blocks = ((rows + 127) / 128) * ((cols + 127) / 128);
    Fp8Buffers q{empty_on(x, {rows, (cols + 15) / 16 * 16}, at::kByte),
                 empty_on(x, {block == ACTCOMP_FP8_TILES ? blocks : blocks * 128}, at::kByte), {}};
    q.desc = fp8_desc(rows, cols, q.codes, q.scales, format, block, block == ACTCOMP_FP8_COLS);
    return q;
}

// (rows, cols, codes and scales by rows or tiles, codes and scales by columns) of the
// joined matrix; what is not asked for is None
std::tuple<int64_t, int64_t, OptTensor, OptTensor, OptTensor, OptTensor> fp8_quantize(const Tensor &x, bool by_rows,
                                                                                     bool by_cols, bool tiles,
                                                                                     int format) {
    need_cuda(x);
    const auto fn = need(api.fp8_quantize, "actcomp_fp8_quantize");
    const int dt = dtype_of(x.scalar_type());
    const Rows r = matrix(x);
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    std::optional<Fp8Buffers> q, qt;
    if (by_rows || tiles) q = empty_fp8(x, rows, cols, format, tiles ? ACTCOMP_FP8_TILES : ACTCOMP_FP8_ROWS);
    if (by_cols) qt = empty_fp8(x, rows, cols, format, ACTCOMP_FP8_COLS);
    const c10::cuda::CUDAGuard guard(x.device());
    check("actcomp_fp8_quantize", fn(ptr(r.t), rows, cols, r.ld, dt, q ? &q->desc : nullptr, qt ? &qt->desc : nullptr,
                                     stream_of(x)));
    const auto c = [](const std::optional<Fp8Buffers> &v) { return v ? OptTensor(v->codes) : OptTensor(); };
    const auto s = [](const std::optional<Fp8Buffers> &v) { return v ? OptTensor(v->scales) : OptTensor(); };
    return {rows, cols, c(q), s(q), c(qt), s(qt)};
}

Tensor fp8_dequantize(int64_t rows, int64_t cols, const Tensor &codes, const Tensor &scales, int format, int block,
                      at::ScalarType dtype) {
    const auto fn = need(api.fp8_dequantize, "actcomp_fp8_dequantize");
    const int dt = dtype_of(dtype);
    const actcomp_fp8 d = fp8_desc(rows, cols, codes, scales, format, block, block == ACTCOMP_FP8_COLS);
    const Tensor out = empty_on(codes, {rows, cols}, dtype);
    const c10::cuda::CUDAGuard guard(codes.device());
    check("actcomp_fp8_dequantize", fn(&d, ptr(out), cols, dt, stream_of(codes)));
    return out;
}

// An operand as Python holds it: stored rows and columns, codes, scales, format, block, transposed.
using Fp8Operand = std::tuple<int64_t, int64_t, Tensor, Tensor, int, int, bool>;
actcomp_fp8 fp8_desc(const Fp8Operand &q) {
    return fp8_desc(std::get<0>(q), std::get<1>(q), std::get<2>(q), std::get<3>(q), std::get<4>(q), std::get<5>(q),
                    std::get<6>(q));
}
Tensor fp8_product(const actcomp_fp8 &a, const actcomp_fp8 &b, const Tensor &like, at::IntArrayRef shape,
                   at::ScalarType dtype) {
    const auto fn = need(api.fp8_gemm, "actcomp_fp8_gemm");
    const int dt = dtype_of(dtype);
    const Tensor out = empty_on(like, shape, dtype);
    const c10::cuda::CUDAGuard guard(like.device());
    check("actcomp_fp8_gemm", fn(&a, &b, ptr(out), b.transposed ? b.cols : b.rows, dt, stream_of(like)));
    return out;
}
Tensor fp8_matmul(const Fp8Operand &a, const Fp8Operand &b, at::ScalarType dtype) {
    const actcomp_fp8 da = fp8_desc(a), db = fp8_desc(b);
    const Tensor &like = std::get<2>(a);
    if (like.device() != std::get<2>(b).device()) bad_value("operands on different devices");
    return fp8_product(da, db, like, {da.transposed ? da.cols : da.rows, db.transposed ? db.cols : db.rows}, dtype);
}
// x . w^T with x quantised by rows on the way
Tensor fp8_linear(const Tensor &x, const Fp8Operand &w, std::optional<at::ScalarType> out_dtype) {
    need_cuda(x);
    const auto fn = need(api.fp8_quantize, "actcomp_fp8_quantize");
    const int dt = dtype_of(x.scalar_type());
    const actcomp_fp8 dw = fp8_desc(w);
    const int64_t k = dw.transposed ? dw.rows : dw.cols, n = dw.transposed ? dw.cols : dw.rows;
    if (x.dim() < 1 || x.size(-1) != k)
        bad_value("x is " + str(x) + ", the weight has " + std::to_string(k) + " columns");
    if (x.device() != std::get<2>(w).device()) bad_value("operands on different devices");
    const Rows r = matrix(x);
    const int64_t tokens = x.numel() / k;
    const at::ScalarType dtype = out_dtype.value_or(x.scalar_type());
    dtype_of(dtype);
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    const Fp8Buffers q = empty_fp8(x, tokens, k, ACTCOMP_FP8_E4M3, ACTCOMP_FP8_ROWS);
    {
        const c10::cuda::CUDAGuard guard(x.device());
        check("actcomp_fp8_quantize", fn(ptr(r.t), tokens, k, r.ld, dt, &q.desc, nullptr, stream_of(x)));
    }
    return fp8_product(q.desc, dw, x, shape, dtype);
}

// ---------------------------------------------------------------- cross entropy of a linear layer
// x as rows that the copies to shared memory can take: 16-byte aligned, with a stride of
// whole 16 bytes; copied where they are not.
Rows rows16(const Tensor &x, int64_t cols) {
    Rows r = rows_of(x, cols);
    if (reinterpret_cast<uintptr_t>(ptr(r.t)) % 16 == 0 && r.ld % 8 == 0) return r;
    const int64_t rows = x.numel() / cols, ld = (cols + 7) / 8 * 8;
    const Tensor t = empty_on(x, {rows, ld}, x.scalar_type());
    t.narrow(1, 0, cols).copy_(r.t.reshape({rows, cols}));
    return {t, ld};
}
struct XentIn {
    Rows x, w;
    Tensor target;
    actcomp_xent_args a;
    std::vector<int64_t> lead;
};
XentIn xent_in(const Tensor &x, const Tensor &weight, const Tensor &target, int64_t ignore_index) {
    need_cuda(x);
    if (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf)
        bad_type(std::string("bfloat16 or float16 expected, got ") + at::toString(x.scalar_type()));
    if (x.dim() < 1 || x.size(-1) == 0) bad_value("x over an empty last dimension: " + str(x));
    const int64_t cols = x.size(-1), tokens = x.numel() / cols;
    if (weight.dim() != 2 || weight.size(1) != cols || weight.size(0) == 0 || weight.scalar_type() != x.scalar_type() ||
        weight.device() != x.device())
        bad_value("weight must be (vocabulary, " + std::to_string(cols) + ") with the dtype and device of x (" + str(x) +
                  "), got " + str(weight));
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    if (target.sizes() != lead || target.scalar_type() != at::kLong || target.device() != x.device())
        bad_value("target must hold one int64 for each row of x (" + str(x) + "), got " + str(target));
    const c10::cuda::CUDAGuard guard(x.device());
    XentIn in{tokens ? rows16(x, cols) : Rows{x, cols}, rows16(weight, cols), target.contiguous(), {},
              std::vector<int64_t>(lead.begin(), lead.end())};
    in.a = {tokens, cols, weight.size(0), ptr(in.x.t), in.x.ld, ptr(in.w.t), in.w.ld,
            static_cast<const int64_t *>(ptr(in.target)), ignore_index, nullptr, nullptr, dtype_of(x.scalar_type()), 0};
    return in;
}

std::tuple<Tensor, Tensor> xent(const Tensor &x, const Tensor &weight, const Tensor &target, int64_t ignore_index) {
    const auto fn = need(api.xent, "actcomp_xent");
    XentIn in = xent_in(x, weight, target, ignore_index);
    const Tensor loss = empty_on(x, in.lead, at::kFloat), lse = empty_on(x, in.lead, at::kFloat);
    const c10::cuda::CUDAGuard guard(x.device());
    const size_t bytes = need(api.xent_workspace, "actcomp_xent_workspace")(in.a.tokens, in.a.vocab);
    const Tensor ws = empty_on(x, {(int64_t)std::max<size_t>(bytes, 1)}, at::kByte);
    in.a.loss = static_cast<float *>(ptr(loss));
    in.a.lse = static_cast<float *>(ptr(lse));
    check("actcomp_xent", fn(&in.a, ptr(ws), bytes, stream_of(x)));
    return {loss, lse};
}

std::tuple<OptTensor, OptTensor> xent_backward(const Tensor &dloss, const Tensor &x, const Tensor &weight,
                                               const Tensor &target, const Tensor &lse, const OptTensor &dlse,
                                               int64_t ignore_index, bool x_grad, bool weight_grad, int64_t piece) {
    const auto fn = need(api.xent_bwd, "actcomp_xent_bwd");
    if (!x_grad && !weight_grad) bad_value("no gradient is asked for");
    if (piece < 0) bad_value("vocab_piece must not be negative");
    XentIn in = xent_in(x, weight, target, ignore_index);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor d = stats(dloss, in.a.tokens, x, "dloss"), l = stats(lse, in.a.tokens, x, "lse");
    const OptTensor dl = dlse ? OptTensor(stats(*dlse, in.a.tokens, x, "dlse")) : OptTensor();
    const OptTensor dx = x_grad ? OptTensor(fresh(x)) : OptTensor();
    const OptTensor dw = weight_grad ? OptTensor(fresh(weight)) : OptTensor();
    const size_t bytes = need(api.xent_bwd_workspace, "actcomp_xent_bwd_workspace")(in.a.tokens, in.a.channels,
                                                                                   in.a.vocab, piece);
    const Tensor ws = empty_on(x, {(int64_t)std::max<size_t>(bytes, 1)}, at::kByte);
    in.a.lse = static_cast<float *>(ptr(l));
    const actcomp_xent_grads g{static_cast<const float *>(ptr(d)), static_cast<const float *>(ptr(dl)), ptr(dx),
                               in.a.channels, ptr(dw), in.a.channels};
    check("actcomp_xent_bwd", fn(&in.a, &g, piece, ptr(ws), bytes, stream_of(x)));
    return {dx, dw};
}

}  // namespace

PYBIND11_MODULE(_host, m) {
    m.def("bind", &bind);
    m.def("dropout", &dropout);
    m.def("layer_norm", &layer_norm);
    m.def("branch", &branch);
    m.def("layer_norm_backward", &layer_norm_backward);
    m.def("branch_backward", &branch_backward);
    m.def("quantize", &quantize);
    m.def("dequantize", &dequantize);
    m.def("matmul", &matmul);
    m.def("linear", &linear);
    m.def("one_kernel", &one_kernel);
    m.def("rms_norm", &rms_norm);
    m.def("add_rms_norm", &add_rms_norm);
    m.def("rms_norm_fp8", &rms_norm_fp8);
    m.def("rms_norm_backward", &rms_norm_backward);
    m.def("fp8_quantize", &fp8_quantize);
    m.def("fp8_dequantize", &fp8_dequantize);
    m.def("fp8_matmul", &fp8_matmul);
    m.def("fp8_linear", &fp8_linear);
    m.def("xent", &xent);
    m.def("xent_backward", &xent_backward);
}
