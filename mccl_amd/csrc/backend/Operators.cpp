// Operators.cpp -- layer norm and dropout over torch tensors without the Python statements between the
// call and the launch, which for a few rows take longer than the kernel (8 rows of 1024: 9.7 us a call from
// Python, 6.0 from here).
//
// What is not the plain case, rows that lie apart or arguments that do not go together, is left to the
// Python form (the functions return None and have done nothing), which copies, or words the error.
#include "backend/Operators.hpp"

#include <torch/extension.h>

#include <optional>

#include "backend/Device.hpp"
#include "mcclx.h"

namespace py = pybind11;

namespace mccl {
namespace {

using Maybe = std::optional<at::Tensor>;

int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return MCCLX_F32;
        case at::kHalf: return MCCLX_F16;
        case at::kBFloat16: return MCCLX_BF16;
        default: return -1;
    }
}
mcclx_ctx* context(uintptr_t handle) { return reinterpret_cast<mcclx_ctx*>(handle); }
// (a norm of 8 rows 6.7 us a call; with at::empty_like, and autograd asked about each, 7.0; 3.8 of it the launch)
at::Tensor fresh_like(const at::Tensor& t) { return at::empty(t.sizes(), t.options()); }
void* address(const Maybe& t) { return t ? t->data_ptr() : nullptr; }

bool here(const at::Tensor& t, int device) { return dev::on_device(t) && t.get_device() == device && t.is_contiguous(); }
// A matrix of adjacent rows of a known type.
bool matrix(const at::Tensor& t, int device) { return t.dim() > 0 && t.size(-1) > 0 && here(t, device) && dtype_code(t) >= 0; }
bool like(const at::Tensor& t, const at::Tensor& x, int device) {
    return here(t, device) && t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes();
}
bool parameter(const Maybe& t, const at::Tensor& x, int device) {
    return !t || (here(*t, device) && t->dim() == 1 && t->size(0) == x.size(-1) && (t->scalar_type() == x.scalar_type() || t->scalar_type() == at::kFloat));
}
bool statistic(const at::Tensor& t, int64_t rows, int device) { return here(t, device) && t.scalar_type() == at::kFloat && t.numel() == rows; }

mcclx_norm arguments(const at::Tensor& x, const Maybe& weight, const Maybe& bias, double p, uint64_t seed, uint64_t offset) {
    mcclx_norm a = {};
    a.dtype = dtype_code(x);
    a.param_dtype = weight ? dtype_code(*weight) : bias ? dtype_code(*bias) : a.dtype;
    a.cols = static_cast<uint64_t>(x.size(-1));
    a.rows = static_cast<uint64_t>(x.numel()) / a.cols;
    a.p = p;
    a.seed = seed;
    a.offset = offset;
    a.weight = address(weight);
    a.bias = address(bias);
    return a;
}

py::object norm_forward(uintptr_t handle, int device, const at::Tensor& x, const Maybe& residual, const Maybe& weight, const Maybe& bias, double p,
                        uint64_t seed, uint64_t offset, double eps, bool keep_sum) {
    if (!matrix(x, device) || (residual && !like(*residual, x, device)) || !parameter(weight, x, device) || !parameter(bias, x, device) ||
        (weight && bias && weight->scalar_type() != bias->scalar_type()))
        return py::none();
    const at::AutoDispatchBelowAutograd guard;
    mcclx_norm a = arguments(x, weight, bias, p, seed, offset);
    a.eps = eps;
    const at::Tensor y = fresh_like(x), mean = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat)), rstd = fresh_like(mean);
    Maybe s;
    if (keep_sum) s = fresh_like(x);
    a.x = x.data_ptr();
    a.residual = address(residual);
    a.y = y.data_ptr();
    a.s = address(s);
    a.mean = mean.data_ptr<float>();
    a.rstd = rstd.data_ptr<float>();
    const int rc = mcclx_layer_norm_forward(context(handle), dev::current_stream(device), &a);
    return py::make_tuple(rc, y, s, mean, rstd);
}

py::object norm_backward(uintptr_t handle, int device, const at::Tensor& dy, const Maybe& ds, const at::Tensor& s, const at::Tensor& mean,
                         const at::Tensor& rstd, const Maybe& weight, double p, uint64_t seed, uint64_t offset, bool with_x, bool with_residual,
                         bool with_weight, int bias_dtype) {
    if (!matrix(s, device) || !like(dy, s, device) || (ds && !like(*ds, s, device)) || !parameter(weight, s, device)) return py::none();
    mcclx_norm a = arguments(s, weight, std::nullopt, p, seed, offset);
    if (bias_dtype != -1) {  // (-1: no gradient of a bias)
        if (bias_dtype != a.param_dtype && (weight || bias_dtype != MCCLX_F32)) return py::none();
        a.param_dtype = bias_dtype;
    }
    if (!statistic(mean, static_cast<int64_t>(a.rows), device) || !statistic(rstd, static_cast<int64_t>(a.rows), device)) return py::none();
    const at::AutoDispatchBelowAutograd guard;
    Maybe dx, dresidual, dweight, dbias;
    if (with_x) dx = fresh_like(s);
    if (with_residual) dresidual = fresh_like(s);
    if (weight && with_weight) dweight = fresh_like(*weight);
    if (bias_dtype != -1) dbias = at::empty({s.size(-1)}, a.param_dtype == a.dtype ? s.options() : s.options().dtype(at::kFloat));
    a.workspace_bytes = mcclx_layer_norm_workspace_bytes(context(handle), a.rows, a.cols);
    const at::Tensor work = dev::empty_bytes(static_cast<int64_t>(a.workspace_bytes), device);
    a.workspace = work.data_ptr();
    a.mean = mean.data_ptr<float>();
    a.rstd = rstd.data_ptr<float>();
    a.s = s.data_ptr();
    a.dy = dy.data_ptr();
    a.ds = address(ds);
    a.dx = address(dx);
    a.dresidual = address(dresidual);
    a.dweight = address(dweight);
    a.dbias = address(dbias);
    const int rc = mcclx_layer_norm_backward(context(handle), dev::current_stream(device), &a);
    return py::make_tuple(rc, dx, dresidual, dweight, dbias);
}

py::object dropout(uintptr_t handle, int device, const at::Tensor& x, const Maybe& residual, double p, uint64_t seed, uint64_t offset) {
    if (!matrix(x, device) || (residual && !like(*residual, x, device))) return py::none();
    const at::AutoDispatchBelowAutograd guard;
    const at::Tensor out = fresh_like(x);
    const uint64_t cols = static_cast<uint64_t>(x.size(-1));
    const int rc = mcclx_dropout(context(handle), dev::current_stream(device), dtype_code(x), static_cast<uint64_t>(x.numel()) / cols, cols, x.data_ptr(),
                                 cols, address(residual), cols, out.data_ptr(), p, seed, offset);
    return py::make_tuple(rc, out);
}

}  // namespace

void bind_operators(py::module_& m) {
    m.def("_norm_forward", &norm_forward);
    m.def("_norm_backward", &norm_backward);
    m.def("_dropout", &dropout);
}

}  // namespace mccl
