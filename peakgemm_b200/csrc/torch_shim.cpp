// libPeakGemm.so: the PyTorch operator surface over the C ABI (include/peakgemm.h).
// Plain C++ (no CUDA code in this file), so it never needs nvcc.
//
// Mirrors the reference project's registration and host code:
//   TORCH_LIBRARY(PeakGemm, m) with the schema string of src/register.cpp:4-7,
//   gemm_peak(Tensor& c, Tensor& a, Tensor& b, int64 m, n, k) of src/ops/gemm.cpp:5-45:
//   contiguity check, device guard on `a`, the current CUDA stream, dispatch on a's dtype,
//   asynchronous launch, nothing returned, `c` written in place.
// Differences, all on the error side: arguments the reference leaves unchecked
// (device, dtype equality, shapes against m/n/k) raise c10::Error here instead of
// reading out of bounds, and fp64 inputs are refused with a message (in the reference
// they fall into the float branch and throw inside data_ptr<float>, gemm.cpp:34-37).
// float32 goes to pg_sgemm, as the reference sends it to sgemm_peak.
//
// rms_norm_fwd / rms_norm_bwd have no counterpart in the reference; they follow
// the same conventions: outputs first, caller-allocated, in place, return ().
//
// The reference's schema does not say that `c` is written (no `Tensor(a!)`), so a tracing
// compiler sees an operator without outputs or side effects and may drop it.  The schema string
// is kept verbatim for compatibility; next to it every operator has a twin `<name>_out` whose schema
// marks the written tensors, registered for the CUDA key only (so fake/meta tracing never reaches the
// kernels; the fake implementations live in the Python package).  gemm_peak_fused and rms_norm_rstd
// (fused epilogue, RMSNorm folded into the projection), gemm_peak_lora (adapters beside the weights) and rms_norm_residual_fwd / _bwd (the norms around a
// block with its gate and the scaled residual) exist only in the annotated form.

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "../../include/peakgemm.h"

namespace {

using at::Tensor;

int dtype_code(const Tensor &t, const char *op) {
    if (t.scalar_type() == at::kHalf) return PG_F16;
    if (t.scalar_type() == at::kBFloat16) return PG_BF16;
    TORCH_CHECK(false, op, ": only float16 and bfloat16 are built for sm_100a, got ", t.scalar_type());
    return -1;
}

void check_status(int st, const char *op) {
    TORCH_CHECK(st == PG_OK, op, ": ", pg_status_string(st),
                st == PG_ERR_CUDA ? " cudaError=" : "", st == PG_ERR_CUDA ? std::to_string(pg_last_cuda_error()) : "");
}

void gemm_peak(Tensor &c, Tensor &a, Tensor &b, int64_t m, int64_t n, int64_t k) {
    TORCH_CHECK(c.is_contiguous() && a.is_contiguous() && b.is_contiguous());
    TORCH_CHECK(a.is_cuda() && b.is_cuda() && c.is_cuda(), "gemm_peak: tensors must be on a CUDA device");
    TORCH_CHECK(a.device() == b.device() && a.device() == c.device(), "gemm_peak: tensors on different devices");
    TORCH_CHECK(a.scalar_type() == b.scalar_type() && a.scalar_type() == c.scalar_type(),
                "gemm_peak: a, b, c must have one dtype");
    TORCH_CHECK(m >= 0 && n >= 0 && k >= 0 && a.numel() == m * k && b.numel() == n * k && c.numel() == m * n,
                "gemm_peak: tensor sizes do not match m, n, k");
    c10::DeviceGuard device_guard(a.device());
    auto stream = at::cuda::getCurrentCUDAStream();
    if (a.scalar_type() == at::kFloat) {      // the reference's sgemm_peak branch (src/ops/gemm.cpp:34-43)
        check_status(pg_sgemm(c.data_ptr<float>(), a.data_ptr<float>(), b.data_ptr<float>(), m, n, k, k, k, n,
                              stream.stream()),
                     "gemm_peak");
        return;
    }
    const int dt = dtype_code(a, "gemm_peak");
    // Shapes whose last wave of tiles is mostly empty run that wave split over k; the scratch for the partial
    // sums comes from torch's caching allocator (stream-ordered, no cudaMalloc in steady state, capturable).
    const size_t ws_bytes = pg_hgemm_workspace_bytes(m, n, k);
    if (ws_bytes > 0) {
        Tensor ws = at::empty({static_cast<int64_t>(ws_bytes)}, a.options().dtype(at::kByte));
        check_status(pg_hgemm_ws(c.data_ptr(), a.data_ptr(), b.data_ptr(), m, n, k, k, k, n, dt, ws.data_ptr(),
                                 ws_bytes, stream.stream()),
                     "gemm_peak");
        return;
    }
    check_status(pg_hgemm(c.data_ptr(), a.data_ptr(), b.data_ptr(), m, n, k, k, k, n, dt, stream.stream()),
                 "gemm_peak");
}

void rms_norm_fwd(Tensor &y, Tensor &x, Tensor &gamma, double eps) {
    TORCH_CHECK(y.is_contiguous() && x.is_contiguous() && gamma.is_contiguous());
    TORCH_CHECK(x.is_cuda() && y.is_cuda() && gamma.is_cuda(), "rms_norm_fwd: tensors must be on a CUDA device");
    TORCH_CHECK(x.device() == y.device() && x.device() == gamma.device(), "rms_norm_fwd: tensors on different devices");
    TORCH_CHECK(x.dim() >= 1 && x.sizes() == y.sizes() && x.scalar_type() == y.scalar_type(),
                "rms_norm_fwd: y must have x's shape and dtype");
    const int64_t h = x.size(-1);
    TORCH_CHECK(gamma.scalar_type() == at::kFloat && gamma.numel() == h, "rms_norm_fwd: gamma must be float32 [h]");
    const int64_t rows = h > 0 ? x.numel() / h : 0;
    const int dt = dtype_code(x, "rms_norm_fwd");
    c10::DeviceGuard device_guard(x.device());
    auto stream = at::cuda::getCurrentCUDAStream();
    check_status(pg_rmsnorm_fwd(y.data_ptr(), x.data_ptr(), gamma.data_ptr<float>(), rows, h,
                                static_cast<float>(eps), dt, stream.stream()),
                 "rms_norm_fwd");
}

void rms_norm_bwd(Tensor &dx, Tensor &dgamma, Tensor &dy, Tensor &x, Tensor &gamma, double eps) {
    TORCH_CHECK(dx.is_contiguous() && dgamma.is_contiguous() && dy.is_contiguous() && x.is_contiguous() &&
                gamma.is_contiguous());
    TORCH_CHECK(x.is_cuda() && dx.is_cuda() && dy.is_cuda() && gamma.is_cuda() && dgamma.is_cuda(),
                "rms_norm_bwd: tensors must be on a CUDA device");
    TORCH_CHECK(x.device() == dx.device() && x.device() == dy.device() && x.device() == gamma.device() &&
                    x.device() == dgamma.device(),
                "rms_norm_bwd: tensors on different devices");
    TORCH_CHECK(x.dim() >= 1 && x.sizes() == dx.sizes() && x.sizes() == dy.sizes() &&
                    x.scalar_type() == dx.scalar_type() && x.scalar_type() == dy.scalar_type(),
                "rms_norm_bwd: dx and dy must have x's shape and dtype");
    const int64_t h = x.size(-1);
    TORCH_CHECK(gamma.scalar_type() == at::kFloat && gamma.numel() == h && dgamma.scalar_type() == at::kFloat &&
                    dgamma.numel() == h,
                "rms_norm_bwd: gamma and dgamma must be float32 [h]");
    const int64_t rows = h > 0 ? x.numel() / h : 0;
    const int dt = dtype_code(x, "rms_norm_bwd");
    c10::DeviceGuard device_guard(x.device());
    auto stream = at::cuda::getCurrentCUDAStream();
    // Scratch for the per-CTA dgamma partial rows comes from torch's caching
    // allocator: stream-ordered, no cudaMalloc in steady state.
    const size_t ws_bytes = pg_rmsnorm_bwd_workspace_bytes(rows, h);
    Tensor ws = at::empty({static_cast<int64_t>(ws_bytes > 0 ? ws_bytes : 16)}, x.options().dtype(at::kByte));
    check_status(pg_rmsnorm_bwd(dx.data_ptr(), dgamma.data_ptr<float>(), dy.data_ptr(), x.data_ptr(),
                                gamma.data_ptr<float>(), rows, h, static_cast<float>(eps), dt, ws.data_ptr(),
                                ws_bytes, stream.stream()),
                 "rms_norm_bwd");
}

void gemm_peak_out(Tensor &c, const Tensor &a, const Tensor &b) {
    TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && c.dim() == 2, "gemm_peak_out: a [m,k], b [n,k], c [m,n]");
    Tensor a2 = a, b2 = b;
    gemm_peak(c, a2, b2, a.size(0), b.size(0), a.size(1));
}

void rms_norm_fwd_out(Tensor &y, const Tensor &x, const Tensor &gamma, double eps) {
    Tensor x2 = x, g2 = gamma;
    rms_norm_fwd(y, x2, g2, eps);
}

void rms_norm_bwd_out(Tensor &dx, Tensor &dgamma, const Tensor &dy, const Tensor &x, const Tensor &gamma,
                      double eps) {
    Tensor dy2 = dy, x2 = x, g2 = gamma;
    rms_norm_bwd(dx, dgamma, dy2, x2, g2, eps);
}

void rms_norm_rstd(Tensor &rstd, const Tensor &x, double eps) {
    TORCH_CHECK(x.is_cuda() && rstd.is_cuda() && x.device() == rstd.device(), "rms_norm_rstd: CUDA tensors on one device");
    TORCH_CHECK(x.is_contiguous() && rstd.is_contiguous() && x.dim() >= 1);
    const int64_t h = x.size(-1);
    const int64_t rows = h > 0 ? x.numel() / h : 0;
    TORCH_CHECK(rstd.scalar_type() == at::kFloat && rstd.numel() == rows, "rms_norm_rstd: rstd must be float32 [rows]");
    const int dt = dtype_code(x, "rms_norm_rstd");
    c10::DeviceGuard device_guard(x.device());
    auto stream = at::cuda::getCurrentCUDAStream();
    check_status(pg_rmsnorm_rstd(rstd.data_ptr<float>(), x.data_ptr(), rows, h, static_cast<float>(eps), dt,
                                 stream.stream()),
                 "rms_norm_rstd");
}

using OptTensor = std::optional<Tensor>;

struct FusedTerms {
    int64_t m, n, k;
    int dtype;
    const float *row_scale = nullptr;
    const void *bias = nullptr, *residual = nullptr;
};

// The arguments that gemm_peak_fused and gemm_peak_lora share.
FusedTerms check_fused_terms(const Tensor &d, const Tensor &a, const Tensor &b, const OptTensor &row_scale,
                             const OptTensor &bias, const OptTensor &residual, const char *op) {
    TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && d.dim() == 2, op, ": a [m,k], b [n,k], d [m,n]");
    TORCH_CHECK(d.is_contiguous() && a.is_contiguous() && b.is_contiguous());
    TORCH_CHECK(a.is_cuda() && b.is_cuda() && d.is_cuda() && a.device() == b.device() && a.device() == d.device(), op,
                ": tensors must be on one CUDA device");
    TORCH_CHECK(a.scalar_type() == b.scalar_type() && a.scalar_type() == d.scalar_type(), op,
                ": a, b, d must have one dtype");
    FusedTerms f;
    f.m = a.size(0);
    f.k = a.size(1);
    f.n = b.size(0);
    TORCH_CHECK(b.size(1) == f.k && d.size(0) == f.m && d.size(1) == f.n, op, ": shapes do not match");
    if (row_scale) {
        TORCH_CHECK(row_scale->is_cuda() && row_scale->device() == a.device() && row_scale->is_contiguous() &&
                        row_scale->scalar_type() == at::kFloat && row_scale->numel() == f.m,
                    op, ": row_scale must be float32 [m] on a's device");
        f.row_scale = row_scale->data_ptr<float>();
    }
    if (bias) {
        TORCH_CHECK(bias->is_cuda() && bias->device() == a.device() && bias->is_contiguous() &&
                        bias->scalar_type() == a.scalar_type() && bias->numel() == f.n,
                    op, ": bias must be [n] of a's dtype on a's device");
        f.bias = bias->data_ptr();
    }
    if (residual) {
        TORCH_CHECK(residual->is_cuda() && residual->device() == a.device() && residual->is_contiguous() &&
                        residual->scalar_type() == a.scalar_type() && residual->dim() == 2 &&
                        residual->size(0) == f.m && residual->size(1) == f.n,
                    op, ": residual must be [m,n] of a's dtype on a's device");
        f.residual = residual->data_ptr();
    }
    f.dtype = dtype_code(a, op);
    return f;
}

// d[m,n] = row_scale[:,None] * (a[m,k] @ b[n,k]^T) + bias[None,:] + residual, each term optional.
void gemm_peak_fused(Tensor &d, const Tensor &a, const Tensor &b, const OptTensor &row_scale, const OptTensor &bias,
                     const OptTensor &residual, bool pdl) {
    const FusedTerms f = check_fused_terms(d, a, b, row_scale, bias, residual, "gemm_peak_fused");
    c10::DeviceGuard device_guard(a.device());
    auto stream = at::cuda::getCurrentCUDAStream();
    check_status(pg_hgemm_fused(d.data_ptr(), a.data_ptr(), b.data_ptr(), f.m, f.n, f.k, f.k, f.k, f.n, f.row_scale,
                                f.bias, f.residual, f.n, f.dtype, pdl ? PG_FUSED_PDL : 0, stream.stream()),
                 "gemm_peak_fused");
}

// The same with every row's adapter beside b: lora_a [L,r,k], lora_b [L,n,r], ids [m].
void gemm_peak_lora(Tensor &d, const Tensor &a, const Tensor &b, const Tensor &lora_a, const Tensor &lora_b,
                    const Tensor &ids, const OptTensor &scale, const OptTensor &row_scale, const OptTensor &bias,
                    const OptTensor &residual) {
    const char *op = "gemm_peak_lora";
    const FusedTerms f = check_fused_terms(d, a, b, row_scale, bias, residual, op);
    TORCH_CHECK(lora_a.dim() == 3 && lora_b.dim() == 3 && ids.dim() == 1, op, ": lora_a [L,r,k], lora_b [L,n,r], ids [m]");
    const int64_t adapters = lora_a.size(0), rank = lora_a.size(1);
    TORCH_CHECK(lora_a.size(2) == f.k && lora_b.size(0) == adapters && lora_b.size(1) == f.n && lora_b.size(2) == rank &&
                    ids.size(0) == f.m,
                op, ": the adapters' shapes do not match");
    TORCH_CHECK(lora_a.device() == a.device() && lora_b.device() == a.device() && ids.device() == a.device(), op,
                ": tensors must be on one CUDA device");
    TORCH_CHECK(lora_a.is_contiguous() && lora_b.is_contiguous() && ids.is_contiguous(), op,
                ": lora_a, lora_b and ids must be contiguous");
    TORCH_CHECK(lora_a.scalar_type() == a.scalar_type() && lora_b.scalar_type() == a.scalar_type(), op,
                ": lora_a and lora_b must have a's dtype");
    TORCH_CHECK(ids.scalar_type() == at::kInt, op, ": ids must be int32");
    if (scale)
        TORCH_CHECK(scale->device() == a.device() && scale->is_contiguous() && scale->scalar_type() == at::kFloat &&
                        scale->numel() == adapters,
                    op, ": scale must be float32 [L] on a's device");
    c10::DeviceGuard device_guard(a.device());
    auto stream = at::cuda::getCurrentCUDAStream();
    // scratch from torch's caching allocator, as for gemm_peak
    const size_t ws_bytes = pg_hgemm_lora_workspace_bytes(f.m, f.n, f.k, adapters, rank);
    Tensor ws = at::empty({static_cast<int64_t>(ws_bytes > 0 ? ws_bytes : 16)}, a.options().dtype(at::kByte));
    check_status(pg_hgemm_lora(d.data_ptr(), a.data_ptr(), b.data_ptr(), f.m, f.n, f.k, f.k, f.k, f.n, lora_a.data_ptr(),
                               lora_b.data_ptr(), ids.data_ptr<int32_t>(), adapters, rank,
                               scale ? scale->data_ptr<float>() : nullptr, f.row_scale, f.bias, f.residual, f.n, f.dtype,
                               ws.data_ptr(), ws_bytes, stream.stream()),
                 op);
}

// ------------------------------------------- norms around a gated residual ----

void *opt_ptr(const OptTensor &t) { return t ? t->data_ptr() : nullptr; }
float *opt_f32(const OptTensor &t) { return t ? t->data_ptr<float>() : nullptr; }

// `t`, where given, is a dense tensor of `type` and shape `sizes` on like's device.
void check_tensor(const Tensor &t, const Tensor &like, at::ScalarType type, at::IntArrayRef sizes, const char *op, const char *what) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), op, ": ", what, " must be on the other tensors' CUDA device");
    TORCH_CHECK(t.is_contiguous() && t.scalar_type() == type && t.sizes() == sizes, op, ": ", what,
                " must be contiguous, of type ", type, " and shape ", sizes);
}
void check_opt(const OptTensor &t, const Tensor &like, at::ScalarType type, at::IntArrayRef sizes, const char *op, const char *what) {
    if (t) check_tensor(*t, like, type, sizes, op, what);
}

struct ResidualTerms {
    int64_t rows, h, gate_rows, res_scale_len;
    int dtype;
};

ResidualTerms check_residual_terms(const Tensor &u, const OptTensor &gamma_post, const OptTensor &gate,
                                   const OptTensor &res_scale, const OptTensor &gamma_pre, const char *op) {
    TORCH_CHECK(u.is_cuda(), op, ": tensors must be on a CUDA device");
    TORCH_CHECK(u.dim() >= 1 && u.is_contiguous(), op, ": tensors must be contiguous [..., h]");
    ResidualTerms t;
    t.dtype = dtype_code(u, op);
    t.h = u.size(-1);
    t.rows = t.h > 0 ? u.numel() / t.h : 0;
    check_opt(gamma_post, u, at::kFloat, {t.h}, op, "gamma_post");
    check_opt(gamma_pre, u, at::kFloat, {t.h}, op, "gamma_pre");
    t.gate_rows = 0;
    if (gate) {
        TORCH_CHECK(gate->dim() >= 1 && gate->size(-1) == t.h, op, ": gate must be [..., h]");
        t.gate_rows = t.h > 0 ? gate->numel() / t.h : 0;
        TORCH_CHECK(t.gate_rows > 0 && t.rows % t.gate_rows == 0, op, ": the rows of gate must divide the rows of u");
        check_tensor(*gate, u, u.scalar_type(), gate->sizes(), op, "gate");
    }
    t.res_scale_len = res_scale ? res_scale->numel() : 0;
    TORCH_CHECK(!res_scale || t.res_scale_len == 1 || t.res_scale_len == t.h, op, ": res_scale must have 1 or h elements");
    check_opt(res_scale, u, at::kFloat, {t.res_scale_len}, op, "res_scale");
    return t;
}

void rms_norm_residual_fwd(Tensor &s, const OptTensor &y, const Tensor &u, const Tensor &residual,
                           const OptTensor &gamma_post, const OptTensor &gate, const OptTensor &res_scale,
                           const OptTensor &gamma_pre, double eps) {
    const char *op = "rms_norm_residual_fwd";
    const ResidualTerms t = check_residual_terms(u, gamma_post, gate, res_scale, gamma_pre, op);
    TORCH_CHECK(y.has_value() == gamma_pre.has_value(), op, ": y and gamma_pre come together");
    check_tensor(s, u, u.scalar_type(), u.sizes(), op, "s");
    check_opt(y, u, u.scalar_type(), u.sizes(), op, "y");
    check_tensor(residual, u, u.scalar_type(), u.sizes(), op, "residual");
    c10::DeviceGuard device_guard(u.device());
    auto stream = at::cuda::getCurrentCUDAStream();
    check_status(pg_rmsnorm_residual_fwd(s.data_ptr(), opt_ptr(y), u.data_ptr(), residual.data_ptr(), opt_f32(gamma_post),
                                         opt_ptr(gate), t.gate_rows, opt_f32(res_scale), t.res_scale_len,
                                         opt_f32(gamma_pre), t.rows, t.h, static_cast<float>(eps), t.dtype,
                                         stream.stream()),
                 op);
}

void rms_norm_residual_bwd(Tensor &du, Tensor &dresidual, const OptTensor &dgamma_post, const OptTensor &dgate,
                           const OptTensor &dres_scale, const OptTensor &dgamma_pre, const OptTensor &dy,
                           const OptTensor &ds, const OptTensor &s, const OptTensor &u, const OptTensor &residual,
                           const OptTensor &gamma_post, const OptTensor &gate, const OptTensor &res_scale,
                           const OptTensor &gamma_pre, double eps) {
    const char *op = "rms_norm_residual_bwd";
    const ResidualTerms t = check_residual_terms(du, gamma_post, gate, res_scale, gamma_pre, op);
    const at::ScalarType type = du.scalar_type();
    const at::IntArrayRef n = du.sizes();
    TORCH_CHECK(dy.has_value() == gamma_pre.has_value(), op, ": dy and gamma_pre come together");
    TORCH_CHECK(dy || ds, op, ": at least one of dy and ds is needed");
    TORCH_CHECK(s || !gamma_pre, op, ": gamma_pre needs s");
    TORCH_CHECK(u || !(gamma_post || dgate), op, ": gamma_post and dgate need u");
    TORCH_CHECK(residual || !dres_scale, op, ": dres_scale needs residual");
    TORCH_CHECK((gamma_post || !dgamma_post) && (gate || !dgate) && (res_scale || !dres_scale) && (gamma_pre || !dgamma_pre),
                op, ": a gradient needs the tensor it is the gradient of");
    check_tensor(dresidual, du, type, n, op, "dresidual");
    check_opt(dy, du, type, n, op, "dy");
    check_opt(ds, du, type, n, op, "ds");
    check_opt(s, du, type, n, op, "s");
    check_opt(u, du, type, n, op, "u");
    check_opt(residual, du, type, n, op, "residual");
    check_opt(dgamma_post, du, at::kFloat, {t.h}, op, "dgamma_post");
    check_opt(dgamma_pre, du, at::kFloat, {t.h}, op, "dgamma_pre");
    if (dgate) check_tensor(*dgate, du, type, gate->sizes(), op, "dgate");
    check_opt(dres_scale, du, at::kFloat, {t.res_scale_len}, op, "dres_scale");
    c10::DeviceGuard device_guard(du.device());
    auto stream = at::cuda::getCurrentCUDAStream();
    const size_t ws_bytes = pg_rmsnorm_residual_bwd_workspace_bytes(t.rows, t.h, t.gate_rows);
    Tensor ws = at::empty({static_cast<int64_t>(ws_bytes > 0 ? ws_bytes : 16)}, du.options().dtype(at::kByte));
    check_status(pg_rmsnorm_residual_bwd(du.data_ptr(), dresidual.data_ptr(), opt_f32(dgamma_post), opt_ptr(dgate),
                                         opt_f32(dres_scale), opt_f32(dgamma_pre), opt_ptr(dy), opt_ptr(ds), opt_ptr(s),
                                         opt_ptr(u), opt_ptr(residual), opt_f32(gamma_post), opt_ptr(gate), t.gate_rows,
                                         opt_f32(res_scale), t.res_scale_len, opt_f32(gamma_pre), t.rows, t.h,
                                         static_cast<float>(eps), t.dtype, ws.data_ptr(), ws_bytes, stream.stream()),
                 op);
}

}  // namespace

TORCH_LIBRARY(PeakGemm, m) {
    m.def("gemm_peak(Tensor c, Tensor a, Tensor b, SymInt m, SymInt n, SymInt k) -> ()");
    m.impl("gemm_peak", &gemm_peak);
    m.def("rms_norm_fwd(Tensor y, Tensor x, Tensor gamma, float eps) -> ()");
    m.impl("rms_norm_fwd", &rms_norm_fwd);
    m.def("rms_norm_bwd(Tensor dx, Tensor dgamma, Tensor dy, Tensor x, Tensor gamma, float eps) -> ()");
    m.impl("rms_norm_bwd", &rms_norm_bwd);
    // annotated forms (see the note at the top of this file)
    m.def("gemm_peak_out(Tensor(a!) c, Tensor a, Tensor b) -> ()");
    m.def("rms_norm_fwd_out(Tensor(a!) y, Tensor x, Tensor gamma, float eps) -> ()");
    m.def("rms_norm_bwd_out(Tensor(a!) dx, Tensor(b!) dgamma, Tensor dy, Tensor x, Tensor gamma, float eps) -> ()");
    m.def("rms_norm_rstd(Tensor(a!) rstd, Tensor x, float eps) -> ()");
    m.def("gemm_peak_fused(Tensor(a!) d, Tensor a, Tensor b, Tensor? row_scale, Tensor? bias, Tensor? residual, "
          "bool pdl=False) -> ()");
    m.def("gemm_peak_lora(Tensor(a!) d, Tensor a, Tensor b, Tensor lora_a, Tensor lora_b, Tensor ids, Tensor? scale, "
          "Tensor? row_scale, Tensor? bias, Tensor? residual) -> ()");
    m.def("rms_norm_residual_fwd(Tensor(a!) s, Tensor(b!)? y, Tensor u, Tensor residual, Tensor? gamma_post, Tensor? gate, "
          "Tensor? res_scale, Tensor? gamma_pre, float eps) -> ()");
    m.def("rms_norm_residual_bwd(Tensor(a!) du, Tensor(b!) dresidual, Tensor(c!)? dgamma_post, Tensor(d!)? dgate, "
          "Tensor(e!)? dres_scale, Tensor(f!)? dgamma_pre, Tensor? dy, Tensor? ds, Tensor? s, Tensor? u, "
          "Tensor? residual, Tensor? gamma_post, Tensor? gate, Tensor? res_scale, Tensor? gamma_pre, float eps) -> ()");
}

TORCH_LIBRARY_IMPL(PeakGemm, CUDA, m) {
    m.impl("gemm_peak_out", &gemm_peak_out);
    m.impl("rms_norm_fwd_out", &rms_norm_fwd_out);
    m.impl("rms_norm_bwd_out", &rms_norm_bwd_out);
    m.impl("rms_norm_rstd", &rms_norm_rstd);
    m.impl("gemm_peak_fused", &gemm_peak_fused);
    m.impl("gemm_peak_lora", &gemm_peak_lora);
    m.impl("rms_norm_residual_fwd", &rms_norm_residual_fwd);
    m.impl("rms_norm_residual_bwd", &rms_norm_residual_bwd);
}
