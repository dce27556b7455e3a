// Binding of the row norm, the 8-bit channel mix and the gradient clipping to torch tensors and autograd.
//
// The kernels are the C entries of libdsw_hip.so (include/dsw_hip.h); this file checks arguments, allocates results on the current
// stream and records backward passes.  It is compiled code because of what the operators are used for: one token is normalised
// in 4 us and multiplied in 5 us on the card, and a training step's norm spends less time there than an interpreter needs to
// run its forward and backward functions on two threads (777 x 1030 fp32, both passes: a Python autograd function 150 us, this
// one 54 us).
//
// Errors: ValueError / TypeError for arguments, RuntimeError for what the path does not offer and for the library's codes.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <c10/hip/HIPGraphsC10Utils.h>

#include <array>
#include <cmath>
#include <optional>
#include <string>
#include <vector>

#include "../../include/dsw_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// the library's entries, by address (dsw_amd._native decides which build of it is loaded)
struct Entries {
    decltype(&dsw_strerror) strerror = nullptr;
    decltype(&dsw_rmsnorm_fwd) rmsnorm_fwd = nullptr;
    decltype(&dsw_rmsnorm_fwd_fp8) rmsnorm_fwd_fp8 = nullptr;
    decltype(&dsw_quant_fp8) quant_fp8 = nullptr;
    decltype(&dsw_quant_fp8_weight) quant_fp8_weight = nullptr;
    decltype(&dsw_rmsnorm_bwd_workspace_bytes) rmsnorm_bwd_workspace_bytes = nullptr;
    decltype(&dsw_rmsnorm_bwd) rmsnorm_bwd = nullptr;
    decltype(&dsw_fp8_mix_workspace_bytes) fp8_mix_workspace_bytes = nullptr;
    decltype(&dsw_fp8_mix) fp8_mix = nullptr;
    decltype(&dsw_grad_norm_workspace_bytes) grad_norm_workspace_bytes = nullptr;
    decltype(&dsw_grad_norm_clip) grad_norm_clip = nullptr;
} lib;

void bind(const std::map<std::string, uint64_t>& at) {
#define ENTRY(name) lib.name = reinterpret_cast<decltype(lib.name)>(at.at("dsw_" #name))
    ENTRY(strerror); ENTRY(rmsnorm_fwd); ENTRY(rmsnorm_fwd_fp8); ENTRY(quant_fp8); ENTRY(quant_fp8_weight);
    ENTRY(rmsnorm_bwd_workspace_bytes); ENTRY(rmsnorm_bwd); ENTRY(fp8_mix_workspace_bytes); ENTRY(fp8_mix);
    ENTRY(grad_norm_workspace_bytes); ENTRY(grad_norm_clip);
#undef ENTRY
}

void check(int64_t rc, const char* what) {
    TORCH_CHECK(rc >= 0, what, " failed: ", lib.strerror((int)rc), " (code ", rc, ")");
}

int code_of(at::ScalarType t) {
    TORCH_CHECK_TYPE(t == at::kFloat || t == at::kBFloat16, "dsw: unsupported dtype ", t, "; the HIP path implements float32 and bfloat16");
    return t == at::kBFloat16 ? DSW_BF16 : DSW_F32;
}
void same_type(const Tensor& a, const Tensor& b) {
    TORCH_CHECK_TYPE(a.scalar_type() == b.scalar_type(), "dsw: mixed dtypes ", a.scalar_type(), " vs ", b.scalar_type());
}
void same_device(const Tensor& a, const Tensor& b) {
    TORCH_CHECK_VALUE(a.device() == b.device(), "dsw: tensors on ", a.device(), " and ", b.device(), " in one call");
}
void on_gpu(const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "dsw: the row norm, the 8-bit channel mix and the gradient clipping run only on a ROCm device (got a ",
                t.device(), " tensor). There is no CPU fallback; move the model and inputs to 'cuda'.");
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
// (a result without a tangent would read as a derivative of zero; no_grad does not switch tangents off)
void no_tangent(at::ArrayRef<const Tensor*> tensors) {
    if (!torch::autograd::ForwardADLevel::try_get_by_idx(0)) return;       // (no tensor of the process has a tangent)
    for (const Tensor* t : tensors)
        TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), "dsw: the row norm, the 8-bit channel mix and the gradient norm have no "
                    "forward-mode derivative; unpack the dual tensor (torch.autograd.forward_ad.unpack_dual)");
}
void no_backward(const char* what, std::initializer_list<const Tensor*> tensors) {
    no_tangent(tensors);
    if (!at::GradMode::is_enabled()) return;
    for (const Tensor* t : tensors)
        TORCH_CHECK(!wants_grad(*t), "dsw: ", what, " is a serving path without a backward pass; call it under torch.no_grad()");
}

// t [..., C] as rows of C neighbouring elements, `step` elements apart: channel slices of wider tensors stay views, any other
// layout is copied.  any_last: the last axis may have any stride of its own.
struct Rows { Tensor t; int64_t rows, step; };
Rows as_rows(const Tensor& t, bool any_last = false) {
    const auto sizes = t.sizes(), strides = t.strides();
    const int64_t C = sizes.back(), rows = C ? t.numel() / C : 0;
    if (t.is_contiguous()) return {t, rows, C};
    bool ok = rows > 0 && (any_last || C == 1 || strides.back() == 1);
    int64_t step = -1, want = -1;
    for (int64_t i = (int64_t)sizes.size() - 2; i >= 0 && ok; --i) {
        if (sizes[i] == 1) continue;
        if (step < 0) step = strides[i];
        else if (strides[i] != want) ok = false;
        want = strides[i] * sizes[i];
    }
    if (step < 0) step = C;
    if (!any_last && step < C) ok = false;             // rows that overlap (a broadcast input)
    if (!ok) return {t.contiguous(), rows, C};
    return {t, rows, step};
}

int64_t blocks_of(int64_t channels) { return (channels + 127) / 128; }

// Uninitialised e4m3 rows: the scales lie block after block with the rows next to each other (whole lines for the product),
// behind a view [..., blocks]
std::array<Tensor, 2> new_rows(const Tensor& x, int64_t rows, int64_t C) {
    std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end()), strides(sizes.size());
    sizes.back() = blocks_of(C);
    strides.back() = rows > 0 ? rows : 1;
    int64_t s = 1;
    for (int64_t i = (int64_t)sizes.size() - 2; i >= 0; --i) { strides[i] = s; s *= sizes[i] > 0 ? sizes[i] : 1; }
    return {at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)), at::empty_strided(sizes, strides, x.options().dtype(at::kFloat))};
}

// ---- row norm --------------------------------------------------------------------------------------------------------------
void check_norm(const Tensor& x, const Tensor& r, const Tensor& w, double eps) {
    TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 1 && x.size(-1) == w.size(0) && w.size(0) >= 1, "expected x [..., C] and weight [C] with C >= 1");
    TORCH_CHECK_VALUE(!r.defined() || r.sizes() == x.sizes(), "expected a residual of the shape of x");
    TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(eps), "eps must be a finite number >= 0");
    code_of(x.scalar_type());
    no_tangent({&x, &r, &w});
    same_type(x, w);
    same_device(x, w);
    if (r.defined()) { same_type(x, r); same_device(x, r); }
}

struct NormOut { Tensor y, h, rstd, x, r; };        // x, r: the rows as the kernel read them
NormOut norm_forward(const Tensor& x, const Tensor& r, const Tensor& w, double eps, bool need_rstd) {
    const c10::DeviceGuard guard(x.device());
    const Rows xr = as_rows(x);
    const Tensor wc = w.contiguous();
    NormOut o;
    o.y = at::empty(x.sizes(), x.options());
    if (need_rstd) o.rstd = at::empty({xr.rows}, x.options().dtype(at::kFloat));
    Rows rr{Tensor(), 0, 0};
    if (r.defined()) { rr = as_rows(r); o.h = at::empty(x.sizes(), x.options()); }
    o.x = xr.t;
    o.r = rr.t;
    check(lib.rmsnorm_fwd(xr.t.data_ptr(), xr.step, r.defined() ? rr.t.data_ptr() : nullptr, rr.step, wc.data_ptr(), o.y.data_ptr(),
                          r.defined() ? o.h.data_ptr() : nullptr, need_rstd ? o.rstd.data_ptr<float>() : nullptr, xr.rows, w.size(0),
                          (float)eps, code_of(x.scalar_type()), stream_of(x)), "dsw_rmsnorm_fwd");
    return o;
}

// A leaf has one gradient accumulator, which belongs to the stream it was created on and lives as long as any graph over the leaf.
// A backward pass captured while such a graph of another stream is alive would hand its gradient over to that stream, which
// then waits for the capture without ever joining it: ending the capture kills the process.  It is refused instead.
void refuse_foreign_leaves(const Tensor& t) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    const c10::Stream here = c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device());
    for (size_t i = 0; i < node->num_outputs(); ++i) {
        auto* leaf = dynamic_cast<torch::autograd::AccumulateGrad*>(node->next_edge(i).function.get());
        if (leaf == nullptr || !node->task_should_compute_output(i)) continue;
        const auto s = leaf->stream();
        if (!s || *s == here) continue;
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;                      // (a stream of the same capture may join it)
        const hipError_t err = hipStreamIsCapturing(c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, *s).stream(), &status);
        if (err != hipSuccess) (void)hipGetLastError();
        TORCH_CHECK(err == hipSuccess && status == hipStreamCaptureStatusActive, "dsw: a backward pass is being captured while an earlier graph over the same leaf (shape ",
                    leaf->variable.sizes(), ") is alive on another stream; drop that graph (its outputs, its loss) before the capture");
    }
}

// gradients that do not differentiate again: an error for whoever tries (create_graph), nothing otherwise
// (their error stands behind everything they were computed from, so that no path past it reads as a missing gradient)
variable_list once(variable_list grads, const variable_list& from, const variable_list& dys) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (Tensor& g : grads) if (g.defined()) in.push_back(g.detach().requires_grad_());
    for (const auto& list : {from, dys})
        for (const Tensor& t : list) if (t.defined()) in.push_back(t);
    auto err = std::make_shared<torch::autograd::DelayedError>("dsw: the row norm differentiates once", (int64_t)in.size());
    in = (*err)(std::move(in));
    size_t k = 0;
    for (Tensor& g : grads) if (g.defined()) g = in[k++];
    return grads;
}

// {dx (of both addends), dw}
std::array<Tensor, 2> norm_backward(const Tensor& x, const Tensor& r, const Tensor& w, const Tensor& rstd, const Tensor& dy, const Tensor& dh,
                                    bool need_x, bool need_w) {
    const at::AutoGradMode off(false);
    refuse_foreign_leaves(x);
    if (!dy.defined())                                // nothing behind y: the stream's own gradient passes through
        return {need_x ? dh : Tensor(), need_w ? at::zeros_like(w) : Tensor()};
    const c10::DeviceGuard guard(x.device());
    const Rows xr = as_rows(x), rr = r.defined() ? as_rows(r) : Rows{Tensor(), 0, 0};
    const Tensor g = dy.contiguous(), d = dh.defined() ? dh.contiguous() : dh;
    const int code = code_of(x.scalar_type());
    const int64_t C = w.size(0);
    Tensor dx, dw, ws;
    int64_t bytes = 0;
    if (need_x) dx = at::empty(x.sizes(), x.options());
    if (need_w) {
        dw = at::empty(w.sizes(), w.options());
        bytes = lib.rmsnorm_bwd_workspace_bytes(xr.rows, C, code);
        check(bytes, "dsw_rmsnorm_bwd_workspace_bytes");
        ws = at::empty({bytes}, x.options().dtype(at::kByte));
    }
    if (need_x || need_w)
        check(lib.rmsnorm_bwd(g.data_ptr(), d.defined() ? d.data_ptr() : nullptr, xr.t.data_ptr(), xr.step, r.defined() ? rr.t.data_ptr() : nullptr,
                              rr.step, w.data_ptr(), rstd.data_ptr<float>(), need_x ? dx.data_ptr() : nullptr, need_w ? dw.data_ptr() : nullptr,
                              need_w ? ws.data_ptr() : nullptr, bytes, xr.rows, C, code, stream_of(x)), "dsw_rmsnorm_bwd");
    return {dx, dw};
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, double eps) {
        const NormOut o = norm_forward(x, Tensor(), w, eps, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({o.x, w.contiguous(), o.rstd});
        return o.y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
        const auto saved = ctx->get_saved_variables();
        const auto g = norm_backward(saved[0], Tensor(), saved[1], saved[2], grads[0], Tensor(), ctx->needs_input_grad(0), ctx->needs_input_grad(1));
        return once({g[0], g[1], Tensor()}, saved, grads);
    }
};

// bf16: backward reads both addends again (the stored stream h is their rounded sum, which dw would show); fp32: it reads h, which
// is alive anyway as the next block's input
struct RmsNormResidual : torch::autograd::Function<RmsNormResidual> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& r, const Tensor& w, double eps) {
        const NormOut o = norm_forward(x, r, w, eps, true);
        ctx->set_materialize_grads(false);
        const bool both = x.scalar_type() == at::kBFloat16;
        ctx->save_for_backward({both ? o.x : o.h, w.contiguous(), o.rstd, both ? o.r : Tensor()});
        return {o.y, o.h};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const bool need_x = ctx->needs_input_grad(0), need_r = ctx->needs_input_grad(1);
        const auto saved = ctx->get_saved_variables();
        const auto g = norm_backward(saved[0], saved[3], saved[1], saved[2], grads[0], grads[1], need_x || need_r, ctx->needs_input_grad(2));
        return once({need_x ? g[0] : Tensor(), need_r ? g[0] : Tensor(), g[1], Tensor()}, saved, grads);
    }
};

Tensor rms_norm(const Tensor& x, const Tensor& w, double eps) {
    check_norm(x, Tensor(), w, eps);
    on_gpu(x);
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w))) return RmsNorm::apply(x, w, eps);
    return norm_forward(x, Tensor(), w, eps, false).y;
}

std::tuple<Tensor, Tensor> rms_norm_residual(const Tensor& x, const Tensor& r, const Tensor& w, double eps) {
    check_norm(x, r, w, eps);
    on_gpu(x);
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(r) || wants_grad(w))) {
        const auto o = RmsNormResidual::apply(x, r, w, eps);
        return {o[0], o[1]};
    }
    const NormOut o = norm_forward(x, r, w, eps, false);
    return {o.y, o.h};
}

std::tuple<Tensor, Tensor, std::optional<Tensor>> rms_norm_fp8(const Tensor& x, const Tensor& w, const std::optional<Tensor>& residual, double eps) {
    const Tensor r = residual.value_or(Tensor());
    check_norm(x, r, w, eps);
    no_backward("rms_norm_fp8", {&x, &r, &w});
    on_gpu(x);
    const c10::DeviceGuard guard(x.device());
    const Rows xr = as_rows(x);
    const Tensor wc = w.contiguous();
    const int64_t C = w.size(0);
    const auto q = new_rows(x, xr.rows, C);
    Rows rr{Tensor(), 0, 0};
    std::optional<Tensor> h;
    if (r.defined()) { rr = as_rows(r); h = at::empty(x.sizes(), x.options()); }
    check(lib.rmsnorm_fwd_fp8(xr.t.data_ptr(), xr.step, r.defined() ? rr.t.data_ptr() : nullptr, rr.step, wc.data_ptr(), q[0].data_ptr(),
                              q[1].data_ptr<float>(), xr.rows, h ? h->data_ptr() : nullptr, xr.rows, C, (float)eps,
                              code_of(x.scalar_type()), stream_of(x)), "dsw_rmsnorm_fwd_fp8");
    return {q[0], q[1], h};
}

// ---- 8-bit channel mix -----------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> quantize_fp8(const Tensor& x) {
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "expected x [..., C] with C >= 1");
    const int code = code_of(x.scalar_type());
    no_backward("quantize_fp8", {&x});
    on_gpu(x);
    const c10::DeviceGuard guard(x.device());
    const Rows xr = as_rows(x);
    const int64_t C = x.size(-1);
    const auto q = new_rows(x, xr.rows, C);
    check(lib.quant_fp8(xr.t.data_ptr(), xr.step, q[0].data_ptr(), q[1].data_ptr<float>(), xr.rows, xr.rows, C, code, stream_of(x)), "dsw_quant_fp8");
    return {q[0], q[1]};
}

std::tuple<Tensor, Tensor> quantize_fp8_weight(const Tensor& w) {
    TORCH_CHECK_VALUE(w.dim() == 2 && w.numel() > 0, "expected weight [Fin, Fout]");
    const int code = code_of(w.scalar_type());
    no_backward("quantize_fp8_weight", {&w});
    on_gpu(w);
    const c10::DeviceGuard guard(w.device());
    const int64_t fin = w.size(0), fout = w.size(1);
    const Tensor q = at::empty({fout, fin}, w.options().dtype(at::kFloat8_e4m3fn));
    const Tensor s = at::empty({blocks_of(fout), blocks_of(fin)}, w.options().dtype(at::kFloat));
    check(lib.quant_fp8_weight(w.data_ptr(), w.stride(0), w.stride(1), q.data_ptr(), s.data_ptr<float>(), fin, fout, code, stream_of(w)), "dsw_quant_fp8_weight");
    return {q, s};
}

Tensor dense_mix_fp8(const Tensor& xq, const Tensor& xs, const Tensor& wq, const Tensor& ws, const std::optional<Tensor>& bias_, at::ScalarType dtype) {
    const Tensor bias = bias_.value_or(Tensor());
    TORCH_CHECK_TYPE(xq.scalar_type() == at::kFloat8_e4m3fn && wq.scalar_type() == at::kFloat8_e4m3fn, "dsw: 8-bit operands are float8_e4m3fn");
    TORCH_CHECK_TYPE(xs.scalar_type() == at::kFloat && ws.scalar_type() == at::kFloat, "dsw: scales are float32");
    const int code = code_of(dtype);
    TORCH_CHECK_VALUE(xq.dim() >= 1 && wq.dim() == 2 && xq.size(-1) == wq.size(1) && wq.numel() > 0, "expected x.q [..., Fin] and weight.q [Fout, Fin]");
    const int64_t n = wq.size(0), k = wq.size(1);
    TORCH_CHECK_VALUE(xs.dim() == xq.dim() && xs.size(-1) == blocks_of(k) && xs.sizes().slice(0, xs.dim() - 1) == xq.sizes().slice(0, xq.dim() - 1),
                      "expected x.scale [..., ceil(Fin / 128)]");
    TORCH_CHECK_VALUE(ws.dim() == 2 && ws.size(0) == blocks_of(n) && ws.size(1) == blocks_of(k), "expected weight.scale [ceil(Fout / 128), ceil(Fin / 128)]");
    same_device(xq, xs);
    same_device(xq, wq);
    same_device(xq, ws);
    if (bias.defined()) {
        TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == n, "expected bias [Fout]");
        TORCH_CHECK_TYPE(bias.scalar_type() == dtype, "dsw: mixed dtypes ", dtype, " vs ", bias.scalar_type());
        same_device(xq, bias);
    }
    no_backward("dense_mix_fp8", {&xs, &ws, &bias});
    on_gpu(xq);
    const c10::DeviceGuard guard(xq.device());
    constexpr int64_t far = 1 << 23;                   // rows further apart are copied (the tiles use 32-bit offsets)
    const bool w_rows = (k == 1 || wq.stride(1) == 1) && (n == 1 || (wq.stride(0) >= k && wq.stride(0) < far));
    const Tensor w = w_rows ? wq : wq.contiguous();
    Rows x = as_rows(xq);
    if (x.step >= far) x = as_rows(xq.contiguous());
    const Rows s = as_rows(xs, true);
    const Tensor wsc = ws.contiguous(), b = bias.defined() ? bias.contiguous() : bias;
    std::vector<int64_t> sizes(xq.sizes().begin(), xq.sizes().end());
    sizes.back() = n;
    const Tensor y = at::empty(sizes, xq.options().dtype(dtype));
    const int64_t w_step = n == 1 ? k : w.stride(0);
    const auto low = [](const void* p) { return (int64_t)(reinterpret_cast<uintptr_t>(p) & 15); };
    const bool aligned = (low(x.t.data_ptr()) | low(w.data_ptr()) | ((x.step | w_step | k) & 15)) == 0;
    const int64_t bytes = lib.fp8_mix_workspace_bytes(x.rows, n, k, aligned);
    check(bytes, "dsw_fp8_mix_workspace_bytes");
    const Tensor work = bytes ? at::empty({bytes}, xq.options().dtype(at::kByte)) : Tensor();
    check(lib.fp8_mix(x.t.data_ptr(), x.step, s.t.data_ptr<float>(), s.step, s.t.stride(-1), w.data_ptr(), w_step, wsc.data_ptr<float>(),
                      b.defined() ? b.data_ptr() : nullptr, y.data_ptr(), x.rows, n, k, code, bytes ? work.data_ptr() : nullptr, bytes, stream_of(xq)),
          "dsw_fp8_mix");
    return y;
}

// ---- gradients -------------------------------------------------------------------------------------------------------------
// covers consecutive elements of its storage, in some dimension order
bool dense(const Tensor& t) { return t.is_contiguous() || t.is_non_overlapping_and_dense(); }

Tensor grad_norm_clip(std::vector<Tensor> grads, const std::optional<std::vector<Tensor>>& out, double norm_type, double max_norm, bool clip) {
    TORCH_CHECK_VALUE(norm_type == 1.0 || norm_type == 2.0 || norm_type == INFINITY, "norm_type must be 1, 2 or inf");
    TORCH_CHECK_VALUE(!clip || max_norm >= 0.0, "max_norm must be >= 0");
    TORCH_CHECK_VALUE(!grads.empty(), "expected at least one gradient tensor");
    const size_t n = grads.size();
    std::vector<int32_t> types(n);
    const c10::Device dev = grads[0].device();
    for (size_t i = 0; i < n; ++i) {
        types[i] = code_of(grads[i].scalar_type());
        TORCH_CHECK_VALUE(grads[i].device() == dev, "dsw: gradients on more than one device in one call");
    }
    const std::vector<Tensor>& to = out ? *out : grads;
    if (clip) {
        TORCH_CHECK_VALUE(to.size() == n, "expected one `out` tensor for each gradient");
        for (size_t i = 0; i < n; ++i) {
            if (out)
                TORCH_CHECK_VALUE(to[i].sizes() == grads[i].sizes() && to[i].scalar_type() == grads[i].scalar_type() && to[i].device() == dev,
                                  "`out` must have the gradients' shapes, types and device");
            TORCH_CHECK_VALUE(dense(to[i]), "dsw: a clipped tensor must be dense (cover consecutive elements, in any dimension order)");
        }
    }
    std::vector<const Tensor*> all;
    all.reserve(2 * n);
    for (const Tensor& t : grads) all.push_back(&t);
    if (clip && out) for (const Tensor& t : to) all.push_back(&t);
    no_tangent(all);
    if (at::GradMode::is_enabled())
        for (const Tensor* t : all)
            TORCH_CHECK(!wants_grad(*t), "dsw: the gradient norm and the clipping have no backward pass; call them under torch.no_grad() or detach() the tensors");
    on_gpu(grads[0]);
    const c10::DeviceGuard guard(dev);
    const at::AutoGradMode off(false);
    std::vector<const void*> g(n);
    std::vector<void*> o(n);
    std::vector<int64_t> sizes(n);
    std::vector<Tensor> copies;                        // the kernels walk a gradient and its output in memory order
    for (size_t i = 0; i < n; ++i) {
        Tensor t = grads[i];
        if (clip && out && !(t.is_contiguous() && to[i].is_contiguous()) && t.strides() != to[i].strides()) {
            copies.push_back(at::empty_strided(to[i].sizes(), to[i].strides(), to[i].options()).copy_(t));
            t = copies.back();
        } else if (!dense(t)) {
            copies.push_back(t.contiguous());
            t = copies.back();
        }
        g[i] = t.data_ptr();
        o[i] = clip ? to[i].data_ptr() : nullptr;
        sizes[i] = t.numel();
    }
    const Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
    const int64_t bytes = lib.grad_norm_workspace_bytes();
    const Tensor ws = at::empty({bytes}, norm.options().dtype(at::kByte));
    check(lib.grad_norm_clip((int)n, g.data(), clip ? o.data() : nullptr, sizes.data(), types.data(), norm_type, max_norm, norm.data_ptr<float>(),
                             ws.data_ptr(), bytes, stream_of(norm)), "dsw_grad_norm_clip");
    if (clip) for (const Tensor& t : to) if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();   // (written behind autograd's back)
    return norm;
}

}  // namespace

PYBIND11_MODULE(_dsw_torch, m) {
    m.def("bind", &bind);
    m.def("as_rows", [](const Tensor& t, bool any_last) { const Rows r = as_rows(t, any_last); return std::make_tuple(r.t, r.rows, r.step); });
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_residual", &rms_norm_residual);
    m.def("rms_norm_fp8", &rms_norm_fp8);
    m.def("quantize_fp8", &quantize_fp8);
    m.def("quantize_fp8_weight", &quantize_fp8_weight);
    m.def("dense_mix_fp8", &dense_mix_fp8);
    m.def("grad_norm_clip", &grad_norm_clip);
}
