// torch binding of the optimizer operators and of the residual norm (module _scx_torch): what their
// calls spend on the host is walking lists of tensors and building an autograd node, which takes
// tens of microseconds in Python and about one per ten tensors here.  The work is libscx.so's C ABI
// (include/scx.h); everything else of the package binds to it with ctypes.
//
// A failed check raises RuntimeError (TORCH_CHECK).
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <vector>

#include "scx.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Tensors = std::vector<Tensor>;

void check_status(int status, const char* what) {
    TORCH_CHECK(status == 0, what, " failed with CUDA status ", status, " (", scx_status_string(status), ")");
}

scx_stream_t stream_of(const at::Device& device) { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }

// A block of its own per call: calls on other streams and captured graphs share nothing.
Tensor workspace(size_t bytes, const at::Device& device) {
    return at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(device));
}

Tensor scalar(const at::Device& device) { return at::empty({}, at::TensorOptions().dtype(at::kFloat).device(device)); }

// Element type code of scx.h, -1 for others; complex64 counts as two float32 per element.
int code_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat:
        case at::kComplexFloat: return SCX_FLOAT32;
        case at::kBFloat16: return SCX_BFLOAT16;
        case at::kHalf: return SCX_FLOAT16;
        default: return -1;
    }
}

// Forward-mode derivatives do not pass through the kernels, and a tangent left out reads as zero.
void check_no_tangent(const Tensor& t, const char* name) {
    TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), name, " must not carry a tangent: there is no forward-mode derivative");
}

// A trace would record the outputs' allocation and not the kernels that fill them.
void check_not_traced() { TORCH_CHECK(!torch::jit::tracer::isTracing(), "the call cannot be traced"); }

at::Device check_tensors(const Tensors& tensors, const char* name) {
    check_not_traced();
    const at::Device device = tensors[0].device();
    for (const Tensor& t : tensors) {
        TORCH_CHECK(t.is_cuda(), name, " must be CUDA tensors");
        TORCH_CHECK(t.layout() == at::kStrided, name, " must not be sparse");
        TORCH_CHECK(code_of(t.scalar_type()) >= 0, name, " must be float32, bfloat16, float16 or complex64, got ",
                    t.scalar_type());
        TORCH_CHECK(t.device() == device, name, " must be on one device");
        check_no_tangent(t, name);
    }
    return device;
}

// Whether the elements of t fill one run of memory, in whatever order, each once.
bool dense(const Tensor& t) { return t.is_non_overlapping_and_dense(); }

bool overlaps_itself(const Tensor& t) {
    std::vector<std::pair<int64_t, int64_t>> axes;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) axes.emplace_back(t.stride(i), t.size(i));
    std::sort(axes.begin(), axes.end());
    int64_t reach = 0;
    for (const auto& [stride, size] : axes) {
        if (stride <= reach) return true;
        reach += stride * (size - 1);
    }
    return false;
}

// Tells autograd (and whoever caches by version) that the kernels wrote these tensors.
void changed(const Tensors& tensors) {
    for (const Tensor& t : tensors)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

template <typename P>
std::vector<P> pointers(const Tensors& tensors) {
    std::vector<P> p;
    p.reserve(tensors.size());
    for (const Tensor& t : tensors) p.push_back(static_cast<P>(t.data_ptr()));
    return p;
}

struct Described {
    std::vector<long long> counts;
    std::vector<int> types;
    explicit Described(const Tensors& tensors) {
        counts.reserve(tensors.size());
        types.reserve(tensors.size());
        for (const Tensor& t : tensors) {
            counts.push_back(t.numel() * (t.is_complex() ? 2 : 1));
            types.push_back(code_of(t.scalar_type()));
        }
    }
};

Tensor run_norm(at::TensorList tensors) {
    const at::Device device = tensors[0].device();
    Tensors flat = tensors.vec();
    for (Tensor& t : flat)
        if (!dense(t)) t = t.contiguous();
    const c10::cuda::CUDAGuard guard(device);
    const int n = static_cast<int>(flat.size());
    const size_t bytes = scx_grad_norm_workspace_size(n);
    const Tensor ws = workspace(bytes, device), norm = scalar(device);
    const Described d(flat);
    check_status(scx_grad_norm(n, pointers<const void*>(flat).data(), d.counts.data(), d.types.data(),
                               static_cast<float*>(norm.data_ptr()), ws.data_ptr(), bytes, stream_of(device)),
                 "scx_grad_norm");
    return norm;
}

// dN/dg = g / N (zero where N is), in torch operations, so that it can be differentiated again.  A norm that is
// differentiated is part of a loss (a penalty on gradients), not of the training step that the kernels are for.
struct GradNorm : torch::autograd::Function<GradNorm> {
    static Tensor forward(AutogradContext* ctx, at::TensorList tensors) {
        const Tensor norm = run_norm(tensors);
        variable_list saved = tensors.vec();
        saved.push_back(norm);
        ctx->save_for_backward(std::move(saved));
        return norm;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list saved = ctx->get_saved_variables();
        const Tensor norm = saved.back();
        saved.pop_back();
        variable_list result(saved.size());
        if (!grads[0].defined()) return result;
        const Tensor factor = grads[0] / norm.masked_fill(norm == 0, 1.0);
        for (size_t i = 0; i < saved.size(); ++i) {
            if (!ctx->needs_input_grad(i)) continue;
            const at::ScalarType type = saved[i].scalar_type();
            const bool narrow = type == at::kBFloat16 || type == at::kHalf;  // rounded once, behind the product
            result[i] = narrow ? (saved[i].to(at::kFloat) * factor).to(type) : saved[i] * factor;
        }
        return result;
    }
};

Tensor grad_norm(const Tensors& tensors) {
    check_tensors(tensors, "tensors");
    bool wanted = false;
    for (const Tensor& t : tensors) wanted = wanted || t.requires_grad();
    return wanted && at::GradMode::is_enabled() ? GradNorm::apply(at::TensorList(tensors)) : run_norm(tensors);
}

Tensor clip_grads(const Tensors& grads, double max_norm) {
    const at::NoGradGuard no_grad;
    const at::Device device = check_tensors(grads, "grads");
    Tensors flat = grads;
    for (Tensor& t : flat) {
        if (dense(t)) continue;
        TORCH_CHECK(!overlaps_itself(t), "grads must not be expanded tensors");
        t = t.contiguous();
    }
    const c10::cuda::CUDAGuard guard(device);
    const int n = static_cast<int>(flat.size());
    const size_t bytes = scx_grad_norm_workspace_size(n);
    const Tensor ws = workspace(bytes, device), norm = scalar(device);
    const Described d(flat);
    check_status(scx_grad_clip(n, pointers<void*>(flat).data(), d.counts.data(), d.types.data(), max_norm,
                               static_cast<float*>(norm.data_ptr()), ws.data_ptr(), bytes, stream_of(device)),
                 "scx_grad_clip");
    for (size_t i = 0; i < grads.size(); ++i)
        if (!flat[i].is_same(grads[i])) grads[i].copy_(flat[i]);
    changed(grads);
    return norm;
}

// Whether t has its elements where p has them.
bool same_layout(const Tensor& t, const Tensor& p) {
    if (t.is_contiguous() && p.is_contiguous()) return true;
    for (int64_t i = 0; i < p.dim(); ++i)
        if (p.size(i) > 1 && t.stride(i) != p.stride(i)) return false;
    return true;
}

std::optional<Tensor> adam_step(const Tensors& params, const Tensors& given_grads, const Tensors& exp_avgs,
                                const Tensors& exp_avg_sqs, const Tensors& steps, double lr,
                                const std::optional<Tensor>& lr_tensor, double beta1, double beta2, double eps,
                                double weight_decay, bool decoupled, std::optional<double> max_norm,
                                const std::optional<Tensor>& total_norm) {
    const at::NoGradGuard no_grad;
    const at::Device device = check_tensors(params, "params");
    const size_t n = params.size();
    auto one_value = [&](const Tensor& t) {
        return t.scalar_type() == at::kFloat && t.numel() == 1 && t.device() == device;
    };
    TORCH_CHECK(!lr_tensor || one_value(*lr_tensor), "lr must be a number or one float32 value on the params' device");
    TORCH_CHECK(!total_norm || one_value(*total_norm), "total_norm must be one float32 value on the params' device");
    Tensors grads = given_grads;
    for (size_t i = 0; i < n; ++i) {
        const Tensor &p = params[i], &m = exp_avgs[i], &v = exp_avg_sqs[i], &t = steps[i];
        Tensor& g = grads[i];
        TORCH_CHECK(g.scalar_type() == p.scalar_type() && g.sizes() == p.sizes() && g.layout() == at::kStrided,
                    "a gradient must have its parameter's type and shape");
        const at::ScalarType kind = p.is_complex() ? at::kComplexFloat : at::kFloat;
        TORCH_CHECK(m.scalar_type() == kind && v.scalar_type() == kind && m.sizes() == p.sizes() && v.sizes() == p.sizes(),
                    "moments must be float32 (complex64 for a complex parameter), of their parameter's shape");
        TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == 1, "steps must be single float32 values");
        TORCH_CHECK(g.device() == device && m.device() == device && v.device() == device && t.device() == device,
                    "gradients, moments and steps must be on the params' device");
        check_no_tangent(g, "gradients");
        check_no_tangent(m, "moments");
        check_no_tangent(v, "moments");
        check_no_tangent(t, "steps");
        TORCH_CHECK(!p.is_conj() && !m.is_conj() && !v.is_conj(), "params and moments must not be conjugate views");
        TORCH_CHECK(!p.is_neg() && !m.is_neg() && !v.is_neg(), "params and moments must not be negated views");
        TORCH_CHECK(dense(p) && same_layout(m, p) && same_layout(v, p),
                    "params must be dense, and moments of their params' strides");
        if (g.is_conj() || g.is_neg() || !same_layout(g, p)) g = at::empty_like(p).copy_(g);
    }
    const c10::cuda::CUDAGuard guard(device);
    const size_t bytes = scx_adam_workspace_size(static_cast<int>(n));
    const Tensor ws = workspace(bytes, device);
    std::optional<Tensor> norm;
    if (max_norm && !total_norm) norm = scalar(device);
    const Described d(params);
    check_status(
        scx_adam_step(static_cast<int>(n), pointers<void*>(params).data(), pointers<const void*>(grads).data(),
                      pointers<float*>(exp_avgs).data(), pointers<float*>(exp_avg_sqs).data(),
                      pointers<float*>(steps).data(), d.counts.data(), d.types.data(), lr,
                      lr_tensor ? static_cast<const float*>(lr_tensor->data_ptr()) : nullptr, beta1, beta2, eps,
                      weight_decay, decoupled, max_norm.value_or(0.0),
                      total_norm ? static_cast<const float*>(total_norm->data_ptr()) : nullptr,
                      norm ? static_cast<float*>(norm->data_ptr()) : nullptr, ws.data_ptr(), bytes, stream_of(device)),
        "scx_adam_step");
    changed(params);
    changed(exp_avgs);
    changed(exp_avg_sqs);
    changed(steps);
    return total_norm ? total_norm : norm;
}

// ---------------------------------------------------------------------------- residual norm

// batch, length, channels, channels_last, dtype, weight_dtype, kind, gate_mode, gate_act, post_norm, pre_norm
using Options = std::vector<int64_t>;

scx_residual_norm_config config_of(const Options& o, double eps, double scale) {
    TORCH_CHECK(o.size() == 11, "residual_norm takes 11 options, got ", o.size());
    scx_residual_norm_config c = {};
    c.batch = o[0];
    c.length = o[1];
    c.channels = static_cast<int>(o[2]);
    c.channels_last = static_cast<int>(o[3]);
    c.dtype = static_cast<int>(o[4]);
    c.weight_dtype = static_cast<int>(o[5]);
    c.kind = static_cast<int>(o[6]);
    c.gate_mode = static_cast<int>(o[7]);
    c.gate_act = static_cast<int>(o[8]);
    c.post_norm = static_cast<int>(o[9]);
    c.pre_norm = static_cast<int>(o[10]);
    c.eps = static_cast<float>(eps);
    c.scale = static_cast<float>(scale);
    return c;
}

const void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// x, y, gate, post_weight, post_bias, pre_weight, pre_bias, scale; undefined where there is none.
constexpr size_t kInputs = 8;

scx_residual_norm_tensors tensors_of(const variable_list& in) {
    return {data(in[0]), data(in[1]), data(in[2]), data(in[3]), data(in[4]), data(in[5]),
            data(in[6]), data(in[7]), nullptr,     nullptr,     nullptr};
}

// t with its values in memory as they read: in one run, and not behind a negation bit (contiguous() leaves that).
Tensor plain(const Tensor& t) { return t.resolve_neg().contiguous(); }

struct Forward {
    Tensor r, n, stats;
};

Forward run_forward(const scx_residual_norm_config& c, const variable_list& in, bool keep_stats) {
    const Tensor& x = in[0];
    const c10::cuda::CUDAGuard guard(x.device());
    Forward f;
    if (in[1].defined()) f.r = at::empty_like(x);
    if (c.pre_norm) f.n = at::empty_like(x);
    if (keep_stats) f.stats = at::empty({c.batch * c.length, 4}, x.options().dtype(at::kFloat));
    scx_residual_norm_tensors t = tensors_of(in);
    t.r = out(f.r);
    t.n = out(f.n);
    t.stats = static_cast<float*>(out(f.stats));
    check_status(scx_residual_norm_fwd(&c, &t, stream_of(x.device())), "scx_residual_norm_fwd");
    return f;
}

// Stands for an input that is not there: autograd's node wants a defined tensor in every place.
const Tensor& nothing() {
    static const Tensor* const t = new Tensor(at::empty({0}));  // never freed: outlives the module's teardown
    return *t;
}

// Keeps the inputs and four statistics per position; r is recomputed in the backward.
struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const Options& options, double eps, double scale, Tensor x,
                                 Tensor y, Tensor gate, Tensor post_w, Tensor post_b, Tensor pre_w, Tensor pre_b,
                                 Tensor scale_w) {
        const scx_residual_norm_config c = config_of(options, eps, scale);
        variable_list in = {x, y, gate, post_w, post_b, pre_w, pre_b, scale_w};
        for (Tensor& t : in)
            if (t.is_same(nothing())) t = Tensor();
        const bool block = in[1].defined();
        const Forward f = run_forward(c, in, true);
        ctx->saved_data["options"] = options;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["scale"] = scale;
        in.push_back(f.stats);
        ctx->save_for_backward(std::move(in));
        ctx->set_materialize_grads(false);
        // without y, r is x: returned from here so that its gradient joins n's before the rounding
        variable_list outs = {block ? f.r : x};
        if (c.pre_norm) outs.push_back(f.n);
        return outs;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        constexpr size_t kBefore = 3;  // the arguments that are not tensors
        variable_list result(kBefore + kInputs);
        variable_list saved = ctx->get_saved_variables();
        const Tensor stats = saved.back();
        saved.pop_back();
        const Tensor& x = saved[0];
        Tensor dr = grads[0], dn = grads.size() > 1 ? grads[1] : Tensor();
        if (!dr.defined() && !dn.defined()) return result;
        bool again = false;
        if (at::GradMode::is_enabled())
            for (const variable_list& list : {saved, variable_list{dr, dn}})
                for (const Tensor& t : list) again = again || (t.defined() && t.requires_grad());
        {
            const at::NoGradGuard no_grad;
            for (size_t i = 0; i < kInputs; ++i)
                if (saved[i].defined() && ctx->needs_input_grad(i))
                    result[kBefore + i] = x.numel() ? at::empty_like(saved[i]) : at::zeros_like(saved[i]);
            if (x.numel()) {
                const c10::cuda::CUDAGuard guard(x.device());
                if (dr.defined()) dr = plain(dr);
                if (dn.defined()) dn = plain(dn);
                const scx_residual_norm_config c =
                    config_of(ctx->saved_data["options"].toIntVector(), ctx->saved_data["eps"].toDouble(),
                              ctx->saved_data["scale"].toDouble());
                const size_t bytes = scx_residual_norm_bwd_workspace_size(&c);
                const Tensor ws = workspace(bytes, x.device());
                scx_residual_norm_tensors t = tensors_of(saved);
                t.stats = static_cast<float*>(out(stats));
                const Tensor* g = &result[kBefore];
                const scx_residual_norm_grads grads_of = {data(dr),  data(dn),  out(g[0]), out(g[1]), out(g[2]),
                                                          out(g[3]), out(g[4]), out(g[5]), out(g[6]), out(g[7])};
                check_status(scx_residual_norm_bwd(&c, &t, &grads_of, ws.data_ptr(), bytes, stream_of(x.device())),
                             "scx_residual_norm_bwd");
            }
        }
        if (again) {  // a graph through this backward ends in an error, not in silence
            variable_list made;
            for (const Tensor& t : result)
                if (t.defined()) made.push_back(t.detach().requires_grad_(true));
            const auto error = std::make_shared<torch::autograd::DelayedError>(
                "residual_norm is differentiable once only", static_cast<int64_t>(made.size()));
            made = (*error)(std::move(made));
            size_t k = 0;
            for (Tensor& t : result)
                if (t.defined()) t = made[k++];
        }
        return result;
    }
};

using MaybeTensor = std::optional<Tensor>;

// (r, n) of contiguous inputs that the caller has checked.
std::pair<MaybeTensor, MaybeTensor> residual_norm(const Options& options, double eps, double scale, const Tensor& x,
                                                  const MaybeTensor& y, const MaybeTensor& gate,
                                                  const MaybeTensor& post_w, const MaybeTensor& post_b,
                                                  const MaybeTensor& pre_w, const MaybeTensor& pre_b,
                                                  const MaybeTensor& scale_w) {
    check_not_traced();
    variable_list in = {x};
    for (const MaybeTensor* t : {&y, &gate, &post_w, &post_b, &pre_w, &pre_b, &scale_w}) in.push_back(t->value_or(Tensor()));
    bool wanted = false;
    for (Tensor& t : in) {
        if (!t.defined()) continue;
        check_no_tangent(t, "inputs of residual_norm");
        t = plain(t);
        wanted = wanted || t.requires_grad();
    }
    if (wanted && at::GradMode::is_enabled()) {
        for (Tensor& t : in)
            if (!t.defined()) t = nothing();
        const variable_list outs =
            ResidualNorm::apply(options, eps, scale, in[0], in[1], in[2], in[3], in[4], in[5], in[6], in[7]);
        return {outs[0], outs.size() > 1 ? MaybeTensor(outs[1]) : std::nullopt};
    }
    const scx_residual_norm_config c = config_of(options, eps, scale);
    const Forward f = run_forward(c, in, false);
    return {f.r.defined() ? MaybeTensor(f.r) : MaybeTensor(x), f.n.defined() ? MaybeTensor(f.n) : std::nullopt};
}

}  // namespace

PYBIND11_MODULE(_scx_torch, m) {
    using release = pybind11::call_guard<pybind11::gil_scoped_release>;
    m.def("dense", &dense);
    m.def("overlaps_itself", &overlaps_itself);
    m.def("grad_norm", &grad_norm, release());
    m.def("clip_grads", &clip_grads, release());
    m.def("adam_step", &adam_step, release());
    m.def("residual_norm", &residual_norm, release());
}
