// torch binding of the sequence operators (pointcloud_rl_amd/sequence.py): argument checks, outputs and scratch from torch's allocator, autograd
// nodes.  In C++ because these calls are short: a step of an acting agent is 3 us of kernel, and a Python autograd function costs tens of
// microseconds in the engine's thread.  The kernels are reached through the C ABI of libpcrl_hip.so, whose entry points are handed in as
// addresses by the ctypes binding (_lib.py) -- this file links neither against that library nor against a HIP runtime of its own.
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>

#include <map>
#include <string>

#include "pcrl.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Opt;

struct Api {
    decltype(&pcrl_last_error) last_error = nullptr;
    decltype(&pcrl_short_conv_fwd) conv_fwd = nullptr;
    decltype(&pcrl_short_conv_bwd_workspace_bytes) conv_bwd_bytes = nullptr;
    decltype(&pcrl_short_conv_bwd) conv_bwd = nullptr;
    decltype(&pcrl_ssm_scan_bytes) scan_bytes = nullptr;
    decltype(&pcrl_ssm_scan_fwd) scan_fwd = nullptr;
    decltype(&pcrl_ssm_scan_bwd) scan_bwd = nullptr;
    decltype(&pcrl_ssm_step) step = nullptr;
    decltype(&pcrl_dropout) dropout = nullptr;
} api;

void bind(const std::map<std::string, uintptr_t>& at) {
    auto get = [&](const char* name) { return at.at(name); };
    api.last_error = (decltype(api.last_error))get("pcrl_last_error");
    api.conv_fwd = (decltype(api.conv_fwd))get("pcrl_short_conv_fwd");
    api.conv_bwd_bytes = (decltype(api.conv_bwd_bytes))get("pcrl_short_conv_bwd_workspace_bytes");
    api.conv_bwd = (decltype(api.conv_bwd))get("pcrl_short_conv_bwd");
    api.scan_bytes = (decltype(api.scan_bytes))get("pcrl_ssm_scan_bytes");
    api.scan_fwd = (decltype(api.scan_fwd))get("pcrl_ssm_scan_fwd");
    api.scan_bwd = (decltype(api.scan_bwd))get("pcrl_ssm_scan_bwd");
    api.step = (decltype(api.step))get("pcrl_ssm_step");
    api.dropout = (decltype(api.dropout))get("pcrl_dropout");
}

void check(int rc) { TORCH_CHECK(rc == 0, "pcrl error ", rc, ": ", api.last_error()); }

// The current stream of the tensors' device, made the current device for the launch.
struct On {
    c10::OptionalDeviceGuard guard;
    void* stream;
    explicit On(const Tensor& t) : guard(t.device()), stream((void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream()) {}
};

Tensor val(const Opt& t) { return t.has_value() ? *t : Tensor(); }
Opt opt(const Tensor& t) { return t.defined() ? Opt(t) : Opt(); }      // (the engine takes no undefined tensors as a node's inputs)
const void* at_(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* to_(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const float* fat(const Tensor& t) { return (const float*)at_(t); }

int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return PCRL_DT_F32;
        case at::kBFloat16: return PCRL_DT_BF16;
        case at::kHalf: return PCRL_DT_F16;
        default: TORCH_CHECK_VALUE(false, "activations are float32, bfloat16 or float16, not ", t.scalar_type());
    }
}
void on_gpu(const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "the sequence operators run on the MI355X (got a tensor on ", t.device(), "); there is no CPU path");
}

// t against a shape and the type and device of `like`; channels made adjacent, step strides within what the kernels' offsets reach.
Tensor activation(const char* name, const Tensor& t, at::IntArrayRef shape, const Tensor& like) {
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " is ", t.sizes(), ", expected ", shape);
    TORCH_CHECK_VALUE(t.scalar_type() == like.scalar_type() && t.device() == like.device(), name, " is ", t.scalar_type(), " on ", t.device(),
                      ", the sequence is ", like.scalar_type(), " on ", like.device());
    return t;
}
Tensor adjacent(const Tensor& t, int batch_and_step) {
    bool ok = t.stride(-1) == 1;
    for (int i = 0; i < batch_and_step; ++i) ok = ok && t.stride(i) >= 0 && (i == 0 || t.stride(i) < (1 << 26));
    return ok ? t : t.contiguous();
}
Tensor parameter(const char* name, const Tensor& t, at::IntArrayRef shape, const Tensor& like) {
    TORCH_CHECK_VALUE(t.sizes() == shape, name, " is ", t.sizes(), ", expected ", shape);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.device() == like.device(), name, " is ", t.scalar_type(), " on ", t.device(), ", expected float32 on ", like.device());
    return t.contiguous();
}
Tensor starts_of(const Opt& starts, at::IntArrayRef rows, const Tensor& like) {
    if (!starts.has_value()) return Tensor();
    TORCH_CHECK_VALUE(starts->sizes() == rows && (starts->scalar_type() == at::kBool || starts->scalar_type() == at::kByte) && starts->device() == like.device(),
                      "starts is ", starts->scalar_type(), " ", starts->sizes(), " on ", starts->device(), ", expected bool ", rows, " on ", like.device());
    return starts->contiguous();
}
Tensor lengths_of(const Opt& lengths, int64_t rows, int64_t steps, const Tensor& like) {
    if (!lengths.has_value()) return Tensor();
    TORCH_CHECK_VALUE(lengths->dim() == 1 && lengths->size(0) == rows && (lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong) && lengths->device() == like.device(),
                      "lengths is ", lengths->scalar_type(), " ", lengths->sizes(), " on ", lengths->device(), ", expected int32 [", rows, "] on ", like.device());
    return lengths->scalar_type() == at::kInt ? lengths->contiguous() : lengths->clamp(0, steps).to(at::kInt);
}
// Stride between steps; 0 where there is only one (a view's stride over an axis of one element may be anything).
int64_t step_stride(const Tensor& t) { return t.size(1) == 1 ? 0 : t.stride(1); }
bool wants_grad(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : ts) if (t.defined() && t.requires_grad()) return true;
    return false;
}
// The kernels carry no tangents: a forward-mode derivative through them would come out as zero.
void no_tangents(std::initializer_list<Tensor> ts) {
    for (const Tensor& t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), "the sequence operators have no forward-mode derivatives (an input is a dual tensor)");
}
// The gradient of an output that may take no part in the loss: zeros that are one row in memory.
Tensor full_grad(const Tensor& g, const Tensor& like) {
    if (!g.defined()) return at::zeros({like.size(-1)}, like.options()).expand(like.sizes());
    return adjacent(g, 2);
}
Tensor twin(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options().requires_grad(false)) : Tensor(); }
void once() { TORCH_CHECK(!at::GradMode::is_enabled(), "the sequence operators are differentiable once (create_graph=True is not supported)"); }
int fits(const char* name, int64_t n) {
    TORCH_CHECK_VALUE(n <= 0x7FFFFFFF, name, " = ", n, " is too large");
    return (int)n;
}

// ---- short convolution -------------------------------------------------------------------------------------------------------------------
pcrl_conv_desc conv_desc(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& state, const Tensor& starts, const Tensor& lengths, bool silu) {
    pcrl_conv_desc d{};
    const bool step = x.dim() == 2;
    d.B = fits("batch", x.size(0)), d.T = step ? 1 : fits("steps", x.size(1)), d.D = fits("channels", x.size(-1)), d.W = (int)weight.size(1);
    d.dtype = dtype_code(x), d.silu = silu;
    d.x = at_(x), d.x_sb = x.stride(0), d.x_st = step ? 0 : step_stride(x);
    d.weight = fat(weight), d.bias = fat(bias), d.state = at_(state);
    d.starts = (const uint8_t*)at_(starts), d.starts_sb = d.T, d.lengths = (const int32_t*)at_(lengths);
    return d;
}
variable_list conv_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& state, const Tensor& starts, const Tensor& lengths, bool silu) {
    Tensor y = at::empty(x.sizes(), x.options().requires_grad(false));
    Tensor last = at::empty({x.size(0), weight.size(1) - 1, x.size(2)}, y.options());
    if (y.numel()) {
        On on(x);
        const pcrl_conv_desc d = conv_desc(x, weight, bias, state, starts, lengths, silu);
        check(api.conv_fwd(&d, to_(y), to_(last), on.stream));
    } else if (state.defined()) last.copy_(state);
    else last.zero_();
    return {y, last};
}
struct ConvNode : Function<ConvNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Opt& bias, const Opt& state, const Opt& starts,
                                 const Opt& lengths, bool silu) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, weight, val(bias), val(state), val(starts), val(lengths)});
        ctx->saved_data["silu"] = silu;
        return conv_forward(x, weight, val(bias), val(state), val(starts), val(lengths), silu);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once();
        const Tensor dy_ = grads[0], dlast_ = grads[1];
        if (!dy_.defined() && !dlast_.defined()) return variable_list(7);
        const auto s = ctx->get_saved_variables();
        const Tensor &x = s[0], &weight = s[1], &bias = s[2], &state = s[3];
        Tensor dx = twin(x), dweight = twin(weight), dbias = twin(bias), dstate = twin(state);
        const Tensor dy = full_grad(dy_, x), dlast = dlast_.defined() ? dlast_.contiguous() : dlast_;
        if (x.numel()) {
            On on(x);
            const pcrl_conv_desc d = conv_desc(x, weight, bias, state, s[4], s[5], ctx->saved_data["silu"].toBool());
            size_t need = 0;
            check(api.conv_bwd_bytes(&d, &need));
            const Tensor work = at::empty({(int64_t)need}, dx.options().dtype(at::kByte));
            check(api.conv_bwd(&d, at_(dy), dy.stride(0), step_stride(dy), at_(dlast), to_(dx), (float*)to_(dweight), (float*)to_(dbias), to_(dstate), to_(work), need, on.stream));
        } else {                                                // no step: the state passes through
            dweight.zero_();
            if (dbias.defined()) dbias.zero_();
            if (dstate.defined()) { if (dlast.defined()) dstate.copy_(dlast); else dstate.zero_(); }
        }
        return {dx, dweight, dbias, dstate, Tensor(), Tensor(), Tensor()};
    }
};

struct ConvArgs { Tensor x, weight, bias, state, starts, lengths; bool silu; };
ConvArgs conv_args(const Tensor& x, const Tensor& weight, const Opt& bias, const Opt& state, const Opt& starts, const Opt& lengths, const std::optional<std::string>& act, int dims) {
    TORCH_CHECK_VALUE(x.dim() == dims, "x is ", x.sizes(), dims == 2 ? ", expected [B, D]" : ", expected [B, T, D]");
    dtype_code(x);
    TORCH_CHECK_VALUE(!act.has_value() || *act == "silu", "activation '", act.value_or(""), "': None or 'silu'");
    const int64_t D = x.size(-1);
    TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(1) >= 1 && weight.size(1) <= 4, "weight is ", weight.sizes(), ", expected [", D, ", W] with 1 to 4 taps");
    ConvArgs a;
    a.x = adjacent(x, dims - 1);
    a.weight = parameter("weight", weight, {D, weight.size(1)}, x);
    if (bias.has_value()) a.bias = parameter("bias", *bias, {D}, x);
    if (state.has_value()) a.state = activation("state", *state, {x.size(0), weight.size(1) - 1, D}, x);
    a.starts = starts_of(starts, x.sizes().slice(0, dims - 1), x);
    a.lengths = lengths_of(lengths, x.size(0), dims == 3 ? x.size(1) : 1, x);
    a.silu = act.has_value();
    return a;
}
// Where a step leaves the new state: `state` itself, or a tensor that does not overlap it.
Tensor state_out_of(const Tensor& state, const Opt& out) {
    TORCH_CHECK_VALUE(state.is_contiguous(), "the state of a step must be contiguous (it is updated in place)");
    if (!out.has_value()) return state;
    TORCH_CHECK_VALUE(out->sizes() == state.sizes() && out->scalar_type() == state.scalar_type() && out->device() == state.device() && out->is_contiguous(),
                      "state_out is ", out->scalar_type(), " ", out->sizes(), " on ", out->device(), ", expected a contiguous twin of the state");
    const char *a = (const char*)at_(state), *b = (const char*)at_(*out);
    TORCH_CHECK_VALUE(a == b || a + state.nbytes() <= b || b + out->nbytes() <= a, "state_out overlaps the state");
    return *out;
}

// A graph that saved the old state must not be differentiated with the new one in its place.
void written(const Tensor& t) { if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); }

std::tuple<Tensor, Tensor> short_conv(const Tensor& x, const Tensor& weight, const Opt& bias, const Opt& state, const Opt& starts, const Opt& lengths,
                                      const std::optional<std::string>& act) {
    ConvArgs a = conv_args(x, weight, bias, state, starts, lengths, act, 3);
    no_tangents({a.x, a.weight, a.bias, a.state});
    on_gpu(x);
    if (a.state.defined()) a.state = a.state.contiguous();
    const variable_list r = wants_grad({a.x, a.weight, a.bias, a.state}) ? ConvNode::apply(a.x, a.weight, opt(a.bias), opt(a.state), opt(a.starts), opt(a.lengths), a.silu)
                                                                        : conv_forward(a.x, a.weight, a.bias, a.state, a.starts, a.lengths, a.silu);
    return {r[0], r[1]};
}
Tensor short_conv_step(const Tensor& x, const Opt& state, const Tensor& weight, const Opt& bias, const Opt& starts, const std::optional<std::string>& act, const Opt& state_out) {
    at::NoGradGuard no_grad;
    TORCH_CHECK_VALUE(state.has_value(), "a step needs a state");
    const ConvArgs a = conv_args(x, weight, bias, state, starts, std::nullopt, act, 2);
    no_tangents({a.x, a.weight, a.bias, a.state});
    const Tensor out = state_out_of(a.state, state_out);
    on_gpu(x);
    Tensor y = at::empty(x.sizes(), x.options().requires_grad(false));
    if (y.numel()) {
        On on(x);
        const pcrl_conv_desc d = conv_desc(a.x, a.weight, a.bias, a.state, a.starts, Tensor(), a.silu);
        check(api.conv_fwd(&d, to_(y), to_(out), on.stream));
    }
    written(out);
    return y;
}

// ---- selective scan ------------------------------------------------------------------------------------------------------------------------
struct ScanArgs { Tensor u, dt, A, B, C, D, z, dt_bias, state, starts, lengths; bool softplus; };

pcrl_ssm_desc scan_desc(const ScanArgs& a) {
    pcrl_ssm_desc d{};
    const bool step = a.u.dim() == 2;
    d.B = fits("batch", a.u.size(0)), d.T = step ? 1 : fits("steps", a.u.size(1)), d.D = fits("channels", a.u.size(-1)), d.N = (int)a.A.size(1);
    d.G = fits("groups", a.B.size(-2)), d.dtype = dtype_code(a.u), d.softplus = a.softplus;
    auto st = [&](const Tensor& t) { return step ? 0 : step_stride(t); };
    d.u = at_(a.u), d.dt = at_(a.dt), d.z = at_(a.z), d.Bm = at_(a.B), d.Cm = at_(a.C);
    d.u_sb = a.u.stride(0), d.u_st = st(a.u), d.dt_sb = a.dt.stride(0), d.dt_st = st(a.dt);
    if (a.z.defined()) d.z_sb = a.z.stride(0), d.z_st = st(a.z);
    d.b_sb = a.B.stride(0), d.b_st = st(a.B), d.b_sg = a.B.stride(-2), d.c_sb = a.C.stride(0), d.c_st = st(a.C), d.c_sg = a.C.stride(-2);
    d.A = fat(a.A), d.D_skip = fat(a.D), d.dt_bias = fat(a.dt_bias), d.state = fat(a.state);
    d.starts = (const uint8_t*)at_(a.starts), d.starts_sb = d.T, d.lengths = (const int32_t*)at_(a.lengths);
    return d;
}
// {y, last state, states kept for a backward (undefined without `keep`)} and the size of the backward's workspace
variable_list scan_forward(const ScanArgs& a, bool keep, int64_t& bwd_bytes) {
    Tensor y = at::empty(a.u.sizes(), a.u.options().requires_grad(false)), kept;
    Tensor last = at::empty({a.u.size(0), a.u.size(2), a.A.size(1)}, y.options().dtype(at::kFloat));
    bwd_bytes = 0;
    if (!y.numel()) {
        if (a.state.defined()) last.copy_(a.state);
        else last.zero_();
        return {y, last, kept};
    }
    On on(a.u);
    const pcrl_ssm_desc d = scan_desc(a);
    size_t need = 0, saved = 0, bwd = 0;
    check(api.scan_bytes(&d, &need, &saved, &bwd));
    bwd_bytes = (int64_t)bwd;
    Tensor work;
    if (need) work = at::empty({(int64_t)need}, y.options().dtype(at::kByte));
    if (keep) kept = at::empty({(int64_t)(saved / 4)}, last.options());
    check(api.scan_fwd(&d, to_(y), (float*)to_(last), (float*)to_(kept), to_(work), need, on.stream));
    return {y, last, kept};
}
struct ScanNode : Function<ScanNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D, const Opt& z,
                                 const Opt& dt_bias, const Opt& state, const Opt& starts, const Opt& lengths, bool softplus) {
        ctx->set_materialize_grads(false);
        int64_t bytes = 0;
        const ScanArgs a{u, dt, A, B, C, val(D), val(z), val(dt_bias), val(state), val(starts), val(lengths), softplus};
        variable_list r = scan_forward(a, true, bytes);
        ctx->save_for_backward({u, dt, A, B, C, a.D, a.z, a.dt_bias, a.state, a.starts, a.lengths, r[2]});
        ctx->saved_data["softplus"] = softplus;
        ctx->saved_data["bytes"] = bytes;
        r.pop_back();
        return r;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once();
        const Tensor dy_ = grads[0], dlast_ = grads[1];
        if (!dy_.defined() && !dlast_.defined()) return variable_list(12);
        const auto s = ctx->get_saved_variables();
        const ScanArgs a{s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], s[10], ctx->saved_data["softplus"].toBool()};
        variable_list g(12);
        for (int i = 0; i < 9; ++i) g[i] = twin(s[i]);          // u, dt, A, B, C, D, z, dt_bias, state
        const Tensor dy = full_grad(dy_, a.u), dlast = dlast_.defined() ? dlast_.contiguous() : dlast_;
        if (a.u.numel()) {
            On on(a.u);
            const pcrl_ssm_desc d = scan_desc(a);
            const int64_t bytes = ctx->saved_data["bytes"].toInt();
            const Tensor work = at::empty({bytes}, g[0].options().dtype(at::kByte));
            pcrl_ssm_grads o{};
            o.du = to_(g[0]), o.ddt = to_(g[1]), o.dz = to_(g[6]), o.dB = to_(g[3]), o.dC = to_(g[4]);
            o.dA = (float*)to_(g[2]), o.dD = (float*)to_(g[5]), o.ddt_bias = (float*)to_(g[7]), o.dstate = (float*)to_(g[8]);
            check(api.scan_bwd(&d, fat(s[11]), at_(dy), dy.stride(0), step_stride(dy), fat(dlast), &o, to_(work), (size_t)bytes, on.stream));
        } else {                                                // no step: the state passes through
            for (int i = 0; i < 8; ++i) if (g[i].defined()) g[i].zero_();
            if (g[8].defined()) { if (dlast.defined()) g[8].copy_(dlast); else g[8].zero_(); }
        }
        return g;
    }
};

ScanArgs scan_args(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D, const Opt& z, const Opt& dt_bias, bool softplus,
                   const Opt& state, const Opt& starts, const Opt& lengths, int dims) {
    TORCH_CHECK_VALUE(u.dim() == dims, "u is ", u.sizes(), dims == 2 ? ", expected [B, D]" : ", expected [B, T, D]");
    dtype_code(u);
    const int64_t width = u.size(-1), N = A.dim() == 2 ? A.size(1) : 0;
    TORCH_CHECK_VALUE(N >= 1 && N <= 32, "A is ", A.sizes(), ", expected [", width, ", N] with 1 to 32 states");
    ScanArgs a;
    a.u = adjacent(u, dims - 1);
    a.dt = adjacent(activation("dt", dt, u.sizes(), u), dims - 1);
    if (z.has_value()) a.z = adjacent(activation("z", *z, u.sizes(), u), dims - 1);
    a.A = parameter("A", A, {width, N}, u);
    if (D.has_value()) a.D = parameter("D", *D, {width}, u);
    if (dt_bias.has_value()) a.dt_bias = parameter("dt_bias", *dt_bias, {width}, u);
    if (state.has_value()) {
        TORCH_CHECK_VALUE(dims == 3 || state->is_contiguous(), "the state of a step must be contiguous (it is updated in place)");
        a.state = parameter("state", *state, {u.size(0), width, N}, u);
    }
    const int64_t G = B.dim() == dims + 1 ? B.size(-2) : 1;
    TORCH_CHECK_VALUE(G >= 1 && width % G == 0, width, " channels are not shared evenly by ", G, " groups");
    std::vector<int64_t> shape(u.sizes().begin(), u.sizes().end() - 1);
    shape.push_back(G), shape.push_back(N);
    a.B = adjacent(activation("B", B.dim() == dims ? B.unsqueeze(-2) : B, shape, u), dims);
    a.C = adjacent(activation("C", C.dim() == dims ? C.unsqueeze(-2) : C, shape, u), dims);
    a.starts = starts_of(starts, u.sizes().slice(0, dims - 1), u);
    a.lengths = lengths_of(lengths, u.size(0), dims == 3 ? u.size(1) : 1, u);
    a.softplus = softplus;
    return a;
}
std::tuple<Tensor, Tensor> ssm_scan(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D, const Opt& z, const Opt& dt_bias,
                                    bool softplus, const Opt& state, const Opt& starts, const Opt& lengths) {
    const ScanArgs a = scan_args(u, dt, A, B, C, D, z, dt_bias, softplus, state, starts, lengths, 3);
    no_tangents({a.u, a.dt, a.A, a.B, a.C, a.D, a.z, a.dt_bias, a.state});
    on_gpu(u);
    int64_t bytes = 0;
    const variable_list r = wants_grad({a.u, a.dt, a.A, a.B, a.C, a.D, a.z, a.dt_bias, a.state})
                                ? ScanNode::apply(a.u, a.dt, a.A, a.B, a.C, opt(a.D), opt(a.z), opt(a.dt_bias), opt(a.state), opt(a.starts), opt(a.lengths), a.softplus)
                                : scan_forward(a, false, bytes);
    return {r[0], r[1]};
}
Tensor ssm_step(const Tensor& u, const Tensor& dt, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& state, const Opt& D, const Opt& z, const Opt& dt_bias,
                bool softplus, const Opt& starts, const Opt& state_out) {
    at::NoGradGuard no_grad;
    TORCH_CHECK_VALUE(state.has_value(), "a step needs a state");
    const ScanArgs a = scan_args(u, dt, A, B, C, D, z, dt_bias, softplus, state, starts, std::nullopt, 2);
    no_tangents({a.u, a.dt, a.A, a.B, a.C, a.D, a.z, a.dt_bias, a.state});
    const Tensor out = state_out_of(a.state, state_out);
    on_gpu(u);
    Tensor y = at::empty(u.sizes(), u.options().requires_grad(false));
    if (y.numel()) {
        On on(u);
        const pcrl_ssm_desc d = scan_desc(a);
        check(api.step(&d, to_(y), (float*)to_(out), on.stream));
    }
    written(out);
    return y;
}

// ---- dropout ---------------------------------------------------------------------------------------------------------------------------------
// t as rows x cols with adjacent columns; what cannot be seen that way is copied.  An axis of one element takes no part: its stride is never
// stepped over and may be anything.
struct Rows { Tensor t; int64_t rows, cols, ld; };
Rows rows_of(const Tensor& t) {
    if (!t.is_contiguous() && t.stride(-1) == 1) {
        int64_t rows = 1, ld = t.size(-1);
        bool flat = true;                                       // the leading axes collapse into one with a single stride
        for (int64_t i = t.dim() - 2; i >= 0 && flat; --i) {
            if (t.size(i) == 1) continue;
            if (rows == 1) ld = t.stride(i);
            else flat = t.stride(i) == ld * rows;
            rows *= t.size(i);
        }
        if (flat && ld >= 0) return {t, rows, t.size(-1), ld};
    }
    const Tensor c = t.contiguous();
    return {c, 1, c.numel(), c.numel()};
}
Tensor dropout_launch(const Tensor& x, const Tensor& residual, int threshold, uint64_t seed, uint64_t offset, const Tensor& offset_t) {
    Tensor out = at::empty(x.sizes(), x.options().requires_grad(false));
    if (!out.numel()) return out;
    Rows a = rows_of(x), r{};
    if (residual.defined()) {
        r = rows_of(residual);
        if (r.cols != a.cols) {                                 // one is dense and the other is not: walk both by the shorter rows
            const int64_t cols = std::min(a.cols, r.cols);
            if (a.cols != cols) a.ld = cols;
            if (r.cols != cols) r.ld = cols;
            a.cols = cols, a.rows = out.numel() / cols;
        }
    }
    On on(out);
    check(api.dropout(at_(a.t), a.ld, at_(r.t), r.ld, to_(out), a.rows, a.cols, dtype_code(out), threshold, seed, offset, (const uint64_t*)at_(offset_t), on.stream));
    return out;
}
struct DropoutNode : Function<DropoutNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Opt& residual, int64_t threshold, int64_t seed, int64_t offset, const Opt& offset_t) {
        ctx->save_for_backward({val(offset_t)});
        ctx->saved_data["threshold"] = threshold;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["residual"] = residual.has_value();
        return dropout_launch(x, val(residual), (int)threshold, (uint64_t)seed, (uint64_t)offset, val(offset_t));
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once();
        variable_list g(6);
        const Tensor dy = grads[0];
        if (!dy.defined()) return g;
        const auto s = ctx->get_saved_variables();
        if (ctx->needs_input_grad(0))
            g[0] = dropout_launch(dy, Tensor(), (int)ctx->saved_data["threshold"].toInt(), (uint64_t)ctx->saved_data["seed"].toInt(), (uint64_t)ctx->saved_data["offset"].toInt(), s[0]);
        if (ctx->saved_data["residual"].toBool()) g[1] = dy;
        return g;
    }
};
Tensor dropout(const Tensor& x, double p, uint64_t seed, uint64_t offset, const Opt& offset_t_, const Opt& residual_) {
    dtype_code(x);
    TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout probability ", p);
    const Tensor residual = val(residual_), offset_t = val(offset_t_);
    if (residual.defined())
        TORCH_CHECK_VALUE(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type() && residual.device() == x.device(), "residual is ", residual.scalar_type(), " ",
                          residual.sizes(), " on ", residual.device(), ", x is ", x.scalar_type(), " ", x.sizes(), " on ", x.device());
    if (offset_t.defined())
        TORCH_CHECK_VALUE(offset_t.scalar_type() == at::kLong && offset_t.numel() == 1 && offset_t.device() == x.device(),
                          "offset: an integer, or an int64 tensor of one element on the device of x");
    no_tangents({x, residual});
    on_gpu(x);
    const int64_t threshold = (int64_t)std::nearbyint(p * 65536.0);
    if (wants_grad({x, residual})) return DropoutNode::apply(x, residual_, threshold, (int64_t)seed, (int64_t)offset, offset_t_);
    return dropout_launch(x, residual, (int)threshold, seed, offset, offset_t);
}

}  // namespace

PYBIND11_MODULE(_sequence, m) {
    m.def("bind", &bind);
    m.def("short_conv", &short_conv);
    m.def("short_conv_step", &short_conv_step);
    m.def("ssm_scan", &ssm_scan);
    m.def("ssm_step", &ssm_step);
    m.def("dropout", &dropout);
    // how dropout walks a tensor (tests): rows, columns, row stride, whether it works on a copy
    m.def("dropout_rows", [](const Tensor& t) {
        const Rows r = rows_of(t);
        return std::make_tuple(r.rows, r.cols, r.ld, !r.t.is_same(t));
    });
}
