// host_nodes.cpp - the host side of the gated linear recurrence and of the AdamW step: argument checks, output allocation, the
// autograd node and the calls of the C ABI (include/megacrn_hip.h), as the Python module megacrn_amd._host.
//
// Why C++: a node written in Python costs 175 us of host time for a forward and a backward pass (its backward runs on the autograd
// engine's thread and waits for the interpreter lock), this one 45 - 75 (8 for the forward; the rest is the engine's hand-over between its
// threads), where the kernels of a METR-LA training window take 60.  A serving step: 18 us before, 4.8 now.
// The library is not linked: `bind` takes the addresses of its entry points from the one that Python has loaded.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>
#include <ATen/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "../../include/megacrn_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Api {
    decltype(&mcrn_last_error) last_error = nullptr;
    decltype(&mcrn_glr_checkpoint_floats) glr_checkpoint_floats = nullptr;
    decltype(&mcrn_glr_workspace_bytes) glr_workspace_bytes = nullptr;
    decltype(&mcrn_glr_forward) glr_forward = nullptr;
    decltype(&mcrn_glr_backward) glr_backward = nullptr;
    decltype(&mcrn_adamw_step) adamw_step = nullptr;
    decltype(&mcrn_adamw_unpack) adamw_unpack = nullptr;
};
Api api;

template <class F> void take(const pybind11::dict& d, const char* name, F& f) { f = reinterpret_cast<F>(d[name].cast<uintptr_t>()); }
void bind(const pybind11::dict& d) {
    take(d, "mcrn_last_error", api.last_error);
    take(d, "mcrn_glr_checkpoint_floats", api.glr_checkpoint_floats);
    take(d, "mcrn_glr_workspace_bytes", api.glr_workspace_bytes);
    take(d, "mcrn_glr_forward", api.glr_forward);
    take(d, "mcrn_glr_backward", api.glr_backward);
    take(d, "mcrn_adamw_step", api.adamw_step);
    take(d, "mcrn_adamw_unpack", api.adamw_unpack);
}

// A backward pass runs on the autograd engine's thread without the interpreter lock, while another thread of the program may take a step: they take
// turns in the library, whose last error is the calling thread's own.
template <class F> void call(const char* what, F f) {
    const int rc = f();
    TORCH_CHECK(rc == 0, what, " failed (rc=", rc, "): ", api.last_error());
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void need_gpu(const Tensor& t, const char* who) {
    TORCH_CHECK(t.is_cuda(), who, ": megacrn_amd runs on MI355X only (got a ", t.device(), " tensor); there is no CPU fallback");
}
// what autograd has saved of a tensor that a kernel writes in place is no longer valid
void changed(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// The kernels write through pointers, so torch sees no operation that could carry a tangent: a dual tensor is refused, not taken as a constant
void no_tangent(const Tensor& t, const char* who) {
    TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), who, " is differentiable in reverse mode only: an input carries a forward gradient (torch.autograd.forward_ad)");
}
int type_of(at::ScalarType t) { return t == at::kFloat ? MCRN_T_F32 : t == at::kBFloat16 ? MCRN_T_BF16 : t == at::kHalf ? MCRN_T_F16 : -1; }

// ---- gated linear recurrence -------------------------------------------------------------------------------------------
int activation_of(const std::string& name, const char* who) {
    TORCH_CHECK_VALUE(name == "tanh" || name == "none", who, ": activation must be 'tanh' or 'none'; got '", name, "'");
    return name == "tanh" ? MCRN_ACT_TANH : MCRN_ACT_NONE;
}

// Everything that the C entry points cannot see in raw pointers; returns the mask expanded to (B, T, N) or (B, N).
Tensor check_inputs(const Tensor& gate, const Tensor& cand, const Tensor& state, const Tensor& mask, const char* who, int64_t lead) {
    TORCH_CHECK(!torch::jit::tracer::isTracing(), who, " cannot be traced: a trace would hold the allocation of its outputs and not what fills them");
    for (const Tensor* t : {&gate, &cand})
        TORCH_CHECK_TYPE(type_of(t->scalar_type()) >= 0, who, ": gate and cand must be float32, bfloat16 or float16; got ", t->scalar_type());
    TORCH_CHECK_VALUE(cand.dim() == lead + 1 && gate.dim() == lead + 1 && gate.sizes().slice(0, lead) == cand.sizes().slice(0, lead), who,
                      ": gate ", gate.sizes(), " and cand ", cand.sizes(), " must agree in all but their last of ", lead + 1, " dimensions");
    TORCH_CHECK_VALUE(gate.scalar_type() == cand.scalar_type() && gate.device() == cand.device(), who, ": gate and cand must have one type and one device");
    const int64_t H = cand.size(-1), G = gate.size(-1);
    TORCH_CHECK_VALUE(H >= 1 && G >= 1 && H % G == 0, who, ": the gates' number ", G, " must divide the channels' ", H);
    for (int64_t i = 0; i <= lead; ++i) TORCH_CHECK_VALUE(cand.size(i) <= (1 << 30), who, ": a dimension of cand ", cand.sizes(), " is above 2^30");
    if (state.defined()) {
        const int64_t want[3] = {cand.size(0), cand.size(-2), H};
        TORCH_CHECK_VALUE(state.scalar_type() == at::kFloat && state.device() == cand.device() && state.sizes() == at::IntArrayRef(want, 3), who,
                          ": state must be a float32 tensor of shape ", at::IntArrayRef(want, 3), " on ", cand.device());
    }
    Tensor m = mask;
    if (m.defined()) {
        TORCH_CHECK_VALUE(m.scalar_type() == at::kBool && m.device() == cand.device(), who, ": mask must be a bool tensor on ", cand.device());
        if (m.dim() == lead - 1) m = m.unsqueeze(-1);      // the same for every node
        bool fits = m.dim() == lead;
        for (int64_t i = 0; fits && i < lead; ++i) fits = m.size(i) == cand.size(i) || m.size(i) == 1;
        TORCH_CHECK_VALUE(fits, who, ": mask must be ", cand.sizes().slice(0, lead), ", with 1 where all share an entry, or lack its last dimension; got ", mask.sizes());
        m = m.expand(cand.sizes().slice(0, lead));
    }
    for (const Tensor* t : {&gate, &cand, &state}) no_tangent(*t, who);
    need_gpu(cand, who);
    return m;
}

// strides over B, T, N (B, N: T = 1); those of dimensions that have one entry do not matter
void strides_of(const Tensor& t, int64_t lead, long long* s) {
    const int64_t at[3] = {0, lead == 3 ? 1 : -1, lead - 1};
    for (int i = 0; i < 3; ++i) s[i] = at[i] < 0 || t.size(at[i]) == 1 ? 0 : t.stride(at[i]);
}
// A view that is negative by a bit (the imaginary part of a conjugate): its memory holds the other sign
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
// The kernels want a last dimension without gaps, and a tile's rows (128 steps at most) within 4 GB of each other: a copy where that is not so.
bool near(const Tensor& t, int64_t lead, int64_t width) {
    long long s[3];
    strides_of(t, lead, s);
    const long long steps = lead == 3 ? std::min<int64_t>(t.size(1), 128) : 1;
    return ((steps - 1) * s[1] + (t.size(lead - 1) - 1) * s[2] + width) * (long long)t.element_size() < (1ll << 32);
}
Tensor rows(const Tensor& t0, int64_t lead) {
    const Tensor t = plain(t0);
    if (!t.defined()) return t;
    return (t.size(-1) == 1 || t.stride(-1) == 1) && near(t, lead, t.size(-1)) ? t : t.contiguous();
}

mcrn_glr_t dims_of(const Tensor& gate, const Tensor& cand, const Tensor& mask, const Tensor& dout, int act, int64_t lead) {
    mcrn_glr_t d = {};
    d.B = (int)cand.size(0);
    d.T = lead == 3 ? (int)cand.size(1) : 1;
    d.N = (int)cand.size(-2);
    d.H = (int)cand.size(-1);
    d.G = (int)gate.size(-1);
    d.dtype = type_of(cand.scalar_type());
    d.activation = act;
    strides_of(gate, lead, d.gate_s);
    strides_of(cand, lead, d.cand_s);
    if (mask.defined()) strides_of(mask, lead, d.mask_s);
    if (dout.defined()) strides_of(dout, lead, d.dout_s);
    return d;
}
// From torch's allocator, call by call: it knows streams and graph captures, and the block is free again once the kernels are queued.
Tensor workspace(const mcrn_glr_t& d, int backward, const Tensor& like, size_t& bytes) {
    bytes = api.glr_workspace_bytes(&d, backward);
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

struct Sequence {
    Tensor out, last, ckpt;
};
Sequence glr_run(const Tensor& gate, const Tensor& cand, const Tensor& state, const Tensor& mask, int act, bool keep) {
    const at::DeviceGuard guard(cand.device());
    const mcrn_glr_t d = dims_of(gate, cand, mask, Tensor(), act, 3);
    Sequence r;
    const auto f32 = cand.options().dtype(at::kFloat);
    r.out = at::empty(cand.sizes(), cand.options());
    r.last = at::empty({d.B, d.N, d.H}, f32);
    if (keep)
        if (const size_t n = api.glr_checkpoint_floats(&d)) r.ckpt = at::empty({(int64_t)n}, f32);
    size_t nb;
    const Tensor ws = workspace(d, 0, cand, nb);
    call("mcrn_glr_forward", [&] {
        return api.glr_forward(&d, ptr(gate), ptr(cand), (const unsigned char*)ptr(mask), (const float*)ptr(state), ws.defined() ? ws.mutable_data_ptr() : nullptr, nb,
                               r.out.mutable_data_ptr(), (float*)r.last.mutable_data_ptr(), r.ckpt.defined() ? (float*)r.ckpt.mutable_data_ptr() : nullptr, stream_of(cand));
    });
    return r;
}

struct GlrNode : torch::autograd::Function<GlrNode> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, Tensor gate, Tensor cand, OptTensor state, OptTensor mask, int64_t act) {
        Tensor h0 = state ? plain(*state).contiguous() : Tensor(), m = mask.value_or(Tensor());
        const Sequence r = glr_run(gate, cand, h0, m, (int)act, true);
        // fp32: the backward reads the states before every 8th step from `out` itself; the 16-bit types keep those in fp32
        ctx->save_for_backward({gate, cand, h0, m, cand.scalar_type() == at::kFloat ? r.out : r.ckpt});
        ctx->saved_data["act"] = act;
        ctx->set_materialize_grads(false);
        return {r.out, r.last};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list g) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "gated_linear_recurrence is differentiable once: its gradient has no graph (create_graph=True)");
        torch::autograd::variable_list out(5);
        if (!g[0].defined() && !g[1].defined()) return out;
        const auto s = ctx->get_saved_variables();
        const Tensor &gate = s[0], &cand = s[1], &h0 = s[2], &mask = s[3], &kept = s[4];
        const at::DeviceGuard guard(cand.device());
        const Tensor dout = rows(g[0], 3), dlast = g[1].defined() ? plain(g[1]).contiguous() : Tensor();
        const mcrn_glr_t d = dims_of(gate, cand, mask, dout, (int)ctx->saved_data["act"].toInt(), 3);
        out[0] = at::empty(gate.sizes(), gate.options());
        out[1] = at::empty(cand.sizes(), cand.options());
        if (h0.defined()) out[2] = at::empty(h0.sizes(), h0.options());
        size_t nb;
        const Tensor ws = workspace(d, 1, cand, nb);
        call("mcrn_glr_backward", [&] {
            return api.glr_backward(&d, ptr(gate), ptr(cand), (const unsigned char*)ptr(mask), (const float*)ptr(h0), ptr(kept), ptr(dout), (const float*)ptr(dlast),
                                    ws.defined() ? ws.mutable_data_ptr() : nullptr, nb, out[0].mutable_data_ptr(), out[1].mutable_data_ptr(),
                                    h0.defined() ? (float*)out[2].mutable_data_ptr() : nullptr, stream_of(cand));
        });
        return out;
    }
};

std::pair<Tensor, Tensor> glr(const Tensor& gate0, const Tensor& cand0, const OptTensor& state, const OptTensor& mask0, const std::string& activation) {
    const char* who = "gated_linear_recurrence";
    const int act = activation_of(activation, who);
    const Tensor h0 = state.value_or(Tensor());
    Tensor mask = check_inputs(gate0, cand0, h0, mask0.value_or(Tensor()), who, 3);
    if (cand0.numel() == 0) {                              // nothing to read, or no step to take
        const Tensor last = h0.defined() ? h0.clone() : at::zeros({cand0.size(0), cand0.size(2), cand0.size(3)}, cand0.options().dtype(at::kFloat));
        if (at::GradMode::is_enabled() && (gate0.requires_grad() || cand0.requires_grad())) {      // a backward pass finds its way: gradients of no elements
            const Tensor out = cand0 + gate0.sum(-1, true);
            return {out, last + out.sum(1, false, at::kFloat)};
        }
        return {at::empty(cand0.sizes(), cand0.options()), last};
    }
    const Tensor gate = rows(gate0, 3), cand = rows(cand0, 3);
    if (mask.defined() && !near(mask, 3, 1)) mask = mask.contiguous();
    if (at::GradMode::is_enabled() && (gate.requires_grad() || cand.requires_grad() || (h0.defined() && h0.requires_grad()))) {
        auto r = GlrNode::apply(gate, cand, state, mask.defined() ? OptTensor(mask) : OptTensor(), (int64_t)act);
        return {r[0], r[1]};
    }
    const Sequence r = glr_run(gate, cand, h0.defined() ? plain(h0).contiguous() : h0, mask, act, false);
    return {r.out, r.last};
}

// The input, or a copy where it lies in memory that the step overwrites: a thread advances its channel while another one still reads
Tensor apart(const Tensor& t, const Tensor& state) {
    if (!t.defined() || !t.is_alias_of(state) || t.numel() == 0) return t;
    int64_t reach = 1;
    for (int64_t i = 0; i < t.dim(); ++i) reach += (t.size(i) - 1) * t.stride(i);
    const auto at = (uintptr_t)t.const_data_ptr(), to = (uintptr_t)state.const_data_ptr();
    return at < to + state.nbytes() && to < at + reach * t.element_size() ? t.clone() : t;
}

Tensor glr_step(const Tensor& gate0, const Tensor& cand0, const OptTensor& state0, const OptTensor& mask0, const std::string& activation) {
    const char* who = "gated_linear_recurrence_step";
    const int act = activation_of(activation, who);
    const Tensor state = state0.value_or(Tensor());
    TORCH_CHECK_VALUE(state.defined() && state.is_contiguous() && !state.is_neg(), who, ": state must be a contiguous tensor; it is advanced in place");
    Tensor mask = check_inputs(gate0, cand0, state, mask0.value_or(Tensor()), who, 2);
    TORCH_CHECK(!(at::GradMode::is_enabled() && (gate0.requires_grad() || cand0.requires_grad() || state.requires_grad())), who,
                " is not differentiable: call it under torch.no_grad()");
    const Tensor gate = rows(apart(gate0, state), 2), cand = rows(apart(cand0, state), 2), out = at::empty(cand.sizes(), cand.options());
    if (out.numel() == 0) return out;
    if (mask.defined() && !near(mask, 2, 1)) mask = mask.contiguous();
    const at::DeviceGuard guard(cand.device());
    const mcrn_glr_t d = dims_of(gate, cand, mask, Tensor(), act, 2);
    float* h = (float*)state.mutable_data_ptr();
    call("mcrn_glr_forward", [&] {
        return api.glr_forward(&d, ptr(gate), ptr(cand), (const unsigned char*)ptr(mask), h, nullptr, 0, out.mutable_data_ptr(), h, nullptr, stream_of(cand));
    });
    changed(state);
    return out;
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------
// cfg, numel, lr, weight_decay, step: addresses of the optimizer's own arrays (lr .. step on the device where cfg says so).
void adamw_step(uintptr_t cfg_at, const std::vector<Tensor>& params, const std::vector<OptTensor>& grads, uintptr_t numel_at, uintptr_t lr, uintptr_t wd,
                uintptr_t step_at, const Tensor& m, const Tensor& v, const OptTensor& ms, const OptTensor& vs, const OptTensor& master, const Tensor& ws,
                const OptTensor& norm) {
    const auto* cfg = reinterpret_cast<const mcrn_adamw_t*>(cfg_at);
    const auto* numel = reinterpret_cast<const long long*>(numel_at);
    const size_t n = params.size();
    TORCH_CHECK_VALUE(grads.size() == n && (size_t)cfg->ntensors == n, "AdamW.step: ", grads.size(), " gradients for ", n, " parameters");
    const auto type = cfg->dtype == MCRN_T_F32 ? at::kFloat : at::kBFloat16;
    const auto dev = m.device();
    std::vector<void*> p(n, nullptr);
    std::vector<const void*> g(n, nullptr);
    std::vector<Tensor> held;                              // contiguous copies live until the kernels are queued
    for (size_t i = 0; i < n; ++i) {
        if (!grads[i] || !grads[i]->defined()) continue;
        const Tensor &a = params[i], &b = *grads[i];
        TORCH_CHECK_VALUE(a.scalar_type() == type && a.device() == dev && a.is_contiguous() && !a.is_neg() && a.numel() == numel[i], "AdamW.step: parameter ", i,
                          " is no longer the contiguous ", type, " tensor that the optimizer was made for");
        TORCH_CHECK_VALUE(b.scalar_type() == type && b.device() == dev && b.layout() == at::kStrided && b.sizes() == a.sizes(), "AdamW.step: gradient ", i,
                          " must be a ", type, " tensor of shape ", a.sizes(), " on ", dev);
        no_tangent(a, "AdamW.step");
        no_tangent(b, "AdamW.step");
        p[i] = a.mutable_data_ptr();
        if (b.is_contiguous() && !b.is_neg()) g[i] = b.const_data_ptr();
        else g[i] = held.emplace_back(plain(b).contiguous()).const_data_ptr();
    }
    auto data = [](const OptTensor& t) { return t ? t->mutable_data_ptr() : nullptr; };
    const at::DeviceGuard guard(dev);
    int* step = reinterpret_cast<int*>(step_at);
    auto count = [&](int by) {
        if (!cfg->on_device)
            for (size_t i = 0; i < n; ++i)
                if (grads[i] && grads[i]->defined() && numel[i]) step[i] += by;      // as the device counts: a tensor without elements has no updates
    };
    if (m.numel() == 0) return;                            // no tensor has any
    call("mcrn_adamw_step", [&] {
        count(1);
        const int rc = api.adamw_step(cfg, p.data(), g.data(), numel, reinterpret_cast<const double*>(lr), reinterpret_cast<const double*>(wd), step,
                                      m.mutable_data_ptr(), v.mutable_data_ptr(), (unsigned char*)data(ms), (unsigned char*)data(vs), (float*)data(master),
                                      ws.mutable_data_ptr(), (size_t)ws.numel(), (float*)data(norm), stream_of(m));
        if (rc) count(-1);                                 // refused before the first launch: nothing was updated
        return rc;
    });
    for (size_t i = 0; i < n; ++i)
        if (p[i]) changed(params[i]);
}

std::pair<Tensor, Tensor> adamw_unpack(const Tensor& m, const Tensor& ms, const Tensor& v, const Tensor& vs) {
    const at::DeviceGuard guard(m.device());
    const Tensor om = at::empty(m.sizes(), m.options().dtype(at::kFloat)), ov = at::empty(v.sizes(), v.options().dtype(at::kFloat));
    if (m.numel() == 0) return {om, ov};
    auto bytes = [](const Tensor& t) { return (const unsigned char*)t.const_data_ptr(); };
    call("mcrn_adamw_unpack", [&] {
        return api.adamw_unpack(bytes(m), bytes(ms), bytes(v), bytes(vs), m.numel(), (float*)om.mutable_data_ptr(), (float*)ov.mutable_data_ptr(), stream_of(m));
    });
    return {om, ov};
}

}  // namespace

PYBIND11_MODULE(_host, mod) {
    mod.def("bind", &bind);
    mod.def("glr", &glr);
    mod.def("glr_step", &glr_step);
    mod.def("adamw_step", &adamw_step);
    mod.def("adamw_unpack", &adamw_unpack);
}
