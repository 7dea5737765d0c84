// The differentiable calls of nanoplm_amd as native autograd nodes (Python module nanoplm_amd._node): plain, gated and
// LayerNorm-fused conv, gated linear recurrence and residual norm, forward and backward through the C ABI of libnplm_dwconv.so.
//
// What bounds a small training step is the host. As torch.autograd.Function the backward runs Python on the engine's
// thread, which first has to get the interpreter lock from the thread that waits for it; as torch.library custom ops (the
// pre-norm door's eager route before) both directions go through Python dispatch as well. Here neither direction runs Python.
// Forward + backward of one call after another, T=2048, 7 taps, bf16, before and now: plain, C=768 65 to 126 us (by how the threads
// meet at the lock) and 34 to 67 (by how soon the waiting thread and the engine's wake each other); gated 124 to 129 and 38 to 68; pre-norm
// 217 to 223 and 79 to 83. A multiplication by a constant takes 24 to 47. Inference, T=776, C=64, 3 taps 15.2 and 7.0; padded door, 32 x 512
// rows 23.9 and 15.8.
//
// A call that is not of the usual form - arguments that the checks below do not settle, tensor subclasses, modes, transforms,
// tracing, forward-mode AD - is answered with None, and the Python route takes it with its own messages. So nothing
// is accepted or refused here that it would treat otherwise.
//
// Replaces no reference code (peymanvahidi/nanoplm 0.1.6 has no convolution); the backward is what autograd runs at
// src/nanoplm/pretraining/pure_pipeline.py:739-742.
#include <torch/extension.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <ATen/record_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <climits>
#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/nplm_dwconv.h"
#include "../../include/nplm_recurrence.h"
#include "../../include/nplm_resnorm.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<at::Tensor>;

// The library has no fused kernel for the call: the Python route composes it.
struct Unsupported : std::runtime_error {
    Unsupported() : std::runtime_error("no fused kernel for this call") {}
};

int dtype_code(const at::Tensor& t) {
    if (t.scalar_type() == at::kFloat) return NPLM_DWCONV_F32;
    if (t.scalar_type() == at::kBFloat16) return NPLM_DWCONV_BF16;
    return -1;
}
// Whether t's values are what lies at its data pointer, one after the other: not so for wrappers (of a batch, of another tensor), for a
// tensor known to be zero, and for a view that negates its values when they are read.
bool dense(const at::Tensor& t, const at::Device& dev) {
    return t.layout() == at::kStrided && t.device() == dev && !at::isTensorSubclassLike(t) && !t.is_neg() && !t._is_zerotensor() &&
           t.is_contiguous();
}
// The same of [T, C] rows that may lie apart: adjacent elements, no row reaching into the next one.
bool rows(const at::Tensor& t, const at::Device& dev, int64_t T, int64_t C) {
    return t.layout() == at::kStrided && t.device() == dev && !at::isTensorSubclassLike(t) && !t.is_neg() && !t._is_zerotensor() && t.dim() == 2 &&
           t.size(0) == T && t.size(1) == C && (t.stride(1) == 1 || C == 1) && (t.stride(0) >= C || T <= 1);
}
int64_t row_stride(const at::Tensor& t) { return t.stride(0) > t.size(1) ? t.stride(0) : t.size(1); }
// a parameter of one value a channel, in w's dtype on its device
bool vector_as(const at::Tensor& t, const at::Tensor& w, int32_t C) {
    return dense(t, w.device()) && t.dim() == 1 && t.size(0) == C && t.scalar_type() == w.scalar_type();
}

struct Sizes {
    int64_t T;
    int32_t C, K, S, act, wdt;
};
// Sizes of a call on x [T, width * C], if everything about its tensors is as the kernels take it.
bool sizes_of(const at::Tensor& x, int width, const at::Tensor& cu, const at::Tensor& w, const OptTensor& b, Sizes* s) {
    if (!x.is_cuda() || x.dim() != 2 || w.dim() != 2 || cu.dim() != 1) return false;
    const at::Device dev = x.device();
    if (!dense(x, dev) || !dense(w, dev) || !dense(cu, dev) || cu.scalar_type() != at::kInt || cu.numel() < 1) return false;
    s->act = dtype_code(x);
    s->wdt = dtype_code(w);
    if (s->act < 0 || s->wdt < 0) return false;
    const int64_t C = x.size(1) / width, K = w.size(1);
    if (x.size(1) % width || w.size(0) != C || K % 2 == 0 || C > INT_MAX || K > INT_MAX || cu.numel() > INT_MAX) return false;
    if (b && !vector_as(*b, w, (int32_t)C)) return false;
    s->T = x.size(0);
    s->C = (int32_t)C;
    s->K = (int32_t)K;
    s->S = (int32_t)(cu.numel() - 1);
    return true;
}

const void* ptr(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }
const int32_t* ints(const at::Tensor& t) { return t.const_data_ptr<int32_t>(); }
bool aligned16(const at::Tensor& t) { return (uintptr_t)t.const_data_ptr() % 16 == 0; }
void* stream_of(const at::Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check(int rc, const char* what) {
    if (rc == -NPLM_DWCONV_EUNSUPPORTED) throw Unsupported();
    if (rc != 0) throw std::runtime_error(std::string(what) + " failed with code " + std::to_string(rc) + ": " + nplm_dwconv_strerror(rc));
}
uint32_t flags_of(bool residual, bool grads_bf16) {
    return (residual ? NPLM_DWCONV_RESIDUAL : 0u) | (grads_bf16 ? NPLM_DWCONV_GRADS_BF16 : 0u);
}
at::Tensor scratch(size_t bytes, const at::Tensor& like) {
    return at::empty({(int64_t)(bytes > 256 ? bytes : 256)}, like.options().dtype(at::kByte));
}
// dy as the kernels take it
at::Tensor incoming(const at::Tensor& dy, const at::Tensor& x) {
    return dy.scalar_type() == x.scalar_type() ? dy.contiguous() : dy.to(x.scalar_type()).contiguous();
}
at::Tensor as(const at::Tensor& t, bool wanted, at::ScalarType dt) {
    return !wanted ? at::Tensor() : t.scalar_type() == dt ? t : t.to(dt);
}

// The Python route of a backward whose call turns out to be of another form (its result as a list of tensors).
template <typename... Args>
variable_list python_backward(const char* module, const char* name, Args&&... args) {
    pybind11::gil_scoped_acquire gil;
    pybind11::object out = pybind11::module_::import(module).attr(name)(std::forward<Args>(args)...);
    variable_list r;
    for (pybind11::handle h : out) r.push_back(h.is_none() ? at::Tensor() : h.cast<at::Tensor>());
    return r;
}

// Calls (and backwards) that something else records, rewrites or looks into go the Python way.
bool observed() {
    return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::PythonTorchFunctionTLS::stack_len() > 0 ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) || torch::jit::tracer::isTracing() ||
           torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
}

// The tensors of a backward are what saved-tensor hooks gave back, which need not be what was saved, and a gradient of whatever kind its
// caller has: whether they are as the kernels take them. If not, the Python route makes them so, takes them apart or refuses them.
bool usual_backward(const at::Tensor& x, int width, const at::Tensor& cu, const at::Tensor& w, const at::Tensor& dy, Sizes* s) {
    return !observed() && x.defined() && cu.defined() && w.defined() && sizes_of(x, width, cu, w, std::nullopt, s) && dense(dy, x.device()) &&
           dy.dim() == 2 && dy.size(0) == s->T && dy.size(1) == s->C;
}

}  // namespace

// The nodes, by the names that profiles and autograd's messages give them; their calls are recorded there as the registered ops are.
namespace nanoplm_amd {
struct VarlenDWConv1d : torch::autograd::Function<VarlenDWConv1d> {
    static at::Tensor run(const at::Tensor& x, const at::Tensor& cu, const at::Tensor& w, const OptTensor& b, bool residual) {
        RECORD_FUNCTION("nanoplm_amd::varlen_dwconv_fwd", {});
        Sizes s;
        sizes_of(x, 1, cu, w, b, &s);
        const c10::DeviceGuard on(x.device());
        at::Tensor y = at::empty({s.T, s.C}, x.options());
        check(nplm_dwconv_fwd_ex(x.const_data_ptr(), ints(cu), w.const_data_ptr(), ptr(b), y.mutable_data_ptr(), s.T, s.C, s.K, s.S, s.act,
                                 s.wdt, flags_of(residual, false), stream_of(x)), "nplm_dwconv_fwd");
        return y;
    }
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& cu, const at::Tensor& w, const OptTensor& b,
                              bool residual) {
        ctx->save_for_backward({x, cu, w});
        ctx->saved_data["bias"] = b.has_value();
        ctx->saved_data["residual"] = residual;
        return run(x, cu, w, b, residual);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        RECORD_FUNCTION("nanoplm_amd::varlen_dwconv_bwd", {});
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &cu = saved[1], &w = saved[2];
        const bool has_bias = ctx->saved_data["bias"].toBool(), residual = ctx->saved_data["residual"].toBool();
        const bool need_dx = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(2), need_b = has_bias && ctx->needs_input_grad(3);
        Sizes s;
        const c10::DeviceGuard on(x.device());
        const at::Tensor dy = incoming(grads[0], x);
        const bool bf16 = w.scalar_type() == at::kBFloat16;
        const at::ScalarType gdt = w.scalar_type();          // (fp32 or bf16: what the reduction kernel writes)
        at::Tensor dx, dw, db, ws;
        if (!usual_backward(x, 1, cu, w, dy, &s)) {
            using namespace pybind11::literals;
            pybind11::gil_scoped_acquire gil;
            const variable_list r = python_backward("nanoplm_amd.dwconv", "varlen_dwconv_bwd", x, dy, cu, w, "need_dx"_a = need_dx,
                                                    "need_dw"_a = need_w || need_b, "residual"_a = residual, "grads_bf16"_a = bf16);
            return {r[0], at::Tensor(), need_w ? r[1] : at::Tensor(), need_b ? r[2] : at::Tensor(), at::Tensor()};
        }
        if (need_dx) dx = at::empty({s.T, s.C}, x.options());
        size_t bytes = 0;
        if (need_w || need_b) {
            dw = at::empty({s.C, s.K}, x.options().dtype(gdt));
            db = at::empty({s.C}, x.options().dtype(gdt));
            bytes = nplm_dwconv_bwd_workspace_bytes(s.T, s.C, s.K, s.act);
            ws = scratch(bytes, x);
        }
        auto at_of = [](const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; };
        check(nplm_dwconv_bwd_ex(x.const_data_ptr(), dy.const_data_ptr(), ints(cu), w.const_data_ptr(), at_of(dx), (float*)at_of(dw),
                                 (float*)at_of(db), at_of(ws), ws.defined() ? (size_t)ws.numel() : 0, s.T, s.C, s.K, s.S, s.act, s.wdt,
                                 flags_of(residual, bf16), stream_of(x)), "nplm_dwconv_bwd");
        return {dx, at::Tensor(), need_w ? dw : at::Tensor(), need_b ? db : at::Tensor(), at::Tensor()};
    }
};

struct GatedVarlenDWConv1d : torch::autograd::Function<GatedVarlenDWConv1d> {
    static at::Tensor run(const at::Tensor& z, const at::Tensor& cu, const at::Tensor& w, const OptTensor& b, bool residual) {
        RECORD_FUNCTION("nanoplm_amd::gated_dwconv_fwd", {});
        Sizes s;
        sizes_of(z, 2, cu, w, b, &s);
        const c10::DeviceGuard on(z.device());
        at::Tensor y = at::empty({s.T, s.C}, z.options());
        check(nplm_dwconv_gated_fwd(z.const_data_ptr(), ints(cu), w.const_data_ptr(), ptr(b), y.mutable_data_ptr(), s.T, s.C, s.K, s.S,
                                    s.act, s.wdt, flags_of(residual, false), stream_of(z)), "nplm_dwconv_gated_fwd");
        return y;
    }
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& z, const at::Tensor& cu, const at::Tensor& w, const OptTensor& b,
                              bool residual) {
        ctx->save_for_backward({z, cu, w});
        ctx->saved_data["bias"] = b.has_value();
        ctx->saved_data["residual"] = residual;
        return run(z, cu, w, b, residual);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        RECORD_FUNCTION("nanoplm_amd::gated_dwconv_bwd", {});
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &z = saved[0], &cu = saved[1], &w = saved[2];
        const bool has_bias = ctx->saved_data["bias"].toBool(), residual = ctx->saved_data["residual"].toBool();
        Sizes s;
        const c10::DeviceGuard on(z.device());
        const at::Tensor dy = incoming(grads[0], z);
        const bool bf16 = w.scalar_type() == at::kBFloat16;
        const at::ScalarType gdt = w.scalar_type();
        const bool usual = usual_backward(z, 2, cu, w, dy, &s);
        const size_t bytes = usual ? nplm_dwconv_gated_bwd_workspace_bytes(s.T, s.C, s.K, s.act) : 0;
        at::Tensor dz, dw, db;
        int rc = -NPLM_DWCONV_EUNSUPPORTED;
        if (bytes > 0) {
            dz = at::empty({s.T, 2 * (int64_t)s.C}, z.options());
            dw = at::empty({s.C, s.K}, z.options().dtype(gdt));
            db = at::empty({s.C}, z.options().dtype(gdt));
            const at::Tensor ws = scratch(bytes, z);
            rc = nplm_dwconv_gated_bwd(z.const_data_ptr(), dy.const_data_ptr(), ints(cu), w.const_data_ptr(), dz.mutable_data_ptr(),
                                       (float*)dw.mutable_data_ptr(), (float*)db.mutable_data_ptr(), ws.mutable_data_ptr(),
                                       (size_t)ws.numel(), s.T, s.C, s.K, s.S, s.act, s.wdt, flags_of(residual, bf16), stream_of(z));
        }
        if (rc == -NPLM_DWCONV_EUNSUPPORTED) {
            using namespace pybind11::literals;
            pybind11::gil_scoped_acquire gil;
            const variable_list r = python_backward("nanoplm_amd.gated", "gated_dwconv_bwd", z, dy, cu, w, "residual"_a = residual, "grads_bf16"_a = bf16);
            dz = r[0], dw = r[1], db = r[2];
        } else {
            check(rc, "nplm_dwconv_gated_bwd");
        }
        return {ctx->needs_input_grad(0) ? dz : at::Tensor(), at::Tensor(), as(dw, ctx->needs_input_grad(2), gdt),
                as(db, has_bias && ctx->needs_input_grad(3), gdt), at::Tensor()};
    }
};

struct LnVarlenDWConv1d : torch::autograd::Function<LnVarlenDWConv1d> {
    // stats [T, 2] come back for the backward
    static at::Tensor run(const at::Tensor& x, const at::Tensor& cu, const at::Tensor& g, const OptTensor& beta, const at::Tensor& w,
                          const OptTensor& b, double eps, bool residual, at::Tensor* stats) {
        RECORD_FUNCTION("nanoplm_amd::ln_dwconv_fwd", {});
        Sizes s;
        sizes_of(x, 1, cu, w, b, &s);
        const c10::DeviceGuard on(x.device());
        at::Tensor y = at::empty({s.T, s.C}, x.options());
        *stats = at::empty({s.T, 2}, x.options().dtype(at::kFloat));
        check(nplm_dwconv_ln_fwd(x.const_data_ptr(), ints(cu), g.const_data_ptr(), ptr(beta), (float)eps, w.const_data_ptr(), ptr(b),
                                 y.mutable_data_ptr(), stats->mutable_data_ptr<float>(), s.T, s.C, s.K, s.S, s.act, s.wdt,
                                 flags_of(residual, false), stream_of(x)), "nplm_dwconv_ln_fwd");
        return y;
    }
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& cu, const at::Tensor& g, const OptTensor& beta,
                              const at::Tensor& w, const OptTensor& b, double eps, bool residual) {
        at::Tensor stats;
        at::Tensor y = run(x, cu, g, beta, w, b, eps, residual, &stats);
        ctx->save_for_backward({x, cu, g, beta ? *beta : at::Tensor(), w, stats});
        ctx->saved_data["bias"] = b.has_value();
        ctx->saved_data["residual"] = residual;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        RECORD_FUNCTION("nanoplm_amd::ln_dwconv_bwd", {});
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &cu = saved[1], &g = saved[2], &beta = saved[3], &w = saved[4], &stats = saved[5];
        const bool has_bias = ctx->saved_data["bias"].toBool(), residual = ctx->saved_data["residual"].toBool();
        Sizes s;
        const c10::DeviceGuard on(x.device());
        const at::Tensor dy = incoming(grads[0], x);
        const bool bf16 = w.scalar_type() == at::kBFloat16;
        const at::ScalarType gdt = w.scalar_type();
        const bool usual = usual_backward(x, 1, cu, w, dy, &s) && vector_as(g, w, s.C) && (!beta.defined() || vector_as(beta, w, s.C)) &&
                           dense(stats, x.device()) && stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == s.T &&
                           stats.size(1) == 2;
        const size_t bytes = usual ? nplm_dwconv_ln_bwd_workspace_bytes(s.T, s.C, s.K, s.act) : 0;
        at::Tensor dx, dw, db, dg, dbeta;
        int rc = -NPLM_DWCONV_EUNSUPPORTED;
        // (under create_graph the op records itself, and says so if it is differentiated once more)
        if (bytes > 0 && !at::GradMode::is_enabled()) {
            const at::TensorOptions go = x.options().dtype(gdt);
            dx = at::empty({s.T, s.C}, x.options());
            dw = at::empty({s.C, s.K}, go);
            db = at::empty({s.C}, go);
            dg = at::empty({s.C}, go);
            if (beta.defined()) dbeta = at::empty({s.C}, go);
            const at::Tensor ws = scratch(bytes, x);
            rc = nplm_dwconv_ln_bwd(x.const_data_ptr(), dy.const_data_ptr(), ints(cu), stats.const_data_ptr<float>(), g.const_data_ptr(),
                                    beta.defined() ? beta.const_data_ptr() : nullptr, w.const_data_ptr(), dx.mutable_data_ptr(),
                                    (float*)dw.mutable_data_ptr(), (float*)db.mutable_data_ptr(), (float*)dg.mutable_data_ptr(),
                                    beta.defined() ? (float*)dbeta.mutable_data_ptr() : nullptr, ws.mutable_data_ptr(), (size_t)ws.numel(),
                                    s.T, s.C, s.K, s.S, s.act, s.wdt, flags_of(residual, bf16), stream_of(x));
        }
        if (rc == -NPLM_DWCONV_EUNSUPPORTED) {
            const OptTensor ob = beta.defined() ? OptTensor(beta) : OptTensor();
            const variable_list r = python_backward("nanoplm_amd.lnconv", "ln_dwconv_bwd_op", x, dy, cu, stats, g, ob, w, residual, bf16);
            dx = r[0], dg = r[1], dbeta = r[2], dw = r[3], db = r[4];
        } else {
            check(rc, "nplm_dwconv_ln_bwd");
        }
        return {dx, at::Tensor(), dg, beta.defined() ? dbeta : at::Tensor(), dw, has_bias ? db : at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

// What a recurrence call is, if everything about its tensors is as the kernels take it.
struct Recurrence {
    int64_t T;
    int32_t C, S, act, wdt;
};
bool recurrence_of(const at::Tensor& x, const at::Tensor& gates, const at::Tensor& cu, const at::Tensor& decay, const OptTensor& initial, Recurrence* r) {
    if (!x.is_cuda() || x.dim() != 2 || cu.dim() != 1 || x.size(1) < 1 || x.size(1) > NPLM_RECURRENCE_MAX_STRIDE / 2) return false;
    const at::Device dev = x.device();
    const int64_t T = x.size(0), C = x.size(1);
    r->act = dtype_code(x);
    r->wdt = dtype_code(decay);
    if (r->act < 0 || r->wdt < 0 || !rows(x, dev, T, C) || !rows(gates, dev, T, 2 * C) || gates.scalar_type() != x.scalar_type()) return false;
    if (!dense(decay, dev) || decay.dim() != 1 || decay.size(0) != C) return false;
    if (!dense(cu, dev) || cu.scalar_type() != at::kInt || cu.numel() < 1 || cu.numel() > INT_MAX) return false;
    const int64_t S = cu.numel() - 1;
    if (initial && (!dense(*initial, dev) || initial->scalar_type() != at::kFloat || initial->dim() != 2 || initial->size(0) != S || initial->size(1) != C))
        return false;
    r->T = T;
    r->C = (int32_t)C;
    r->S = (int32_t)S;
    return true;
}
at::Tensor workspace(size_t bytes, const at::Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}
void* at_of(const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const void* in_of(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct VarlenRecurrence : torch::autograd::Function<VarlenRecurrence> {
    // y and, if wanted, the last states; carries come back for the backward if there is to be one
    static variable_list run(const at::Tensor& x, const at::Tensor& gates, const at::Tensor& cu, const at::Tensor& decay, const OptTensor& initial,
                             double scale, bool reverse, bool want_state, at::Tensor* carries) {
        RECORD_FUNCTION("nanoplm_amd::varlen_recurrence_fwd", {});
        Recurrence r;
        recurrence_of(x, gates, cu, decay, initial, &r);
        const c10::DeviceGuard on(x.device());
        const at::TensorOptions f32 = x.options().dtype(at::kFloat);
        variable_list out{at::empty({r.T, r.C}, x.options())};
        if (want_state) out.push_back(at::empty({r.S, r.C}, f32));
        if (carries) *carries = at::empty({(r.T + NPLM_RECURRENCE_CHUNK - 1) / NPLM_RECURRENCE_CHUNK, r.C}, f32);
        const size_t bytes = nplm_recurrence_fwd_workspace_bytes(r.T, r.C, r.S, r.act);
        const at::Tensor ws = workspace(bytes, x);
        check(nplm_recurrence_fwd(x.const_data_ptr(), row_stride(x), gates.const_data_ptr(), row_stride(gates), ints(cu), decay.const_data_ptr(),
                                  (float)scale, (const float*)ptr(initial), out[0].mutable_data_ptr(), want_state ? out[1].mutable_data_ptr<float>() : nullptr,
                                  carries ? carries->mutable_data_ptr<float>() : nullptr, at_of(ws), bytes, r.T, r.C, r.S, r.act, r.wdt,
                                  reverse ? NPLM_RECURRENCE_REVERSE : 0u, stream_of(x)), "nplm_recurrence_fwd");
        return out;
    }
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gates, const at::Tensor& cu, const at::Tensor& decay,
                                 const OptTensor& initial, double scale, bool reverse, bool want_state) {
        at::Tensor carries;
        variable_list out = run(x, gates, cu, decay, initial, scale, reverse, want_state, &carries);
        ctx->save_for_backward({x, gates, cu, decay, initial ? *initial : at::Tensor(), carries});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["reverse"] = reverse;
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        RECORD_FUNCTION("nanoplm_amd::varlen_recurrence_bwd", {});
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &gates = saved[1], &cu = saved[2], &decay = saved[3], &initial = saved[4], &carries = saved[5];
        const double scale = ctx->saved_data["scale"].toDouble();
        const bool reverse = ctx->saved_data["reverse"].toBool(), want_initial = initial.defined() && ctx->needs_input_grad(4);
        const c10::DeviceGuard on(x.device());
        at::Tensor dy = !grads[0].defined() ? at::zeros_like(x) : grads[0].scalar_type() == x.scalar_type() ? grads[0] : grads[0].to(x.scalar_type());
        const at::Tensor dstate = grads.size() > 1 ? grads[1] : at::Tensor();
        auto state_like = [&](const at::Tensor& t, int64_t n) {
            return dense(t, x.device()) && t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == n && t.size(1) == x.size(1);
        };
        Recurrence r;
        // (under create_graph the op records itself, and says so if it is differentiated once more)
        if (observed() || at::GradMode::is_enabled() || !x.defined() || !recurrence_of(x, gates, cu, decay, opt(initial), &r) ||
            !state_like(carries, (r.T + NPLM_RECURRENCE_CHUNK - 1) / NPLM_RECURRENCE_CHUNK) || (dstate.defined() && !state_like(dstate, r.S)) ||
            dy.dim() != 2 || dy.size(0) != r.T || dy.size(1) != r.C || !rows(dy.stride(1) == 1 ? dy : dy = dy.contiguous(), x.device(), r.T, r.C)) {
            const variable_list out = python_backward("nanoplm_amd.recurrence", "varlen_recurrence_bwd_op", x, gates, dy, cu, decay, carries, opt(initial),
                                                      opt(dstate), scale, reverse);
            return {out[0], out[1], at::Tensor(), out[2], initial.defined() ? out[3] : at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        }
        const bool bf16 = decay.scalar_type() == at::kBFloat16;
        at::Tensor dx = at::empty({r.T, r.C}, x.options()), dgates = at::empty({r.T, 2 * (int64_t)r.C}, x.options());
        at::Tensor ddecay = at::empty({r.C}, decay.options()), dinitial;
        if (want_initial) dinitial = at::empty({r.S, r.C}, x.options().dtype(at::kFloat));
        const size_t bytes = nplm_recurrence_bwd_workspace_bytes(r.T, r.C, r.S, r.act);
        const at::Tensor ws = workspace(bytes, x);
        check(nplm_recurrence_bwd(x.const_data_ptr(), row_stride(x), gates.const_data_ptr(), row_stride(gates), dy.const_data_ptr(), row_stride(dy),
                                  ints(cu), decay.const_data_ptr(), (float)scale, (const float*)in_of(initial), (const float*)in_of(dstate),
                                  carries.const_data_ptr<float>(), dx.mutable_data_ptr(), dgates.mutable_data_ptr(), ddecay.mutable_data_ptr(),
                                  (float*)at_of(dinitial), at_of(ws), bytes, r.T, r.C, r.S, r.act, r.wdt,
                                  (reverse ? NPLM_RECURRENCE_REVERSE : 0u) | (bf16 ? NPLM_RECURRENCE_GRADS_BF16 : 0u), stream_of(x)), "nplm_recurrence_bwd");
        return {dx, dgates, at::Tensor(), ddecay, dinitial, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

// u, residual, gate and the five parameters of a residual norm, if they are as the kernels take them: parameters in one dtype.
struct ResNorm {
    int64_t T;
    int32_t C, act, st, wdt;
};
bool resnorm_of(const at::Tensor& u, const at::Tensor& residual, const at::Tensor& gate, const at::Tensor* const (&par)[5], ResNorm* r) {
    if (!u.is_cuda() || u.dim() != 2 || u.size(1) < 1 || u.size(1) > NPLM_RESNORM_MAX_C) return false;
    const at::Device dev = u.device();
    const int64_t T = u.size(0), C = u.size(1);
    r->act = dtype_code(u);
    r->st = dtype_code(residual);
    r->wdt = NPLM_DWCONV_F32;
    if (r->act < 0 || r->st < 0 || (r->act == NPLM_DWCONV_F32 && r->st != NPLM_DWCONV_F32)) return false;
    if (!rows(u, dev, T, C) || !rows(residual, dev, T, C)) return false;
    if (gate.defined() && (!rows(gate, dev, T, C) || gate.scalar_type() != u.scalar_type())) return false;
    const at::Tensor* first = nullptr;
    for (const at::Tensor* t : par)
        if (t->defined()) {
            if (!dense(*t, dev) || t->dim() != 1 || t->size(0) != C || (first && t->scalar_type() != first->scalar_type())) return false;
            first = t;
        }
    if (first && (r->wdt = dtype_code(*first)) < 0) return false;
    if ((par[1]->defined() && !par[0]->defined()) || (par[4]->defined() && !par[3]->defined())) return false;
    r->T = T;
    r->C = (int32_t)C;
    return true;
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list run(const at::Tensor& u, const at::Tensor& residual, const at::Tensor& gate, const at::Tensor& pw, const at::Tensor& pb,
                             const at::Tensor& scale, const at::Tensor& qw, const at::Tensor& qb, bool rms, double eps, at::Tensor* stats) {
        RECORD_FUNCTION("nanoplm_amd::residual_norm_fwd", {});
        ResNorm r;
        resnorm_of(u, residual, gate, {&pw, &pb, &scale, &qw, &qb}, &r);
        const c10::DeviceGuard on(u.device());
        variable_list out{at::empty({r.T, r.C}, residual.options())};
        if (qw.defined()) out.push_back(at::empty({r.T, r.C}, u.options()));
        if (stats) *stats = at::empty({r.T, 4}, u.options().dtype(at::kFloat));
        check(nplm_resnorm_fwd(u.const_data_ptr(), row_stride(u), in_of(gate), gate.defined() ? row_stride(gate) : 0, residual.const_data_ptr(),
                               row_stride(residual), in_of(pw), in_of(pb), in_of(scale), in_of(qw), in_of(qb), (float)eps, out[0].mutable_data_ptr(),
                               qw.defined() ? out[1].mutable_data_ptr() : nullptr, stats ? stats->mutable_data_ptr<float>() : nullptr, r.T, r.C, r.act,
                               r.st, r.wdt, rms ? NPLM_RESNORM_RMS : 0u, stream_of(u)), "nplm_resnorm_fwd");
        return out;
    }
    static variable_list forward(AutogradContext* ctx, const at::Tensor& u, const at::Tensor& residual, const OptTensor& gate, const OptTensor& pw,
                                 const OptTensor& pb, const OptTensor& scale, const OptTensor& qw, const OptTensor& qb, bool rms, double eps) {
        auto t = [](const OptTensor& o) { return o ? *o : at::Tensor(); };
        at::Tensor stats;
        variable_list out = run(u, residual, t(gate), t(pw), t(pb), t(scale), t(qw), t(qb), rms, eps, &stats);
        ctx->save_for_backward({u, residual, t(gate), t(pw), t(pb), t(scale), t(qw), t(qb), stats});
        ctx->saved_data["rms"] = rms;
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        RECORD_FUNCTION("nanoplm_amd::residual_norm_bwd", {});
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &u = saved[0], &residual = saved[1], &gate = saved[2], &stats = saved[8];
        const at::Tensor* const par[5] = {&saved[3], &saved[4], &saved[5], &saved[6], &saved[7]};
        const bool rms = ctx->saved_data["rms"].toBool();
        const c10::DeviceGuard on(u.device());
        auto incoming_or_none = [](const at::Tensor& d, const at::Tensor& like) { return !d.defined() || d.scalar_type() == like.scalar_type() ? d : d.to(like.scalar_type()); };
        at::Tensor dout = incoming_or_none(grads[0], residual), dn = grads.size() > 1 ? incoming_or_none(grads[1], u) : at::Tensor();
        ResNorm r;
        bool usual = !observed() && !at::GradMode::is_enabled() && u.defined() && resnorm_of(u, residual, gate, par, &r) && dense(stats, u.device()) &&
                     stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == r.T && stats.size(1) == 4;
        for (at::Tensor* d : {&dout, &dn})
            if (usual && d->defined()) {
                if (d->dim() == 2 && d->stride(1) != 1) *d = d->contiguous();
                usual = rows(*d, u.device(), r.T, r.C);
            }
        bool bf16 = true, wanted = false;
        int edge = gate.defined() ? 3 : 2;                  // (of the inputs that there are, in order)
        for (const at::Tensor* t : par)
            if (t->defined()) {
                bf16 = bf16 && t->scalar_type() == at::kBFloat16;
                wanted = ctx->needs_input_grad(edge++) || wanted;
            }
        variable_list out(10);
        if (!usual) {
            const variable_list g = python_backward("nanoplm_amd.resnorm", "residual_norm_bwd_op", u, residual, opt(gate), opt(*par[0]), opt(*par[1]),
                                                    opt(*par[2]), opt(*par[3]), stats, opt(dout), opt(dn), rms ? "rms" : "layer", par[4]->defined(), bf16);
            out[0] = g[0], out[1] = g[1];
            if (gate.defined()) out[2] = g[2];
            for (int i = 0; i < 5; ++i)
                if (par[i]->defined()) out[3 + i] = g[3 + i].to(par[i]->scalar_type());
            return out;
        }
        out[0] = at::empty({r.T, r.C}, u.options());
        out[1] = at::empty({r.T, r.C}, residual.options());
        if (gate.defined()) out[2] = at::empty({r.T, r.C}, u.options());
        for (int i = 0; i < 5; ++i)
            if (wanted && par[i]->defined()) out[3 + i] = at::empty({r.C}, par[i]->options());       // (all in one dtype)
        const size_t bytes = wanted ? nplm_resnorm_bwd_workspace_bytes(r.T, r.C) : 0;
        const at::Tensor ws = workspace(bytes, u);
        auto stride = [](const at::Tensor& t) { return t.defined() ? row_stride(t) : 0; };
        check(nplm_resnorm_bwd(u.const_data_ptr(), row_stride(u), in_of(gate), stride(gate), residual.const_data_ptr(), row_stride(residual), in_of(dout),
                               stride(dout), in_of(dn), stride(dn), stats.const_data_ptr<float>(), in_of(*par[0]), in_of(*par[1]), in_of(*par[2]),
                               in_of(*par[3]), out[0].mutable_data_ptr(), at_of(out[2]), out[1].mutable_data_ptr(), at_of(out[3]), at_of(out[4]),
                               at_of(out[5]), at_of(out[6]), at_of(out[7]), at_of(ws), bytes, r.T, r.C, r.act, r.st, r.wdt,
                               (rms ? NPLM_RESNORM_RMS : 0u) | (wanted && bf16 ? NPLM_RESNORM_GRADS_BF16 : 0u), stream_of(u)), "nplm_resnorm_bwd");
        return out;
    }
};
}  // namespace nanoplm_amd

namespace {

bool tensor_arg(PyObject* o, at::Tensor* t) {
    if (!THPVariable_CheckExact(o)) return false;
    *t = THPVariable_Unpack(o);
    return true;
}
bool tensor_arg(PyObject* o, OptTensor* t) {
    if (o == Py_None) return true;
    if (!THPVariable_CheckExact(o)) return false;
    *t = THPVariable_Unpack(o);
    return true;
}
bool wants_grad(const OptTensor& t) { return t && t->requires_grad(); }

// (x or z, cu_seqlens, weight, bias or None, residual) -> y, or None
template <typename Node, int WIDTH>
PyObject* conv(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 5, "5 arguments");
    at::Tensor x, cu, w, y;
    OptTensor b;
    Sizes s;
    if (observed() || !tensor_arg(a[0], &x) || !tensor_arg(a[1], &cu) || !tensor_arg(a[2], &w) || !tensor_arg(a[3], &b)) Py_RETURN_NONE;
    const int residual = PyObject_IsTrue(a[4]);
    if (residual < 0) return nullptr;
    if (!sizes_of(x, WIDTH, cu, w, b, &s)) Py_RETURN_NONE;
    // (asked first: a forward of the composed route would start with an allocation and an exception here, 4 us)
    if (WIDTH == 2 && (s.T == 0 || !aligned16(x) || nplm_dwconv_gated_bwd_workspace_bytes(s.T, s.C, s.K, s.act) == 0)) Py_RETURN_NONE;
    try {
        pybind11::gil_scoped_release no_gil;
        const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || wants_grad(b));
        y = grad ? Node::apply(x, cu, w, b, residual != 0) : Node::run(x, cu, w, b, residual != 0);
    } catch (const Unsupported&) {
        Py_RETURN_NONE;
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// (x, cu_seqlens, ln_weight, ln_bias or None, weight, bias or None, eps, residual) -> y, or None
PyObject* prenorm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 8, "8 arguments");
    at::Tensor x, cu, g, w, y, stats;
    OptTensor beta, b;
    Sizes s;
    if (observed() || !tensor_arg(a[0], &x) || !tensor_arg(a[1], &cu) || !tensor_arg(a[2], &g) || !tensor_arg(a[3], &beta) ||
        !tensor_arg(a[4], &w) || !tensor_arg(a[5], &b)) Py_RETURN_NONE;
    const double eps = PyFloat_AsDouble(a[6]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    const int residual = PyObject_IsTrue(a[7]);
    if (residual < 0) return nullptr;
    if (!sizes_of(x, 1, cu, w, b, &s) || s.T == 0 || !aligned16(x)) Py_RETURN_NONE;
    for (const at::Tensor& t : {g, beta ? *beta : g})        // (one dtype for all parameters)
        if (!vector_as(t, w, s.C)) Py_RETURN_NONE;
    if (nplm_dwconv_ln_bwd_workspace_bytes(s.T, s.C, s.K, s.act) == 0) Py_RETURN_NONE;
    try {
        pybind11::gil_scoped_release no_gil;
        const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || g.requires_grad() || wants_grad(beta) || wants_grad(b));
        y = grad ? nanoplm_amd::LnVarlenDWConv1d::apply(x, cu, g, beta, w, b, eps, residual != 0) : nanoplm_amd::LnVarlenDWConv1d::run(x, cu, g, beta, w, b, eps, residual != 0, &stats);
    } catch (const Unsupported&) {
        Py_RETURN_NONE;
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

PyObject* pair_of(const variable_list& out) {
    PyObject* second = out.size() > 1 ? THPVariable_Wrap(out[1]) : (Py_INCREF(Py_None), Py_None);
    return Py_BuildValue("(NN)", THPVariable_Wrap(out[0]), second);
}

// (x, gates, cu_seqlens, decay, initial_state or None, scale, reverse, return_state) -> (y, state or None), or None
PyObject* recurrence(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 8, "8 arguments");
    at::Tensor x, gates, cu, decay;
    OptTensor initial;
    nanoplm_amd::Recurrence r;
    if (observed() || !tensor_arg(a[0], &x) || !tensor_arg(a[1], &gates) || !tensor_arg(a[2], &cu) || !tensor_arg(a[3], &decay) || !tensor_arg(a[4], &initial))
        Py_RETURN_NONE;
    const double scale = PyFloat_AsDouble(a[5]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    const int reverse = PyObject_IsTrue(a[6]), want_state = PyObject_IsTrue(a[7]);
    if (reverse < 0 || want_state < 0) return nullptr;
    if (!(scale > 0.0 && scale < INFINITY) || !nanoplm_amd::recurrence_of(x, gates, cu, decay, initial, &r)) Py_RETURN_NONE;
    for (const at::Tensor* t : {&x, &gates})                // (a stride that the library refuses is refused with its message)
        if (row_stride(*t) > NPLM_RECURRENCE_MAX_STRIDE) Py_RETURN_NONE;
    variable_list out;
    {
        pybind11::gil_scoped_release no_gil;
        const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || gates.requires_grad() || decay.requires_grad() || wants_grad(initial));
        out = grad ? nanoplm_amd::VarlenRecurrence::apply(x, gates, cu, decay, initial, scale, reverse != 0, want_state != 0)
                   : nanoplm_amd::VarlenRecurrence::run(x, gates, cu, decay, initial, scale, reverse != 0, want_state != 0, nullptr);
    }
    return pair_of(out);
    END_HANDLE_TH_ERRORS
}

// (u, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias, each of the last six or None, rms, eps) -> (stream, normed or None), or None
PyObject* residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 10, "10 arguments");
    at::Tensor u, residual;
    OptTensor o[6];
    nanoplm_amd::ResNorm r;
    if (observed() || !tensor_arg(a[0], &u) || !tensor_arg(a[1], &residual)) Py_RETURN_NONE;
    bool grad = u.requires_grad() || residual.requires_grad();
    at::Tensor t[6];
    for (int i = 0; i < 6; ++i) {
        if (!tensor_arg(a[2 + i], &o[i])) Py_RETURN_NONE;
        if (o[i]) t[i] = *o[i];
        grad = grad || wants_grad(o[i]);
    }
    const int rms = PyObject_IsTrue(a[8]);
    const double eps = PyFloat_AsDouble(a[9]);
    if (rms < 0 || (eps == -1.0 && PyErr_Occurred())) return nullptr;
    if (!(eps >= 0.0 && eps < INFINITY) || !nanoplm_amd::resnorm_of(u, residual, t[0], {&t[1], &t[2], &t[3], &t[4], &t[5]}, &r)) Py_RETURN_NONE;
    variable_list out;
    {
        pybind11::gil_scoped_release no_gil;
        out = grad && at::GradMode::is_enabled() ? nanoplm_amd::ResidualNorm::apply(u, residual, o[0], o[1], o[2], o[3], o[4], o[5], rms != 0, eps)
                                                 : nanoplm_amd::ResidualNorm::run(u, residual, t[0], t[1], t[2], t[3], t[4], t[5], rms != 0, eps, nullptr);
    }
    return pair_of(out);
    END_HANDLE_TH_ERRORS
}

// (x, gates, decay, state, slots or None, scale, out_state or None) -> y, or None
PyObject* recurrence_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK_TYPE(n == 7, "7 arguments");
    at::Tensor x, gates, decay, state;
    OptTensor slots, other;
    if (observed() || !tensor_arg(a[0], &x) || !tensor_arg(a[1], &gates) || !tensor_arg(a[2], &decay) || !tensor_arg(a[3], &state) ||
        !tensor_arg(a[4], &slots) || !tensor_arg(a[6], &other)) Py_RETURN_NONE;
    const double scale = PyFloat_AsDouble(a[5]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    if (!x.is_cuda() || x.dim() != 2 || x.size(1) < 1 || x.size(1) > NPLM_RECURRENCE_MAX_STRIDE / 2 || x.size(0) > INT_MAX) Py_RETURN_NONE;
    const at::Device dev = x.device();
    const int64_t B = x.size(0), C = x.size(1);
    const int act = dtype_code(x), wdt = dtype_code(decay);
    if (!(scale > 0.0 && scale < INFINITY) || act < 0 || wdt < 0 || !rows(x, dev, B, C) || !rows(gates, dev, B, 2 * C) || gates.scalar_type() != x.scalar_type() ||
        !dense(decay, dev) || decay.dim() != 1 || decay.size(0) != C) Py_RETURN_NONE;
    const at::Tensor out_state = other ? *other : state;
    for (const at::Tensor* t : {(const at::Tensor*)&state, &out_state})
        if (!dense(*t, dev) || t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(1) != C || t->size(0) != state.size(0) || t->size(0) > INT_MAX) Py_RETURN_NONE;
    const uintptr_t from = (uintptr_t)state.const_data_ptr(), to = (uintptr_t)out_state.const_data_ptr();
    if (from != to && (from < to ? to - from : from - to) < state.nbytes()) Py_RETURN_NONE;      // (two tables, but not apart)
    if (slots ? B > NPLM_RECURRENCE_MAX_SLOTS || !dense(*slots, dev) || slots->scalar_type() != at::kInt || slots->dim() != 1 || slots->size(0) != B : B > state.size(0)) Py_RETURN_NONE;
    if (at::GradMode::is_enabled() && (x.requires_grad() || gates.requires_grad() || decay.requires_grad() || state.requires_grad() || out_state.requires_grad()))
        Py_RETURN_NONE;
    for (const at::Tensor* t : {&x, &gates})
        if (row_stride(*t) > NPLM_RECURRENCE_MAX_STRIDE) Py_RETURN_NONE;
    at::Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        RECORD_FUNCTION("nanoplm_amd::recurrence_step", {});
        const c10::DeviceGuard on(dev);
        y = at::empty({B, C}, x.options());
        if (!out_state.is_inference()) out_state.unsafeGetTensorImpl()->bump_version();      // (a graph that has saved the table says so)
        check(nplm_recurrence_step(x.const_data_ptr(), row_stride(x), gates.const_data_ptr(), row_stride(gates), decay.const_data_ptr(), (float)scale,
                                   state.const_data_ptr<float>(), out_state.mutable_data_ptr<float>(), slots ? ints(*slots) : nullptr, y.mutable_data_ptr(), B,
                                   (int32_t)C, state.size(0), act, wdt, stream_of(x)), "nplm_recurrence_step");
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"dwconv", (PyCFunction)(void (*)(void))&conv<nanoplm_amd::VarlenDWConv1d, 1>, METH_FASTCALL, "y = conv(x), differentiable; None: take the Python route"},
    {"gated_dwconv", (PyCFunction)(void (*)(void))&conv<nanoplm_amd::GatedVarlenDWConv1d, 2>, METH_FASTCALL, "y = conv(u * silu(g)), differentiable; None: take the Python route"},
    {"ln_dwconv", (PyCFunction)(void (*)(void))&prenorm, METH_FASTCALL, "y = conv(layer_norm(x)), differentiable; None: take the Python route"},
    {"recurrence", (PyCFunction)(void (*)(void))&recurrence, METH_FASTCALL, "(y, state), differentiable; None: take the Python route"},
    {"recurrence_step", (PyCFunction)(void (*)(void))&recurrence_step, METH_FASTCALL, "y of one token of each sequence; None: take the Python route"},
    {"residual_norm", (PyCFunction)(void (*)(void))&residual_norm, METH_FASTCALL, "(stream, normed), differentiable; None: take the Python route"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_node", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__node() {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) != 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
