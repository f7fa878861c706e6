// The common calls of flash_attention_v100() as a native autograd operator: fp16, bf16 or fp32 tensors on one GPU as the
// kernels take them, without bias or dropout.  attention() checks whether a call is one of these and answers None where
// it is not; ops/attention.py's Function then takes the call, with its messages, its other options and its error cases.
//
// What it is for: the Python operator is 40 us of host work around a forward and 150 around a training step (argument
// checks, a ctypes block, the Python side of autograd), more than the kernels of a short call take.  B200: a prompt of
// B1 N128 H8 D64 39 -> 10 us, a training step of B32 N197 H12 D64 157 -> 95 (bound by its kernels then).
//
// Beside it attention_rules(), rotary() and key_ranges(), the common forms of flash_attention_v100_with_rules(),
// rotary_embedding() and build_key_ranges(), whose small calls are host work alone.
//
// Replaces, for the first, the reference's autograd.Function (ops/attention.py:36-333).
#include <ATen/FunctionalTensorWrapper.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/PythonFallbackKernel.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <atomic>
#include <cmath>
#include <cstring>
#include "../../include/fa_b200.h"

namespace py = pybind11;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

constexpr int kMaxDevices = 64;
constexpr size_t kF32PlanesMaxBytes = (size_t)8 << 30;      // as F32_PLANES_MAX_BYTES in ops/attention.py
std::atomic<int32_t*> g_status_word[kMaxDevices];           // pinned, one per device, held by ops/attention.py

// The exception types of kernels/_cabi.py; may run in an autograd thread.
void raise_for_status(int rc, const char* what) {
    if (rc == FA_OK) return;
    const std::string msg = std::string(what) + ": " + fa_b200_strerror(rc) + ": " + fa_b200_last_error();
    py::gil_scoped_acquire gil;
    const bool value = rc == FA_EINVAL || rc == FA_EUNSUPPORTED || rc == FA_EALIGN;
    PyErr_SetString(value ? PyExc_ValueError : PyExc_RuntimeError, msg.c_str());
    python_error err;
    err.persist();
    throw err;
}

// Unit stride on the head dimension, 16-byte rows: what utils.py passes to the kernels untouched.
bool rows_fit(const at::Tensor& t) {
    uintptr_t bits = (uintptr_t)t.const_data_ptr();
    for (int i = 0; i < 3; ++i) bits |= (uintptr_t)(t.stride(i) * t.element_size());
    return t.stride(3) == 1 && (bits & 15u) == 0;
}

fa_b200_tensor operand(const at::Tensor& t) { return {const_cast<void*>(t.const_data_ptr()), t.stride(0), t.stride(1), t.stride(2)}; }

struct Call {
    double scale;
    bool causal, fast;
    int64_t shift;
    at::Tensor lengths;         // may be undefined
};

fa_b200_params params_of(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& o, const at::Tensor& lse, const Call& c) {
    fa_b200_params p;
    memset(&p, 0, sizeof(p));
    p.struct_bytes = sizeof(p);
    p.q = operand(q); p.k = operand(k); p.v = operand(v); p.o = operand(o);
    p.lse = lse.mutable_data_ptr<float>();
    const int device = q.device().index();
    p.status_word = g_status_word[device].load(std::memory_order_acquire);
    p.stream = c10::cuda::getCurrentCUDAStream(device).stream();
    p.B = (int32_t)q.size(0); p.Nq = (int32_t)q.size(1); p.Nk = (int32_t)k.size(1);
    p.H = (int32_t)q.size(2); p.Hkv = (int32_t)k.size(2); p.D = (int32_t)q.size(3);
    p.dtype = q.scalar_type() == at::kHalf ? FA_B200_F16 : (q.scalar_type() == at::kBFloat16 ? FA_B200_BF16 : FA_B200_F32);
    p.causal = c.causal;
    p.variant = FA_B200_VARIANT_AUTO;
    p.device = device;
    p.scale = (float)c.scale;
    p.causal_shift = c.causal ? (int32_t)c.shift : 0;
    if (c.lengths.defined()) p.kv_lengths = c.lengths.const_data_ptr<int32_t>();
    return p;
}

at::Tensor bytes_like(const at::Tensor& q, size_t n) { return at::empty({(int64_t)n}, q.options().dtype(at::kByte)); }

// o, lse and, for a bf16 call whose gradients will be asked for, what rounding o dropped.  `split`: the keys of a call with
// few queries may be shared out over the SMs (calls whose inputs want gradients keep whole pairs of tiles).
void forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Call& c, bool split, bool residual, at::Tensor& o, at::Tensor& lse,
             at::Tensor& o_lo) {
    o = at::empty(q.sizes(), q.options());
    lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    fa_b200_params p = params_of(q, k, v, o, lse, c);
    if (residual) { o_lo = at::empty(q.sizes(), q.options()); p.o_lo = operand(o_lo); }
    const size_t n = split ? fa_b200_fwd_workspace_bytes(&p) : 0;
    if (n) {
        const at::Tensor ws = bytes_like(q, n);
        raise_for_status(fa_b200_fwd_with_workspace(&p, ws.mutable_data_ptr(), n), "fa_b200_fwd");
    } else {
        raise_for_status(fa_b200_fwd(&p), "fa_b200_fwd");
    }
}

void backward(at::Tensor d_o, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& o, const at::Tensor& lse,
              const at::Tensor& o_lo, const Call& c, at::Tensor& dq, at::Tensor& dk, at::Tensor& dv) {
    if (!rows_fit(d_o)) d_o = d_o.contiguous();
    dq = at::empty(q.sizes(), q.options()); dk = at::empty(k.sizes(), k.options()); dv = at::empty(v.sizes(), v.options());
    fa_b200_params p = params_of(q, k, v, o, lse, c);
    p.d_o = operand(d_o); p.dq = operand(dq); p.dk = operand(dk); p.dv = operand(dv);
    const bool f32 = q.scalar_type() == at::kFloat;
    if (c.fast && !f32 && q.size(3) == 64) p.variant = FA_B200_VARIANT_TCGEN05;
    if (o_lo.defined()) p.o_lo = operand(o_lo);
    if (f32) {
        // planes for the tensor-core kernels, up to a limit and as far as the allocator goes
        const size_t n = fa_b200_bwd_scratch_bytes(&p);
        at::Tensor ws;
        if (n && n <= kF32PlanesMaxBytes) {
            try { ws = bytes_like(q, n); } catch (const c10::OutOfMemoryError&) {}
        }
        if (ws.defined()) { raise_for_status(fa_b200_bwd_with_scratch(&p, ws.mutable_data_ptr(), n), "fa_b200_bwd"); return; }
    }
    const size_t n = fa_b200_bwd_workspace_bytes(&p);
    const at::Tensor ws = bytes_like(q, n);
    p.workspace = ws.mutable_data_ptr();
    p.workspace_bytes = n;
    raise_for_status(fa_b200_bwd(&p), "fa_b200_bwd");
}

// A gradient computed outside of autograd where its own gradient may be asked for (create_graph): it would look like a constant,
// and a loss that uses it would lose its part without a word.  A node that throws between it and what it is made of.  (As
// last_derivative in utils.py.)
struct LastGradient : torch::autograd::Function<LastGradient> {
    static at::Tensor forward(AutogradContext*, const at::Tensor& gradient, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&) {
        return gradient.variable_data();                 // (no view: a caller may write to it)
    }
    static variable_list backward(AutogradContext*, variable_list) {
        TORCH_CHECK(false, "these kernels have no gradient of a gradient: a second derivative through attention is not available");
    }
};
variable_list last_derivative(variable_list out, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& d_o) {
    if (at::GradMode::is_enabled())
        for (at::Tensor& g : out)
            if (g.defined()) g = LastGradient::apply(g, q, k, v, d_o);
    return out;
}

struct Attention : torch::autograd::Function<Attention> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Call& c) {
        at::Tensor o, lse, o_lo;
        ::forward(q, k, v, c, false, q.scalar_type() == at::kBFloat16, o, lse, o_lo);
        variable_list kept{q, k, v, o, lse};
        if (o_lo.defined()) kept.push_back(o_lo);
        ctx->save_for_backward(std::move(kept));
        ctx->saved_data["scale"] = c.scale;
        ctx->saved_data["flags"] = (int64_t)c.causal | ((int64_t)c.fast << 1) | (c.shift << 2);
        if (c.lengths.defined()) ctx->saved_data["lengths"] = c.lengths;
        ctx->mark_non_differentiable({lse});
        ctx->set_materialize_grads(false);             // (lse's would be a launch of zeros)
        return {o, lse};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list kept = ctx->get_saved_variables();
        const int64_t flags = ctx->saved_data["flags"].toInt();
        const auto lengths = ctx->saved_data.find("lengths");
        const Call c{ctx->saved_data["scale"].toDouble(), (flags & 1) != 0, (flags & 2) != 0, flags >> 2,
                     lengths == ctx->saved_data.end() ? at::Tensor() : lengths->second.toTensor()};
        variable_list out(4);
        {
            at::Tensor d[3];
            at::AutoDispatchBelowADInplaceOrView below;          // (allocations and a copy: nothing of this is recorded)
            if (!grads[0].defined()) grads[0] = at::zeros_like(kept[3]);
            ::backward(grads[0], kept[0], kept[1], kept[2], kept[3], kept[4], kept.size() > 5 ? kept[5] : at::Tensor(), c, d[0], d[1], d[2]);
            for (int i = 0; i < 3; ++i)
                if (ctx->needs_input_grad(i)) out[i] = d[i];
        }
        return last_derivative(std::move(out), kept[0], kept[1], kept[2], grads[0]);
    }
};

// ---- calls with rules (ops/rules.py), rotary positions (ops/rotary.py), key ranges (ops/key_ranges.py): the same division,
// their Python forms take what is refused here ----
struct Ruled {
    double scale, cap;
    int64_t plan_batch, max_keys;
    at::Tensor slopes, plan;    // slopes may be undefined
};

fa_b200_rules rules_of(const Ruled& r) {
    return {sizeof(fa_b200_rules), r.plan.const_data_ptr(), (int32_t)r.plan_batch, (float)r.cap,
            r.slopes.defined() ? r.slopes.const_data_ptr<float>() : nullptr, (int32_t)r.max_keys, 0};
}

void ruled_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Ruled& r, bool split, bool residual, at::Tensor& o, at::Tensor& lse,
                   at::Tensor& o_lo) {
    o = at::empty(q.sizes(), q.options());
    lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    fa_b200_params p = params_of(q, k, v, o, lse, Call{r.scale, false, false, 0, {}});
    if (residual) { o_lo = at::empty(q.sizes(), q.options()); p.o_lo = operand(o_lo); }
    const fa_b200_rules u = rules_of(r);
    const size_t n = split ? fa_b200_fwd_rules_workspace_bytes(&p, &u) : 0;
    at::Tensor ws;
    if (n) ws = bytes_like(q, n);
    raise_for_status(fa_b200_fwd_with_rules(&p, &u, n ? ws.mutable_data_ptr() : nullptr, n), "fa_b200_fwd_with_rules");
}

void ruled_backward(at::Tensor d_o, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& o, const at::Tensor& lse,
                    const at::Tensor& o_lo, const Ruled& r, at::Tensor& dq, at::Tensor& dk, at::Tensor& dv) {
    if (!rows_fit(d_o)) d_o = d_o.contiguous();
    dq = at::empty(q.sizes(), q.options()); dk = at::empty(k.sizes(), k.options()); dv = at::empty(v.sizes(), v.options());
    fa_b200_params p = params_of(q, k, v, o, lse, Call{r.scale, false, false, 0, {}});
    p.d_o = operand(d_o); p.dq = operand(dq); p.dk = operand(dk); p.dv = operand(dv);
    if (o_lo.defined()) p.o_lo = operand(o_lo);
    const fa_b200_rules u = rules_of(r);
    const size_t n = fa_b200_bwd_rules_workspace_bytes(&p);
    const at::Tensor ws = bytes_like(q, n);
    p.workspace = ws.mutable_data_ptr();
    p.workspace_bytes = n;
    raise_for_status(fa_b200_bwd_with_rules(&p, &u), "fa_b200_bwd_with_rules");
}

struct RuledAttention : torch::autograd::Function<RuledAttention> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Ruled& r) {
        at::Tensor o, lse, o_lo;
        ruled_forward(q, k, v, r, false, q.scalar_type() != at::kFloat, o, lse, o_lo);
        ctx->save_for_backward({q, k, v, o, lse, r.plan, o_lo, r.slopes});
        ctx->saved_data["scale"] = r.scale;
        ctx->saved_data["cap"] = r.cap;
        ctx->saved_data["batch"] = r.plan_batch;
        ctx->mark_non_differentiable({lse});
        ctx->set_materialize_grads(false);
        return {o, lse};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(4);
        if (!grads[0].defined()) return out;
        const variable_list kept = ctx->get_saved_variables();
        const Ruled r{ctx->saved_data["scale"].toDouble(), ctx->saved_data["cap"].toDouble(), ctx->saved_data["batch"].toInt(), 0, kept[7], kept[5]};
        {
            at::Tensor d[3];
            at::AutoDispatchBelowADInplaceOrView below;
            ruled_backward(grads[0], kept[0], kept[1], kept[2], kept[3], kept[4], kept[6], r, d[0], d[1], d[2]);
            for (int i = 0; i < 3; ++i)
                if (ctx->needs_input_grad(i)) out[i] = d[i];
        }
        return last_derivative(std::move(out), kept[0], kept[1], kept[2], grads[0]);
    }
};

struct Turn {
    at::Tensor positions, inv_freq;      // positions may be undefined
    int64_t offset;
    bool interleaved, inverse;
    double factor;
};

void turn(const at::Tensor* x, const at::Tensor* y, int n, const Turn& t) {
    fa_b200_rotary_params p;
    memset(&p, 0, sizeof(p));
    p.struct_bytes = sizeof(p);
    for (int i = 0; i < n; ++i) { p.x[i] = operand(x[i]); p.y[i] = operand(y[i]); p.heads[i] = (int32_t)x[i].size(2); }
    if (t.positions.defined()) {
        p.positions = t.positions.const_data_ptr();
        p.positions_64bit = t.positions.scalar_type() == at::kLong;
        p.positions_stride_n = t.positions.stride(-1);
        p.positions_stride_b = t.positions.dim() == 2 && t.positions.size(0) > 1 ? t.positions.stride(0) : 0;
    }
    p.position0 = t.offset;
    p.inv_freq = t.inv_freq.const_data_ptr<double>();
    p.B = (int32_t)x[0].size(0); p.N = (int32_t)x[0].size(1); p.D = (int32_t)x[0].size(3); p.half = (int32_t)t.inv_freq.size(0);
    p.interleaved = t.interleaved; p.inverse = t.inverse; p.factor = (float)t.factor;
    const auto type = x[0].scalar_type();
    p.dtype = type == at::kHalf ? FA_B200_F16 : (type == at::kBFloat16 ? FA_B200_BF16 : FA_B200_F32);
    p.device = x[0].device().index();
    p.stream = c10::cuda::getCurrentCUDAStream(p.device).stream();
    raise_for_status(fa_b200_rotary(&p), "fa_b200_rotary");
}

// One or two tensors turned, and their gradients: the turn back, which has a gradient of its own.
template <int N>
struct Rotary : torch::autograd::Function<Rotary<N>> {
    template <typename... Tensors>
    static variable_list forward(AutogradContext* ctx, const Turn& t, const Tensors&... xs) {
        const at::Tensor x[N] = {xs...};
        at::Tensor y[N];
        for (int i = 0; i < N; ++i) y[i] = at::empty(x[i].sizes(), x[i].options());
        turn(x, y, N, t);
        ctx->save_for_backward({t.positions, t.inv_freq});
        ctx->saved_data["offset"] = t.offset;
        ctx->saved_data["interleaved"] = t.interleaved;
        ctx->saved_data["inverse"] = t.inverse;
        ctx->saved_data["factor"] = t.factor;
        ctx->set_materialize_grads(false);
        return variable_list(y, y + N);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads);
};
variable_list turned(const at::Tensor* x, int n, const Turn& t) { return n == 1 ? Rotary<1>::apply(t, x[0]) : Rotary<2>::apply(t, x[0], x[1]); }

template <int N>
variable_list Rotary<N>::backward(AutogradContext* ctx, variable_list grads) {
    const variable_list kept = ctx->get_saved_variables();
    const Turn t{kept[0], kept[1], ctx->saved_data["offset"].toInt(), ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool(),
                 ctx->saved_data["factor"].toDouble()};
    at::Tensor g[N], d[N];
    int which[N], n = 0;
    bool again = false;                  // (create_graph)
    for (int i = 0; i < N; ++i)
        if (grads[i].defined() && ctx->needs_input_grad(i)) {          // (counts tensors)
            g[n] = grads[i].stride(3) == 1 ? grads[i] : grads[i].contiguous();
            again |= at::GradMode::is_enabled() && g[n].requires_grad();
            which[n++] = i;
        }
    variable_list out(N + 1);            // (counts arguments)
    if (again) {
        const variable_list back = turned(g, n, t);
        for (int i = 0; i < n; ++i) out[which[i] + 1] = back[i];
    } else if (n) {
        at::AutoDispatchBelowADInplaceOrView below;
        for (int i = 0; i < n; ++i) d[i] = at::empty(g[i].sizes(), g[i].options());
        turn(g, d, n, t);
        for (int i = 0; i < n; ++i) out[which[i] + 1] = d[i];
    }
    return out;
}

// A plain tensor on a GPU: no subclass, no wrapper, no dual number, no bits to be resolved first.
bool plain(PyObject* obj, const at::Tensor*& t) {
    if (!THPVariable_CheckExact(obj)) return false;
    t = &THPVariable_Unpack(obj);
    const auto keys = t->key_set();
    return t->is_cuda() && t->layout() == at::kStrided && !t->is_conj() && !t->is_neg() && !t->_is_zerotensor() &&
           !keys.has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched,
                                              c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched})) &&
           !t->_fw_grad(0).defined();
}

// Whether something else wants to see the call's operators: a transform, a tracer, a mode.
bool watched() {
    return c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchVmapMode) ||
           c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Functionalize) || at::tracer::impl::is_dispatch_enabled();
}

py::object wrap(at::Tensor t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(t))); }

// q, k and v of a call the kernels take as they are.
bool served(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
    const auto type = q.scalar_type();
    if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || k.sizes() != v.sizes() || q.size(0) != k.size(0) || q.size(3) != k.size(3) ||
        k.size(2) == 0 || q.size(2) % k.size(2) != 0 || q.numel() == 0 || k.numel() == 0 || q.size(3) > 128 ||
        (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) || k.scalar_type() != type || v.scalar_type() != type ||
        k.device() != q.device() || v.device() != q.device() || !rows_fit(q) || !rows_fit(k) || !rows_fit(v))
        return false;
    for (const at::Tensor* t : {&q, &k})
        if (t->size(0) > INT32_MAX || t->size(1) > INT32_MAX || t->size(2) > INT32_MAX) return false;
    return true;
}

// (o, lse), or None where the call is not one of those served here.
py::object attention(py::handle q_, py::handle k_, py::handle v_, py::handle scale_, bool causal, bool bottom_right, py::handle lengths_, bool fast) {
    const at::Tensor *qp, *kp, *vp, *lp = nullptr;
    if (watched() || !plain(q_.ptr(), qp) || !plain(k_.ptr(), kp) || !plain(v_.ptr(), vp)) return py::none();
    const at::Tensor q = *qp, k = *kp, v = *vp;          // (own references: other threads run during the call)
    if (!served(q, k, v)) return py::none();
    const int device = q.device().index();
    if (device >= kMaxDevices || !g_status_word[device].load(std::memory_order_acquire)) return py::none();
    Call c{std::pow((double)q.size(3), -0.5), causal, fast, 0, {}};
    if (!scale_.is_none()) {
        if (!PyFloat_CheckExact(scale_.ptr())) return py::none();
        c.scale = PyFloat_AS_DOUBLE(scale_.ptr());
    }
    if (!lengths_.is_none()) {
        if (!plain(lengths_.ptr(), lp) || lp->scalar_type() != at::kInt || lp->device() != q.device() || lp->dim() != 1 || lp->size(0) != q.size(0) ||
            !lp->is_contiguous())
            return py::none();
        c.lengths = lp->detach();
    }
    if (causal && bottom_right) {
        if (k.size(1) < q.size(1) || lp) return py::none();
        c.shift = k.size(1) - q.size(1);
    }
    const bool wants = q.requires_grad() || k.requires_grad() || v.requires_grad();
    at::Tensor o, lse, o_lo;
    try {
        // Allocation and launches may have to wait (for memory, for room in the launch queue): other Python threads, which
        // may be what the GPU waits for, run meanwhile.
        py::gil_scoped_release others_run;
        if (wants && at::GradMode::is_enabled()) {
            variable_list out = Attention::apply(q, k, v, c);
            o = std::move(out[0]); lse = std::move(out[1]);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            forward(q, k, v, c, !wants, false, o, lse, o_lo);
        }
    } catch (python_error& e) {
        e.restore();
        throw py::error_already_set();
    }
    return py::make_tuple(wrap(std::move(o)), wrap(std::move(lse)));
}

// Runs what may have to wait without the lock, and gives its Python exceptions back.
template <typename F> void unlocked(F f) {
    try {
        py::gil_scoped_release others_run;
        f();
    } catch (python_error& e) {
        e.restore();
        throw py::error_already_set();
    }
}

// (o, lse) of flash_attention_v100_with_rules, or None.  seq_q, seq_k: the plan's.
py::object attention_rules(py::handle q_, py::handle k_, py::handle v_, py::handle scale_, py::handle cap_, py::handle slopes_, py::handle plan_, int64_t batch,
                           int64_t seq_q, int64_t seq_k, int64_t max_keys) {
    const at::Tensor *qp, *kp, *vp, *sp, *pp;
    if (watched() || !plain(q_.ptr(), qp) || !plain(k_.ptr(), kp) || !plain(v_.ptr(), vp) || !plain(plan_.ptr(), pp)) return py::none();
    const at::Tensor q = *qp, k = *kp, v = *vp;
    if (!served(q, k, v)) return py::none();
    const int device = q.device().index();
    if (device >= kMaxDevices || !g_status_word[device].load(std::memory_order_acquire)) return py::none();
    Ruled r{std::pow((double)q.size(3), -0.5), 0.0, batch, max_keys, {}, *pp};
    if (q.size(1) != seq_q || k.size(1) != seq_k || (batch != 1 && batch != q.size(0)) || r.plan.device() != q.device() || r.plan.scalar_type() != at::kInt ||
        !r.plan.is_contiguous() || (size_t)r.plan.numel() * 4 < fa_b200_key_ranges_bytes((int)batch, (int)seq_q, (int)seq_k))
        return py::none();
    if (!scale_.is_none()) {
        if (!PyFloat_CheckExact(scale_.ptr())) return py::none();
        r.scale = PyFloat_AS_DOUBLE(scale_.ptr());
    }
    if (!cap_.is_none()) {
        if (!PyFloat_CheckExact(cap_.ptr())) return py::none();
        r.cap = PyFloat_AS_DOUBLE(cap_.ptr());
        if (!((float)r.cap > 0.f && r.cap < 1e30)) return py::none();
    }
    if (!slopes_.is_none()) {
        if (!plain(slopes_.ptr(), sp) || sp->scalar_type() != at::kFloat || sp->device() != q.device() || sp->dim() != 1 || sp->size(0) != q.size(2) ||
            !sp->is_contiguous() || sp->requires_grad())
            return py::none();
        r.slopes = *sp;
    }
    const bool wants = q.requires_grad() || k.requires_grad() || v.requires_grad();
    at::Tensor o, lse, o_lo;
    unlocked([&] {
        if (wants && at::GradMode::is_enabled()) {
            variable_list out = RuledAttention::apply(q, k, v, r);
            o = std::move(out[0]); lse = std::move(out[1]);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            ruled_forward(q, k, v, r, true, false, o, lse, o_lo);
        }
    });
    return py::make_tuple(wrap(std::move(o)), wrap(std::move(lse)));
}

// The turned q, or (q, k), or None.
py::object rotary(py::handle q_, py::handle k_, py::handle positions_, py::handle inv_freq_, bool interleaved, double factor) {
    const at::Tensor *qp, *kp = nullptr, *pp = nullptr, *fp;
    if (watched() || !plain(q_.ptr(), qp) || !plain(inv_freq_.ptr(), fp)) return py::none();
    if (!k_.is_none() && !plain(k_.ptr(), kp)) return py::none();
    Turn t{{}, *fp, 0, interleaved, false, factor};
    if (!positions_.is_none()) {
        if (PyLong_CheckExact(positions_.ptr())) {
            t.offset = PyLong_AsLongLong(positions_.ptr());
            if (t.offset == -1 && PyErr_Occurred()) { PyErr_Clear(); return py::none(); }
        } else {
            if (!plain(positions_.ptr(), pp)) return py::none();
            t.positions = *pp;
        }
    }
    const at::Tensor q = *qp, k = kp ? *kp : at::Tensor();
    const auto type = q.scalar_type();
    auto fits = [&](const at::Tensor& x) {
        return x.dim() == 4 && x.scalar_type() == type && x.device() == q.device() && x.size(0) == q.size(0) && x.size(1) == q.size(1) && x.size(3) == q.size(3) &&
               x.stride(3) == 1 && x.numel() > 0 && x.size(0) <= INT32_MAX && x.size(1) <= INT32_MAX && x.size(2) <= INT32_MAX;
    };
    if ((type != at::kHalf && type != at::kBFloat16 && type != at::kFloat) || !fits(q) || (kp && !fits(k)) || q.size(3) > 128 ||
        t.inv_freq.scalar_type() != at::kDouble || t.inv_freq.dim() != 1 || !t.inv_freq.is_contiguous() || 2 * t.inv_freq.size(0) > q.size(3) ||
        t.inv_freq.device() != q.device() || t.inv_freq.requires_grad())
        return py::none();
    if (pp) {
        const at::Tensor& x = t.positions;
        if ((x.scalar_type() != at::kInt && x.scalar_type() != at::kLong) || x.device() != q.device() || x.dim() < 1 || x.dim() > 2 || x.size(-1) != q.size(1) ||
            (x.dim() == 2 && x.size(0) != 1 && x.size(0) != q.size(0)))
            return py::none();
    }
    const bool wants = at::GradMode::is_enabled() && (q.requires_grad() || (kp && k.requires_grad()));
    at::Tensor y[2];
    unlocked([&] {
        if (wants) {
            const at::Tensor x[2] = {q, k};
            variable_list out = turned(x, kp ? 2 : 1, t);
            for (size_t i = 0; i < out.size(); ++i) y[i] = std::move(out[i]);
        } else {
            at::AutoDispatchBelowADInplaceOrView below;
            const at::Tensor x[2] = {q, k};
            for (int i = 0; i < (kp ? 2 : 1); ++i) y[i] = at::empty(x[i].sizes(), x[i].options());
            turn(x, y, kp ? 2 : 1, t);
        }
    });
    if (!kp) return wrap(std::move(y[0]));
    return py::make_tuple(wrap(std::move(y[0])), wrap(std::move(y[1])));
}

// (plan, positions, first, end) of build_key_ranges, or None.
py::object key_ranges(int64_t seq_q, int64_t seq_k, int64_t batch, bool causal, int64_t window, py::handle offsets_, py::handle prefixes_, py::handle lengths_,
                      py::handle starts_, int64_t start, int device) {
    if (watched() || seq_q < 0 || seq_k < 0 || batch < 0 || seq_q > INT32_MAX || seq_k > INT32_MAX || batch > INT32_MAX || window < 0 || window > INT32_MAX ||
        start < INT32_MIN || start > INT32_MAX)
        return py::none();
    at::Tensor t[4];
    const py::handle h[4] = {offsets_, prefixes_, lengths_, starts_};
    for (int i = 0; i < 4; ++i) {
        if (h[i].is_none()) continue;
        const at::Tensor* x;
        if (!plain(h[i].ptr(), x) || x->scalar_type() != at::kInt || x->device().index() != device || !x->is_contiguous()) return py::none();
        t[i] = *x;
    }
    fa_b200_ranges_params p;
    memset(&p, 0, sizeof(p));
    p.struct_bytes = sizeof(p);
    if (t[0].defined()) {
        const int64_t n = t[0].dim() ? t[0].size(-1) - 1 : 0;
        if (n < 1 || n > INT32_MAX || !(t[0].dim() == 1 || (t[0].dim() == 2 && t[0].size(0) == batch))) return py::none();
        p.n_documents = (int32_t)n;
        p.offsets_stride_b = t[0].dim() == 2 ? n + 1 : 0;
        p.document_offsets = t[0].const_data_ptr<int32_t>();
    }
    if (t[1].defined()) {
        const int64_t n = p.n_documents;
        if (!causal || window || !(n ? (t[1].dim() == 1 && t[1].size(0) == n) || (t[1].dim() == 2 && t[1].size(0) == batch && t[1].size(1) == n)
                                     : t[1].dim() == 1 && t[1].size(0) == batch))
            return py::none();
        p.prefix_stride_b = n ? (t[1].dim() == 2 ? n : 0) : 1;
        p.prefix_lengths = t[1].const_data_ptr<int32_t>();
    }
    for (int i = 2; i < 4; ++i)
        if (t[i].defined() && (t[i].dim() != 1 || t[i].size(0) != batch)) return py::none();
    if (t[2].defined()) p.key_lengths = t[2].const_data_ptr<int32_t>();
    if (t[3].defined()) p.query_offsets = t[3].const_data_ptr<int32_t>();
    p.query_offset = (int32_t)start; p.causal = causal; p.window = (int32_t)window;
    p.B = (int32_t)batch; p.Nq = (int32_t)seq_q; p.Nk = (int32_t)seq_k; p.device = device;
    at::Tensor plan, positions;
    unlocked([&] {
        at::AutoDispatchBelowADInplaceOrView below;
        const auto options = at::TensorOptions().dtype(at::kInt).device(at::kCUDA, (c10::DeviceIndex)device);
        p.plan_bytes = fa_b200_key_ranges_bytes(p.B, p.Nq, p.Nk);
        plan = at::empty({(int64_t)(p.plan_bytes / 4)}, options);
        positions = at::empty({batch, seq_q}, options);
        p.plan = plan.mutable_data_ptr();
        p.positions = positions.mutable_data_ptr<int32_t>();
        p.stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
        raise_for_status(fa_b200_key_ranges(&p), "fa_b200_key_ranges");
    });
    const int64_t pitch = 2 * ((seq_q + 127) / 128 * 128);
    at::Tensor first, end;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        first = plan.as_strided({batch, seq_q}, {pitch, 2}, 0);
        end = plan.as_strided({batch, seq_q}, {pitch, 2}, seq_q > 0 && batch > 0 ? 1 : 0);
    }
    return py::make_tuple(wrap(std::move(plan)), wrap(std::move(positions)), wrap(std::move(first)), wrap(std::move(end)));
}

}  // namespace

#ifndef FA_TORCH_VERSION
#error "the build names the torch whose headers these are (FA_TORCH_VERSION)"
#endif
// Read by kernels/_cabi.py before Python imports the module: what stands above is laid out for this torch and no other.
extern "C" __attribute__((visibility("default"))) const char* fa_b200_torch_built_for() { return FA_TORCH_VERSION; }

PYBIND11_MODULE(fa_b200_torch, m) {
    m.def("attention", &attention);
    m.def("attention_rules", &attention_rules);
    m.def("rotary", &rotary);
    m.def("key_ranges", &key_ranges);
    m.def("set_status_word", [](int device, uintptr_t word) {
        if (device >= 0 && device < kMaxDevices) g_status_word[device].store((int32_t*)word, std::memory_order_release);
    });
}
