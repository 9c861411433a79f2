// Differentiable class-head operators (layer_norm, linear, label_log_probs) over the detbox C ABI: argument checks,
// allocation and the autograd nodes, in C++ because a training step on few rows is host work: the same in Python took 145 us
// for a layer_norm forward and backward of 64 x 256, the kernels of which run 15 us.
//
// The entry points of libdetbox.so are handed over as addresses (bind), so that there is one loaded library, the one the
// Python layer's ctypes binding holds.  Scratch memory comes from the caching allocator for the time of a call: calls on
// different streams never share it, and a captured graph has its own.
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <map>
#include <string>

#include "../../include/detbox.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

struct Api {
    decltype(&detbox_last_error) last_error;
    decltype(&detbox_layer_norm_forward) layer_norm_forward;
    decltype(&detbox_layer_norm_backward) layer_norm_backward;
    decltype(&detbox_layer_norm_backward_workspace_bytes) layer_norm_backward_workspace_bytes;
    decltype(&detbox_linear_forward) linear_forward;
    decltype(&detbox_linear_workspace_bytes) linear_workspace_bytes;
    decltype(&detbox_linear_backward) linear_backward;
    decltype(&detbox_linear_backward_workspace_bytes) linear_backward_workspace_bytes;
    decltype(&detbox_label_log_probs_forward) label_log_probs_forward;
    decltype(&detbox_label_log_probs_workspace_bytes) label_log_probs_workspace_bytes;
    decltype(&detbox_label_log_probs_backward) label_log_probs_backward;
} api;
PyObject *device_error = nullptr;       // the package's DetboxError
bool poison = false;                    // tests: every call finds its scratch memory filled with garbage

void bind(const std::map<std::string, uintptr_t> &at, py::object error, bool fill) {
#define DETBOX_BIND(name) api.name = reinterpret_cast<decltype(api.name)>(at.at("detbox_" #name))
    DETBOX_BIND(last_error);
    DETBOX_BIND(layer_norm_forward);
    DETBOX_BIND(layer_norm_backward);
    DETBOX_BIND(layer_norm_backward_workspace_bytes);
    DETBOX_BIND(linear_forward);
    DETBOX_BIND(linear_workspace_bytes);
    DETBOX_BIND(linear_backward);
    DETBOX_BIND(linear_backward_workspace_bytes);
    DETBOX_BIND(label_log_probs_forward);
    DETBOX_BIND(label_log_probs_workspace_bytes);
    DETBOX_BIND(label_log_probs_backward);
#undef DETBOX_BIND
    device_error = error.release().ptr();
    poison = fill;
}

// ---- checks --------------------------------------------------------------------------------------------------------------

template <typename... A>
[[noreturn]] void refuse(const A &...parts) { throw py::value_error(c10::str(parts...)); }

int dtype_of(at::ScalarType t) {
    return t == at::kFloat ? DETBOX_F32 : t == at::kBFloat16 ? DETBOX_BF16 : t == at::kHalf ? DETBOX_F16 : -1;
}

void check_input(const char *name, const char *what, const Tensor &t, const Tensor *like = nullptr) {
    if (!t.is_cuda()) {
        PyErr_SetString(device_error, c10::str(name, " runs on a ROCm device only").c_str());
        throw py::error_already_set();
    }
    if (like && t.device() != like->device()) refuse(name, ": ", what, " is on ", t.device(), ", not on ", like->device());
    if (dtype_of(t.scalar_type()) < 0)
        refuse(name, ": ", what, " is ", t.scalar_type(), "; float32, bfloat16 and float16 are supported");
}

// Called with Python's lock held (a forward call) an error of the library is the package's DetboxError, like everywhere else;
// in autograd's threads it is a C++ exception, which arrives in Python as RuntimeError, DetboxError's base.
void check(int rc, const char *what) {
    if (!rc) return;
    const std::string text = c10::str(what, " failed with code ", rc, ": ", api.last_error());
    if (!PyGILState_Check()) throw std::runtime_error(text);
    PyErr_SetString(device_error, text.c_str());
    throw py::error_already_set();
}

// ---- layout, streams, scratch --------------------------------------------------------------------------------------------

// t as a matrix of its last axis: a view where the rows have one stride and unit element stride, a copy elsewhere (expanded
// gradients, transposed inputs).
Tensor rows_of(const Tensor &t) {
    if (t.dim() == 2 && t.is_contiguous()) return t;
    const Tensor m = t.reshape({-1, t.size(-1)});
    if ((m.stride(1) == 1 || m.size(1) == 1) && (m.size(0) <= 1 || m.stride(0) >= m.size(1))) return m;
    return m.contiguous();
}
int64_t stride_of(const Tensor &m) { return m.size(0) > 1 ? std::max(m.stride(0), m.size(1)) : m.size(1); }

void *ptr(const Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
float *fptr(const Tensor &t) { return static_cast<float *>(ptr(t)); }

void *stream_of(const Tensor &t) {
    return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

struct Scratch {
    Tensor t;
    Scratch(const Tensor &like, size_t bytes) {
        if (!bytes) return;
        t = at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
        if (poison) t.fill_(0xA5);
    }
    void *p() const { return ptr(t); }
    size_t bytes() const { return t.defined() ? (size_t)t.numel() : 0; }
};

// The sizes of t with the last axis replaced (none: dropped).  Outputs are allocated in their final shape: a view made inside a
// node could not be changed in place by the caller.
std::vector<int64_t> with_last(const Tensor &t, std::optional<int64_t> last) {
    auto sizes = t.sizes().vec();
    sizes.pop_back();
    if (last) sizes.push_back(*last);
    return sizes;
}

// The gradients of a node that has none of its own: asking for a second derivative raises, as it must.
variable_list only_once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list has;
    for (auto &g : grads)
        if (g.defined()) has.push_back(g.detach().set_requires_grad(true));
    auto error = std::make_shared<torch::autograd::DelayedError>("the class-head operators have no second derivative", (int64_t)has.size());
    const variable_list out = (*error)(std::move(has));
    size_t i = 0;
    for (auto &g : grads)
        if (g.defined()) g = out[i++];
    return grads;
}

bool wants_grad(std::initializer_list<const MaybeTensor *> inputs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const auto *t : inputs)
        if (t->has_value() && (*t)->requires_grad()) return true;
    return false;
}

// Tangents are not carried through.  A call without a node would drop them without a word, which reads as a derivative of zero;
// whether gradients are enabled or asked for does not matter to them.
void refuse_tangents(const char *name, std::initializer_list<const MaybeTensor *> inputs) {
    for (const auto *t : inputs)
        if (t->has_value() && (*t)->_fw_grad(0).defined()) {
            PyErr_SetString(PyExc_NotImplementedError, c10::str(name, " has no forward-mode derivative").c_str());
            throw py::error_already_set();
        }
}

// ---- layer_norm ----------------------------------------------------------------------------------------------------------

struct NormResult { Tensor y, m, weight, stats; };
NormResult norm_forward(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps, bool keep) {
    const Tensor m = rows_of(x), w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
    const int64_t rows = m.size(0), D = m.size(1);
    Tensor y = at::empty(x.sizes(), x.options()), stats;
    if (keep) stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
    const int pdt = dtype_of(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type());
    c10::DeviceGuard guard(x.device());
    check(api.layer_norm_forward(dtype_of(x.scalar_type()), ptr(m), stride_of(m), pdt, ptr(w), ptr(b), rows, D, (float)eps, ptr(y),
                                 fptr(stats), stream_of(x)), "detbox_layer_norm_forward");
    return {y, m, w, stats};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps) {
        NormResult r = norm_forward(x, weight, bias, eps, true);
        ctx->save_for_backward({r.m, r.weight, r.stats});
        ctx->saved_data["shape"] = x.sizes();
        ctx->saved_data["param"] = (int64_t)(weight ? weight->scalar_type() : bias ? bias->scalar_type() : x.scalar_type());
        ctx->saved_data["need"] = (int64_t)(x.requires_grad() | (weight && weight->requires_grad()) << 1 | (bias && bias->requires_grad()) << 2);
        return r.y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &m = saved[0], &weight = saved[1], &stats = saved[2];
        const int64_t rows = m.size(0), D = m.size(1), need = ctx->saved_data["need"].toInt();
        const auto param = (at::ScalarType)ctx->saved_data["param"].toInt();
        Tensor gx, gw, gb;
        {
            at::NoGradGuard none;
            const Tensor g = rows_of(grads[0]);
            if (need & 1) gx = at::empty(ctx->saved_data["shape"].toIntVector(), m.options());
            if (need & 2) gw = at::empty({D}, m.options().dtype(param));
            if (need & 4) gb = at::empty({D}, m.options().dtype(param));
            c10::DeviceGuard guard(m.device());
            const Scratch ws(m, need & 6 ? api.layer_norm_backward_workspace_bytes(rows, D) : 0);
            check(api.layer_norm_backward(dtype_of(m.scalar_type()), ptr(g), stride_of(g), ptr(m), stride_of(m), dtype_of(param), ptr(weight),
                                          fptr(stats), rows, D, ptr(gx), ptr(gw), ptr(gb), ws.p(), ws.bytes(), stream_of(m)),
                  "detbox_layer_norm_backward");
        }
        return only_once({gx, gw, gb, Tensor()});
    }
};

Tensor layer_norm(const Tensor &x, const MaybeTensor &weight, const MaybeTensor &bias, double eps) {
    check_input("layer_norm", "x", x);
    if (x.dim() < 1 || x.size(-1) < 1) refuse("layer_norm: x needs a last axis of at least one element");
    for (const auto *p : {&weight, &bias}) {
        if (!p->has_value()) continue;
        const char *what = p == &weight ? "weight" : "bias";
        check_input("layer_norm", what, **p, &x);
        if ((*p)->dim() != 1 || (*p)->size(0) != x.size(-1)) refuse("layer_norm: ", what, " ", (*p)->sizes(), " does not fit rows of ", x.size(-1));
    }
    if (weight && bias && weight->scalar_type() != bias->scalar_type()) refuse("layer_norm: weight and bias differ in type");
    const MaybeTensor xx(x);
    refuse_tangents("layer_norm", {&xx, &weight, &bias});
    if (wants_grad({&xx, &weight, &bias})) return LayerNorm::apply(x, weight, bias, eps);
    return norm_forward(x, weight, bias, eps, false).y;
}

// ---- linear --------------------------------------------------------------------------------------------------------------

struct LinearResult { Tensor y, m, w, pre; };
LinearResult linear_forward(const Tensor &x, const Tensor &weight, const MaybeTensor &bias, int64_t act, const MaybeTensor &residual,
                            at::ScalarType out, bool keep) {
    const Tensor m = rows_of(x), w = rows_of(weight), b = bias ? bias->contiguous() : Tensor(), r = residual ? rows_of(*residual) : Tensor();
    const int64_t M = m.size(0), K = m.size(1), N = w.size(0);
    const int dt = dtype_of(x.scalar_type());
    Tensor y = at::empty(with_last(x, N), x.options().dtype(out)), pre;
    if (keep && act) pre = at::empty({M, N}, x.options());
    c10::DeviceGuard guard(x.device());
    const Scratch ws(x, api.linear_workspace_bytes(dt, M, N, K));
    check(api.linear_forward(dt, (int)act, ptr(m), stride_of(m), ptr(w), stride_of(w), b.defined() ? dtype_of(b.scalar_type()) : 0, ptr(b), ptr(r),
                             r.defined() ? stride_of(r) : 0, M, N, K, dtype_of(out), ptr(y), ptr(pre), ws.p(), ws.bytes(), stream_of(x)),
          "detbox_linear_forward");
    return {y, m, w, pre};
}

struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, const MaybeTensor &bias, const MaybeTensor &residual,
                          int64_t act, int64_t out) {
        const bool need_x = x.requires_grad(), need_w = weight.requires_grad(), need_b = bias && bias->requires_grad();
        LinearResult r = linear_forward(x, weight, bias, act, residual, (at::ScalarType)out, need_x || need_w || need_b);
        ctx->save_for_backward({need_w ? r.m : Tensor(), need_x ? r.w : Tensor(), r.pre});
        ctx->saved_data["need"] = (int64_t)(need_x | need_w << 1 | need_b << 2 | (residual && residual->requires_grad()) << 3);
        ctx->saved_data["shape"] = x.sizes();
        ctx->saved_data["N"] = weight.size(0);
        ctx->saved_data["act"] = act;
        ctx->saved_data["dtype"] = (int64_t)x.scalar_type();
        ctx->saved_data["bias"] = (int64_t)(bias ? bias->scalar_type() : x.scalar_type());
        return r.y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const int64_t need = ctx->saved_data["need"].toInt();
        Tensor gx, gw, gb;
        if (need & 7) {
            at::NoGradGuard none;
            const auto saved = ctx->get_saved_variables();
            const Tensor &m = saved[0], &w = saved[1], &pre = saved[2];
            const Tensor g = rows_of(grads[0]);
            const auto shape = ctx->saved_data["shape"].toIntVector();
            const int64_t M = g.size(0), N = ctx->saved_data["N"].toInt(), K = shape.back(), act = ctx->saved_data["act"].toInt();
            const auto type = (at::ScalarType)ctx->saved_data["dtype"].toInt(), btype = (at::ScalarType)ctx->saved_data["bias"].toInt();
            const int dt = dtype_of(type), gdt = dtype_of(g.scalar_type());
            if (need & 1) gx = at::empty(shape, g.options().dtype(type));
            if (need & 2) gw = at::empty({N, K}, g.options().dtype(type));
            if (need & 4) gb = at::empty({N}, g.options().dtype(btype));
            c10::DeviceGuard guard(g.device());
            const Scratch ws(g, api.linear_backward_workspace_bytes(dt, (int)act, gdt, M, N, K));
            check(api.linear_backward(dt, (int)act, gdt, ptr(g), stride_of(g), ptr(pre), ptr(m), m.defined() ? stride_of(m) : K, ptr(w),
                                      w.defined() ? stride_of(w) : K, M, N, K, ptr(gx), ptr(gw), dtype_of(btype), ptr(gb), ws.p(), ws.bytes(),
                                      stream_of(g)), "detbox_linear_backward");
        }
        return only_once({gx, gw, gb, need & 8 ? grads[0] : Tensor(), Tensor(), Tensor()});
    }
};

Tensor linear(const Tensor &x, const Tensor &weight, const MaybeTensor &bias, int64_t act, const MaybeTensor &residual,
              const std::optional<at::ScalarType> &out_dtype) {
    check_input("linear", "x", x);
    check_input("linear", "weight", weight, &x);
    if (weight.dim() != 2 || x.dim() < 1 || weight.size(1) != x.size(-1) || weight.size(0) < 1 || weight.size(1) < 1)
        refuse("linear: x ", x.sizes(), " and weight ", weight.sizes(), " do not fit");
    if (weight.scalar_type() != x.scalar_type()) refuse("linear: x and weight differ in type");
    const at::ScalarType out = out_dtype.value_or(x.scalar_type());
    if (out != x.scalar_type() && out != at::kFloat) refuse("linear: out_dtype ", out, " is neither the type of x nor float32");
    if (bias) {
        check_input("linear", "bias", *bias, &x);
        if (bias->dim() != 1 || bias->size(0) != weight.size(0)) refuse("linear: bias ", bias->sizes(), " does not fit weight ", weight.sizes());
    }
    if (residual) {
        check_input("linear", "residual", *residual, &x);
        bool fits = residual->scalar_type() == out && residual->dim() == x.dim() && residual->size(-1) == weight.size(0);
        for (int64_t i = 0; fits && i + 1 < x.dim(); ++i) fits = residual->size(i) == x.size(i);
        if (!fits) refuse("linear: residual ", residual->sizes(), " of ", residual->scalar_type(), " does not fit the output");
    }
    const MaybeTensor xx(x), ww(weight);
    refuse_tangents("linear", {&xx, &ww, &bias, &residual});
    if (wants_grad({&xx, &ww, &bias, &residual})) return Linear::apply(x, weight, bias, residual, act, (int64_t)out);
    return linear_forward(x, weight, bias, act, residual, out, false).y;
}

// ---- label_log_probs -----------------------------------------------------------------------------------------------------

struct LogProbResult { Tensor lp, ent, tv, ti, m, t, stats; };
LogProbResult logprob_forward(const Tensor &logits, const Tensor &labels, int64_t top_k, bool entropy, bool keep) {
    const Tensor m = rows_of(logits);
    const int64_t rows = m.size(0), C = m.size(1);
    Tensor t = labels.scalar_type() == at::kLong ? labels : labels.to(at::kLong);
    t = t.reshape({-1}).contiguous();
    const auto f32 = logits.options().dtype(at::kFloat);
    LogProbResult r{at::empty(with_last(logits, std::nullopt), f32), {}, {}, {}, m, t, {}};
    if (entropy) r.ent = at::empty_like(r.lp);
    if (top_k) {
        r.tv = at::empty(with_last(logits, top_k), f32);
        r.ti = at::empty(with_last(logits, top_k), f32.dtype(at::kLong));
    }
    if (keep) r.stats = at::empty({rows, 2}, f32);
    c10::DeviceGuard guard(logits.device());
    const Scratch ws(logits, api.label_log_probs_workspace_bytes(rows, C, (int)top_k));
    check(api.label_log_probs_forward(dtype_of(m.scalar_type()), ptr(m), stride_of(m), static_cast<int64_t *>(ptr(t)), rows, C, (int)top_k,
                                      fptr(r.lp), fptr(r.ent), fptr(r.tv), static_cast<int64_t *>(ptr(r.ti)), fptr(r.stats), ws.p(), ws.bytes(),
                                      stream_of(logits)), "detbox_label_log_probs_forward");
    return r;
}

struct LogProbs : torch::autograd::Function<LogProbs> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &labels, int64_t top_k, bool entropy) {
        LogProbResult r = logprob_forward(logits, labels, top_k, entropy, true);
        ctx->save_for_backward({r.m, r.t, r.stats, r.ent});
        ctx->saved_data["shape"] = logits.sizes();
        ctx->set_materialize_grads(false);
        variable_list out{r.lp};
        if (entropy) out.push_back(r.ent);
        if (top_k) {
            out.push_back(r.tv);
            out.push_back(r.ti);
            ctx->mark_non_differentiable({r.tv, r.ti});
        }
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &m = saved[0], &t = saved[1], &stats = saved[2], &ent = saved[3];
        const Tensor none, grad_ent = ent.defined() ? grads[1] : none;
        if (!grads[0].defined() && !grad_ent.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        Tensor gx;
        {
            at::NoGradGuard guard_grad;
            const Tensor g = grads[0].defined() ? grads[0].reshape({-1}).contiguous() : none;
            const Tensor h = grad_ent.defined() ? grad_ent.reshape({-1}).contiguous() : none;
            gx = at::empty(ctx->saved_data["shape"].toIntVector(), m.options());
            c10::DeviceGuard guard(m.device());
            check(api.label_log_probs_backward(dtype_of(m.scalar_type()), ptr(m), stride_of(m), static_cast<int64_t *>(ptr(t)), m.size(0),
                                               m.size(1), fptr(stats), fptr(ent), fptr(g), fptr(h), ptr(gx), stream_of(m)),
                  "detbox_label_log_probs_backward");
        }
        return only_once({gx, Tensor(), Tensor(), Tensor()});
    }
};

// (log_probs, entropy or None, top_log_probs or None, top_ids or None)
py::tuple label_log_probs(const Tensor &logits, const Tensor &labels, int64_t top_k, bool entropy, int64_t most) {
    check_input("label_log_probs", "logits", logits);
    if (logits.dim() < 1 || logits.size(-1) < 1) refuse("label_log_probs: logits need a last axis of at least one class");
    if (labels.device() != logits.device()) refuse("label_log_probs: labels are on ", labels.device(), ", not on ", logits.device());
    bool fits = labels.dim() == logits.dim() - 1 && at::isIntegralType(labels.scalar_type(), false);
    for (int64_t i = 0; fits && i < labels.dim(); ++i) fits = labels.size(i) == logits.size(i);
    if (!fits) refuse("label_log_probs: labels ", labels.sizes(), " of ", labels.scalar_type(), " do not fit logits ", logits.sizes());
    if (top_k < 0 || top_k > std::min(most, logits.size(-1)))
        refuse("label_log_probs: top_k ", top_k, " is outside 0 .. min(", most, ", ", logits.size(-1), ")");
    const MaybeTensor x(logits);
    refuse_tangents("label_log_probs", {&x});
    Tensor lp, ent, tv, ti;
    if (wants_grad({&x})) {
        const variable_list out = LogProbs::apply(logits, labels, top_k, entropy);
        size_t i = 0;
        lp = out[i++];
        if (entropy) ent = out[i++];
        if (top_k) {
            tv = out[i++];
            ti = out[i];
        }
    } else {
        LogProbResult r = logprob_forward(logits, labels, top_k, entropy, false);
        lp = r.lp;
        ent = r.ent;
        tv = r.tv;
        ti = r.ti;
    }
    auto or_none = [](const Tensor &t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
    return py::make_tuple(lp, or_none(ent), or_none(tv), or_none(ti));
}

}  // namespace

PYBIND11_MODULE(_heads, m) {
    m.def("bind", &bind);
    m.def("layer_norm", &layer_norm);
    m.def("linear", &linear);
    m.def("label_log_probs", &label_log_probs);
}
