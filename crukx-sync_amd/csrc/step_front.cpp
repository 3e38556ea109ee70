// The Python face of the training step (crukx_sync/step.py): argument checks, output tensors, autograd and the
// calls of the crx_* entry points, as a torch C++ extension.  A call of a few tokens takes less time on the GPU
// than these checks take in Python (a loss of 14 positions with its gradient: 12 us of kernels; its call 39 us
// when step.py did this work, and 147 us for a score with its backward pass).
//
// The entry points are those of the library that crukx_sync/_native.py has loaded: their addresses are given to
// init(), and nothing is linked.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/crukx.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    decltype(&crx_rows_scratch) rows_scratch = nullptr;
    decltype(&crx_token_logprobs) token_logprobs = nullptr;
    decltype(&crx_token_logprobs_grad) token_logprobs_grad = nullptr;
    decltype(&crx_policy_loss) policy_loss = nullptr;
    decltype(&crx_policy_loss_grad) policy_loss_grad = nullptr;
    decltype(&crx_norm_scratch) norm_scratch = nullptr;
    decltype(&crx_grad_norm) grad_norm = nullptr;
    decltype(&crx_clip_grads) clip_grads = nullptr;
    decltype(&crx_adamw_step) adamw_step = nullptr;
};
Api g_api;
py::object *g_stream = nullptr;  // device index -> the current stream's handle; never freed (the interpreter may be gone)
bool g_any_device = false;       // the CPU model of the library: tensors in host memory, stream 0

[[noreturn]] void bad(const std::string &m) { throw std::invalid_argument(m); }

// -------------------------------------------------------------------- devices and calls

int64_t index_of(const Tensor &t) { return g_any_device ? 0 : t.is_cuda() ? (int64_t)t.device().index() : -1; }

// Under a tracer the calls must not run: it sees the allocation of their results and not the kernels, and what it records
// would return memory that nothing has written.  (Modes that only look on, as profilers do, are not meant.)
void not_traced() {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    bool traced = torch::jit::tracer::isTracing();
    for (auto mode : {TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FAKE, TorchDispatchModeKey::FUNCTIONAL})
        traced = traced || TorchDispatchModeTLS::get_mode(mode).has_value();
    if (traced) throw std::runtime_error("the training step's calls cannot be traced");
}

// t with its data as they are meant: torch keeps some negations as a flag beside the data.  (Differentiable.)
Tensor resolved(const Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
optional<Tensor> resolved(const optional<Tensor> &t) { return t.has_value() ? optional<Tensor>(resolved(*t)) : t; }

// An upstream gradient as data: torch may hand down one of nothing but zeros without any storage.
Tensor upstream(const Tensor &t) { return t.defined() && t._is_zerotensor() ? at::zeros(t.sizes(), t.options()) : resolved(t); }

// What holds no data itself (distributed, fake and zero tensors): a null address would read as an argument left out.
constexpr const char *kNoStorage = "the tensor has no storage of its own";
bool without_storage(const Tensor &t) { return !t.data_ptr() && t.numel(); }

// A dual tensor's tangent would be lost without a word: no operator here has a forward-mode derivative.
constexpr const char *kNoTangent = "forward-mode derivatives are not supported, got a dual tensor";

void check_hip(const char *name, const Tensor &t) {
    if (!t.defined()) bad(std::string(name) + ": expected a torch tensor");
    if (t._fw_grad(0).defined()) bad(std::string(name) + ": " + kNoTangent);
    if (index_of(t) < 0) bad(std::string(name) + ": expected a tensor on a HIP device, got one on " + t.device().str());
}

// One call of the library on the tensors' device and its current stream.
struct Call {
    c10::OptionalDeviceGuard guard;
    void *stream = nullptr;
    char err[512] = "";
    explicit Call(const Tensor &t) {
        if (g_any_device) return;
        guard.reset_device(t.device());
        py::gil_scoped_acquire gil;  // (a backward pass runs without it)
        stream = reinterpret_cast<void *>((*g_stream)(t.device().index()).cast<uintptr_t>());
    }
    void done(int32_t rc) const {
        if (rc == CRX_OK) return;
        if (rc == CRX_INVALID) bad(err);
        if (rc == CRX_NOMEM) throw std::bad_alloc();
        throw std::runtime_error(std::string("HIP error: ") + err);
    }
};

Tensor floats(at::IntArrayRef shape, const Tensor &like) { return at::empty(shape, like.options().dtype(at::kFloat).requires_grad(false)); }
Tensor bytes(uint64_t n, const Tensor &like) {
    return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false));
}

template <typename T = float>
T *data(const Tensor &t) {
    return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr;
}

std::string shape_of(at::IntArrayRef s) {
    std::string o = "(";
    for (size_t i = 0; i < s.size(); ++i) o += (i ? ", " : "") + std::to_string(s[i]);
    return o + (s.size() == 1 ? ",)" : ")");
}

int32_t type_of(const Tensor &t) {
    switch (t.scalar_type()) {
    case at::kBFloat16: return CRX_BF16;
    case at::kHalf: return CRX_F16;
    case at::kFloat: return CRX_F32;
    default: return -1;
    }
}

// -------------------------------------------------------------------- logits and positions

// One value per position of `like`, at t's own strides (0 where it is broadcast).
crx_positions positions(const char *name, const Tensor &t, const Tensor &like, at::ScalarType type, at::ScalarType other,
                        bool broadcast) {
    check_hip(name, t);
    const auto st = t.scalar_type();
    if (st != type && st != other)
        bad(std::string(name) + ": expected " + c10::toString(type) + (type == other ? "" : std::string(" or ") + c10::toString(other)) +
            ", got " + c10::toString(st));
    if (t.layout() != at::kStrided) bad(std::string(name) + ": expected a strided tensor");
    if (without_storage(t)) bad(std::string(name) + ": " + kNoStorage);
    if (index_of(t) != index_of(like)) bad(std::string(name) + ": all tensors must be on one device");
    const auto want = like.sizes().slice(0, like.dim() - 1);
    bool fits = t.dim() == (int64_t)want.size();
    int64_t stride[2] = {0, 0};
    for (size_t k = 0; fits && k < want.size(); ++k) {
        const int64_t n = t.size((int64_t)k);
        fits = n == want[k] || (broadcast && n == 1);
        stride[2 - want.size() + k] = n == want[k] ? t.stride((int64_t)k) : 0;
    }
    if (!fits) bad(std::string(name) + ": expected shape " + shape_of(want) + ", got " + shape_of(t.sizes()));
    return crx_positions{t.data_ptr(), stride[0], stride[1]};
}
crx_positions floats_at(const char *name, const Tensor &t, const Tensor &like) {
    return t.defined() ? positions(name, t, like, at::kFloat, at::kFloat, true) : crx_positions{nullptr, 0, 0};
}

crx_logits logits_of(const Tensor &x, const Tensor &tokens, const Tensor &mask, double temperature) {
    check_hip("logits", x);
    const int32_t type = type_of(x);
    if (type < 0) bad(std::string("logits: expected bfloat16, float16 or float32, got ") + c10::toString(x.scalar_type()));
    if (x.layout() != at::kStrided) bad("logits: expected a strided tensor");
    if (without_storage(x)) bad(std::string("logits: ") + kNoStorage);
    const int64_t dim = x.dim();
    if (dim != 2 && dim != 3)
        bad("logits: expected [tokens, vocabulary] or [sequences, tokens, vocabulary], got " + shape_of(x.sizes()));
    if (x.stride(dim - 1) != 1 && x.size(dim - 1) > 1) bad("logits: the vocabulary must be contiguous");
    crx_logits o{};
    o.x = x.data_ptr();
    o.seqs = dim == 2 ? 1 : (uint64_t)x.size(0);
    o.tokens = (uint64_t)x.size(dim - 2);
    o.vocab = (uint64_t)x.size(dim - 1);
    // (the library's own check comes after the results' allocation)
    if (o.tokens && o.seqs > ((1ULL << 31) - 1) / o.tokens) bad("logits of 2^31 or more positions are not supported");
    o.stride_seq = dim == 2 ? 0 : x.stride(0);
    o.stride_token = x.stride(dim - 2);
    o.dtype = type;
    o.ids = positions("tokens", tokens, x, at::kLong, at::kInt, false);
    o.id_bytes = (int32_t)tokens.element_size();
    if (mask.defined()) o.mask = positions("mask", mask, x, at::kBool, at::kByte, false);
    o.temperature = temperature;
    return o;
}

Tensor new_grad(const Tensor &x) { return at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous)); }

Tensor or_none(const optional<Tensor> &t) { return t.has_value() ? *t : Tensor(); }

// A gradient that was asked for with a graph of its own: differentiating it again raises an error.
Tensor once(Tensor g) {
    if (!at::GradMode::is_enabled() || !g.defined()) return g;
    g.set_requires_grad(true);
    const auto stop = std::make_shared<torch::autograd::DelayedError>("the training step's gradients cannot be differentiated again", 1);
    return (*stop)({g})[0];
}

// -------------------------------------------------------------------- scores

struct Scored {
    Tensor logp, entropy, stats;
};

Scored score(const Tensor &x, const Tensor &tokens, const Tensor &mask, double temperature, bool entropy, bool keep) {
    const crx_logits in = logits_of(x, tokens, mask, temperature);
    const auto shape = x.sizes().slice(0, x.dim() - 1);
    Call call(x);
    Scored o;
    o.logp = floats(shape, x);
    if (entropy) o.entropy = floats(shape, x);
    if (keep) o.stats = floats({(int64_t)(in.seqs * in.tokens), 2}, x);
    const Tensor scratch = bytes(g_api.rows_scratch(in.seqs, in.tokens, in.vocab), x);
    call.done(g_api.token_logprobs(&in, data(o.logp), data(o.entropy), data(o.stats), data<void>(scratch), call.stream,
                                   call.err, sizeof call.err));
    return o;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &tokens, const optional<Tensor> &mask,
                                 double temperature, bool entropy) {
        const Scored o = score(x, tokens, or_none(mask), temperature, entropy, true);
        ctx->save_for_backward({x, tokens, or_none(mask), o.stats, o.entropy});
        ctx->saved_data["temperature"] = temperature;
        ctx->set_materialize_grads(false);
        if (entropy) return {o.logp, o.entropy};
        return {o.logp};
    }
    static variable_list backward(AutogradContext *ctx, variable_list up) {
        not_traced();
        const auto kept = ctx->get_saved_variables();
        const Tensor &x = kept[0];
        Tensor grad;
        const Tensor up_logp = upstream(up[0]), up_entropy = up.size() > 1 ? upstream(up[1]) : Tensor();
        if (up_logp.defined() || up_entropy.defined()) {
            const crx_logits in = logits_of(x, kept[1], kept[2], ctx->saved_data["temperature"].toDouble());
            const crx_positions a = floats_at("gradient", up_logp, x), h = floats_at("gradient", up_entropy, x);
            Call call(x);
            grad = new_grad(x);
            call.done(g_api.token_logprobs_grad(&in, data(kept[3]), data(kept[4]), &a, &h, data<void>(grad), call.stream,
                                                call.err, sizeof call.err));
        }
        return {once(grad), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

py::object token_logprobs(const Tensor &x_, const Tensor &tokens_, const optional<Tensor> &mask_, double temperature, bool entropy) {
    not_traced();
    const Tensor x = resolved(x_), tokens = resolved(tokens_);
    const optional<Tensor> mask = resolved(mask_);
    Tensor logp, ent;
    if (x.defined() && x.requires_grad() && at::GradMode::is_enabled()) {
        const variable_list o = TokenLogprobs::apply(x, tokens, mask, temperature, entropy);
        logp = o[0];
        if (entropy) ent = o[1];
    } else {
        const Scored o = score(x, tokens, or_none(mask), temperature, entropy, false);
        logp = o.logp;
        ent = o.entropy;
    }
    if (entropy) return py::make_tuple(logp, ent);
    return py::cast(logp);
}

// -------------------------------------------------------------------- policy loss

struct Options {
    double low, high, kl_coef, temperature, scale;
    int64_t reduction;
};

struct PolicyOut {
    Tensor loss, logp, kl, clipped, kept, grad;
};

PolicyOut policy(const Tensor &x, const Tensor &tokens, const Tensor &old, const Tensor &adv, const Tensor &mask,
                 const Tensor &ref, const Options &opt, bool keep, bool want_grad) {
    const crx_logits in = logits_of(x, tokens, mask, opt.temperature);
    crx_policy p{};
    check_hip("old_logprobs", old);
    check_hip("advantages", adv);
    p.old = floats_at("old_logprobs", old, x);
    p.advantages = floats_at("advantages", adv, x);
    p.ref = floats_at("ref_logprobs", ref, x);
    p.clip_low = opt.low;
    p.clip_high = opt.high;
    p.kl_coef = opt.kl_coef;
    p.scale = opt.scale;
    p.reduction = (int32_t)opt.reduction;
    const int64_t n = (int64_t)(in.seqs * in.tokens);
    Call call(x);
    PolicyOut o;
    o.loss = floats({}, x);
    o.kl = floats({}, x);
    o.clipped = floats({}, x);
    o.logp = floats(x.sizes().slice(0, x.dim() - 1), x);
    if (keep) o.kept = floats({3, n}, x);  // the statistics (two each), then the slopes
    if (want_grad) o.grad = new_grad(x);
    const Tensor scratch = bytes(g_api.rows_scratch(in.seqs, in.tokens, in.vocab), x);
    float *const kept = data(o.kept);
    call.done(g_api.policy_loss(&in, &p, data(o.loss), data(o.kl), data(o.clipped), data(o.logp), kept, kept ? kept + 2 * n : nullptr,
                                data<void>(o.grad), data<void>(scratch), call.stream, call.err, sizeof call.err));
    return o;
}

// The gradient is written by the forward call, which has every row at hand; the backward call only has to compute
// it anew where the loss's own gradient is not 1 (which the device decides), or where it is asked for a second time.
struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &tokens, const Tensor &old, const Tensor &adv,
                                 const optional<Tensor> &mask, const optional<Tensor> &ref, const Options &opt) {
        PolicyOut o = policy(x, tokens, old, adv, or_none(mask), or_none(ref), opt, true, true);
        ctx->save_for_backward({x, tokens, or_none(mask), o.kept});
        ctx->saved_data["temperature"] = opt.temperature;
        ctx->saved_data["grad"] = o.grad;
        ctx->mark_non_differentiable({o.logp, o.kl, o.clipped});
        ctx->set_materialize_grads(false);
        return {o.loss, o.logp, o.kl, o.clipped};
    }
    static variable_list backward(AutogradContext *ctx, variable_list up) {
        not_traced();
        const auto kept = ctx->get_saved_variables();
        const Tensor &x = kept[0];
        Tensor grad;
        if (up[0].defined()) {
            const Tensor factor = upstream(up[0]);
            check_hip("gradient", factor);
            const crx_logits in = logits_of(x, kept[1], kept[2], ctx->saved_data["temperature"].toDouble());
            const auto made = ctx->saved_data.find("grad");
            const bool first = made != ctx->saved_data.end();
            Call call(x);
            if (first) {
                grad = made->second.toTensor();
                ctx->saved_data.erase(made);
            } else {
                grad = new_grad(x);
            }
            const float *const stats = data(kept[3]);
            call.done(g_api.policy_loss_grad(&in, stats, stats + 2 * in.seqs * in.tokens, data(factor), first ? 1 : 0,
                                             data<void>(grad), call.stream, call.err, sizeof call.err));
        }
        variable_list r(7);
        r[0] = once(grad);
        return r;
    }
};

Options options(const py::object &clip, double kl_coef, double temperature, const std::string &reduction, double scale, bool has_ref) {
    Options o{};
    const auto number = [](const py::handle &v) {
        const double d = PyFloat_AsDouble(v.ptr());
        if (d == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            bad("clip: expected a number or a pair of numbers");
        }
        return d;
    };
    if (PySequence_Check(clip.ptr())) {
        const py::sequence pair = py::reinterpret_borrow<py::sequence>(clip);
        if (pair.size() != 2) bad("clip: expected a number or a pair of numbers");
        o.low = number(pair[0]);
        o.high = number(pair[1]);
    } else {
        o.low = o.high = number(clip);
    }
    if (!(o.low >= 0) || !(o.high >= 0)) bad("clip: the range must not be negative");
    o.reduction = reduction == "token" ? CRX_MEAN_TOKEN : reduction == "sequence" ? CRX_MEAN_SEQUENCE : reduction == "sum" ? CRX_SUM : -1;
    if (o.reduction < 0) bad("reduction: expected one of token, sequence, sum, got '" + reduction + "'");
    if (kl_coef != 0 && !has_ref) bad("kl_coef: a KL term needs ref_logprobs");
    o.kl_coef = kl_coef;
    o.temperature = temperature;
    o.scale = scale;
    return o;
}

// (loss, logprobs, kl, clipped) with the loss's gradient by autograd, or (direct) the gradient as a fifth
py::tuple policy_loss(const Tensor &x_, const Tensor &tokens_, const Tensor &old_, const Tensor &adv_, const optional<Tensor> &mask_,
                      const optional<Tensor> &ref_, const py::object &clip, double kl_coef, double temperature,
                      const std::string &reduction, double scale, bool direct) {
    not_traced();
    const Options opt = options(clip, kl_coef, temperature, reduction, scale, ref_.has_value());
    const Tensor x = resolved(x_), tokens = resolved(tokens_), old = resolved(old_), adv = resolved(adv_);
    const optional<Tensor> mask = resolved(mask_), ref = resolved(ref_);
    if (!direct && x.requires_grad() && at::GradMode::is_enabled()) {
        const variable_list o = PolicyLoss::apply(x, tokens, old, adv, mask, ref, opt);
        return py::make_tuple(o[0], o[1], o[2], o[3]);
    }
    const PolicyOut o = policy(x, tokens, old, adv, or_none(mask), or_none(ref), opt, false, direct);
    if (direct) return py::make_tuple(o.loss, o.logp, o.kl, o.clipped, o.grad);
    return py::make_tuple(o.loss, o.logp, o.kl, o.clipped);
}

// -------------------------------------------------------------------- lists of tensors

// The tensors of a list, checked, with what the entry points take of them.  They are borrowed from the Python objects that
// the caller holds: a step of 338 tensors looks at 1690, and taking and giving up a reference to each costs as much as
// the checks.
struct List {
    std::vector<c10::TensorImpl *> t;
    std::vector<void *> ptr;
    std::vector<uint64_t> numel;
    std::vector<int32_t> type;
    Tensor one;  // the first of them
    const bool duals = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;  // whether any tensor can be one

    explicit List(size_t n) {
        if (n > (size_t)INT32_MAX) bad("too many tensors");
        t.reserve(n), ptr.reserve(n), numel.reserve(n), type.reserve(n);
    }
    int32_t n() const { return (int32_t)t.size(); }
    // `name` of the list `what`: an error names it (no name: its place in the list)
    void add(const char *what, PyObject *name, PyObject *item, bool floats_only) {
        auto fail = [&](const std::string &m) {
            bad(std::string(what) + " " + (name ? py::str(name).cast<std::string>() : std::to_string(t.size())) + ": " + m);
        };
        if (!THPVariable_Check(item)) fail("expected a torch tensor, got " + std::string(Py_TYPE(item)->tp_name));
        const Tensor &v = THPVariable_Unpack(item);
        if (!v.defined()) fail("expected a torch tensor");
        c10::TensorImpl *const impl = v.unsafeGetTensorImpl();
        if (t.empty()) {
            if (index_of(v) < 0) fail("all tensors must be on one HIP device, got one on " + v.device().str());
            one = v;
        } else if (impl->device() != one.device()) {
            fail("all tensors must be on one HIP device, got one on " + v.device().str());
        }
        if (duals && v._fw_grad(0).defined()) fail(kNoTangent);
        if (impl->layout() != at::kStrided || !impl->is_contiguous()) fail("tensor must be contiguous");
        const int32_t k = type_of(v);
        if (k < 0 || (floats_only && k != CRX_F32)) fail(std::string("unexpected type ") + c10::toString(v.scalar_type()));
        void *const at = v.data_ptr();
        const uint64_t n = (uint64_t)impl->numel();
        if (!at && n) fail(kNoStorage);
        t.push_back(impl);
        ptr.push_back(at);
        numel.push_back(n);
        type.push_back(k);
    }
};

// A mapping's values (a dict) or a sequence's items (a list).
List list_of(const char *what, const py::object &tensors) {
    if (PyDict_Check(tensors.ptr())) {
        List l((size_t)PyDict_Size(tensors.ptr()));
        PyObject *name, *item;
        Py_ssize_t at = 0;
        while (PyDict_Next(tensors.ptr(), &at, &name, &item)) l.add(what, name, item, false);
        return l;
    }
    const py::list items(tensors);
    List l(items.size());
    for (size_t i = 0; i < items.size(); ++i) l.add(what, nullptr, PyList_GET_ITEM(items.ptr(), (Py_ssize_t)i), false);
    return l;
}

void written(const List &l) {  // in place: the tensors' versions move, as after a torch operation
    for (c10::TensorImpl *t : l.t)
        if (!t->is_inference()) t->bump_version();
}

// the norm of an empty list is on the current device
Tensor place_of(const List &l, const py::object &current) {
    if (l.n()) return l.one;
    return at::empty({0}, at::TensorOptions().device(g_any_device ? at::Device(at::kCPU) : at::Device(at::kCUDA, (c10::DeviceIndex)current().cast<int>())));
}

Tensor norm_of(const List &l, const Tensor &place) {
    Call call(place);
    const Tensor norm = floats({}, place), scratch = bytes(g_api.norm_scratch(), place);
    call.done(g_api.grad_norm(l.n(), l.ptr.data(), l.numel.data(), l.type.data(), data(norm), data<void>(scratch), call.stream,
                              call.err, sizeof call.err));
    return norm;
}

Tensor grad_norm(const py::object &grads, const py::object &current) {
    not_traced();
    const List l = list_of("grads", grads);
    return norm_of(l, place_of(l, current));
}

double checked_norm(double max_norm) {
    if (!(max_norm >= 0)) bad("max_norm must not be negative");
    return max_norm;
}

Tensor clip_grad_norm(const py::object &grads, double max_norm, const py::object &current) {
    not_traced();
    checked_norm(max_norm);
    const List l = list_of("grads", grads);
    const Tensor place = place_of(l, current), norm = norm_of(l, place);
    Call call(place);
    call.done(g_api.clip_grads(l.n(), l.ptr.data(), l.numel.data(), l.type.data(), data(norm), max_norm, call.stream, call.err,
                               sizeof call.err));
    written(l);
    return norm;
}

// dicts: weights, masters, exp_avg, exp_avg_sq, grads, of the same names in any order
void adamw_step(const std::vector<py::dict> &dicts, int64_t step, double lr, double beta1, double beta2, double eps,
                double weight_decay, const optional<Tensor> &norm_, double max_norm) {
    not_traced();
    static const char *const what[5] = {"weights", "masters", "exp_avg", "exp_avg_sq", "grads"};
    if (dicts.size() != 5) bad("adamw_step: expected five mappings");
    if (step < 1) bad("step counts from 1, got " + std::to_string(step));
    const size_t n = dicts[0].size();
    std::vector<List> l(5, List(n));
    auto missing = [&](int k, PyObject *name) {
        bad(std::string(what[k]) + " and weights differ in tensor names" + (name ? ": " + py::str(name).cast<std::string>() : ""));
    };
    auto negated = [&](int k, PyObject *name) {  // (a norm does not see signs, and a scale keeps them)
        bad(std::string(what[k]) + " " + py::str(name).cast<std::string>() + ": the tensor is negated by a flag; pass its resolve_neg()");
    };
    for (int k = 1; k < 5; ++k)
        if (dicts[k].size() != n) missing(k, nullptr);
    Py_ssize_t at[5] = {};
    bool in_order[5] = {true, true, true, true, true};  // so far the names come in the weights' order
    PyObject *name, *weight;
    while (PyDict_Next(dicts[0].ptr(), &at[0], &name, &weight)) {
        l[0].add(what[0], name, weight, false);
        const c10::TensorImpl *const w = l[0].t.back();
        if (w->is_neg()) negated(0, name);
        for (int k = 1; k < 5; ++k) {
            PyObject *other, *item = nullptr;
            if (in_order[k]) in_order[k] = PyDict_Next(dicts[k].ptr(), &at[k], &other, &item) && (other == name || PyObject_RichCompareBool(other, name, Py_EQ) == 1);
            if (!in_order[k]) item = PyDict_GetItemWithError(dicts[k].ptr(), name);
            if (PyErr_Occurred()) throw py::error_already_set();
            if (!item) missing(k, name);
            l[k].add(what[k], name, item, k < 4);
            const c10::TensorImpl *const o = l[k].t.back();
            if (o->is_neg()) negated(k, name);
            if (o->sizes() != w->sizes()) bad(py::str(name).cast<std::string>() + ": " + what[k] + " and weights differ in shape");
            if (o->device() != w->device()) bad("all tensors must be on one device");
        }
    }
    crx_adamw a{lr, beta1, beta2, eps, weight_decay, (uint64_t)step, nullptr, 0.0};
    const Tensor norm = resolved(or_none(norm_));
    if (norm_.has_value()) {
        check_hip("grad_norm", norm);
        if (norm.scalar_type() != at::kFloat || norm.numel() != 1) bad("grad_norm: expected one float32 value");
        if (without_storage(norm)) bad(std::string("grad_norm: ") + kNoStorage);
        if (n && norm.device() != l[0].one.device()) bad("all tensors must be on one device");
        a.norm = data(norm);
        a.max_norm = checked_norm(max_norm);
    }
    if (!n) return;
    Call call(l[0].one);
    auto as_floats = [](List &v) { return reinterpret_cast<float *const *>(v.ptr.data()); };
    call.done(g_api.adamw_step(l[0].n(), l[0].ptr.data(), as_floats(l[1]), as_floats(l[2]), as_floats(l[3]), l[4].ptr.data(),
                               l[0].numel.data(), l[0].type.data(), l[4].type.data(), &a, call.stream, call.err, sizeof call.err));
    for (int k = 0; k < 4; ++k) written(l[k]);
}

void init(const py::dict &at, py::object stream, bool any_device) {
    auto set = [&](auto &f, const char *name) {
        f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(at[name].cast<uintptr_t>());
    };
    set(g_api.rows_scratch, "crx_rows_scratch");
    set(g_api.token_logprobs, "crx_token_logprobs");
    set(g_api.token_logprobs_grad, "crx_token_logprobs_grad");
    set(g_api.policy_loss, "crx_policy_loss");
    set(g_api.policy_loss_grad, "crx_policy_loss_grad");
    set(g_api.norm_scratch, "crx_norm_scratch");
    set(g_api.grad_norm, "crx_grad_norm");
    set(g_api.clip_grads, "crx_clip_grads");
    set(g_api.adamw_step, "crx_adamw_step");
    delete g_stream;
    g_stream = new py::object(std::move(stream));
    g_any_device = any_device;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("init", &init, "the library's entry points, the current stream of a device, and whether any device will do");
    m.def("token_logprobs", &token_logprobs);
    m.def("policy_loss", &policy_loss);
    m.def("grad_norm", &grad_norm);
    m.def("clip_grad_norm", &clip_grad_norm);
    m.def("adamw_step", &adamw_step);
}
