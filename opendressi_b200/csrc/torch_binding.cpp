// The learning operators on torch tensors: argument checks, output and
// workspace allocation, autograd, and one C ABI call (include/dressi_b200.h)
// each. In C++ because these calls are made per layer and per tensor of a
// training step: a group norm's forward and backward cost 166 us of host time
// through Python and ctypes, and a step over 150 tensors 300 us, several times
// what their kernels take.
#include <c10/core/AutogradState.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <limits>
#include <string>
#include <vector>

#include "../../include/dressi_b200.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using c10::optional;

// Becomes opendressi_b200.DressiError.
struct Refused : std::runtime_error {
    int code;
    Refused(int c, const std::string& m) : std::runtime_error(m), code(c) {}
};

[[noreturn]] void refuse(const std::string& m) {
    throw Refused(DRESSI_ERR_INVALID, m);
}

void done(int rc, const char* what) {
    if (rc == DRESSI_OK) return;
    char text[1024];
    dressi_last_error(text, sizeof text);
    throw Refused(rc, std::string(what) + ": " + text);
}

std::string shape_of(const Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); i++)
        s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + ")";
}

int32_t dtype_of(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return DRESSI_F32;
        case at::kHalf: return DRESSI_F16;
        case at::kBFloat16: return DRESSI_BF16;
        default:
            refuse(std::string(name) +
                   " must be float32, float16 or bfloat16, got " +
                   c10::toString(t.scalar_type()));
    }
}

void on_cuda(const Tensor& t, const char* name) {
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided)
        refuse(std::string(name) + " must be a dense CUDA tensor");
}

// t's values packed in memory, a lazy negation (of an imaginary part) done.
Tensor packed(const Tensor& t) { return t.contiguous().resolve_neg(); }

void* stream_of(const Tensor& t) {
    return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

Tensor bytes_on(const Tensor& like, size_t n) {
    return at::empty({int64_t(n)}, like.options().dtype(at::kByte));
}

// Tells autograd that t's values were written: a graph that has kept the ones
// before refuses its backward pass.
void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

const float* floats(const Tensor& t) {
    return t.defined() ? static_cast<const float*>(t.const_data_ptr())
                       : nullptr;
}

// --------------------------------------------------------------- group norm

Tensor table(const Tensor& t, const char* name, const Tensor& x) {
    if (!t.defined()) return t;
    on_cuda(t, name);
    if (t.scalar_type() != at::kFloat)
        refuse(std::string(name) + " must be float32");
    if (t.dim() != 1 || t.size(0) != x.size(-1) || t.device() != x.device())
        refuse(std::string(name) + " must be [" + std::to_string(x.size(-1)) +
               "] on " + x.device().str() + ", got " + shape_of(t) + " on " +
               t.device().str());
    return packed(t);
}

int activation_of(const std::string& name) {
    if (name == "none") return DRESSI_ACT_NONE;
    if (name == "relu") return DRESSI_ACT_RELU;
    if (name == "silu") return DRESSI_ACT_SILU;
    refuse("activation must be \"none\", \"relu\" or \"silu\", got \"" + name +
           "\"");
}

dressi_group_norm_desc norm_desc(const Tensor& x, int64_t groups, double eps,
                                 int activation) {
    on_cuda(x, "x");
    dressi_group_norm_desc d{};
    d.struct_size = sizeof d;
    d.dtype = dtype_of(x, "x");
    if (x.dim() < 2) refuse("x must be [N, ..., C], got " + shape_of(x));
    const int64_t c = x.size(-1);
    if (c < 1 || groups < 1 || c % groups != 0)
        refuse(std::to_string(groups) + " groups do not divide " +
               std::to_string(c) + " channels");
    if (c > std::numeric_limits<int32_t>::max())
        refuse("too many channels");
    d.activation = activation;
    d.channels = uint32_t(c);
    d.groups = uint32_t(groups);
    d.eps = float(eps);
    d.n = uint64_t(x.size(0));
    d.rows = 1;
    for (int64_t i = 1; i + 1 < x.dim(); i++) d.rows *= uint64_t(x.size(i));
    return d;
}

// y and, with stats, mean and rstd [N, groups].
std::vector<Tensor> norm_forward(const Tensor& x_, int64_t groups,
                                 const Tensor& weight_, const Tensor& bias_,
                                 double eps, int activation, bool stats) {
    const dressi_group_norm_desc d = norm_desc(x_, groups, eps, activation);
    const Tensor x = packed(x_);
    const Tensor weight = table(weight_, "weight", x);
    const Tensor bias = table(bias_, "bias", x);
    Tensor y = at::empty_like(x), mean, rstd;
    if (stats) {
        // zeros for a sample without pixels
        const auto opt = x.options().dtype(at::kFloat);
        for (Tensor* t : {&mean, &rstd})
            *t = x.numel() ? at::empty({x.size(0), groups}, opt)
                           : at::zeros({x.size(0), groups}, opt);
    }
    const c10::cuda::CUDAGuard guard(x.device());
    size_t need = 0;
    done(dressi_group_norm_workspace(&d, 0, &need), "group_norm");
    const Tensor space = bytes_on(x, need);
    done(dressi_group_norm(&d, x.const_data_ptr(), floats(weight),
                           floats(bias), y.mutable_data_ptr(),
                           const_cast<float*>(floats(mean)),
                           const_cast<float*>(floats(rstd)),
                           space.mutable_data_ptr(), need, stream_of(x)),
         "group_norm");
    return {y, mean, rstd};
}

// dx, dweight, dbias; undefined where not wanted or without a table.
std::vector<Tensor> norm_backward(const Tensor& dy_, const Tensor& x_,
                                  int64_t groups, const Tensor& weight_,
                                  const Tensor& bias_, const Tensor& mean_,
                                  const Tensor& rstd_, double eps,
                                  int activation, bool want_x,
                                  bool want_weight, bool want_bias) {
    const dressi_group_norm_desc d = norm_desc(x_, groups, eps, activation);
    on_cuda(dy_, "dy");
    if (dy_.sizes() != x_.sizes() || dy_.scalar_type() != x_.scalar_type() ||
        dy_.device() != x_.device())
        refuse("dy must be like x");
    const Tensor x = packed(x_), dy = packed(dy_);
    const Tensor weight = table(weight_, "weight", x);
    const Tensor bias = table(bias_, "bias", x);
    for (const Tensor* t : {&mean_, &rstd_}) {
        on_cuda(*t, "mean / rstd");
        if (t->scalar_type() != at::kFloat || t->dim() != 2 ||
            t->size(0) != x.size(0) || t->size(1) != groups ||
            t->device() != x.device())
            refuse("mean and rstd must be float32 [N, groups] on " +
                   x.device().str() + ", got " + shape_of(*t));
    }
    const Tensor mean = packed(mean_), rstd = packed(rstd_);
    const auto opt = x.options().dtype(at::kFloat);
    Tensor dx, dw, db;
    if (want_x) dx = at::empty_like(x);
    if (want_weight && weight.defined()) dw = at::empty({x.size(-1)}, opt);
    if (want_bias && bias.defined()) db = at::empty({x.size(-1)}, opt);
    const c10::cuda::CUDAGuard guard(x.device());
    size_t need = 0;
    done(dressi_group_norm_workspace(&d, 1, &need), "group_norm_grad");
    const Tensor space = bytes_on(x, need);
    done(dressi_group_norm_grad(
                 &d, dy.const_data_ptr(), x.const_data_ptr(), floats(weight),
                 floats(bias), floats(mean), floats(rstd),
                 dx.defined() ? dx.mutable_data_ptr() : nullptr,
                 const_cast<float*>(floats(dw)),
                 const_cast<float*>(floats(db)), space.mutable_data_ptr(),
                 need, stream_of(x)),
         "group_norm_grad");
    return {dx, dw, db};
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static Tensor forward(torch::autograd::AutogradContext* ctx,
                          const Tensor& x_, int64_t groups,
                          const optional<Tensor>& weight_,
                          const optional<Tensor>& bias_, double eps,
                          int64_t activation) {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor x = x_.contiguous();
        const Tensor weight = weight_.value_or(Tensor());
        const Tensor bias = bias_.value_or(Tensor());
        auto out = norm_forward(x, groups, weight, bias, eps, int(activation),
                                true);
        ctx->save_for_backward({x, weight, bias, out[1], out[2]});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["activation"] = activation;
        return out[0];
    }

    static torch::autograd::variable_list backward(
            torch::autograd::AutogradContext* ctx,
            torch::autograd::variable_list dy) {
        const auto s = ctx->get_saved_variables();
        torch::autograd::variable_list g;
        // edges are counted over the tensors that were given
        const size_t at_bias = s[1].defined() ? 2 : 1;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            g = norm_backward(dy[0], s[0], ctx->saved_data["groups"].toInt(),
                              s[1], s[2], s[3], s[4],
                              ctx->saved_data["eps"].toDouble(),
                              int(ctx->saved_data["activation"].toInt()),
                              ctx->needs_input_grad(0),
                              s[1].defined() && ctx->needs_input_grad(1),
                              s[2].defined() &&
                                      ctx->needs_input_grad(at_bias));
        }
        if (at::GradMode::is_enabled()) {
            // a second derivative is an error, not a silent zero
            auto error = std::make_shared<torch::autograd::Error>(
                    "group_norm is differentiable once",
                    torch::autograd::collect_next_edges(dy[0], s[0], s[1],
                                                        s[2]));
            for (const Tensor& t : g)
                if (t.defined()) torch::autograd::set_history(t, error);
        }
        return {g[0], Tensor(), g[1], g[2], Tensor(), Tensor()};
    }
};

// Whether t carries a tangent that forward-mode differentiation expects a
// result to carry on.
bool has_tangent(const Tensor& t) {
    return c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
           t._fw_grad(/*level=*/0).defined();
}

// Whether something looks at the operators of this thread as they are called
// (a tracer, a dispatch mode, a transform), or t stands for other values than
// its memory holds (a subclass, a transform's wrapper, a lazy negation). What
// is computed past the dispatcher would be missing from a trace.
bool dispatched() {
    for (const auto k :
         {c10::DispatchKey::Python, c10::DispatchKey::PythonDispatcher,
          c10::DispatchKey::Tracer, c10::DispatchKey::Functionalize,
          c10::DispatchKey::FuncTorchDynamicLayerFrontMode})
        if (c10::impl::tls_is_dispatch_key_included(k)) return true;
    return false;
}
bool dispatched(const Tensor& t) {
    return t.key_set().has_any(c10::DispatchKeySet(
            {c10::DispatchKey::Python, c10::DispatchKey::Functionalize,
             c10::DispatchKey::FuncTorchBatched,
             c10::DispatchKey::FuncTorchGradWrapper,
             c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor}));
}

// None where the call has to go through the dispatcher.
optional<Tensor> group_norm(const Tensor& x, int64_t groups,
                            optional<Tensor> weight, optional<Tensor> bias,
                            double eps, const std::string& activation) {
    const int act = activation_of(activation);
    bool grad = x.requires_grad(), tangent = has_tangent(x);
    bool dispatch = dispatched() || dispatched(x);
    for (const optional<Tensor>* t : {&weight, &bias})
        if (t->has_value()) {
            tangent |= has_tangent(**t);
            dispatch |= dispatched(**t);
        }
    // dropped, it would read as a derivative of zero
    if (tangent) refuse("group_norm has no forward-mode derivative");
    if (dispatch) return c10::nullopt;
    for (optional<Tensor>* t : {&weight, &bias})
        if (t->has_value()) {
            on_cuda(**t, t == &weight ? "weight" : "bias");
            *t = (*t)->to(at::kFloat);
            grad |= (*t)->requires_grad();
        }
    if (grad && at::GradMode::is_enabled())
        return GroupNorm::apply(x, groups, weight, bias, eps, int64_t(act));
    return norm_forward(x, groups, weight.value_or(Tensor()),
                        bias.value_or(Tensor()), eps, act, false)[0];
}

// ------------------------------------------------------------------- traces

// The norm and the step below are no operators that a trace could hold: it
// would be left without their result, and without what they write. Modes that
// look on while real tensors are computed are welcome.
void not_traced(const char* what) {
    using Mode = c10::impl::TorchDispatchModeKey;
    bool traced =
            c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::Tracer);
    for (const auto k : {Mode::FAKE, Mode::PROXY, Mode::FUNCTIONAL})
        traced |= c10::impl::TorchDispatchModeTLS::get_mode(k).has_value();
    if (traced) refuse(std::string(what) + " cannot be traced");
}

// --------------------------------------------------------------------- norm

struct Addresses {
    std::vector<const void*> p;
    std::vector<uint64_t> n;
    std::vector<int32_t> type;
    void add(const Tensor& t, int32_t dtype) {
        p.push_back(t.const_data_ptr());
        n.push_back(uint64_t(t.numel()));
        type.push_back(dtype);
    }
};

void norm_of(const Addresses& a, const Tensor& out) {
    size_t need = 0;
    done(dressi_grad_norm_workspace(&need), "grad_norm");
    const Tensor space = bytes_on(out, need);
    done(dressi_grad_norm(uint32_t(a.p.size()), a.p.data(), a.n.data(),
                          a.type.data(),
                          static_cast<float*>(out.mutable_data_ptr()),
                          space.mutable_data_ptr(), need, stream_of(out)),
         "grad_norm");
    written(out);
}

Tensor grad_norm(const std::vector<Tensor>& tensors,
                 const optional<Tensor>& out_) {
    not_traced("grad_norm");
    at::NoGradGuard none;
    Addresses a;
    std::vector<Tensor> held;  // copies of what is not contiguous
    for (const Tensor& t : tensors) {
        on_cuda(t, "tensor");
        const int32_t dtype = dtype_of(t, "tensor");
        if (t.device() != tensors[0].device())
            refuse("tensors on several devices");
        if (t.is_contiguous()) {
            a.add(t, dtype);
        } else {
            held.push_back(t.contiguous());
            a.add(held.back(), dtype);
        }
    }
    const at::Device dev =
            tensors.empty()
                    ? at::Device(at::kCUDA, c10::cuda::current_device())
                    : tensors[0].device();
    const c10::cuda::CUDAGuard guard(dev);
    Tensor out;
    if (out_.has_value()) {
        out = *out_;
        on_cuda(out, "out");
        if (out.scalar_type() != at::kFloat || out.numel() != 1 ||
            out.device() != dev || out.is_neg())
            refuse("out must hold one float32 on " + dev.str());
        if (out.requires_grad()) refuse("out requires a gradient");
    } else {
        out = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(dev));
    }
    norm_of(a, out);
    return out;
}

// -------------------------------------------------------------------- AdamW

// The parameters of a group and where their state is.
struct Pack {
    struct Row {
        Tensor p, g;
        int32_t dtype;
        uint64_t n;
        std::vector<int64_t> sizes, strides;
        void* m;
        void* v;
        float* sm;
        float* sv;
        int32_t* step;
        uint32_t index;
    };
    std::vector<Row> rows;
    std::vector<Tensor> state;  // what the rows' addresses are in
    int32_t state_bits;

    Pack(const std::vector<Tensor>& params, const std::vector<int64_t>& blocks,
         const Tensor& step, const Tensor& m, const Tensor& v,
         const optional<Tensor>& sm, const optional<Tensor>& sv,
         int64_t index, int64_t bits)
        : state{step, m, v}, state_bits(int32_t(bits)) {
        if (bits == 8) state.insert(state.end(), {*sm, *sv});
        for (size_t i = 0; i < params.size(); i++) {
            Row r;
            r.p = params[i];
            r.dtype = dtype_of(r.p, "parameter");
            r.n = uint64_t(r.p.numel());
            r.sizes = r.p.sizes().vec();
            r.strides = r.p.strides().vec();
            const int64_t at = blocks[i] * 256 * m.element_size();
            r.m = static_cast<char*>(m.mutable_data_ptr()) + at;
            r.v = static_cast<char*>(v.mutable_data_ptr()) + at;
            r.sm = r.sv = nullptr;
            if (bits == 8) {
                r.sm = static_cast<float*>(sm->mutable_data_ptr()) + blocks[i];
                r.sv = static_cast<float*>(sv->mutable_data_ptr()) + blocks[i];
            }
            r.step = static_cast<int32_t*>(step.mutable_data_ptr()) + i;
            r.index = uint32_t(index + int64_t(i));
            rows.push_back(std::move(r));
        }
    }

    // Takes each parameter's gradient, in the parameter's order of memory.
    void gather(const at::Device& dev) {
        at::NoGradGuard none;
        for (Row& r : rows) {
            // as many values and the same strides could still be a view that
            // is not dense: the kernel writes numel values in a row
            if (dtype_of(r.p, "parameter") != r.dtype ||
                r.p.device() != dev || r.p.is_neg() ||
                r.p.sizes() != at::IntArrayRef(r.sizes) ||
                r.p.strides() != at::IntArrayRef(r.strides)) {
                refuse("a parameter changed its type, shape or device; make a "
                       "new optimizer");
            }
            r.g = r.p.grad();
            if (!r.g.defined()) continue;
            if (r.g.layout() != at::kStrided || !r.g.is_cuda() ||
                r.g.scalar_type() != r.p.scalar_type() ||
                r.g.sizes() != r.p.sizes() || r.g.device() != dev) {
                refuse("a gradient must be dense and like its parameter");
            }
            if (r.g.is_neg() ||
                (r.g.strides() != r.p.strides() &&
                 !(r.g.is_contiguous() && r.p.is_contiguous()))) {
                r.g = at::empty_strided(r.p.sizes(), r.p.strides(),
                                        r.p.options())
                              .copy_(r.g);
            }
        }
    }

    void release() {
        for (Row& r : rows) r.g = Tensor();
    }

    void step(double lr, const optional<Tensor>& lr_device, double beta1,
              double beta2, double eps, double weight_decay, double lo,
              double hi, double max_norm, const optional<Tensor>& norm,
              int64_t seed, const Tensor& ticket) {
        for (int32_t dtype : {DRESSI_F32, DRESSI_F16, DRESSI_BF16}) {
            std::vector<uint64_t> n;
            std::vector<void*> p, m, v;
            std::vector<const void*> g;
            std::vector<float*> sm, sv;
            std::vector<int32_t*> steps;
            std::vector<uint32_t> index;
            for (const Row& r : rows) {
                if (r.dtype != dtype || !r.g.defined()) continue;
                n.push_back(r.n);
                p.push_back(r.p.mutable_data_ptr());
                g.push_back(r.g.const_data_ptr());
                m.push_back(r.m);
                v.push_back(r.v);
                sm.push_back(r.sm);
                sv.push_back(r.sv);
                steps.push_back(r.step);
                index.push_back(r.index);
            }
            if (n.empty()) continue;
            dressi_adamw_desc d{};
            d.struct_size = sizeof d;
            d.n_tensors = uint32_t(n.size());
            d.dtype = dtype;
            d.state_bits = state_bits;
            d.numel = n.data();
            d.params = p.data();
            d.grads = g.data();
            d.exp_avg = m.data();
            d.exp_avg_sq = v.data();
            d.exp_avg_scale = sm.data();
            d.exp_avg_sq_scale = sv.data();
            d.steps = steps.data();
            d.index = index.data();
            d.lr = lr;
            d.beta1 = beta1;
            d.beta2 = beta2;
            d.eps = eps;
            d.weight_decay = weight_decay;
            d.lr_device = lr_device ? floats(*lr_device) : nullptr;
            d.max_norm = max_norm;
            d.grad_norm = norm ? floats(*norm) : nullptr;
            d.clamp_lo = float(lo);
            d.clamp_hi = float(hi);
            d.seed = uint32_t(seed);
            d.ticket = static_cast<uint32_t*>(ticket.mutable_data_ptr());
            done(dressi_adamw_step(&d, stream_of(ticket)), "adamw");
            for (const Row& r : rows)
                if (r.dtype == dtype && r.g.defined()) written(r.p);
            for (const Tensor& t : state) written(t);
        }
    }
};

// One step of an optimizer: each pack with its group's numbers.
using Numbers = std::tuple<double, optional<Tensor>, double, double, double,
                           double, double, double>;

void adamw_step(const std::vector<Pack*>& packs,
                const std::vector<Numbers>& numbers, double max_norm,
                const optional<Tensor>& norm, int64_t seed,
                const Tensor& ticket) {
    not_traced("an AdamW step");
    const c10::cuda::CUDAGuard guard(ticket.device());
    struct Release {
        const std::vector<Pack*>& packs;
        ~Release() {
            for (Pack* p : packs) p->release();
        }
    } release{packs};
    for (Pack* p : packs) p->gather(ticket.device());
    if (norm) {
        Addresses a;
        for (Pack* p : packs)
            for (const Pack::Row& r : p->rows)
                if (r.g.defined()) a.add(r.g, r.dtype);
        norm_of(a, *norm);
    }
    for (size_t i = 0; i < packs.size(); i++) {
        const auto& [lr, lr_device, b1, b2, eps, wd, lo, hi] = numbers[i];
        packs[i]->step(lr, lr_device, b1, b2, eps, wd, lo, hi, max_norm, norm,
                       seed, ticket);
    }
}

// Whether the values of t fill its extent in memory once, in some order.
bool dense(const Tensor& t) {
    return t.is_non_overlapping_and_dense() && !t.is_neg();
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    // never released: it is used until the interpreter is gone
    static py::object& error = *new py::object(
            py::module_::import("opendressi_b200._native").attr("DressiError"));
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Refused& e) {
            py::object made = error(e.code, std::string(e.what()));
            PyErr_SetObject(error.ptr(), made.ptr());
        }
    });
    m.def("group_norm", &group_norm);
    m.def("group_norm_forward",
          [](const Tensor& x, int64_t groups, const optional<Tensor>& w,
             const optional<Tensor>& b, double eps, const std::string& act,
             bool stats) {
              at::NoGradGuard none;
              return norm_forward(x, groups, w.value_or(Tensor()),
                                  b.value_or(Tensor()), eps,
                                  activation_of(act), stats);
          });
    m.def("group_norm_backward",
          [](const Tensor& dy, const Tensor& x, int64_t groups,
             const optional<Tensor>& w, const optional<Tensor>& b,
             const Tensor& mean, const Tensor& rstd, double eps,
             const std::string& act, bool wx, bool ww, bool wb) {
              at::NoGradGuard none;
              return norm_backward(dy, x, groups, w.value_or(Tensor()),
                                   b.value_or(Tensor()), mean, rstd, eps,
                                   activation_of(act), wx, ww, wb);
          });
    m.def("grad_norm", &grad_norm);
    m.def("dense", &dense);
    m.def("adamw_step", &adamw_step);
    py::class_<Pack>(m, "Pack")
            .def(py::init<const std::vector<Tensor>&,
                          const std::vector<int64_t>&, const Tensor&,
                          const Tensor&, const Tensor&,
                          const optional<Tensor>&, const optional<Tensor>&,
                          int64_t, int64_t>());
}
