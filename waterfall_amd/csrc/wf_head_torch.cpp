// The output head's operators as autograd nodes (waterfall_amd/head.py checks the arguments and calls them).  Kernels are reached
// through the C entry points alone; what is here allocates and keeps tensors.  In C++ because short calls are bound by the
// host: a backward pass runs on the autograd engine's own thread, where Python took several times its usual time (a layer norm
// of 8 x 16 x 64, forward and backward: 131 us with Python nodes).
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <ATen/TensorUtils.h>
#include <c10/core/StreamGuard.h>

#include <unordered_set>

#include "../../include/wf_dwfst.h"

extern "C" int wf_stream_captures(void* stream);                 // wf_head.hip: 1 while a graph is captured from it

namespace {
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;                             // (an argument that may be absent, as autograd takes it)
Tensor get(const Maybe& t) { return t ? *t : Tensor(); }

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return WF_F32;
        case at::kBFloat16: return WF_BF16;
        case at::kHalf: return WF_F16;
        default: TORCH_CHECK(false, "unknown element type ", t.scalar_type());
    }
}
void check(int rc) { TORCH_CHECK(rc == WF_OK, "libwfdwfst error ", rc, ": ", wf_last_error()); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor workspace(size_t n, const Tensor& like) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte)); }

constexpr int64_t kMaxStride = (int64_t)1 << 30;                // elements between rows that the entry points take

// Rows of the last dimension with unit stride inside a row, `ld` elements apart: t itself where its leading dimensions collapse
// into one, else a contiguous copy.
struct Rows {
    Tensor t;
    int64_t n, d, ld;
    explicit Rows(const Tensor& x) : t(x), d(x.size(-1)), ld(x.size(-1)) {
        n = d > 0 ? x.numel() / d : 0;
        if (x.is_contiguous()) return;
        if (x.stride(-1) == 1 || d == 1) {
            const at::DimVector to{n, d};
            const auto s = at::detail::computeStride(x.sizes(), x.strides(), to);
            if (s && (d == 1 || (*s)[1] == 1)) {
                ld = n > 1 ? (*s)[0] : d;
                if (ld < kMaxStride) return;
                ld = d;
            }
        }
        t = x.contiguous();
    }
    void* p() const { return t.data_ptr(); }
};

// No second derivative: asked for one (create_graph), the gradients raise when they are differentiated.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (auto& g : grads)
        if (g.defined()) in.push_back(g.detach().set_requires_grad(true));
    auto node = std::make_shared<torch::autograd::DelayedError>("waterfall_amd.head: no second derivative", (int64_t)in.size());
    variable_list out = (*node)(std::move(in));
    size_t k = 0;
    for (auto& g : grads)
        if (g.defined()) g = out[k++];
    return grads;
}
// A saved tensor as hooks hand it back: it has to be where the gradient is, of the type and shape it had (the entry points take their
// sizes from it); strides and address may be others.
const Tensor& back(const Tensor& t, const Tensor& grad, int64_t type, at::IntArrayRef shape) {
    TORCH_CHECK(!t.defined() || (t.device() == grad.device() && (int64_t)t.scalar_type() == type && t.sizes() == shape),
                "waterfall_amd.head: a saved tensor came back on another device, of another type or in another shape");
    return t;
}
Tensor back_whole(const Tensor& t, const Tensor& grad, int64_t type, at::IntArrayRef shape) {
    return back(t, grad, type, shape).defined() ? t.contiguous() : t;
}
int64_t of(const Tensor& t) { return t.defined() ? (int64_t)t.scalar_type() : 0; }
constexpr int64_t kF32 = (int64_t)at::kFloat;
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }
void* as_stream(int64_t s) { return (void*)(uintptr_t)s; }

// the device's own handle of a stream (asked for under capture alone)
void* handle_of(const c10::Stream& s) {
    const c10::StreamGuard guard(s);
    const pybind11::gil_scoped_acquire gil;
    return as_stream(pybind11::module_::import("torch._C").attr("_cuda_getCurrentRawStream")((int)s.device_index()).cast<int64_t>());
}
// A backward pass that is being captured hands its gradients to the nodes behind it, on the streams where those were made.  The
// accumulator of a leaf that an eager graph uses too is that graph's: the engine would draw the default stream into the capture, or
// another one that nothing joins again, and the process ends when the capture does.  Said here, before it happens.
void no_eager_leaves(int64_t stream) {
    if (!wf_stream_captures(as_stream(stream))) return;
    using torch::autograd::Node;
    const auto* runs = torch::autograd::get_current_graph_task_exec_info();      // empty: everything runs
    std::unordered_set<Node*> seen;
    std::vector<Node*> next{torch::autograd::get_current_node().get()};
    while (!next.empty()) {
        Node* at = next.back();
        next.pop_back();
        if (!at) continue;
        for (const auto& e : at->next_edges()) {
            Node* to = e.function.get();
            if (!to || !seen.insert(to).second) continue;
            bool taken = false;                                  // its gradient is asked for, and it is not run itself
            if (runs && !runs->empty()) {
                const auto it = runs->find(to);
                if (it == runs->end() || !it->second.should_execute()) continue;
                taken = !it->second.needed_;
            }
            if (const auto own = to->stream()) {
                void* s = handle_of(*own);
                TORCH_CHECK(s == as_stream(stream) || (s && !taken) || wf_stream_captures(s),
                            "waterfall_amd.head: a backward pass cannot be captured while an eager graph of the same leaves is alive (", to->name(),
                            " belongs to another stream): delete its outputs first");
            }
            if (!taken) next.push_back(to);
        }
    }
}

// (the engine runs backward with the forward's device and stream current: the stream is kept as it came)
struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight_, const Maybe& bias_, double eps, int64_t stream) {
        const Tensor weight = get(weight_), bias = get(bias_);
        const Rows v(x);
        Tensor y = at::empty(x.sizes(), x.options()), stats;
        const Tensor& par = weight.defined() ? weight : bias.defined() ? bias : x;
        const bool keep = wants(x) || wants(weight) || wants(bias);
        if (keep) stats = at::empty({v.n, 2}, x.options().dtype(at::kFloat));
        check(wf_layer_norm(v.p(), v.ld, v.n, (int32_t)v.d, type_of(x), ptr(weight), ptr(bias), type_of(par), (float)eps, y.data_ptr(),
                            (float*)ptr(stats), as_stream(stream)));
        if (keep) {
            ctx->save_for_backward({v.t, weight, stats});
            ctx->saved_data["a"] = std::vector<int64_t>{wants(weight), wants(bias), of(par), stream, of(x), v.n, v.d};
        }
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto a = ctx->saved_data["a"].toIntVector();
        no_eager_leaves(a[3]);
        const Rows v(back(saved[0], grads[0], a[4], grads[0].sizes())), g(grads[0]);
        const Tensor weight = back_whole(saved[1], grads[0], a[2], {a[6]}), stats = back_whole(saved[2], grads[0], kF32, {a[5], 2});
        Tensor dx = at::empty(v.t.sizes(), v.t.options()), dw, db, ws;
        const auto par = v.t.options().dtype((at::ScalarType)a[2]);
        size_t n = 0;
        if (a[0]) dw = at::empty({v.d}, par);
        if (a[1]) db = at::empty({v.d}, par);
        if (a[0] || a[1]) {
            check(wf_layer_norm_backward_workspace_bytes(v.n, (int32_t)v.d, type_of(v.t), &n));
            ws = workspace(n, v.t);
        }
        const int ptype = (at::ScalarType)a[2] == at::kFloat ? WF_F32 : (at::ScalarType)a[2] == at::kHalf ? WF_F16 : WF_BF16;
        check(wf_layer_norm_backward(g.p(), g.ld, v.p(), v.ld, v.n, (int32_t)v.d, type_of(v.t), ptr(weight), ptype,
                                     (const float*)stats.data_ptr(), dx.data_ptr(), ptr(dw), ptr(db), ptr(ws), n, as_stream(a[3])));
        return once({dx, dw, db, Tensor(), Tensor()});
    }
};

Tensor drop(const Tensor& from, double p, uint64_t seed, const Tensor& at_device, int64_t stream) {
    const Tensor x = from.contiguous();
    Tensor y = at::empty(x.sizes(), x.options());
    check(wf_dropout(x.data_ptr(), x.numel(), type_of(x), p, seed, (const uint64_t*)ptr(at_device), y.data_ptr(), as_stream(stream)));
    return y;
}
struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, int64_t seed, const Maybe& at_device, int64_t stream) {
        ctx->save_for_backward({get(at_device)});
        ctx->saved_data["p"] = p;
        ctx->saved_data["a"] = std::vector<int64_t>{seed, stream};
        return drop(x, p, (uint64_t)seed, get(at_device), stream);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto a = ctx->saved_data["a"].toIntVector();
        no_eager_leaves(a[1]);
        const Tensor seed = ctx->get_saved_variables()[0];
        if (seed.defined()) back(seed.reshape({-1}), grads[0], (int64_t)at::kLong, {1});
        const Tensor dx = drop(grads[0], ctx->saved_data["p"].toDouble(), (uint64_t)a[0], seed, a[1]);
        return once({dx, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

enum { kLogFwd = 0, kLogBwd = 1, kCeFwd = 2, kCeBwd = 3 };
size_t linear_bytes(int what, const Rows& x, const Rows& w) {
    size_t n = 0;
    check(wf_linear_workspace_bytes(what, x.n, (int32_t)x.d, (int32_t)w.n, type_of(x.t), &n));
    return n;
}
at::DimVector rows_of(const Tensor& x, int64_t last) {           // x's shape with another last dimension (0: without it)
    at::DimVector s(x.sizes().begin(), x.sizes().end() - 1);
    if (last) s.push_back(last);
    return s;
}
struct Grads {
    Tensor dx, dw, db;
    Grads(const std::vector<int64_t>& a, const Rows& x, const Rows& w, const Tensor& bias) {
        if (a[0]) dx = at::empty(x.t.sizes(), x.t.options());
        if (a[1]) dw = at::empty(w.t.sizes(), w.t.options());
        if (a[2]) db = at::empty(bias.sizes(), bias.options());
    }
};

struct LogSoftmax : torch::autograd::Function<LogSoftmax> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias_, int64_t stream) {
        const Tensor bias = get(bias_);
        const Rows v(x), w(weight);
        Tensor lp = at::empty(rows_of(x, w.n), x.options().dtype(at::kFloat));
        const size_t n = linear_bytes(kLogFwd, v, w);
        const Tensor ws = workspace(n, x);
        check(wf_linear_log_softmax(v.p(), v.ld, v.n, (int32_t)v.d, w.p(), w.ld, (int32_t)w.n, type_of(x), ptr(bias),
                                    bias.defined() ? type_of(bias) : WF_F32, (float*)lp.data_ptr(), ws.data_ptr(), n, as_stream(stream)));
        ctx->save_for_backward({v.t, w.t, bias, lp});
        ctx->saved_data["a"] = std::vector<int64_t>{wants(x), wants(weight), wants(bias), stream, of(x), of(bias), v.n, v.d, w.n};
        return lp;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto a = ctx->saved_data["a"].toIntVector();
        no_eager_leaves(a[3]);
        const Rows v(back(saved[0], grads[0], a[4], rows_of(grads[0], a[7]))), w(back(saved[1], grads[0], a[4], {a[8], a[7]})), g(grads[0]);
        const Tensor bias = back(saved[2], grads[0], a[5], {a[8]}), lp = back_whole(saved[3], grads[0], kF32, grads[0].sizes());
        const Grads o(a, v, w, bias);
        const size_t n = linear_bytes(kLogBwd, v, w);
        const Tensor ws = workspace(n, v.t);
        check(wf_linear_log_softmax_backward((const float*)lp.data_ptr(), (const float*)g.p(), g.ld, v.p(), v.ld, v.n, (int32_t)v.d,
                                             w.p(), w.ld, (int32_t)w.n, type_of(v.t), bias.defined() ? type_of(bias) : WF_F32, ptr(o.dx),
                                             ptr(o.dw), ptr(o.db), ws.data_ptr(), n, as_stream(a[3])));
        return once({o.dx, o.dw, o.db, Tensor()});
    }
};

enum { kNone = 0, kSum = 1, kMean = 2 };
struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& targets, const Maybe& bias_,
                          int64_t ignore, double smoothing, int64_t reduction, int64_t stream) {
        const Tensor bias = get(bias_);
        const Rows v(x), w(weight);
        const auto f32 = x.options().dtype(at::kFloat);
        Tensor loss = at::empty(rows_of(x, 0), f32), lse = at::empty({v.n}, f32), total;
        if (reduction != kNone) total = at::empty({}, f32);
        const size_t n = linear_bytes(kCeFwd, v, w);
        const Tensor ws = workspace(n, x);
        check(wf_linear_cross_entropy(v.p(), v.ld, v.n, (int32_t)v.d, w.p(), w.ld, (int32_t)w.n, type_of(x), ptr(bias),
                                      bias.defined() ? type_of(bias) : WF_F32, targets.data_ptr(), targets.scalar_type() == at::kLong, ignore,
                                      (float)smoothing, (float*)loss.data_ptr(), (float*)lse.data_ptr(), (float*)ptr(total),
                                      reduction == kMean, ws.data_ptr(), n, as_stream(stream)));
        ctx->save_for_backward({v.t, w.t, targets, bias, lse});
        std::vector<int64_t> a{wants(x), wants(weight), wants(bias), stream, ignore, reduction, of(x), of(bias), of(targets), v.n, v.d, w.n};
        a.insert(a.end(), x.sizes().begin(), x.sizes().end());
        ctx->saved_data["a"] = std::move(a);
        ctx->saved_data["s"] = smoothing;
        return total.defined() ? total : loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const auto a = ctx->saved_data["a"].toIntVector();
        no_eager_leaves(a[3]);
        const auto shape = at::IntArrayRef(a).slice(12);
        const Rows v(back(saved[0], grads[0], a[6], shape)), w(back(saved[1], grads[0], a[6], {a[11], a[10]}));
        const Tensor targets = back_whole(saved[2], grads[0], a[8], shape.slice(0, shape.size() - 1));
        const Tensor bias = back_whole(saved[3], grads[0], a[7], {a[11]}), lse = back_whole(saved[4], grads[0], kF32, {a[9]});
        const Tensor g = grads[0].contiguous();
        const Grads o(a, v, w, bias);
        const size_t n = linear_bytes(kCeBwd, v, w);
        const Tensor ws = workspace(n, v.t);
        check(wf_linear_cross_entropy_backward((const float*)g.data_ptr(), a[5] == kNone, a[5] == kMean, (const float*)lse.data_ptr(),
                                               v.p(), v.ld, v.n, (int32_t)v.d, w.p(), w.ld, (int32_t)w.n, type_of(v.t), ptr(bias),
                                               bias.defined() ? type_of(bias) : WF_F32, targets.data_ptr(),
                                               targets.scalar_type() == at::kLong, a[4], (float)ctx->saved_data["s"].toDouble(), ptr(o.dx),
                                               ptr(o.dw), ptr(o.db), ws.data_ptr(), n, as_stream(a[3])));
        return once({o.dx, o.dw, Tensor(), o.db, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

}  // namespace

PYBIND11_MODULE(_head, m) {
    m.def("layer_norm", [](const Tensor& x, const Maybe& w, const Maybe& b, double eps, int64_t s) { return LayerNorm::apply(x, w, b, eps, s); });
    m.def("dropout", [](const Tensor& x, double p, uint64_t seed, const Maybe& at_device, int64_t s) { return Dropout::apply(x, p, (int64_t)seed, at_device, s); });
    m.def("linear_log_softmax", [](const Tensor& x, const Tensor& w, const Maybe& b, int64_t s) { return LogSoftmax::apply(x, w, b, s); });
    m.def("linear_cross_entropy", [](const Tensor& x, const Tensor& w, const Tensor& t, const Maybe& b, int64_t ignore, double smoothing,
                                     int64_t reduction, int64_t s) { return CrossEntropy::apply(x, w, t, b, ignore, smoothing, reduction, s); });
}
