// torch binding of the layer operators (epi_dropout, epi_layer_norm_* of include/epi.h): argument checks, the tensors a
// call needs, and the autograd nodes.  In C++ because a training step of a small layer is all host time: 512 x 128
// doubles, forward and gradients through torch.autograd.grad, take 60 us this way and 118 with nodes written in
// Python, whose backward pass waits for the interpreter in another thread; the kernels of both together take 12.
//
// The entry points are handed over as addresses, so this module needs no libepi.so of its own beside the one that is
// loaded already.
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <string>
#include <tuple>

#include "../../include/epi.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

namespace {

struct Entries {
    decltype(&epi_dropout) dropout = nullptr;
    decltype(&epi_layer_norm_forward) forward = nullptr;
    decltype(&epi_layer_norm_backward_workspace) workspace = nullptr;
    decltype(&epi_layer_norm_backward) backward = nullptr;
    decltype(&epi_last_error) last_error = nullptr;
} lib;

// Becomes an EpiError in Python.
struct Failure : std::runtime_error {
    int32_t status;
    Failure(int32_t s, const std::string& text) : std::runtime_error(text), status(s) {}
};
[[noreturn]] void refuse(const std::string& text) { throw Failure(EPI_ERR_BAD_ARGUMENT, text); }
void check(int32_t status) {
    if (status == EPI_OK) return;
    char text[1024] = "";
    lib.last_error(text, sizeof text);
    throw Failure(status, text);
}
template <class T>
std::string str(const T& v) { return c10::str(v); }

int32_t dtype_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kDouble: return EPI_F64;
        case at::kFloat: return EPI_F32;
        case at::kBFloat16: return EPI_BF16;
        case at::kHalf: return EPI_F16;
        default: return -1;
    }
}

void check_x(const char* name, const Tensor& x) {
    if (!x.defined()) refuse(std::string(name) + " is missing");
    if (!x.is_cuda()) refuse(std::string(name) + " is on " + str(x.device()) + ": the operators run on the GPU only");
    if (x.layout() != at::kStrided) refuse(std::string(name) + " is not a strided tensor");
    if (dtype_of(x) < 0) refuse(std::string(name) + " holds " + str(x.scalar_type()) + ": float64, float32, bfloat16 and float16 are implemented");
    if (x.dim() < 1 || x.size(-1) < 1) refuse(std::string(name) + " has the shape " + str(x.sizes()) + ": at least one column is needed");
}
void check_like(const char* name, const Tensor& t, const Tensor& x) {
    if (t.device() != x.device()) refuse(std::string(name) + " is on " + str(t.device()) + ", x on " + str(x.device()));
    if (t.scalar_type() != x.scalar_type()) refuse(std::string(name) + " holds " + str(t.scalar_type()) + ", x holds " + str(x.scalar_type()));
}

// A tensor whose rows (the last dimension) are evenly spaced, and their distance: t itself, or a copy.
std::pair<Tensor, int64_t> rows_of(const Tensor& t) {
    const int64_t cols = t.size(-1);
    if (t.is_neg()) return {t.resolve_neg().contiguous(), cols};   // a view whose values are the memory's, negated
    if (t.is_contiguous()) return {t, cols};
    if (cols == 1 || t.stride(-1) == 1) {
        // distance of the last leading dimension of more than one index; the others have to follow from it
        int64_t step = cols, span = 0;
        bool even = true;
        for (int64_t d = t.dim() - 2; d >= 0 && even; --d) {
            if (t.size(d) == 1) continue;
            if (span == 0) { step = t.stride(d); span = step * t.size(d); }
            else { even = t.stride(d) == span; span *= t.size(d); }
        }
        // rows of distance zero have a span of zero: only their neighbours' zero would follow
        if (even && step > 0) return {t, step};
        if (even && t.dim() == 2) return {t, step};
    }
    return {t.contiguous(), cols};
}

Tensor vector_of(const char* name, const Tensor& w, const Tensor& x) {
    if (!w.defined()) return w;
    check_like(name, w, x);
    if (w.dim() != 1 || w.size(0) != x.size(-1)) refuse(std::string(name) + " has the shape " + str(w.sizes()) + " for " + str(x.size(-1)) + " columns");
    return (w.is_neg() ? w.resolve_neg() : w).contiguous();
}

// What a call drops with; `offset_dev` may be undefined.
struct Drop {
    double p = 0.0;
    int64_t seed = 0, offset = 0;
    Tensor offset_dev;
};

epi_layer_desc desc_of(const Tensor& x, double eps, const Drop& drop) {
    epi_layer_desc d{};
    d.cols = x.size(-1);
    d.rows = x.numel() / d.cols;
    d.eps = eps;
    d.dropout = drop.p; d.seed = drop.seed; d.offset = drop.offset;
    if (drop.offset_dev.defined()) {
        const Tensor& o = drop.offset_dev;
        if (o.device() != x.device() || o.scalar_type() != at::kLong || o.numel() != 1)
            refuse("offset is a number, or a tensor of one int64 on " + str(x.device()));
        d.offset_dev = o.data_ptr<int64_t>();
    }
    d.dtype = dtype_of(x);
    d.device = x.get_device();
    return d;
}
void* stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.get_device()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor empty_like_rows(const Tensor& x) { return at::empty(x.sizes(), x.options()); }

// ---- the calls ------------------------------------------------------------------------------------------
Tensor run_dropout(const Tensor& t, const Drop& drop) {
    const auto [x, stride] = rows_of(t);
    epi_layer_desc d = desc_of(x, 0.0, drop);
    Tensor y = empty_like_rows(x);
    d.x_stride = stride; d.y_stride = d.cols;
    check(lib.dropout(&d, x.data_ptr(), y.data_ptr(), stream_of(x)));
    return y;
}

// (y, stats): stats holds the rows' means, then their 1 / deviation
std::pair<Tensor, Tensor> run_forward(const Tensor& t, const Tensor& w, const Tensor& b, double eps, const Drop& drop, bool want_stats) {
    const auto [x, stride] = rows_of(t);
    const Tensor weight = vector_of("weight", w, x), bias = vector_of("bias", b, x);
    epi_layer_desc d = desc_of(x, eps, drop);
    Tensor y = empty_like_rows(x), stats;
    d.x_stride = stride; d.y_stride = d.cols;
    void *mean = nullptr, *rstd = nullptr;
    if (want_stats) {
        stats = at::empty({2, d.rows}, x.options().dtype(d.dtype == EPI_F64 ? at::kDouble : at::kFloat));
        mean = stats.data_ptr();
        rstd = static_cast<char*>(mean) + d.rows * stats.element_size();
    }
    check(lib.forward(&d, x.data_ptr(), ptr(weight), ptr(bias), y.data_ptr(), mean, rstd, stream_of(x)));
    return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> run_backward(const Tensor& g, const Tensor& t, const Tensor& w, const void* mean, const void* rstd,
                                                const Drop& drop, bool want_x, bool want_weight, bool want_bias) {
    const auto [x, stride] = rows_of(t);
    const auto [dy, dy_stride] = rows_of(g);
    const Tensor weight = vector_of("weight", w, x);
    epi_layer_desc d = desc_of(x, 0.0, drop);
    d.x_stride = stride; d.dy_stride = dy_stride; d.y_stride = d.cols;
    Tensor dx, dweight, dbias, work;
    if (want_x) dx = empty_like_rows(x);
    if (want_weight) dweight = at::empty({d.cols}, x.options());
    if (want_bias) dbias = at::empty({d.cols}, x.options());
    size_t need = 0;
    if (want_weight || want_bias) check(lib.workspace(&d, &need));
    if (need) work = at::empty({(int64_t)need}, x.options().dtype(at::kByte));
    check(lib.backward(&d, x.data_ptr(), dy.data_ptr(), ptr(weight), mean, rstd, ptr(dx), ptr(dweight), ptr(dbias), ptr(work), need,
                       stream_of(x)));
    return {dx, dweight, dbias};
}

// ---- autograd -----------------------------------------------------------------------------------------------
// Gradients are values only: asked to differentiate them again (create_graph), the node behind them refuses.
variable_list once(variable_list grads, bool again) {
    if (!again) return grads;
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    auto error = std::make_shared<torch::autograd::DelayedError>("the gradients of layer operators cannot be differentiated again", (int)grads.size());
    return (*error)(std::move(grads));
}

// The nodes of the graph, with what their backward passes need.
struct DropoutNode : torch::autograd::Node {
    Drop drop;
    SavedVariable offset_dev;
    variable_list apply(variable_list&& grads) override {
        const bool again = at::GradMode::is_enabled();
        at::AutoGradMode off(false);
        variable_list out(1);
        if (grads[0].defined()) {
            Drop d = drop;
            d.offset_dev = offset_dev.unpack();
            out[0] = run_dropout(grads[0], d);
        }
        at::AutoGradMode on(again);
        return once(std::move(out), again);
    }
    void release_variables() override { offset_dev.reset_data(); }
    std::string name() const override { return "EpiDropoutBackward"; }
};

struct NormNode : torch::autograd::Node {
    Drop drop;
    SavedVariable x, weight, stats, offset_dev;
    variable_list apply(variable_list&& grads) override {
        const bool again = at::GradMode::is_enabled();
        at::AutoGradMode off(false);
        variable_list out(3);
        if (grads[0].defined()) {
            const Tensor s = stats.unpack();
            Drop d = drop;
            d.offset_dev = offset_dev.unpack();
            const char* mean = static_cast<const char*>(s.data_ptr());
            std::tie(out[0], out[1], out[2]) =
                run_backward(grads[0], x.unpack(), weight.unpack(), mean, mean + s.size(1) * s.element_size(), d, task_should_compute_output(0),
                             task_should_compute_output(1), task_should_compute_output(2));
        }
        at::AutoGradMode on(again);
        return once(std::move(out), again);
    }
    void release_variables() override {
        x.reset_data(); weight.reset_data(); stats.reset_data(); offset_dev.reset_data();
    }
    std::string name() const override { return "EpiLayerNormBackward"; }
};

// A leaf that an eager graph still holds collects its gradient on that graph's stream.  A backward pass captured into a
// HIP graph meanwhile would wait across the two streams, which is no part of a capture and ends the process: refused
// while the forward pass is being captured.
void check_capture(std::initializer_list<Tensor> leaves, const Tensor& x) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto here = c10::hip::getCurrentHIPStream(x.get_device()).id();
    for (const Tensor& t : leaves) {
        if (!t.defined() || !t.requires_grad() || !t.is_leaf()) continue;
        const auto collects = torch::autograd::impl::try_get_grad_accumulator(t);
        if (collects && collects->stream() && collects->stream()->id() != here)
            refuse("an eager graph of the same leaf is alive: drop its outputs before capturing, or capture layer_norm_forward and layer_norm_backward");
    }
}

template <class N>
std::shared_ptr<N> new_node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }

Tensor record_dropout(const Tensor& x, const Drop& drop) {
    check_capture({x}, x);
    Tensor y;
    {
        at::AutoGradMode off(false);
        y = run_dropout(x, drop);
    }
    auto node = new_node<DropoutNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->drop = drop;
    node->drop.offset_dev.reset();
    node->offset_dev = SavedVariable(drop.offset_dev, false);
    torch::autograd::set_history(y, node);
    return y;
}
Tensor record_norm(const Tensor& x, const Tensor& w, const Tensor& b, double eps, const Drop& drop) {
    check_capture({x, w, b}, x);
    std::pair<Tensor, Tensor> r;
    {
        at::AutoGradMode off(false);
        r = run_forward(x, w, b, eps, drop, true);
    }
    auto node = new_node<NormNode>();
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    node->drop = drop;
    node->drop.offset_dev.reset();
    node->x = SavedVariable(x, false);
    node->weight = SavedVariable(w, false);
    node->stats = SavedVariable(r.second, false);
    node->offset_dev = SavedVariable(drop.offset_dev, false);
    torch::autograd::set_history(r.first, node);
    return r.first;
}

// ---- what Python calls ------------------------------------------------------------------------------------
// Any integer, taken modulo 2^64.
int64_t word(const py::handle& v) {
    const unsigned long long w = PyLong_AsUnsignedLongLongMask(v.ptr());
    if (PyErr_Occurred()) throw py::error_already_set();
    return (int64_t)w;
}
// Seed and offset as numbers, or the offset as a tensor.
Drop drop_of(double p, const py::handle& seed, const py::handle& offset) {
    Drop d;
    d.p = p;
    d.seed = word(seed);
    if (THPVariable_Check(offset.ptr())) d.offset_dev = THPVariable_Unpack(offset.ptr());
    else d.offset = word(offset);
    return d;
}
Tensor tensor_of(const char* name, const py::handle& v, bool optional) {
    if (optional && v.is_none()) return Tensor();
    if (!THPVariable_Check(v.ptr())) refuse(std::string(name) + " is not a tensor");
    return THPVariable_Unpack(v.ptr());
}
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

Tensor dropout(const py::handle& x_, double p, const py::handle& seed, const py::handle& offset) {
    const Tensor x = tensor_of("x", x_, false);
    const Drop drop = drop_of(p, seed, offset);
    py::gil_scoped_release free;
    check_x("x", x);
    return at::GradMode::is_enabled() && wants(x) ? record_dropout(x, drop) : run_dropout(x, drop);
}
Tensor layer_norm(const py::handle& x_, const py::handle& w_, const py::handle& b_, double eps, double p, const py::handle& seed, const py::handle& offset) {
    const Tensor x = tensor_of("x", x_, false), w = tensor_of("weight", w_, true), b = tensor_of("bias", b_, true);
    const Drop drop = drop_of(p, seed, offset);
    py::gil_scoped_release free;
    check_x("x", x);
    if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b))) return record_norm(x, w, b, eps, drop);
    return run_forward(x, w, b, eps, drop, false).first;
}
std::tuple<Tensor, Tensor, Tensor> layer_norm_forward(const py::handle& x_, const py::handle& w_, const py::handle& b_, double eps, double p,
                                                      const py::handle& seed, const py::handle& offset) {
    const Tensor x = tensor_of("x", x_, false), w = tensor_of("weight", w_, true), b = tensor_of("bias", b_, true);
    const Drop drop = drop_of(p, seed, offset);
    py::gil_scoped_release free;
    at::AutoGradMode off(false);
    check_x("x", x);
    const auto [y, stats] = run_forward(x, w, b, eps, drop, true);
    return {y, stats.select(0, 0), stats.select(0, 1)};
}
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const py::handle& dy_, const py::handle& x_, const py::handle& w_, const py::handle& mean_,
                                                       const py::handle& rstd_, double p, const py::handle& seed, const py::handle& offset) {
    const Tensor dy = tensor_of("dy", dy_, false), x = tensor_of("x", x_, false), w = tensor_of("weight", w_, true);
    const Tensor mean = tensor_of("mean", mean_, false), rstd = tensor_of("rstd", rstd_, false);
    const Drop drop = drop_of(p, seed, offset);
    py::gil_scoped_release free;
    at::AutoGradMode off(false);
    check_x("x", x);
    check_x("dy", dy);
    check_like("dy", dy, x);
    if (dy.sizes() != x.sizes()) refuse("dy has the shape " + str(dy.sizes()) + ", x " + str(x.sizes()));
    const auto wide = x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
    const int64_t rows = x.numel() / x.size(-1);
    for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"mean", mean}, {"rstd", rstd}})
        if (t.device() != x.device() || t.scalar_type() != wide || !t.is_contiguous() || t.numel() != rows)
            refuse(std::string(name) + " is not the forward pass's: " + str(rows) + " numbers of " + str(wide) + " on " + str(x.device()));
    return run_backward(dy, x, w, mean.data_ptr(), rstd.data_ptr(), drop, true, true, true);
}

template <class F>
void take(F& slot, const py::dict& addresses, const char* name) {
    slot = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

}  // namespace

PYBIND11_MODULE(_layers, m) {
    py::register_exception_translator([](std::exception_ptr e) {
        try {
            if (e) std::rethrow_exception(e);
        } catch (const Failure& f) {
            const py::object type = py::module_::import("epidemicsimulator_amd._capi").attr("EpiError");
            PyErr_SetObject(type.ptr(), type(f.status, f.what()).ptr());
        }
    });
    m.def("bind", [](const py::dict& a) {
        take(lib.dropout, a, "epi_dropout");
        take(lib.forward, a, "epi_layer_norm_forward");
        take(lib.workspace, a, "epi_layer_norm_backward_workspace");
        take(lib.backward, a, "epi_layer_norm_backward");
        take(lib.last_error, a, "epi_last_error");
    });
    m.def("dropout", &dropout);
    m.def("layer_norm", &layer_norm);
    m.def("layer_norm_forward", &layer_norm_forward);
    m.def("layer_norm_backward", &layer_norm_backward);
}
