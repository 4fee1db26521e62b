// torch binding of the layer operators (epi_dropout, epi_layer_norm_* of include/epi.h): argument checks, the tensors a
// call needs, and the autograd nodes.  In C++ because a training step of a small layer is all host time: 512 x 128
// doubles, forward and gradients through torch.autograd.grad, take 58 to 67 us this way and 118 with nodes written in
// Python, whose backward pass waits for the interpreter in another thread; the kernels of both together take 12, and
// torch's engine 23 to 43 for a node that does nothing.
//
// The calls bypass torch's dispatcher: what it would do by itself (views that are negated, tangents, captures) is done or
// refused here.
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

#include <algorithm>
#include <mutex>
#include <optional>
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
    if (!lib.dropout) refuse("import epidemicsimulator_amd.layers: this module is a part of it");
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

// Fake and zero tensors have shapes and strides, and no memory: a view of one has an address all the same.
const Tensor& check_memory(const Tensor& t) {
    if (t.numel() && !t.storage().data()) refuse("a tensor has no memory (a fake tensor, or zeros that were never stored)");
    return t;
}

// The distance between rows (the last dimension) that are evenly spaced over all leading dimensions, the last of them
// running fastest; nothing where they are not, or where a row's columns do not lie next to each other.
std::optional<int64_t> row_distance(at::IntArrayRef sizes, at::IntArrayRef strides) {
    const int64_t cols = sizes.back();
    if (std::find(sizes.begin(), sizes.end(), 0) != sizes.end()) return cols;   // no rows
    if (cols != 1 && strides.back() != 1) return std::nullopt;
    // The innermost leading dimension of more than one index sets the distance; the others have to follow from it.  A
    // distance of zero counts like any other: what is expanded inside and moves outside is not evenly spaced.
    int64_t step = cols, next = 0;
    bool seen = false;
    for (int64_t d = (int64_t)sizes.size() - 2; d >= 0; --d) {
        if (sizes[d] == 1) continue;
        if (!seen) { step = next = strides[d]; seen = true; }
        if (strides[d] != next) return std::nullopt;
        next *= sizes[d];
    }
    return step;
}

// A tensor whose rows are evenly spaced, and their distance: t itself, or a copy.
std::pair<Tensor, int64_t> rows_of(const Tensor& t) {
    check_memory(t);
    if (t.is_neg()) return {t.resolve_neg().contiguous(), t.size(-1)};   // a view whose values are the memory's, negated
    if (const auto step = row_distance(t.sizes(), t.strides())) return {t, *step};
    return {t.contiguous(), t.size(-1)};
}

Tensor vector_of(const char* name, const Tensor& w, const Tensor& x) {
    if (!w.defined()) return w;
    check_like(name, w, x);
    if (w.dim() != 1 || w.size(0) != x.size(-1)) refuse(std::string(name) + " has the shape " + str(w.sizes()) + " for " + str(x.size(-1)) + " columns");
    return (check_memory(w).is_neg() ? w.resolve_neg() : w).contiguous();
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
        d.offset_dev = check_memory(o).data_ptr<int64_t>();
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

// Gradients are taken backwards only: the tangent of a dual tensor (forward-mode derivatives) would be lost, which reads
// as a derivative of zero.  Refused, unless forward mode is switched off.
template <class... T>
void refuse_tangents(const T&... inputs) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    if (((inputs.defined() && inputs._fw_grad(/*level=*/0).defined()) || ...)) refuse("layer operators have no forward-mode derivatives");
}

// The nodes of the graph, with what their backward passes need; a pass holds the node's mutex, so that one that releases
// the graph's tensors waits for another that reads them.
struct DropoutNode : torch::autograd::Node {
    Drop drop;
    SavedVariable offset_dev;
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const bool again = at::GradMode::is_enabled();
        at::AutoGradMode off(false);
        variable_list out(1);
        if (grads[0].defined()) {
            refuse_tangents(grads[0]);
            Drop d = drop;
            d.offset_dev = offset_dev.unpack();
            out[0] = run_dropout(grads[0], d);
        }
        at::AutoGradMode on(again);
        return once(std::move(out), again);
    }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        offset_dev.reset_data();
    }
    std::string name() const override { return "EpiDropoutBackward"; }
};

struct NormNode : torch::autograd::Node {
    Drop drop;
    SavedVariable x, weight, stats, offset_dev;
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        const bool again = at::GradMode::is_enabled();
        at::AutoGradMode off(false);
        variable_list out(3);
        if (grads[0].defined()) {
            refuse_tangents(grads[0]);
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
        std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data(); weight.reset_data(); stats.reset_data(); offset_dev.reset_data();
    }
    std::string name() const override { return "EpiLayerNormBackward"; }
};

// A leaf that an eager graph still holds collects its gradient on that graph's stream.  A backward pass captured into a
// HIP graph meanwhile would wait across the two streams, which is no part of a capture and ends the process: refused
// while the forward pass is being captured, for the leaves among the inputs and those that the inputs are views of.
void check_capture(std::initializer_list<Tensor> inputs, const Tensor& x) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    const auto here = c10::hip::getCurrentHIPStream(x.get_device()).id();
    for (const Tensor& t : inputs) {
        if (!t.defined() || !t.requires_grad()) continue;
        const Tensor leaf = !t.is_leaf() && t.is_view() ? Tensor(t._base()) : t;
        if (!leaf.is_leaf() || !leaf.requires_grad()) continue;
        const auto collects = torch::autograd::impl::try_get_grad_accumulator(leaf);
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
// Plain functions of the interpreter's fast call: a small call is mostly its way here and back.

// Positional and named arguments into slots; `required` of them have to be there.
template <size_t N>
bool parse(const char* function, const char* const (&names)[N], size_t required, PyObject* const* args, Py_ssize_t count, PyObject* keywords,
           PyObject* (&slots)[N]) {
    for (auto& s : slots) s = nullptr;
    if (count > (Py_ssize_t)N) {
        PyErr_Format(PyExc_TypeError, "%s() takes at most %zu arguments, %zd given", function, N, count);
        return false;
    }
    for (Py_ssize_t k = 0; k < count; ++k) slots[k] = args[k];
    const Py_ssize_t named = keywords ? PyTuple_GET_SIZE(keywords) : 0;
    for (Py_ssize_t k = 0; k < named; ++k) {
        PyObject* key = PyTuple_GET_ITEM(keywords, k);
        size_t at = 0;
        while (at < N && PyUnicode_CompareWithASCIIString(key, names[at]) != 0) ++at;
        if (at == N || slots[at]) {
            PyErr_Format(PyExc_TypeError, at == N ? "%s() has no argument named %R" : "%s() got argument %R twice", function, key);
            return false;
        }
        slots[at] = args[count + k];
    }
    for (size_t k = 0; k < required; ++k)
        if (!slots[k]) {
            PyErr_Format(PyExc_TypeError, "%s() needs the argument '%s'", function, names[k]);
            return false;
        }
    return true;
}

double number(PyObject* v, double otherwise) {
    if (!v) return otherwise;
    const double d = PyFloat_AsDouble(v);
    if (d == -1.0 && PyErr_Occurred()) throw python_error();
    return d;
}
// Any integer, taken modulo 2^64.
int64_t word(PyObject* v) {
    if (!v) return 0;
    const unsigned long long w = PyLong_AsUnsignedLongLongMask(v);
    if (w == (unsigned long long)-1 && PyErr_Occurred()) throw python_error();
    return (int64_t)w;
}
// Seed and offset as numbers, or the offset as a tensor.
Drop drop_of(PyObject* p, PyObject* seed, PyObject* offset) {
    Drop d;
    d.p = number(p, 0.0);
    d.seed = word(seed);
    if (offset && THPVariable_Check(offset)) d.offset_dev = THPVariable_Unpack(offset);
    else d.offset = word(offset);
    return d;
}
Tensor tensor_of(const char* name, PyObject* v, bool optional) {
    if (optional && (!v || v == Py_None)) return Tensor();
    if (!THPVariable_Check(v)) refuse(std::string(name) + " is not a tensor");
    return THPVariable_Unpack(v);
}
bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Runs f; a Failure becomes the package's EpiError, everything else what torch makes of it.
template <class F>
PyObject* guarded(F f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Failure& e) {
        const py::object type = py::module_::import("epidemicsimulator_amd._capi").attr("EpiError");
        PyErr_SetObject(type.ptr(), type(e.status, e.what()).ptr());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}
PyObject* triple(const std::tuple<Tensor, Tensor, Tensor>& t) {
    py::tuple out(3);
    out[0] = py::reinterpret_steal<py::object>(THPVariable_Wrap(std::get<0>(t)));
    out[1] = py::reinterpret_steal<py::object>(THPVariable_Wrap(std::get<1>(t)));
    out[2] = py::reinterpret_steal<py::object>(THPVariable_Wrap(std::get<2>(t)));
    return out.release().ptr();
}

PyObject* dropout(PyObject*, PyObject* const* args, Py_ssize_t count, PyObject* keywords) {
    static const char* const names[] = {"x", "p", "seed", "offset"};
    PyObject* v[4];
    if (!parse("dropout", names, 3, args, count, keywords, v)) return nullptr;
    return guarded([&] {
        const Tensor x = tensor_of("x", v[0], false);
        const Drop drop = drop_of(v[1], v[2], v[3]);
        Tensor y;
        {
            py::gil_scoped_release free;
            refuse_tangents(x);
            check_x("x", x);
            y = at::GradMode::is_enabled() && wants(x) ? record_dropout(x, drop) : run_dropout(x, drop);
        }
        return THPVariable_Wrap(std::move(y));
    });
}

const char* const kNormNames[] = {"x", "weight", "bias", "eps", "dropout", "seed", "offset"};

PyObject* layer_norm(PyObject*, PyObject* const* args, Py_ssize_t count, PyObject* keywords) {
    PyObject* v[7];
    if (!parse("layer_norm", kNormNames, 1, args, count, keywords, v)) return nullptr;
    return guarded([&] {
        const Tensor x = tensor_of("x", v[0], false), w = tensor_of("weight", v[1], true), b = tensor_of("bias", v[2], true);
        const double eps = number(v[3], 1e-5);
        const Drop drop = drop_of(v[4], v[5], v[6]);
        Tensor y;
        {
            py::gil_scoped_release free;
            refuse_tangents(x, w, b);
            check_x("x", x);
            y = at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b)) ? record_norm(x, w, b, eps, drop)
                                                                                : run_forward(x, w, b, eps, drop, false).first;
        }
        return THPVariable_Wrap(std::move(y));
    });
}

PyObject* layer_norm_forward(PyObject*, PyObject* const* args, Py_ssize_t count, PyObject* keywords) {
    PyObject* v[7];
    if (!parse("layer_norm_forward", kNormNames, 1, args, count, keywords, v)) return nullptr;
    return guarded([&] {
        const Tensor x = tensor_of("x", v[0], false), w = tensor_of("weight", v[1], true), b = tensor_of("bias", v[2], true);
        const double eps = number(v[3], 1e-5);
        const Drop drop = drop_of(v[4], v[5], v[6]);
        std::tuple<Tensor, Tensor, Tensor> out;
        {
            py::gil_scoped_release free;
            at::AutoGradMode off(false);
            check_x("x", x);
            const auto [y, stats] = run_forward(x, w, b, eps, drop, true);
            out = {y, stats.select(0, 0), stats.select(0, 1)};
        }
        return triple(out);
    });
}

PyObject* layer_norm_backward(PyObject*, PyObject* const* args, Py_ssize_t count, PyObject* keywords) {
    static const char* const names[] = {"dy", "x", "weight", "mean", "rstd", "dropout", "seed", "offset"};
    PyObject* v[8];
    if (!parse("layer_norm_backward", names, 5, args, count, keywords, v)) return nullptr;
    return guarded([&] {
        const Tensor dy = tensor_of("dy", v[0], false), x = tensor_of("x", v[1], false), w = tensor_of("weight", v[2], true);
        const Tensor mean = tensor_of("mean", v[3], false), rstd = tensor_of("rstd", v[4], false);
        const Drop drop = drop_of(v[5], v[6], v[7]);
        std::tuple<Tensor, Tensor, Tensor> out;
        {
            py::gil_scoped_release free;
            at::AutoGradMode off(false);
            check_x("x", x);
            check_x("dy", dy);
            check_like("dy", dy, x);
            if (dy.sizes() != x.sizes()) refuse("dy has the shape " + str(dy.sizes()) + ", x " + str(x.sizes()));
            const auto wide = x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
            const int64_t rows = x.numel() / x.size(-1);
            for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"mean", mean}, {"rstd", rstd}})
                if (t.device() != x.device() || t.scalar_type() != wide || !t.is_contiguous() || t.is_neg() || t.numel() != rows)
                    refuse(std::string(name) + " is not the forward pass's: " + str(rows) + " numbers of " + str(wide) + " on " + str(x.device()));
                else
                    check_memory(t);
            out = run_backward(dy, x, w, mean.data_ptr(), rstd.data_ptr(), drop, true, true, true);
        }
        return triple(out);
    });
}

template <class F>
void take(F& slot, const py::dict& addresses, const char* name) {
    slot = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

PyMethodDef functions[] = {
    {"dropout", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&dropout)), METH_FASTCALL | METH_KEYWORDS,
     R"(dropout($module, x, p, seed, offset=0)
--

Each element dropped with probability p (rounded to a multiple of 2^-16), the others multiplied so that the mean
stays; differentiable, backwards.  The mask is a function of (seed, offset, row, column) alone: calls that are to draw
independently -- layers, steps -- take different offsets or seeds.  `offset` may be a tensor of one int64 on x's
device, read when the kernels run: a captured graph then drops other elements on every replay if the program
changes it between replays (not between a forward pass and its backward pass).)"},
    {"layer_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&layer_norm)), METH_FASTCALL | METH_KEYWORDS,
     R"(layer_norm($module, x, weight=None, bias=None, eps=1e-05, dropout=0.0, seed=0, offset=0)
--

(h - mean h) / sqrt(mean (h - mean h)^2 + eps) * weight + bias over the last dimension, with h = x, or
h = dropout(x, dropout, seed, offset) in the same pass; differentiable, backwards, in x, weight and bias.  weight and bias hold
x's type; sums are taken in float32 (float64 for float64) and y is rounded once.  Captured into a graph with its
backward pass while an eager graph of the same leaves is alive, the call is refused: of the leaves that it is given or
given views of; further up, other operators meet the same limit of captures.)"},
    {"layer_norm_forward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&layer_norm_forward)), METH_FASTCALL | METH_KEYWORDS,
     R"(layer_norm_forward($module, x, weight=None, bias=None, eps=1e-05, dropout=0.0, seed=0, offset=0)
--

layer_norm without autograd: (y, mean, 1 / standard deviation), the latter two one number a row.)"},
    {"layer_norm_backward", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&layer_norm_backward)), METH_FASTCALL | METH_KEYWORDS,
     R"(layer_norm_backward($module, dy, x, weight, mean, rstd, dropout=0.0, seed=0, offset=0)
--

(dx, dweight, dbias) from dy and what layer_norm_forward took and gave; without autograd, so it can be captured
into a graph whatever else holds on to the leaves.)"},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(_layers, m) {
    m.def("bind", [](const py::dict& a) {
        take(lib.dropout, a, "epi_dropout");
        take(lib.forward, a, "epi_layer_norm_forward");
        take(lib.workspace, a, "epi_layer_norm_backward_workspace");
        take(lib.backward, a, "epi_layer_norm_backward");
        take(lib.last_error, a, "epi_last_error");
    });
    // which tensors the calls read where they are, for tests without a GPU
    m.def("row_distance", [](const Tensor& t) {
        if (t.dim() < 1) throw py::value_error("at least one dimension is needed");
        return row_distance(t.sizes(), t.strides());
    });
    if (PyModule_AddFunctions(m.ptr(), functions) != 0) throw py::error_already_set();
}
