// erfnet_pytorch_amd._host: the host side of the calls that are shorter than their Python would be.
//   layer_norm, log_probs: autograd nodes over the C ABI (with a backward pass that enters Python from autograd's
//     thread, log probabilities of 256 x 1000 with gradients took 117 us around 15 us of kernels; 67 so);
//   adamw_step: one pass over the parameters (229 of them, 20 us of GPU work: 583 us a step in Python, 33 so).
// Arguments come checked from functional.py / optim.py.  Nothing is kept between calls.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <deque>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "../../include/erfnet_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The library's entry points for fp32 and bf16 tensors, handed over once by bind() (the library that the package has loaded,
// wherever it lies).
struct Library {
    decltype(&erf_last_error) last_error;
    decltype(&erf_layer_norm_workspace_bytes) norm_ws;
    decltype(&erf_log_probs_workspace_bytes) logp_ws;
    decltype(&erf_layer_norm_forward_bf16) norm_fwd[2];
    decltype(&erf_layer_norm_backward_bf16) norm_bwd[2];
    decltype(&erf_log_probs_forward_bf16) logp_fwd[2];
    decltype(&erf_log_probs_backward_bf16) logp_bwd[2];
    decltype(&erf_adamw_step_bf16) adamw[2];
    decltype(&erf_adamw8_step_bf16) adamw8[2];
} lib;

// Other Python threads run while this lives: allocations may call the driver, and a launch waits where the queue is full.
struct Unlocked {
    PyThreadState *state = PyEval_SaveThread();
    Unlocked() = default;
    Unlocked(const Unlocked &) = delete;
    ~Unlocked() { PyEval_RestoreThread(state); }
};

int kind(const Tensor &t) { return t.scalar_type() == at::kBFloat16; }
void check(int rc)
{
    if (rc) throw std::runtime_error(std::string("erfnet_hip: ") + lib.last_error());
}
void *stream(const c10::Device &d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }
float *floats(const Tensor &t) { return t.defined() ? (float *)t.data_ptr() : nullptr; }
// (not through the dispatcher, which takes as long as the allocation: there are up to seven of these in a call)
Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const Tensor &beside, bool image = false)
{
    return Tensor(at::detail::empty_cuda(shape, type, beside.device(),
                                         image ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous));
}
// The numbers themselves, where t is a view that stands for its negative (the imaginary part of a conjugate; such a view of one
// number counts as contiguous).
Tensor numbers(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor parameter(const Tensor &t) { return t.defined() ? numbers(t.to(at::kFloat).contiguous()) : t; }

// What backward returns, from an operator whose gradient has none: where a graph of the backward pass is recorded
// (`recorded`), the results hang on a node that raises, in front of everything that they depend on: the upstream gradients,
// and the inputs by the edges of the node that is running (the tensors it has saved may be copies and views of the inputs,
// made without a graph: autograd would find no way from them to the inputs, and leave the node out).
variable_list first_order(variable_list grads, bool recorded, const variable_list &upstream)
{
    if (!recorded) return grads;
    torch::autograd::edge_list edges = torch::autograd::collect_next_edges(upstream);
    if (const auto running = torch::autograd::get_current_node())
        edges.insert(edges.end(), running->next_edges().begin(), running->next_edges().end());
    if (std::none_of(edges.begin(), edges.end(), [](const torch::autograd::Edge &e) { return e.is_valid(); })) return grads;
    const at::AutoGradMode on(true);
    auto node = std::make_shared<torch::autograd::Error>(
        "erfnet_pytorch_amd: the gradient of layer_norm / log_probs is not differentiable", std::move(edges));
    for (Tensor &g : grads)
        if (g.defined()) torch::autograd::set_history(g, node);
    return grads;
}

// The operators and their gradients have no forward derivative; where no node is left there is none to say so.
void no_tangents(const char *what, at::ArrayRef<Tensor> inputs)
{
    for (const Tensor &t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(t), "erfnet_pytorch_amd: ", what,
                                    " has no forward-mode derivative");
}

// A tracer sees nothing of calls past the dispatcher: the results would be constants of its graph.
void no_tracing(const char *what)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() &&
                                    !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
                                "erfnet_pytorch_amd: ", what, " cannot be traced");
}

// ---------------------------------------------------------------------------------------------- layer norm
// Rows of C contiguous channels: the last axis as it is, axis 1 of an image as NHWC memory.
Tensor norm_rows(const Tensor &x, bool image)
{
    return numbers(image ? x.contiguous(at::MemoryFormat::ChannelsLast) : x.contiguous());
}

Tensor norm_forward(const Tensor &x, const Tensor &w, const Tensor &b, double eps, bool image, Tensor *stat)
{
    const int64_t c = x.size(image ? 1 : -1), rows = x.numel() / c;
    const c10::DeviceGuard guard(x.device());
    const Tensor wf = parameter(w), bf = parameter(b);
    Tensor y = fresh(x.sizes(), x.scalar_type(), x, image);
    if (stat) *stat = fresh({2, rows}, at::kFloat, x);
    float *kept = stat ? floats(*stat) : nullptr;
    check(lib.norm_fwd[kind(x)](x.data_ptr(), floats(wf), floats(bf), y.data_ptr(), kept, kept ? kept + rows : nullptr, rows,
                                (int)c, (float)eps, stream(x.device())));
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x0, const std::optional<Tensor> &w0, const std::optional<Tensor> &b0,
                          double eps, bool image)
    {
        const Tensor x = norm_rows(x0, image), w = w0.value_or(Tensor()), b = b0.value_or(Tensor());
        Tensor stat;
        Tensor y = norm_forward(x, w, b, eps, image, &stat);
        ctx->save_for_backward({x, w, stat});
        ctx->saved_data["image"] = image;
        ctx->saved_data["bias"] = b.defined() ? (int64_t)b.scalar_type() : (int64_t)-1;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        no_tangents("the gradient of layer_norm", grads);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &stat = saved[2];
        const bool image = ctx->saved_data["image"].toBool();
        const int64_t bias = ctx->saved_data["bias"].toInt();
        const int64_t c = x.size(image ? 1 : -1), rows = stat.size(1);
        const c10::DeviceGuard guard(x.device());
        const bool recorded = at::GradMode::is_enabled();
        const at::AutoGradMode off(false);
        const Tensor gy = norm_rows(grads[0].to(x.scalar_type()), image), wf = parameter(w);
        Tensor dx, dw, db, ws;
        if (ctx->needs_input_grad(0)) dx = fresh(x.sizes(), x.scalar_type(), x, image);
        // (an absent weight has no edge)
        if (w.defined() && ctx->needs_input_grad(1)) dw = fresh({c}, at::kFloat, x);
        if (bias >= 0 && ctx->needs_input_grad(w.defined() ? 2 : 1)) db = fresh({c}, at::kFloat, x);
        int64_t n_ws = 0;
        if (dw.defined() || db.defined()) {
            n_ws = (int64_t)lib.norm_ws(rows, (int)c);
            ws = fresh({n_ws}, at::kByte, x);
        }
        check(lib.norm_bwd[kind(x)](x.data_ptr(), floats(wf), floats(stat), floats(stat) + rows, gy.data_ptr(),
                                    dx.defined() ? dx.data_ptr() : nullptr, floats(dw), floats(db), rows, (int)c,
                                    ws.defined() ? ws.data_ptr() : nullptr, (size_t)n_ws, stream(x.device())));
        if (dw.defined()) dw = dw.to(w.scalar_type());
        if (db.defined()) db = db.to((at::ScalarType)bias);
        return first_order({dx, dw, db, Tensor(), Tensor()}, recorded, grads);
    }
};

// ---------------------------------------------------------------------------------------------- log probabilities
struct LogpShape {
    int64_t outer, v, inner, ld, top_k, ignore, axis;
    bool moved;                     // the class axis was brought to the end
};

// The results in the caller's shapes; what backward needs goes to kept, if it is wanted: the logits as the kernels read them, the targets,
// the statistics, the entropy and the alternatives' indices as the kernels wrote them.
variable_list logp_forward(const Tensor &logits, const Tensor &target0, LogpShape &s, variable_list *kept)
{
    const int64_t nd = logits.dim();
    s.v = logits.size(s.axis);
    s.inner = 1;
    for (int64_t i = s.axis + 1; i < nd; ++i) s.inner *= logits.size(i);
    Tensor x;
    const Tensor target = target0.contiguous();
    const int64_t pixels = target.numel();
    const c10::DeviceGuard guard(logits.device());
    std::vector<int64_t> full;
    // The pixel kernel gives a thread a pixel: its time goes with the class count until the pixels fill the card.  Bringing
    // the classes together first and giving a wave a row goes with the pixels (fp32, top 2, 150 classes: 20 and 13 us at
    // 4096 pixels, 20 and 36 at 16384; 20 classes: 4.5 and 8.5 at 1024, 4.8 and 24 at 16384).
    const bool plane = s.inner > 1 && s.top_k <= ERF_LOG_PROBS_MAX_TOP_PIXELS && (s.v <= 32 || pixels >= 64 * s.v);
    s.moved = !plane && s.axis != nd - 1;
    if (plane) {
        x = logits.contiguous();
        s.outer = pixels / s.inner;
        s.ld = 0;
    } else {
        x = s.moved ? logits.movedim(s.axis, -1) : logits;
        if (nd != 2) x = x.reshape({pixels, s.v});
        s.outer = pixels;
        s.inner = 1;
        if (x.stride(1) != 1 || (pixels > 1 && x.stride(0) < s.v)) x = x.contiguous();
        s.ld = pixels > 1 ? x.stride(0) : s.v;
    }
    x = numbers(x);
    for (int64_t i = 0; i < nd; ++i)
        if (i != s.axis) full.push_back(logits.size(i));
        else if (!s.moved) full.push_back(s.top_k);
    if (s.moved) full.push_back(s.top_k);
    const Tensor lp = fresh(target.sizes(), at::kFloat, x), ent = fresh(target.sizes(), at::kFloat, x);
    const Tensor top = fresh(full, at::kFloat, x), idx = fresh(full, at::kLong, x);
    Tensor stats, ws;
    if (kept) stats = fresh({2 * pixels}, at::kFloat, x);
    const int64_t n_ws = (int64_t)lib.logp_ws(s.outer, (int)s.v, s.inner, (int)s.top_k);
    if (n_ws) ws = fresh({n_ws}, at::kByte, x);
    check(lib.logp_fwd[kind(x)](x.data_ptr(), (const long long *)target.data_ptr(), floats(lp), floats(ent), floats(stats), floats(top),
                                (long long *)idx.data_ptr(), s.outer, (int)s.v, s.inner, s.ld, (int)s.top_k, s.ignore,
                                ws.defined() ? ws.data_ptr() : nullptr, (size_t)n_ws, stream(x.device())));
    if (kept) *kept = {x, target, stats, ent, idx};
    if (s.moved) return {lp, ent, top.movedim(-1, s.axis), idx.movedim(-1, s.axis)};
    return {lp, ent, top, idx};
}

struct LogProbs : torch::autograd::Function<LogProbs> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &target0, int64_t top_k,
                                 int64_t ignore, int64_t axis)
    {
        LogpShape s{0, 0, 0, 0, top_k, ignore, axis, false};
        variable_list kept, out = logp_forward(logits, target0, s, &kept);
        ctx->save_for_backward(kept);
        ctx->saved_data["shape"] = std::vector<int64_t>{s.outer, s.v, s.inner, s.ld, s.top_k, s.ignore, s.axis, s.moved};
        ctx->saved_data["logits"] = logits.sizes().vec();
        ctx->mark_non_differentiable({out[3]});
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads)
    {
        no_tangents("the gradient of log_probs", grads);
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &target = saved[1], &stats = saved[2], &ent = saved[3], &idx = saved[4];
        const std::vector<int64_t> s = ctx->saved_data["shape"].toIntVector();
        std::vector<int64_t> shape = ctx->saved_data["logits"].toIntVector();
        const int64_t axis = s[6];
        const bool moved = s[7] != 0;
        const c10::DeviceGuard guard(x.device());
        const bool recorded = at::GradMode::is_enabled();
        const at::AutoGradMode off(false);
        Tensor g[3];
        for (int i = 0; i < 3; ++i)
            if (grads[i].defined())
                g[i] = numbers((moved && i == 2 ? grads[i].movedim(axis, -1) : grads[i]).to(at::kFloat).contiguous());
        if (moved) {
            shape.push_back(shape[axis]);
            shape.erase(shape.begin() + axis);
        }
        Tensor dx = fresh(shape, x.scalar_type(), x);
        check(lib.logp_bwd[kind(x)](x.data_ptr(), (const long long *)target.data_ptr(), floats(ent), floats(stats),
                                    (const long long *)idx.data_ptr(), floats(g[0]), floats(g[1]), floats(g[2]), dx.data_ptr(),
                                    s[0], (int)s[1], s[2], s[3], (int)s[4], s[5], stream(x.device())));
        if (moved) dx = dx.movedim(-1, axis);
        return first_order({dx, Tensor(), Tensor(), Tensor(), Tensor()}, recorded, grads);
    }
};

bool wanted(std::initializer_list<Tensor> inputs)
{
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor &t : inputs)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}
Tensor unpack(PyObject *o) { return o == Py_None ? Tensor() : THPVariable_Unpack(o); }

// layer_norm(x, weight or None, bias or None, eps, image)
PyObject *layer_norm(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 5 || !THPVariable_Check(args[0])) {
        PyErr_SetString(PyExc_TypeError, "layer_norm: (tensor, weight, bias, eps, image)");
        return nullptr;
    }
    const Tensor x = unpack(args[0]), w = unpack(args[1]), b = unpack(args[2]);
    const double eps = PyFloat_AsDouble(args[3]);
    const bool image = PyObject_IsTrue(args[4]);
    if (PyErr_Occurred()) return nullptr;
    no_tracing("layer_norm");
    no_tangents("layer_norm", {x, w, b});
    auto given = [](const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    Tensor y;
    {
        const Unlocked unlocked;
        y = wanted({x, w, b}) ? LayerNorm::apply(x, given(w), given(b), eps, image)
                              : norm_forward(norm_rows(x, image), w, b, eps, image, nullptr);
    }
    return THPVariable_Wrap(y);
    END_HANDLE_TH_ERRORS
}

// log_probs(logits, target, top_k, ignore_index, axis) -> (log_prob, entropy, top, indices)
PyObject *log_probs(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 5 || !THPVariable_Check(args[0]) || !THPVariable_Check(args[1])) {
        PyErr_SetString(PyExc_TypeError, "log_probs: (tensor, tensor, top_k, ignore_index, axis)");
        return nullptr;
    }
    const Tensor logits = unpack(args[0]), target = unpack(args[1]);
    const int64_t top_k = PyLong_AsLongLong(args[2]), ignore = PyLong_AsLongLong(args[3]), axis = PyLong_AsLongLong(args[4]);
    if (PyErr_Occurred()) return nullptr;
    no_tracing("log_probs");
    no_tangents("log_probs", {logits});
    variable_list out;
    if (const Unlocked unlocked; wanted({logits})) {
        out = LogProbs::apply(logits, target, top_k, ignore, axis);
    } else {
        LogpShape s{0, 0, 0, 0, top_k, ignore, axis, false};
        out = logp_forward(logits, target, s, nullptr);
    }
    THPObjectPtr tuple(PyTuple_New(4));
    if (!tuple) return nullptr;
    for (int i = 0; i < 4; ++i) {
        PyObject *o = THPVariable_Wrap(out[i]);
        if (!o) return nullptr;
        PyTuple_SET_ITEM(tuple.get(), i, o);
    }
    return tuple.release();
    END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------------------------- AdamW
struct Batch {                      // the tensors of one launch list: a device, a type and a step count
    c10::Device device;
    at::ScalarType type;
    long long step;
    std::vector<void *> p, s[4];        // (scale tables pass through as void *)
    std::vector<const void *> g;
    std::vector<long long> n;
    std::vector<float *> counts;
    std::vector<c10::TensorImpl *> changed;
};

const char kWho[] = "erfnet_pytorch_amd.optim: ";

// False with a Python error set if the kernels cannot take t.
bool usable(const at::Tensor &t, const char *what)
{
    if (!t.is_cuda()) {
        PyErr_Format(PyExc_RuntimeError, "%s%s lives on %s; the update kernels run on the GPU only (use torch.optim for host "
                     "tensors)", kWho, what, t.device().str().c_str());
        return false;
    }
    if (!t.is_contiguous() || t.is_neg()) {
        PyErr_Format(PyExc_ValueError, "%s%s is %s", kWho, what, t.is_neg() ? "a view of its negative" : "not contiguous");
        return false;
    }
    return true;
}

// Stretches of GPU memory (addresses are unique over the devices).
struct Spans {
    std::vector<std::pair<const char *, size_t>> of;
    explicit Spans(size_t most) { of.reserve(most); }
    void add(const void *p, size_t bytes) { of.emplace_back((const char *)p, bytes); }
    bool overlap()
    {
        if (!std::is_sorted(of.begin(), of.end())) std::sort(of.begin(), of.end());
        for (size_t i = 1; i < of.size(); ++i)
            if (of[i - 1].first + of[i - 1].second > of[i].first) return true;
        return false;
    }
};

// A dict read in its own order, which is the order of the questions as a rule, and looked up where it is not.
struct Walk {
    PyObject *dict, *key = nullptr, *value = nullptr;
    Py_ssize_t pos = 0;
    bool more;
    explicit Walk(PyObject *d) : dict(d) { more = PyDict_Next(dict, &pos, &key, &value); }
    PyObject *next_if(PyObject *k)
    {
        if (!more || key != k) return nullptr;
        PyObject *v = value;
        more = PyDict_Next(dict, &pos, &key, &value);
        return v;
    }
    PyObject *find(PyObject *k)             // (null without an error: not there)
    {
        PyObject *v = next_if(k);
        return v ? v : PyDict_GetItemWithError(dict, k);
    }
};

// adamw_step(params, state, keys, bits, lr, beta1, beta2, eps, weight_decay)
//   params: list of Parameters; state: the optimiser's {Parameter: {key: tensor}}; keys: moments in the order of the
//   library's tables.
// The interpreter stays locked: that keeps the tensors whose addresses are taken here (references to all of them instead, and
// the launches unlocked: 229 tensors 34 -> 55 us a step).
// Returns the parameters that have a gradient and no state; where there are any, nothing has been launched.
// Otherwise an empty list.
PyObject *adamw_step(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 9 || !PyList_Check(args[0]) || !PyDict_Check(args[1]) || !PyTuple_Check(args[2])) {
        PyErr_SetString(PyExc_TypeError, "adamw_step: (list, dict, tuple, ...)");
        return nullptr;
    }
    PyObject *params = args[0], *state = args[1], *keys = args[2];
    const long bits = PyLong_AsLong(args[3]);
    double hp[5];
    for (int i = 0; i < 5; ++i) hp[i] = PyFloat_AsDouble(args[4 + i]);
    if (PyErr_Occurred()) return nullptr;
    const Py_ssize_t nkeys = PyTuple_GET_SIZE(keys);
    if (nkeys != (bits == 8 ? 4 : 2)) {
        PyErr_SetString(PyExc_TypeError, "adamw_step: keys do not fit bits");
        return nullptr;
    }
    static PyObject *step_key = PyUnicode_InternFromString("step");
    THPObjectPtr missing(PyList_New(0));
    if (!missing) return nullptr;
    std::vector<Batch> batches;
    std::deque<Tensor> resolved;            // gradients that are written for the launch (on its stream, as they are read)
    Spans spans((size_t)PyList_GET_SIZE(params));
    Walk states(state);
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); ++i) {
        PyObject *obj = PyList_GET_ITEM(params, i);
        if (!THPVariable_Check(obj)) {
            PyErr_SetString(PyExc_TypeError, "adamw_step: a parameter is not a tensor");
            return nullptr;
        }
        PyObject *st = states.next_if(obj);
        const at::Tensor &p = THPVariable_Unpack(obj);
        const at::Tensor *grad = &p.grad();
        if (!grad->defined()) continue;
        if (grad->is_neg()) {
            const at::NoGradGuard no_grad;
            resolved.push_back(grad->resolve_neg());
            grad = &resolved.back();
        }
        const at::Tensor &g = *grad;
        if (g.is_sparse()) {
            PyErr_Format(PyExc_RuntimeError, "%ssparse gradients are not supported", kWho);
            return nullptr;
        }
        if (!usable(p, "a parameter") || !usable(g, "a gradient")) return nullptr;
        const at::ScalarType type = p.scalar_type();
        if ((type != at::kFloat && type != at::kBFloat16) || g.scalar_type() != type) {
            PyErr_Format(PyExc_TypeError, "%sa parameter is %s and its gradient %s; parameters and gradients are fp32 or bf16, one "
                         "type for both", kWho, c10::toString(type), c10::toString(g.scalar_type()));
            return nullptr;
        }
        const long long n = p.numel();
        if (g.device() != p.device() || g.numel() != n) {
            PyErr_Format(PyExc_ValueError, "%sa gradient does not match its parameter", kWho);
            return nullptr;
        }
        if (n) spans.add(p.const_data_ptr(), p.nbytes());
        if (!st) {
            st = states.find(obj);
            if (!st && PyErr_Occurred()) return nullptr;
        }
        if (!st || !PyDict_Check(st) || PyDict_GET_SIZE(st) == 0) {
            if (PyList_Append(missing, obj)) return nullptr;
            continue;
        }
        Walk entries(st);
        PyObject *count = entries.find(step_key);
        if (!count || !THPVariable_Check(count)) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, "step");
            return nullptr;
        }
        const at::Tensor &c = THPVariable_Unpack(count);
        if (!c.is_cpu() || c.scalar_type() != at::kFloat || c.numel() != 1) {
            PyErr_Format(PyExc_ValueError, "%sstep is a host tensor of one fp32 number", kWho);
            return nullptr;
        }
        float *count_ptr = c.data_ptr<float>();
        const long long step = (long long)*count_ptr;
        void *s[4] = {nullptr, nullptr, nullptr, nullptr};
        for (Py_ssize_t k = 0; k < nkeys; ++k) {
            PyObject *o = entries.find(PyTuple_GET_ITEM(keys, k));
            if (!o || !THPVariable_Check(o)) {
                if (!PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "%U", PyTuple_GET_ITEM(keys, k));
                return nullptr;
            }
            const at::Tensor &t = THPVariable_Unpack(o);
            const bool scale = bits == 8 && (k & 1), code = bits == 8 && !scale;
            if (!usable(t, "optimiser state")) return nullptr;
            if (t.device() != p.device() || t.scalar_type() != (code ? at::kFloat8_e4m3fn : at::kFloat) ||
                t.numel() != (scale ? (n + 255) / 256 : n)) {
                PyErr_Format(PyExc_ValueError, "%s%U does not match its parameter", kWho, PyTuple_GET_ITEM(keys, k));
                return nullptr;
            }
            s[k] = t.data_ptr();
        }
        Batch *b = nullptr;
        for (Batch &x : batches)
            if (x.step == step && x.type == type && x.device == p.device()) b = &x;
        if (!b) {
            batches.push_back(Batch{p.device(), type, step, {}, {}, {}, {}, {}, {}});
            b = &batches.back();
            const size_t most = (size_t)(PyList_GET_SIZE(params) - i);
            b->p.reserve(most);
            b->g.reserve(most);
            for (auto &v : b->s) v.reserve(most);
            b->n.reserve(most);
            b->counts.reserve(most);
            b->changed.reserve(most);
        }
        b->p.push_back(p.data_ptr());
        b->g.push_back(g.data_ptr());
        for (int k = 0; k < 4; ++k) b->s[k].push_back(s[k]);
        b->n.push_back(n);
        b->counts.push_back(count_ptr);
        b->changed.push_back(p.unsafeGetTensorImpl());
    }
    // (at every step: memory moves with .data, .to() and state dicts behind the optimiser's back)
    if (spans.overlap()) {
        PyErr_SetString(PyExc_ValueError, "AdamW: two parameters of one group share memory; their updates would race");
        return nullptr;
    }
    if (PyList_GET_SIZE(missing.get())) return missing.release();
    for (const Batch &b : batches) {
        const c10::DeviceGuard guard(b.device);
        const int which = b.type == at::kBFloat16, count = (int)b.p.size();
        check(bits == 8
                  ? lib.adamw8[which](count, b.p.data(), b.g.data(), b.s[0].data(), (float *const *)b.s[1].data(), b.s[2].data(),
                                      (float *const *)b.s[3].data(), b.n.data(), hp[0], hp[1], hp[2], hp[3], hp[4], b.step + 1,
                                      stream(b.device))
                  : lib.adamw[which](count, b.p.data(), b.g.data(), (float *const *)b.s[0].data(),
                                     (float *const *)b.s[1].data(), b.n.data(), hp[0], hp[1], hp[2], hp[3], hp[4], b.step + 1,
                                     stream(b.device)));
        for (float *f : b.counts) *f = (float)(b.step + 1);
        // the parameters have changed behind torch's back: copies kept of them go by the version
        for (c10::TensorImpl *t : b.changed) t->bump_version();
    }
    return missing.release();
    END_HANDLE_TH_ERRORS
}

// share_memory(list of tensors) -> whether two GPU tensors of it overlap
PyObject *share_memory(PyObject *, PyObject *list)
{
    HANDLE_TH_ERRORS
    if (!PyList_Check(list)) {
        PyErr_SetString(PyExc_TypeError, "share_memory: (list)");
        return nullptr;
    }
    Spans spans((size_t)PyList_GET_SIZE(list));
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(list); ++i) {
        PyObject *o = PyList_GET_ITEM(list, i);
        if (!THPVariable_Check(o)) continue;
        const Tensor &t = THPVariable_Unpack(o);
        if (t.is_cuda() && t.numel()) spans.add(t.const_data_ptr(), t.nbytes());
    }
    return PyBool_FromLong(spans.overlap());
    END_HANDLE_TH_ERRORS
}

// bind(name -> address): see Library
PyObject *bind(PyObject *, PyObject *of)
{
    HANDLE_TH_ERRORS
    auto take = [&](auto &fn, const std::string &name) {
        THPObjectPtr address(PyObject_CallFunction(of, "s", name.c_str()));
        if (!address) throw python_error();
        fn = (std::remove_reference_t<decltype(fn)>)PyLong_AsVoidPtr(address);
    };
    take(lib.last_error, "erf_last_error");
    take(lib.norm_ws, "erf_layer_norm_workspace_bytes");
    take(lib.logp_ws, "erf_log_probs_workspace_bytes");
    for (int bf16 = 0; bf16 < 2; ++bf16) {
        const std::string tail = bf16 ? "_bf16" : "";
        take(lib.norm_fwd[bf16], "erf_layer_norm_forward" + tail);
        take(lib.norm_bwd[bf16], "erf_layer_norm_backward" + tail);
        take(lib.logp_fwd[bf16], "erf_log_probs_forward" + tail);
        take(lib.logp_bwd[bf16], "erf_log_probs_backward" + tail);
        take(lib.adamw[bf16], "erf_adamw_step" + tail);
        take(lib.adamw8[bf16], "erf_adamw8_step" + tail);
    }
    if (PyErr_Occurred()) throw python_error();
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// Which torch this file was compiled against: _lib.py looks for it in the file before it loads it.
__attribute__((used)) const char kBuiltFor[] = "erfnet_pytorch_amd._host for torch " ERF_TORCH_VERSION;

PyMethodDef methods[] = {{"bind", bind, METH_O, nullptr},
                         {"layer_norm", (PyCFunction)(void (*)(void))layer_norm, METH_FASTCALL, nullptr},
                         {"log_probs", (PyCFunction)(void (*)(void))log_probs, METH_FASTCALL, nullptr},
                         {"adamw_step", (PyCFunction)(void (*)(void))adamw_step, METH_FASTCALL, nullptr},
                         {"share_memory", share_memory, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
