// erfnet_pytorch_amd._host: the part of an optimiser step that looks at every parameter, in C++.
//
// A step over the 229 parameter tensors of the 20-class network is 20 us of GPU work; gathering their pointers
// through Python attributes took 560 us.  Nothing is kept between calls: every step reads the gradients,
// the state tensors and their pointers anew.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <vector>

namespace {

typedef int (*adamw32_fn)(int, void *const *, const void *const *, void *const *, void *const *, const long long *, double,
                          double, double, double, double, long long, void *);
typedef int (*adamw8_fn)(int, void *const *, const void *const *, void *const *, void *const *, void *const *, void *const *,
                         const long long *, double, double, double, double, double, long long, void *);

struct Batch {                      // the tensors of one launch list: a device, a type and a step count
    c10::Device device;
    at::ScalarType type;
    long long step;
    std::vector<void *> p, s[4];
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
    if (!t.is_contiguous()) {
        PyErr_Format(PyExc_ValueError, "%s%s is not contiguous", kWho, what);
        return false;
    }
    return true;
}

// adamw_step(params, state, keys, bits, fp32 entry point, bf16 entry point, lr, beta1, beta2, eps, weight_decay, stream_of)
//   params: list of Parameters; state: the optimiser's {Parameter: {key: tensor}}; keys: moments in the order of the
//   library's tables; stream_of(device index) -> raw stream.
// Returns the parameters that have a gradient and no state; where there are any, nothing has been launched.
// Otherwise an empty list, or the library's nonzero status.
PyObject *adamw_step(PyObject *, PyObject *const *args, Py_ssize_t nargs)
{
    HANDLE_TH_ERRORS
    if (nargs != 12 || !PyList_Check(args[0]) || !PyDict_Check(args[1]) || !PyTuple_Check(args[2])) {
        PyErr_SetString(PyExc_TypeError, "adamw_step: (list, dict, tuple, ...)");
        return nullptr;
    }
    PyObject *params = args[0], *state = args[1], *keys = args[2];
    const long bits = PyLong_AsLong(args[3]);
    void *fn32 = PyLong_AsVoidPtr(args[4]), *fn16 = PyLong_AsVoidPtr(args[5]);
    double hp[5];
    for (int i = 0; i < 5; ++i) hp[i] = PyFloat_AsDouble(args[6 + i]);
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
    // the state dict holds the parameters in the order of the groups as a rule: walk along it and look up the others
    Py_ssize_t pos = 0;
    PyObject *next_key = nullptr, *next_value = nullptr;
    bool more = PyDict_Next(state, &pos, &next_key, &next_value);
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(params); ++i) {
        PyObject *obj = PyList_GET_ITEM(params, i);
        if (!THPVariable_Check(obj)) {
            PyErr_SetString(PyExc_TypeError, "adamw_step: a parameter is not a tensor");
            return nullptr;
        }
        PyObject *st = nullptr;
        if (more && next_key == obj) {
            st = next_value;
            more = PyDict_Next(state, &pos, &next_key, &next_value);
        }
        const at::Tensor &p = THPVariable_Unpack(obj);
        const at::Tensor &g = p.grad();
        if (!g.defined()) continue;
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
        if (!st) {
            st = PyDict_GetItemWithError(state, obj);
            if (!st && PyErr_Occurred()) return nullptr;
        }
        if (!st || !PyDict_Check(st) || PyDict_GET_SIZE(st) == 0) {
            if (PyList_Append(missing, obj)) return nullptr;
            continue;
        }
        void *s[4] = {nullptr, nullptr, nullptr, nullptr};
        for (Py_ssize_t k = 0; k < nkeys; ++k) {
            PyObject *o = PyDict_GetItemWithError(st, PyTuple_GET_ITEM(keys, k));
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
        PyObject *count = PyDict_GetItemWithError(st, step_key);
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
        Batch *b = nullptr;
        for (Batch &x : batches)
            if (x.step == step && x.type == type && x.device == p.device()) b = &x;
        if (!b) {
            batches.push_back(Batch{p.device(), type, step, {}, {}, {}, {}, {}, {}});
            b = &batches.back();
        }
        b->p.push_back(p.data_ptr());
        b->g.push_back(g.data_ptr());
        for (int k = 0; k < 4; ++k) b->s[k].push_back(s[k]);
        b->n.push_back(n);
        b->counts.push_back(count_ptr);
        b->changed.push_back(p.unsafeGetTensorImpl());
    }
    if (PyList_GET_SIZE(missing.get())) return missing.release();
    for (const Batch &b : batches) {
        c10::DeviceGuard guard(b.device);
        THPObjectPtr stream(PyObject_CallFunction(args[11], "i", (int)b.device.index()));
        if (!stream) return nullptr;
        void *st = PyLong_AsVoidPtr(stream);
        if (PyErr_Occurred()) return nullptr;
        void *fn = b.type == at::kBFloat16 ? fn16 : fn32;
        const int count = (int)b.p.size();
        const int rc = bits == 8
            ? ((adamw8_fn)fn)(count, b.p.data(), b.g.data(), b.s[0].data(), b.s[1].data(), b.s[2].data(), b.s[3].data(),
                              b.n.data(), hp[0], hp[1], hp[2], hp[3], hp[4], b.step + 1, st)
            : ((adamw32_fn)fn)(count, b.p.data(), b.g.data(), b.s[0].data(), b.s[1].data(), b.n.data(), hp[0], hp[1], hp[2],
                               hp[3], hp[4], b.step + 1, st);
        if (rc) return PyLong_FromLong(rc);
        for (float *f : b.counts) *f = (float)(b.step + 1);
        // the parameters have changed behind torch's back: copies kept of them go by the version
        for (c10::TensorImpl *t : b.changed) t->bump_version();
    }
    return missing.release();
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"adamw_step", (PyCFunction)(void (*)(void))adamw_step, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&module); }
