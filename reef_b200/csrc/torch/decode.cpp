// The calls of reef_b200/decode.py from the second one of a signature on: looks up what the first one has checked and resolved, allocates
// outputs and workspace, launches.  In Python this took 20 us a call, more than most of the kernels; here 4 to 7.
//
// A signature is the operator, its whole-number options, and type, device, sizes and strides of every tensor.  Nothing of a tensor's
// identity or contents is kept.  The last kMaxPlans signatures are: a server whose prompts have every length would else fill its memory with
// them; one that is asked for again is defined again.
#include <ATen/ops/empty.h>
#include <Python.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <deque>
#include <memory>
#include <string>
#include <unordered_map>
#include <vector>

#include "reef_cuda.h"

namespace {

constexpr int kMaxTensors = 12;

struct Launch {
    reef_kernel_t kernel;
    uint32_t dims[6], smem;
    std::vector<int> args;      // tensors by position, inputs first, then outputs; -1: the workspace
};
struct Output {
    std::vector<int64_t> sizes;
    at::ScalarType type;
};
struct Plan {
    std::vector<Launch> launches;
    std::vector<Output> outputs;
    std::vector<int> aligned;                   // tensors that begin at a 16-byte boundary
    std::vector<std::pair<int, int>> apart;     // tensors that do not lie over each other
    size_t workspace;
    PyObject* owner = nullptr;                  // keeps the kernels (everything here runs under the interpreter's lock)
    Plan() = default;
    Plan(const Plan&) = delete;
    ~Plan() { Py_XDECREF(owner); }
};
constexpr size_t kMaxPlans = 4096;
typedef std::vector<int64_t> Key;
struct Hash {
    size_t operator()(const Key& k) const {
        uint64_t h = 1469598103934665603ull;
        for (int64_t x : k) h = (h ^ (uint64_t)x) * 1099511628211ull;
        return (size_t)(h ^ (h >> 29));
    }
};
struct Plans {
    std::unordered_map<Key, std::shared_ptr<const Plan>, Hash> of;
    std::deque<Key> order;      // the oldest first
};
Plans* plans() {
    static auto* p = new Plans;     // (never freed: nothing is given back to an interpreter that has ended)
    return p;
}

struct Call {
    const at::Tensor* t[2 * kMaxTensors];
    int inputs = 0, n = 0;
    bool made = false;          // outputs were given
    Key key;
};

// tuple of tensors and None -> the call's tensors and key; false: something else is among them
bool collect(PyObject* tuple, Call* c) {
    const Py_ssize_t n = PyTuple_GET_SIZE(tuple);
    if (n > kMaxTensors) return false;
    for (Py_ssize_t i = 0; i < n; i++) {
        PyObject* o = PyTuple_GET_ITEM(tuple, i);
        if (o == Py_None) {
            c->t[c->n++] = nullptr;
            c->key.push_back(-1);
            continue;
        }
        if (!THPVariable_Check(o)) return false;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.is_cuda() || t.layout() != at::kStrided || t.is_neg()) return false;
        c->t[c->n++] = &t;
        c->key.push_back((int64_t)t.scalar_type() << 16 | (int64_t)t.get_device() << 8 | t.dim());
        for (int64_t s : t.sizes()) c->key.push_back(s);
        for (int64_t s : t.strides()) c->key.push_back(s);
    }
    return true;
}

// (operator, inputs, outputs or None, options)
bool parse(PyObject* const* args, Call* c) {
    if (!PyLong_Check(args[0]) || !PyTuple_Check(args[1]) || !PyTuple_Check(args[3])) return false;
    c->key.reserve(64);
    c->key.push_back(PyLong_AsLongLong(args[0]));
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[3]); i++) {
        PyObject* o = PyTuple_GET_ITEM(args[3], i);
        if (!PyLong_CheckExact(o)) return false;
        int overflow = 0;
        c->key.push_back(PyLong_AsLongLongAndOverflow(o, &overflow));
        if (overflow) return false;
    }
    if (!collect(args[1], c)) return false;
    c->inputs = c->n;
    if (args[2] != Py_None) {
        if (!PyTuple_Check(args[2])) return false;
        c->made = true;
        c->key.push_back(-2);
        if (!collect(args[2], c)) return false;
    }
    return true;
}

bool overlap(const at::Tensor& a, const at::Tensor& b) {
    auto span = [](const at::Tensor& t, uintptr_t* lo, uintptr_t* hi) {
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); d++) {
            if (t.size(d) == 0) return false;
            last += (t.size(d) - 1) * t.stride(d);
        }
        *lo = (uintptr_t)t.data_ptr();
        *hi = *lo + (size_t)(last + 1) * t.element_size();
        return true;
    };
    uintptr_t a0, a1, b0, b1;
    return span(a, &a0, &a1) && span(b, &b0, &b1) && a0 < b1 && b0 < a1;
}

// None: no such signature; a text: why the call is refused or has failed; else the outputs
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 4) {
        PyErr_SetString(PyExc_TypeError, "call(operator, inputs, outputs, options)");
        return nullptr;
    }
    try {
        Call c;
        if (!parse(args, &c)) {
            PyErr_Clear();
            Py_RETURN_NONE;
        }
        auto it = plans()->of.find(c.key);
        if (it == plans()->of.end() || c.n == 0 || c.t[0] == nullptr) Py_RETURN_NONE;
        const std::shared_ptr<const Plan> plan = it->second;        // (an allocation may run other code, which may define others)
        const Plan& p = *plan;
        if (c10::GradMode::is_enabled())
            for (int i = 0; i < c.n; i++)
                if (c.t[i] && c.t[i]->requires_grad())
                    return PyUnicode_FromString("inputs require gradients and there is no backward pass (use torch.no_grad)");
        if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
            for (int i = 0; i < c.n; i++)
                if (c.t[i] && c.t[i]->_fw_grad(0).defined())
                    return PyUnicode_FromString("inputs carry tangents and there is no forward-mode derivative");
        const c10::cuda::CUDAGuard guard(c.t[0]->device());
        at::Tensor fresh[kMaxTensors];
        if (!c.made)
            for (size_t i = 0; i < p.outputs.size(); i++) {
                fresh[i] = at::empty(p.outputs[i].sizes, at::TensorOptions().dtype(p.outputs[i].type).device(c.t[0]->device()));
                c.t[c.n++] = &fresh[i];
            }
        for (int i : p.aligned)
            if ((uintptr_t)c.t[i]->data_ptr() & 15) return PyUnicode_FromString("a tensor does not begin at a 16-byte boundary");
        if (c.made || p.outputs.empty())
            for (auto& pair : p.apart)
                if (overlap(*c.t[pair.first], *c.t[pair.second])) return PyUnicode_FromString("an output lies over an input or another output");
        c10::DataPtr workspace;
        if (p.workspace) workspace = c10::GetAllocator(c10::kCUDA)->allocate(p.workspace);
        const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(c.t[0]->get_device()).stream();
        for (const Launch& l : p.launches) {
            uint64_t words[16];
            void* pointers[16];
            for (size_t i = 0; i < l.args.size(); i++) {
                words[i] = (uint64_t)(uintptr_t)(l.args[i] < 0 ? workspace.get() : c.t[l.args[i]]->data_ptr());
                pointers[i] = &words[i];
            }
            if (reef_launch(l.kernel, l.dims, l.smem, (reef_stream_t)stream, pointers) != REEF_SUCC) return PyUnicode_FromString(reef_last_error());
        }
        const int n = c.made ? c.n - c.inputs : (int)p.outputs.size();
        PyObject* out = PyTuple_New(n);
        if (!out) return nullptr;
        for (int i = 0; i < n; i++) {
            PyObject* o;
            if (c.made) {
                o = PyTuple_GET_ITEM(args[2], i);
                Py_INCREF(o);
            } else {
                o = THPVariable_Wrap(fresh[i]);
                if (!o) {
                    Py_DECREF(out);
                    return nullptr;
                }
            }
            PyTuple_SET_ITEM(out, i, o);
        }
        return out;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "reef_b200._decode: unknown error");
        return nullptr;
    }
}

bool numbers(PyObject* o, std::vector<int64_t>* out) {
    PyObject* seq = PySequence_Fast(o, "a sequence of numbers");
    if (!seq) return false;
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq); i++) {
        const long long x = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
        if (x == -1 && PyErr_Occurred()) {
            Py_DECREF(seq);
            return false;
        }
        out->push_back(x);
    }
    Py_DECREF(seq);
    return true;
}

// define(operator, inputs, outputs, options, launches, allocate, workspace, aligned, apart, owner): launches = [(handle, dims, smem, args)],
// allocate = [(type of input i or -1 for int32, sizes)], owner: what has to live as long as the handles are used
PyObject* define(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    if (nargs != 10) {
        PyErr_SetString(PyExc_TypeError, "define: ten arguments");
        return nullptr;
    }
    try {
        Call c;
        if (!parse(args, &c)) {
            PyErr_SetString(PyExc_TypeError, "define: not a signature");
            return nullptr;
        }
        const std::shared_ptr<Plan> made = std::make_shared<Plan>();
        Plan& p = *made;
        for (Py_ssize_t i = 0; i < PyList_Size(args[4]); i++) {
            PyObject* l = PyList_GetItem(args[4], i);
            std::vector<int64_t> one, dims, a;
            if (!PyTuple_Check(l) || PyTuple_GET_SIZE(l) != 4 || !numbers(PyTuple_GET_ITEM(l, 1), &dims) || !numbers(PyTuple_GET_ITEM(l, 3), &a)) return nullptr;
            Launch x;
            x.kernel = (reef_kernel_t)(uintptr_t)PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(l, 0));
            x.smem = (uint32_t)PyLong_AsUnsignedLong(PyTuple_GET_ITEM(l, 2));
            if (PyErr_Occurred()) return nullptr;
            for (int d = 0; d < 6; d++) x.dims[d] = (uint32_t)dims.at(d);
            for (int64_t v : a) x.args.push_back((int)v);
            p.launches.push_back(x);
        }
        for (Py_ssize_t i = 0; i < PyList_Size(args[5]); i++) {
            PyObject* o = PyList_GetItem(args[5], i);
            Output x;
            if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2 || !numbers(PyTuple_GET_ITEM(o, 1), &x.sizes)) return nullptr;
            const long like = PyLong_AsLong(PyTuple_GET_ITEM(o, 0));
            x.type = like < 0 ? at::kInt : c.t[like]->scalar_type();
            p.outputs.push_back(x);
        }
        p.workspace = (size_t)PyLong_AsUnsignedLongLong(args[6]);
        std::vector<int64_t> aligned, apart;
        if (PyErr_Occurred() || !numbers(args[7], &aligned) || !numbers(args[8], &apart)) return nullptr;
        for (int64_t i : aligned) p.aligned.push_back((int)i);
        for (size_t i = 0; i + 1 < apart.size(); i += 2) p.apart.emplace_back((int)apart[i], (int)apart[i + 1]);
        Py_INCREF(args[9]);
        p.owner = args[9];
        Plans* all = plans();
        std::shared_ptr<const Plan> gone = made;            // given up at the end, when what that runs finds everything in order
        auto at = all->of.find(c.key);
        if (at != all->of.end()) {
            at->second.swap(gone);
        } else {
            all->order.push_back(c.key);
            all->of.emplace(c.key, made);
            gone.reset();
            if (all->of.size() > kMaxPlans) {
                at = all->of.find(all->order.front());
                gone.swap(at->second);
                all->of.erase(at);
                all->order.pop_front();
            }
        }
        Py_RETURN_NONE;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyObject* count(PyObject*, PyObject*) { return PyLong_FromSize_t(plans()->of.size()); }

PyMethodDef methods[] = {{"call", (PyCFunction)(void (*)())call, METH_FASTCALL, nullptr},
                         {"define", (PyCFunction)(void (*)())define, METH_FASTCALL, nullptr},
                         {"count", count, METH_NOARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_decode", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__decode() { return PyModule_Create(&module_def); }
