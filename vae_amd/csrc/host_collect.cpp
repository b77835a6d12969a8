// The host side of a many-tensor call: walks a list of parameters and fills the table of vae_mt_tensor that the library
// takes (include/vae_hip.h).  In Python that walk costs about 0.7 us a tensor, more than the kernels take for models of up to
// some ten million parameters (52 tensors of 4.1 M: 36 us beside 28 us of kernels); here it is 0.03.  It handles the ordinary case only --
// dense tensors of the expected type, size and device in the order of the state -- and says so when it meets another: the caller then
// takes its general way, which copies or raises.  A CPython extension (vae_amd/_host.so) because it looks into torch tensors;
// libvae_hip.so itself knows nothing of torch.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/version.h>

#include <algorithm>
#include <vector>

#include "../../include/vae_hip.h"

namespace {

struct Buffer {      // a writable (or readable) contiguous buffer of a numpy array
    Py_buffer b{};
    bool ok;
    Buffer(PyObject* o, bool write) { ok = PyObject_GetBuffer(o, &b, write ? PyBUF_CONTIG : PyBUF_CONTIG_RO) == 0; }
    ~Buffer() { if (ok) PyBuffer_Release(&b); }
    Buffer(const Buffer&) = delete;
    Buffer& operator=(const Buffer&) = delete;
};

// -1: not a dense fp32 / bf16 tensor on that device (index < 0: the host's memory); else whether it is bf16
int kind(const at::Tensor& t, int device) {
    if (t.layout() != at::kStrided || t.is_conj() || t.is_neg()) return -1;
    if (device >= 0 ? !t.is_cuda() || t.get_device() != device : !t.is_cpu()) return -1;
    if (t.scalar_type() == at::kFloat) return 0;
    if (t.scalar_type() == at::kBFloat16) return 1;
    return -1;
}

void bump(const at::Tensor& t) { t.unsafeGetTensorImpl()->bump_version(); }

// collect_step(params, jobs, layout, device) -> number of tensors with a gradient, or -1 for the general way.
// layout: int64[n][4]: elements, first block, slot, VAE_MT_* flags (and STRIDED) of the parameter the state was made for.  The parameters' version
// counters are advanced: the launch that follows writes them through their addresses.
// collect_params: the same for all parameters, with or without a gradient, to be read only.
constexpr int64_t STRIDED = 256;      // the state is in the order of a tensor that was not contiguous: a contiguous one is not it
template <bool STEP>
PyObject* collect(PyObject*, PyObject* args) {
    PyObject *list, *jobs_o, *layout_o;
    int device;
    if (!PyArg_ParseTuple(args, "O!OOi", &PyList_Type, &list, &jobs_o, &layout_o, &device)) return nullptr;
    try {
        Buffer jobs(jobs_o, true), layout(layout_o, false);
        if (!jobs.ok || !layout.ok) return nullptr;
        const Py_ssize_t n = PyList_GET_SIZE(list);
        if ((size_t)jobs.b.len < n * sizeof(vae_mt_tensor) || (size_t)layout.b.len < n * 4 * sizeof(int64_t)) {
            PyErr_SetString(PyExc_ValueError, "the tables are shorter than the list");
            return nullptr;
        }
        vae_mt_tensor* job = (vae_mt_tensor*)jobs.b.buf;
        const int64_t* row = (const int64_t*)layout.b.buf;
        long live = 0;
        std::vector<const at::Tensor*> written;
        written.reserve(n);
        for (Py_ssize_t k = 0; k < n; ++k, row += 4) {
            PyObject* o = PyList_GET_ITEM(list, k);
            if (!THPVariable_Check(o)) return PyLong_FromLong(-1);
            const at::Tensor& p = THPVariable_Unpack(o);
            const at::Tensor& g = STEP ? p.grad() : p;
            if (!g.defined()) continue;
            const int pk = kind(p, device), gk = STEP ? kind(g, device) : pk;
            if (pk < 0 || gk < 0 || pk != (int)(row[3] & VAE_MT_PARAM_BF16) || (row[3] & STRIDED) || p.numel() != row[0] ||
                g.numel() != row[0] || !p.is_contiguous() || !g.is_contiguous() || (STEP && (p.is_inference() || p.sizes() != g.sizes())))
                return PyLong_FromLong(-1);
            // mutable: a lazily cloned tensor gets memory of its own
            job[live] = {STEP ? p.mutable_data_ptr() : const_cast<void*>(p.const_data_ptr()), g.const_data_ptr(), row[0], (unsigned)row[1], (unsigned)row[2],
                         (pk ? VAE_MT_PARAM_BF16 : 0u) | (gk ? VAE_MT_GRAD_BF16 : 0u), 0u};
            ++live;
            if (STEP) written.push_back(&p);
        }
        for (const at::Tensor* p : written) bump(*p);
        return PyLong_FromLong(live);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// collect_grads(params, jobs, device, write) -> number of gradients, or -1 for the general way.  write: they will be written in place,
// so no two may overlap, and their version counters are advanced.
PyObject* collect_grads(PyObject*, PyObject* args) {
    PyObject *list, *jobs_o;
    int device, write;
    if (!PyArg_ParseTuple(args, "O!Oip", &PyList_Type, &list, &jobs_o, &device, &write)) return nullptr;
    try {
        Buffer jobs(jobs_o, true);
        if (!jobs.ok) return nullptr;
        const Py_ssize_t n = PyList_GET_SIZE(list);
        if ((size_t)jobs.b.len < n * sizeof(vae_mt_tensor)) {
            PyErr_SetString(PyExc_ValueError, "collect_grads: the table is shorter than the list");
            return nullptr;
        }
        vae_mt_tensor* job = (vae_mt_tensor*)jobs.b.buf;
        std::vector<std::pair<const char*, const char*>> spans;
        std::vector<const at::Tensor*> grads;
        spans.reserve(n);
        grads.reserve(n);
        for (Py_ssize_t k = 0; k < n; ++k) {
            PyObject* o = PyList_GET_ITEM(list, k);
            if (!THPVariable_Check(o)) return PyLong_FromLong(-1);
            const at::Tensor& g = THPVariable_Unpack(o).grad();
            if (!g.defined()) continue;
            const int gk = kind(g, device);
            if (gk < 0 || !g.is_contiguous() || g.is_inference()) return PyLong_FromLong(-1);
            const char* a = write ? (const char*)g.mutable_data_ptr() : (const char*)g.const_data_ptr();
            job[grads.size()] = {nullptr, a, g.numel(), 0u, 0u, gk ? VAE_MT_GRAD_BF16 : 0u, 0u};
            grads.push_back(&g);
            if (write && g.numel()) spans.emplace_back(a, a + g.nbytes());
        }
        if (write) {
            std::sort(spans.begin(), spans.end());
            for (size_t k = 1; k < spans.size(); ++k)
                if (spans[k].first < spans[k - 1].second) return PyLong_FromLong(-1);
            for (const at::Tensor* g : grads) bump(*g);
        }
        return PyLong_FromLong((long)grads.size());
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// same_tensors(now, held): whether two sequences hold the same objects in the same order
PyObject* same_tensors(PyObject*, PyObject* args) {
    PyObject *now, *held;
    if (!PyArg_ParseTuple(args, "OO!", &now, &PyList_Type, &held)) return nullptr;
    PyObject* seq = PySequence_Fast(now, "same_tensors: not a sequence");
    if (!seq) return nullptr;
    const Py_ssize_t n = PyList_GET_SIZE(held);
    bool same = PySequence_Fast_GET_SIZE(seq) == n;
    for (Py_ssize_t k = 0; same && k < n; ++k) same = PySequence_Fast_GET_ITEM(seq, k) == PyList_GET_ITEM(held, k);
    Py_DECREF(seq);
    return PyBool_FromLong(same);
}

PyMethodDef methods[] = {
    {"collect_step", collect<true>, METH_VARARGS, "table of the parameters that have a gradient"},
    {"collect_params", collect<false>, METH_VARARGS, "table of all parameters"},
    {"collect_grads", collect_grads, METH_VARARGS, "table of the gradients"},
    {"same_tensors", same_tensors, METH_VARARGS, "whether two sequences hold the same objects"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) {
    PyObject* m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) { Py_DECREF(m); return nullptr; }
    return m;
}
