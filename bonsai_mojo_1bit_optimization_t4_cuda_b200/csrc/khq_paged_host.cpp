// khq_paged_host.cpp -- the look at a step's tensors for paged.py, as a CPython extension.
//
// A property of a torch tensor costs Python some 0.1 us and a call of a step has up to nine tensors to look at: 6 of its 13 us.  Here
// they are a few nanoseconds each.  Every function checks its tensors against the plan, fills the launcher's argument struct and
// calls it on the plan's device and torch's current stream.  It returns the launcher's code, or NO_FIT when a tensor is not what the plan
// asks for; paged.py then says which and why.
#include <Python.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "khq_b200.h"

namespace {

constexpr long NO_FIT = -1000;

// What a PagedPlan knows; paged.py keeps it in a buffer of its own and passes the address.
struct PlanInfo {
    int64_t device, H_q, H_kv, d, page_size, max_requests, max_tokens, max_new;
    int64_t requests, max_pages;  // of the last build
    void *cu_new, *kv_lens, *positions, *slots, *info, *schedule, *workspace;
    int64_t schedule_bytes, workspace_bytes;
    int (*launch_plan)(const khq_paged_plan_args*, khq_stream_t);
    int (*launch_prestep[2])(const khq_paged_prestep_args*, khq_stream_t);  // fp16, bf16
    int (*launch_attn[2])(const khq_paged_attn_args*, khq_stream_t);
};

PlanInfo* plan_of(PyObject* o) { return static_cast<PlanInfo*>(PyLong_AsVoidPtr(o)); }

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool is(const at::Tensor* t, at::ScalarType type, int64_t device, int64_t dim) {
    return t && t->scalar_type() == type && t->is_cuda() && t->get_device() == device && t->dim() == dim && t->layout() == at::kStrided;
}

// (tokens, heads, d)
bool rows(PyObject* o, const PlanInfo& p, int64_t tokens, int64_t heads, at::ScalarType type, const void*& at, int64_t (&stride)[2]) {
    const at::Tensor* t = tensor_of(o);
    if (!is(t, type, p.device, 3) || t->size(0) != tokens || t->size(1) != heads || t->size(2) != p.d || t->stride(2) != 1) return false;
    at = t->data_ptr();
    stride[0] = t->stride(0);
    stride[1] = t->stride(1);
    return true;
}
// (n_pages, page_size, H_kv, d); n_pages < 0: any
bool cache(PyObject* o, const PlanInfo& p, int64_t& n_pages, at::ScalarType type, const void*& at, int64_t (&stride)[3]) {
    const at::Tensor* t = tensor_of(o);
    if (!is(t, type, p.device, 4) || t->size(1) != p.page_size || t->size(2) != p.H_kv || t->size(3) != p.d || t->stride(3) != 1) return false;
    if (n_pages >= 0 && t->size(0) != n_pages) return false;
    n_pages = t->size(0);
    at = t->data_ptr();
    for (int i = 0; i < 3; ++i) stride[i] = t->stride(i);
    return true;
}
// contiguous with `numel` entries (< 0: any)
bool flat(PyObject* o, const PlanInfo& p, at::ScalarType type, int64_t numel, const void*& at) {
    const at::Tensor* t = tensor_of(o);
    if (!t || t->scalar_type() != type || !t->is_cuda() || t->get_device() != p.device || !t->is_contiguous() || (numel >= 0 && t->numel() != numel)) return false;
    at = t->data_ptr();
    return true;
}

template <class Args>
PyObject* launch(const PlanInfo& p, int (*fn)(const Args*, khq_stream_t), const Args& a) {
    const auto dev = static_cast<c10::DeviceIndex>(p.device);
    int rc;
    if (c10::cuda::current_device() == dev) {
        rc = fn(&a, c10::cuda::getCurrentCUDAStream(dev).stream());
    } else {
        const c10::cuda::CUDAGuard guard(dev);
        rc = fn(&a, c10::cuda::getCurrentCUDAStream(dev).stream());
    }
    return PyLong_FromLong(rc);
}

PyObject* no_fit() { return PyLong_FromLong(NO_FIT); }

// plan, ctx_lens, new_lens, block_table, free_list | None, free_count | None, free_count_out | None
PyObject* build_impl(PyObject* const* v) {
    PlanInfo& p = *plan_of(v[0]);
    khq_paged_plan_args a = {};
    const at::Tensor *ctx = tensor_of(v[1]), *table = tensor_of(v[3]);
    if (!ctx || !is(table, at::kInt, p.device, 2)) return no_fit();
    const int64_t n = ctx->numel();
    if (n < 1 || n > p.max_requests || table->size(0) != n || table->size(1) < 1 || table->stride(1) != 1) return no_fit();
    if (!flat(v[1], p, at::kInt, n, a.ctx_lens) || !flat(v[2], p, at::kInt, n, a.new_lens)) return no_fit();
    if (v[4] != Py_None) {
        const void *list, *out;
        if (!flat(v[4], p, at::kInt, -1, list) || !flat(v[5], p, at::kInt, 1, a.free_count)) return no_fit();
        out = a.free_count;
        if (v[6] != Py_None && !flat(v[6], p, at::kInt, 1, out)) return no_fit();
        a.free_list = const_cast<void*>(list);
        a.free_count_out = const_cast<void*>(out);
        a.n_pages = static_cast<int32_t>(tensor_of(v[4])->numel());
    } else if (v[5] != Py_None || v[6] != Py_None) {
        return no_fit();
    }
    a.block_table = table->data_ptr();
    a.table_stride = n > 1 ? table->stride(0) : table->size(1);
    a.cu_new = p.cu_new;
    a.kv_lens = p.kv_lens;
    a.positions = p.positions;
    a.slots = p.slots;
    a.info = p.info;
    a.schedule = p.schedule;
    a.schedule_bytes = static_cast<size_t>(p.schedule_bytes);
    a.requests = static_cast<int32_t>(n);
    a.max_pages = static_cast<int32_t>(table->size(1));
    a.page_size = static_cast<int32_t>(p.page_size);
    a.max_tokens = static_cast<int32_t>(p.max_tokens);
    a.max_new = static_cast<int32_t>(p.max_new);
    a.H_q = static_cast<int32_t>(p.H_q);
    a.H_kv = static_cast<int32_t>(p.H_kv);
    a.d = static_cast<int32_t>(p.d);
    PyObject* rc = launch(p, p.launch_plan, a);
    if (rc && PyLong_AsLong(rc) == 0) {
        p.requests = n;
        p.max_pages = table->size(1);
    }
    return rc;
}

// The 16-bit type that the call is in, by its first tensor: 0 fp16, 1 bf16, -1 neither; and the rows of the call.
int type_of(PyObject* o, const PlanInfo& p, at::ScalarType& type, int64_t& tokens) {
    const at::Tensor* t = tensor_of(o);
    if (!t || t->dim() != 3 || p.requests == 0) return -1;
    type = t->scalar_type();
    tokens = t->size(0);
    if (tokens < 1 || tokens > p.max_tokens) return -1;
    return type == at::kHalf ? 0 : type == at::kBFloat16 ? 1 : -1;
}

// plan, q, k, v, q_norm_w | None, k_norm_w | None, q_out, k_cache, v_cache, u_cache | None, rotary_dim, rope_theta, rms_eps
PyObject* prestep_impl(PyObject* const* v) {
    const PlanInfo& p = *plan_of(v[0]);
    at::ScalarType type;
    int64_t T, n_pages = -1;
    const int which = type_of(v[1], p, type, T);
    if (which < 0) return no_fit();
    khq_paged_prestep_args a = {};
    const void *q_out, *kc, *vc, *uc = nullptr;
    if (!rows(v[1], p, T, p.H_q, type, a.q, a.q_stride) || !rows(v[2], p, T, p.H_kv, type, a.k, a.k_stride) || !rows(v[3], p, T, p.H_kv, type, a.v, a.v_stride) ||
        !rows(v[6], p, T, p.H_q, type, q_out, a.q_out_stride) || !cache(v[7], p, n_pages, type, kc, a.k_cache_stride) ||
        !cache(v[8], p, n_pages, type, vc, a.v_cache_stride) || (v[9] != Py_None && !cache(v[9], p, n_pages, type, uc, a.u_cache_stride)) ||
        (v[4] != Py_None && !flat(v[4], p, at::kFloat, p.d, a.q_norm_w)) || (v[5] != Py_None && !flat(v[5], p, at::kFloat, p.d, a.k_norm_w)))
        return no_fit();
    a.q_out = const_cast<void*>(q_out);
    a.k_cache = const_cast<void*>(kc);
    a.v_cache = const_cast<void*>(vc);
    a.u_cache = const_cast<void*>(uc);
    a.positions = p.positions;
    a.slots = p.slots;
    a.tokens = static_cast<int32_t>(T);
    a.n_pages = static_cast<int32_t>(n_pages);
    a.page_size = static_cast<int32_t>(p.page_size);
    a.H_q = static_cast<int32_t>(p.H_q);
    a.H_kv = static_cast<int32_t>(p.H_kv);
    a.d = static_cast<int32_t>(p.d);
    a.rotary_dim = static_cast<int32_t>(PyLong_AsLong(v[10]));
    a.rope_theta = static_cast<float>(PyFloat_AsDouble(v[11]));
    a.rms_eps = static_cast<float>(PyFloat_AsDouble(v[12]));
    if (PyErr_Occurred()) return nullptr;
    return launch(p, p.launch_prestep[which], a);
}

// plan, q, k_cache, v_cache, block_table, out, scale, gate | None, lse | None, workspace | None
PyObject* attention_impl(PyObject* const* v) {
    const PlanInfo& p = *plan_of(v[0]);
    at::ScalarType type;
    int64_t T, n_pages = -1;
    const int which = type_of(v[1], p, type, T);
    const at::Tensor* table = tensor_of(v[4]);
    if (which < 0 || !is(table, at::kInt, p.device, 2) || table->size(0) != p.requests || table->size(1) != p.max_pages || table->stride(1) != 1) return no_fit();
    khq_paged_attn_args a = {};
    const void *out, *lse = nullptr, *ws = p.workspace;
    int64_t ws_bytes = p.workspace_bytes;
    if (!rows(v[1], p, T, p.H_q, type, a.q, a.q_stride) || !cache(v[2], p, n_pages, type, a.k_cache, a.k_cache_stride) ||
        !cache(v[3], p, n_pages, type, a.v_cache, a.v_cache_stride) || !rows(v[5], p, T, p.H_q, type, out, a.out_stride) ||
        (v[7] != Py_None && !rows(v[7], p, T, p.H_q, type, a.gate, a.gate_stride)) || (v[8] != Py_None && !flat(v[8], p, at::kFloat, T * p.H_q, lse)) ||
        (v[9] != Py_None && !flat(v[9], p, at::kByte, -1, ws)))
        return no_fit();
    if (v[9] != Py_None) ws_bytes = tensor_of(v[9])->numel();
    a.block_table = table->data_ptr();
    a.table_stride = p.requests > 1 ? table->stride(0) : p.max_pages;
    a.out = const_cast<void*>(out);
    a.lse = const_cast<void*>(lse);
    a.workspace = const_cast<void*>(ws);
    a.schedule = p.schedule;
    a.schedule_bytes = static_cast<size_t>(p.schedule_bytes);
    a.workspace_bytes = static_cast<size_t>(ws_bytes);
    a.tokens = static_cast<int32_t>(T);
    a.max_tokens = static_cast<int32_t>(p.max_tokens);
    a.max_new = static_cast<int32_t>(p.max_new);
    a.requests = static_cast<int32_t>(p.requests);
    a.max_pages = static_cast<int32_t>(p.max_pages);
    a.n_pages = static_cast<int32_t>(n_pages);
    a.page_size = static_cast<int32_t>(p.page_size);
    a.H_q = static_cast<int32_t>(p.H_q);
    a.H_kv = static_cast<int32_t>(p.H_kv);
    a.d = static_cast<int32_t>(p.d);
    a.scale = static_cast<float>(PyFloat_AsDouble(v[6]));
    if (PyErr_Occurred()) return nullptr;
    return launch(p, p.launch_attn[which], a);
}

// No C++ exception leaves the extension.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) return PyErr_Format(PyExc_TypeError, "%d arguments, not %zd", N, n);
    try {
        return F(args);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

PyObject* info_bytes(PyObject*, PyObject* const*, Py_ssize_t) { return PyLong_FromSize_t(sizeof(PlanInfo)); }

using Fast = PyObject* (*)(PyObject*, PyObject* const*, Py_ssize_t);
PyCFunction method(Fast f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {
    {"build", method(entry<build_impl, 7>), METH_FASTCALL, nullptr},
    {"prestep", method(entry<prestep_impl, 13>), METH_FASTCALL, nullptr},
    {"attention", method(entry<attention_impl, 10>), METH_FASTCALL, nullptr},
    {"info_bytes", method(info_bytes), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_khq_paged_host", "Calls of the paged operators without Python's look at the tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__khq_paged_host() { return PyModule_Create(&module); }
