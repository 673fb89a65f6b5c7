// paged_torch.cpp - the torch side of bnn_b200.paged: reads the tensors,
// checks them, fills the C argument blocks and makes the call.
//
// In C++ because a serving step calls these operators some hundred times per
// token: the same work through the interpreter cost 15-20 us a call, several
// times the kernels of a small batch. The functions are positional
// (bnn_b200/paged.py has the signatures and their documentation); the C entry
// points come as addresses from the library that bnn_b200 has loaded.
#include <Python.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <vector>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "bnn_b200_paged.h"

namespace {

using AppendFn = BNN_Status (*)(BNN_Device, const BNN_PagedAppend*, void*);
using AttentionFn = BNN_Status (*)(BNN_Device, const BNN_PagedAttention*, void*);
AppendFn g_append;
AttentionFn g_attention;
PyObject* g_error;  // accel.BnnError

struct Refused {};  // the Python error is set

[[noreturn]] void refuse(int status, const char* format, ...) {
    char text[256];
    va_list list;
    va_start(list, format);
    std::vsnprintf(text, sizeof text, format, list);
    va_end(list);
    if (PyObject* e = PyObject_CallFunction(g_error, "is", status, text)) {
        PyErr_SetObject(g_error, e);
        Py_DECREF(e);
    }
    throw Refused{};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o))
        refuse(BNN_EINVAL, "%s: a tensor is wanted", name);
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o, const char* name) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(BNN_EINVAL, "%s: an integer is wanted", name);
    }
    return v;
}

double number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(BNN_EINVAL, "%s: a number is wanted", name);
    }
    return v;
}

bool truth(PyObject* o, const char* name) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        refuse(BNN_EINVAL, "%s: true or false is wanted", name);
    }
    return v == 1;
}

int64_t type_of(at::ScalarType t) {
    return t == at::kFloat ? BNN_PAGED_F32 : t == at::kBFloat16 ? BNN_PAGED_BF16 : t == at::kHalf ? BNN_PAGED_F16 : 0;
}

void on_device(const at::Tensor& x, int device, const char* name) {
    if (!x.is_cuda() || x.get_device() != device)
        refuse(BNN_EINVAL, "%s: not on cuda:%d", name, device);
}

// These operators have no derivative: a tensor that wants one, of either mode, is
// refused wherever it would be dropped.
void no_gradient(const at::Tensor& x, const char* name) {
    if (!x.unsafeGetTensorImpl()->autograd_meta())
        return;  // most tensors here: ten such questions a call
    if (x.requires_grad() && c10::GradMode::is_enabled())
        refuse(BNN_EINVAL, "%s requires a gradient, and the paged operators have no backward pass", name);
    if (x._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
        refuse(BNN_EINVAL, "%s has a tangent, and the paged operators have no forward-mode derivative", name);
}

void set_cache(const at::Tensor& k, const at::Tensor& v, int device, BNN_PagedCache* c) {
    if (k.dim() != 4 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type())
        refuse(BNN_EINVAL, "k_pages and v_pages: one shape [pages, kv_heads, page_size, head_dim] and type");
    c->type = type_of(k.scalar_type());
    if (c->type != BNN_PAGED_BF16 && c->type != BNN_PAGED_F16)
        refuse(BNN_EINVAL, "k_pages: bfloat16 or float16");
    on_device(k, device, "k_pages");
    on_device(v, device, "v_pages");
    no_gradient(k, "k_pages");
    no_gradient(v, "v_pages");
    c->pages = k.size(0);
    c->kv_heads = k.size(1);
    c->page_size = k.size(2);
    c->head_dim = k.size(3);
    if (k.stride(3) != 1 || v.stride(3) != 1)
        refuse(BNN_EINVAL, "the cache's last dimension has to be adjacent");
    // the stride of a dimension of one is free: nothing steps over it
    auto stride = [&](const at::Tensor& x, int i) { return x.size(i) > 1 ? x.stride(i) : c->head_dim; };
    c->k = k.data_ptr();
    c->v = v.data_ptr();
    c->k_page_stride = stride(k, 0);
    c->k_head_stride = stride(k, 1);
    c->k_row_stride = stride(k, 2);
    c->v_page_stride = stride(v, 0);
    c->v_head_stride = stride(v, 1);
    c->v_row_stride = stride(v, 2);
}

void rows(const at::Tensor& x, const char* name, int64_t tokens, int64_t heads, int64_t dim, int device, int64_t* token_stride,
          int64_t* head_stride) {
    if (x.dim() != 3 || x.size(0) != tokens || x.size(1) != heads || x.size(2) != dim)
        refuse(BNN_EINVAL, "%s: [%lld, %lld, %lld] is wanted", name, (long long)tokens, (long long)heads, (long long)dim);
    on_device(x, device, name);
    if (x.stride(2) != 1)
        refuse(BNN_EINVAL, "%s: the last dimension has to be adjacent", name);
    // as in the cache, the stride of a dimension of one is free
    *head_stride = heads > 1 ? x.stride(1) : dim;
    *token_stride = tokens > 1 ? x.stride(0) : heads * dim;
}

// A result of the caller's: every value has a place of its own.
const at::Tensor& given_out(PyObject* o) {
    const at::Tensor& x = tensor(o, "out");
    no_gradient(x, "out");
    for (int64_t i = 0; i < x.dim(); ++i)
        if (x.size(i) > 1 && x.stride(i) == 0)
            refuse(BNN_EINVAL, "out: expanded, its rows share memory");
    return x;
}

// A call has been launched that writes x: what autograd saved of it is stale
// (inference tensors keep no count).
void written(const at::Tensor& x) {
    if (!x.is_inference())
        x.unsafeGetTensorImpl()->bump_version();
}

template <typename E>
const E* vector(PyObject* o, const char* name, at::ScalarType type, int64_t count, int device) {
    const at::Tensor& x = tensor(o, name);
    if (x.scalar_type() != type || x.dim() != 1 || x.size(0) != count || (count > 1 && x.stride(0) != 1))
        refuse(BNN_EINVAL, "%s: %lld adjacent %s are wanted", name, (long long)count, at::toString(type));
    on_device(x, device, name);
    no_gradient(x, name);
    return static_cast<const E*>(x.data_ptr());
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, int device) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)device), std::nullopt));
}

template <typename F>
PyObject* guarded(F&& f) {
    HANDLE_TH_ERRORS
    try {
        return f();
    } catch (const Refused&) {
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

constexpr char kOrderName[] = "bnn_b200.paged.order";
const cudaStream_t kNoStream = reinterpret_cast<cudaStream_t>(~(uintptr_t)0);  // compares unlike any

// Who used a workspace last. Calls of unlike captures, and a captured call and
// one outside, are ordered by whoever replays the graph.
struct Order {
    at::Tensor workspace;
    cudaStream_t home;  // where the allocator orders what it hands the memory out for next
    cudaStream_t recent;  // the last call's
    cudaStream_t last;    // the last call's outside captures
    cudaStream_t captured;  // the last noted call's inside one,
    unsigned long long capture;  // and its capture (0: none yet)
    cudaEvent_t event;
};

void cuda_ok(cudaError_t e, const char* what) {
    if (e != cudaSuccess) {
        cudaGetLastError();
        refuse(BNN_EIO, "%s: %s", what, cudaGetErrorString(e));
    }
}

// The capture that `stream` is part of, 0 where it is in none.
unsigned long long capture_of(cudaStream_t stream) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(stream, &status, &id) != cudaSuccess) {
        cudaGetLastError();  // the legacy stream beside somebody's capture
        return 0;
    }
    return status == cudaStreamCaptureStatusActive ? id : 0;
}

void after(cudaStream_t now, cudaStream_t before, cudaEvent_t event) {
    cuda_ok(cudaEventRecord(event, before), "workspace order");
    cuda_ok(cudaStreamWaitEvent(now, event, 0), "workspace order");
}

// Workspaces whose object went while their last call, on another stream than
// their own, may have been in flight. That stream may be gone as well, so it is
// not asked (asking one that is gone ended the process): the memory stays here
// until the next object on the device takes it over. Never destroyed, as CUDA
// may be gone before this library.
std::vector<at::Tensor>& left_behind() {
    static auto* all = new std::vector<at::Tensor>;
    return *all;
}

void drop_order(PyObject* capsule) {
    Order* u = static_cast<Order*>(PyCapsule_GetPointer(capsule, kOrderName));
    if (!u)
        return;
    if (u->last != u->home)
        left_behind().push_back(u->workspace);
    cudaEventDestroy(u->event);
    delete u;
}

// A left workspace of this size, all work on the device done.
at::Tensor left_workspace(c10::DeviceIndex device, int64_t bytes, cudaStream_t now) {
    auto& all = left_behind();
    for (size_t i = 0; i < all.size(); ++i)
        if (all[i].get_device() == device && all[i].numel() == bytes && capture_of(now) == 0) {
            cuda_ok(cudaDeviceSynchronize(), "workspace");
            at::Tensor x = all[i];
            all.erase(all.begin() + (ptrdiff_t)i);
            return x;
        }
    return at::Tensor();
}

// new_order(device, bytes) -> (a zeroed workspace, its order), of the current stream
PyObject* new_order(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 2)
            refuse(BNN_EINVAL, "new_order: 2 arguments");
        const auto d = (c10::DeviceIndex)integer(o[0], "device");
        const int64_t bytes = integer(o[1], "bytes");
        const c10::cuda::CUDAGuard guard(d);
        const cudaStream_t now = c10::cuda::getCurrentCUDAStream(d).stream();
        at::Tensor workspace = left_workspace(d, bytes, now);
        const bool taken_over = workspace.defined();
        if (!taken_over)
            workspace = empty({bytes}, at::kByte, d);
        cuda_ok(cudaMemsetAsync(workspace.data_ptr(), 0, (size_t)bytes, now), "workspace");
        cudaEvent_t event;
        cuda_ok(cudaEventCreateWithFlags(&event, cudaEventDisableTiming), "workspace order");
        // one taken over belongs to a stream that is not known here: it is left behind again
        Order* u = new Order{workspace, taken_over ? kNoStream : now, now, now, nullptr, 0, event};
        PyObject* capsule = PyCapsule_New(u, kOrderName, drop_order);
        if (!capsule)
            return nullptr;
        PyObject* x = THPVariable_Wrap(workspace);
        PyObject* both = x ? PyTuple_Pack(2, x, capsule) : nullptr;
        Py_XDECREF(x);
        Py_DECREF(capsule);
        return both;
    });
}

// The stream's next work runs after the work that used the workspace before.
void in_order(Order* u, cudaStream_t now, c10::DeviceIndex device) {
    if (now == u->recent && now == u->last)
        return;  // whether it is captured by now or not (a query costs more than all else here)
    const c10::cuda::CUDAGuard guard(device);
    if (const unsigned long long capture = capture_of(now)) {
        // branches of one graph: an edge from the earlier to the later; `last` may have
        // been drawn into the capture since
        if (u->capture == capture && u->captured != now)
            after(now, u->captured, u->event);
        if (u->last != now && capture_of(u->last) == capture)
            after(now, u->last, u->event);
        u->capture = capture;
        u->captured = now;
    } else if (u->last != now) {
        // waiting for a stream that is being captured would draw this one in
        if (capture_of(u->last) != 0)
            refuse(BNN_EBUSY, "the stream of the last call is being captured");
        after(now, u->last, u->event);
        u->last = now;
    }
    u->recent = now;
}

// append(handle, device, q, k, v, cos, sin, positions, slots, k_pages, v_pages,
//        q_norm, k_norm, eps, interleaved, out) -> q
PyObject* append(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 16)
            refuse(BNN_EINVAL, "append: 16 arguments");
        const int device = (int)integer(o[1], "device");
        BNN_PagedAppend d = {};
        const at::Tensor &q = tensor(o[2], "q"), &k = tensor(o[3], "k"), &v = tensor(o[4], "v");
        const at::Tensor &k_pages = tensor(o[9], "k_pages"), &v_pages = tensor(o[10], "v_pages");
        set_cache(k_pages, v_pages, device, &d.cache);
        if (q.dim() != 3)
            refuse(BNN_EINVAL, "q: [tokens, heads, head_dim]");
        d.tokens = q.size(0);
        d.heads = q.size(1);
        d.type = type_of(q.scalar_type());
        if (d.type == 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
            refuse(BNN_EINVAL, "q, k and v: one type, float32, bfloat16 or float16");
        no_gradient(q, "q");
        no_gradient(k, "k");
        no_gradient(v, "v");
        const int64_t dim = d.cache.head_dim;
        rows(q, "q", d.tokens, d.heads, dim, device, &d.q_token_stride, &d.q_head_stride);
        rows(k, "k", d.tokens, d.cache.kv_heads, dim, device, &d.k_token_stride, &d.k_head_stride);
        rows(v, "v", d.tokens, d.cache.kv_heads, dim, device, &d.v_token_stride, &d.v_head_stride);
        d.q = q.data_ptr();
        d.k = k.data_ptr();
        d.v = v.data_ptr();
        if (o[5] != Py_None) {
            const at::Tensor &cos = tensor(o[5], "cos"), &sin = tensor(o[6], "sin");
            if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat || cos.dim() != 2 || cos.sizes() != sin.sizes() ||
                !cos.is_contiguous() || !sin.is_contiguous())
                refuse(BNN_EINVAL, "cos and sin: contiguous float32 [positions, rotary_dim / 2]");
            on_device(cos, device, "cos");
            on_device(sin, device, "sin");
            no_gradient(cos, "cos");
            no_gradient(sin, "sin");
            d.cos = static_cast<const float*>(cos.data_ptr());
            d.sin = static_cast<const float*>(sin.data_ptr());
            d.table_rows = cos.size(0);
            d.rotary_dim = 2 * cos.size(1);
        }
        d.positions = vector<int32_t>(o[7], "positions", at::kInt, d.tokens, device);
        d.slots = vector<int32_t>(o[8], "slots", at::kInt, d.tokens, device);
        d.q_norm = o[11] == Py_None ? nullptr : vector<float>(o[11], "q_norm", at::kFloat, dim, device);
        d.k_norm = o[12] == Py_None ? nullptr : vector<float>(o[12], "k_norm", at::kFloat, dim, device);
        d.eps = number(o[13], "eps");
        d.interleaved = truth(o[14], "interleaved");
        at::Tensor out;
        if (o[15] == Py_None) {
            out = empty({d.tokens, d.heads, dim}, k_pages.scalar_type(), device);
        } else {
            out = given_out(o[15]);
            if (out.scalar_type() != k_pages.scalar_type())
                refuse(BNN_EINVAL, "out: the cache's type");
        }
        rows(out, "out", d.tokens, d.heads, dim, device, &d.out_token_stride, &d.out_head_stride);
        d.q_out = out.data_ptr();
        const BNN_Status st = g_append(reinterpret_cast<BNN_Device>(PyLong_AsVoidPtr(o[0])), &d,
                                       c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream());
        if (st != BNN_OK)
            refuse(st, "bnn_b200_paged_append");
        written(k_pages);
        written(v_pages);
        if (o[15] != Py_None)
            written(out);
        return THPVariable_Wrap(out);
    });
}

// attention(handle, device, workspace, q, k_pages, v_pages, page_table, kv_lens,
//           q_starts, max_q, scale, window, sinks, out, out_is_f32, return_lse, order)
// -> out or (out, lse). The interpreter's lock is held from the order to the
// launch: another thread's call on this workspace comes before both or after both.
PyObject* attention(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        if (n != 17)
            refuse(BNN_EINVAL, "attention: 17 arguments");
        const int device = (int)integer(o[1], "device");
        BNN_PagedAttention d = {};
        const at::Tensor &workspace = tensor(o[2], "workspace"), &q = tensor(o[3], "q"), &k_pages = tensor(o[4], "k_pages");
        set_cache(k_pages, tensor(o[5], "v_pages"), device, &d.cache);
        const int64_t dim = d.cache.head_dim;
        if (q.dim() != 3 || q.scalar_type() != k_pages.scalar_type())
            refuse(BNN_EINVAL, "q: [tokens, heads, head_dim] of the cache's type");
        no_gradient(q, "q");
        d.tokens = q.size(0);
        d.heads = q.size(1);
        rows(q, "q", d.tokens, d.heads, dim, device, &d.q_token_stride, &d.q_head_stride);
        d.q = q.data_ptr();
        const at::Tensor& table = tensor(o[6], "page_table");
        if (table.dim() != 2 || table.scalar_type() != at::kInt || (table.size(1) > 1 && table.stride(1) != 1))
            refuse(BNN_EINVAL, "page_table: int32 [batch, width], rows adjacent");
        on_device(table, device, "page_table");
        d.batch = table.size(0);
        d.table_width = table.size(1);
        d.table_stride = d.batch > 1 ? table.stride(0) : d.table_width;
        d.page_table = static_cast<const int32_t*>(table.data_ptr());
        d.kv_lens = vector<int32_t>(o[7], "kv_lens", at::kInt, d.batch, device);
        d.q_starts = vector<int32_t>(o[8], "q_starts", at::kInt, d.batch + 1, device);
        d.max_q = integer(o[9], "max_q");
        d.scale = o[10] == Py_None ? 1.0 / std::sqrt((double)dim) : number(o[10], "scale");
        d.window = integer(o[11], "window");
        d.sinks = integer(o[12], "sinks");
        at::Tensor out, lse;
        if (o[13] == Py_None) {
            out = empty({d.tokens, d.heads, dim}, truth(o[14], "out_is_f32") ? at::kFloat : q.scalar_type(), device);
        } else {
            out = given_out(o[13]);
        }
        rows(out, "out", d.tokens, d.heads, dim, device, &d.out_token_stride, &d.out_head_stride);
        d.out = out.data_ptr();
        d.out_type = type_of(out.scalar_type());
        const bool want_lse = truth(o[15], "return_lse");
        if (want_lse) {
            lse = empty({d.tokens, d.heads}, at::kFloat, device);
            d.lse = static_cast<float*>(lse.data_ptr());
            d.lse_token_stride = d.heads;
        }
        d.workspace = workspace.data_ptr();
        d.workspace_bytes = (int64_t)workspace.nbytes();
        Order* order = static_cast<Order*>(PyCapsule_GetPointer(o[16], kOrderName));
        if (!order)
            return nullptr;
        const cudaStream_t now = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
        in_order(order, now, (c10::DeviceIndex)device);
        const BNN_Status st = g_attention(reinterpret_cast<BNN_Device>(PyLong_AsVoidPtr(o[0])), &d, now);
        if (st != BNN_OK)
            refuse(st, "bnn_b200_paged_attention");
        if (o[13] != Py_None)
            written(out);
        if (!want_lse)
            return THPVariable_Wrap(out);
        PyObject *a = THPVariable_Wrap(out), *b = a ? THPVariable_Wrap(lse) : nullptr;
        PyObject* both = b ? PyTuple_Pack(2, a, b) : nullptr;
        Py_XDECREF(a);
        Py_XDECREF(b);
        return both;
    });
}

// The raw current stream of a device, as an integer.
PyObject* stream(PyObject*, PyObject* device) {
    return guarded([&]() -> PyObject* {
        return PyLong_FromVoidPtr(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)integer(device, "device")).stream());
    });
}

// bind(address of bnn_b200_paged_append, of bnn_b200_paged_attention, BnnError)
PyObject* bind(PyObject*, PyObject* args) {
    PyObject *f, *g, *error;
    if (!PyArg_ParseTuple(args, "OOO", &f, &g, &error))
        return nullptr;
    g_append = reinterpret_cast<AppendFn>(PyLong_AsVoidPtr(f));
    g_attention = reinterpret_cast<AttentionFn>(PyLong_AsVoidPtr(g));
    Py_INCREF(error);
    Py_XDECREF(g_error);
    g_error = error;
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
    {"stream", stream, METH_O, nullptr},
    {"new_order", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(new_order)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_torch() { return PyModule_Create(&module); }
