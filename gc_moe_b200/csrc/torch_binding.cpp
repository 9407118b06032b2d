// Calls of the operators in front of the layer, from torch tensors to the C ABI
// (include/gcmoe.h): argument checks, output allocation, current stream, launch.
//
// These calls are a few microseconds of GPU work in a decode step, and the same steps in
// Python cost 8 to 14 us a call (tensor attributes, ctypes conversions, four allocations).
// The addresses of the C functions come from the library that the package has loaded
// (`bind`), so that there is one library and one place that chooses it.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>

#include "../../include/gcmoe.h"

namespace {

int (*rms_norm_fn)(const gcmoe_norm_args*, void*) = nullptr;
int (*router_logits_fn)(const gcmoe_logits_args*, void*) = nullptr;
int (*route_fn)(const gcmoe_route_args*, void*) = nullptr;
const char* (*last_error_fn)() = nullptr;

// A refusal: a Python exception is set, the call returns null.
template <typename... Args>
PyObject* refuse(const char* format, Args... args) {
    PyErr_Format(PyExc_ValueError, format, args...);
    return nullptr;
}

// The exception types of _native.raise_for.
PyObject* raise_for(int code) {
    PyErr_SetString(code == GCMOE_ERR_INVALID       ? PyExc_ValueError
                    : code == GCMOE_ERR_UNSUPPORTED ? PyExc_NotImplementedError
                                                    : PyExc_RuntimeError,
                    last_error_fn());
    return nullptr;
}

const at::Tensor* tensor_of(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

uint64_t address(const at::Tensor& t) { return reinterpret_cast<uint64_t>(t.data_ptr()); }

bool on_device(const at::Tensor& t, int device) { return t.is_cuda() && t.get_device() == device; }

bool is_float(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }

// [rows, columns] on the device, contiguous in the last dimension.
bool is_rows(const at::Tensor& t, int64_t rows, int64_t columns, int device) {
    return t.dim() == 2 && t.size(0) == rows && t.size(1) == columns && on_device(t, device) &&
           (columns <= 1 || t.stride(1) == 1);
}
// Elements between rows; a single row has no stride of its own.
uint64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// Counts are 32 bits wide below this binding; what does not fit is refused, not cut off.
constexpr int64_t kMaxCount = 0x7fffffff;
PyObject* refuse_tokens(int64_t tokens) {
    return refuse("%lld tokens are too many: at most %lld", (long long)tokens, (long long)kMaxCount);
}

at::Tensor new_rows(int64_t rows, int64_t columns, at::ScalarType type, const at::Tensor& like) {
    return at::detail::empty_strided_cuda({rows, columns}, {columns, 1}, type, like.device());
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* none() { Py_RETURN_NONE; }

const char* const kXMessage = "x must be a 2-D CUDA bfloat16 tensor, contiguous in its last dimension";

// rms_norm(x, weight, residual, eps, normed, residual_out, x_q, x_sf, shared_sf, block_m)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 10) return refuse("rms_norm takes 10 arguments, got %zd", count);
    const at::Tensor* const x = tensor_of(args[0]);
    if (x == nullptr || x->dim() != 2 || x->scalar_type() != at::kBFloat16 || !x->is_cuda()) return refuse(kXMessage);
    const int64_t tokens = x->size(0), hidden = x->size(1);
    const int device = x->get_device();
    if (!is_rows(*x, tokens, hidden, device)) return refuse(kXMessage);
    if (hidden == 0 || hidden % 32 || hidden > 32768)
        return refuse("hidden %lld must be a positive multiple of 32 up to 32768", (long long)hidden);
    if (tokens > kMaxCount) return refuse_tokens(tokens);
    const at::Tensor* const weight = tensor_of(args[1]);
    if (weight == nullptr || !is_float(*weight) || weight->dim() != 1 || weight->size(0) != hidden ||
        !on_device(*weight, device) || !weight->is_contiguous())
        return refuse("weight must be contiguous bfloat16 or float32 [%lld] on the device of x", (long long)hidden);
    gcmoe_norm_args a = {};
    a.eps = static_cast<float>(PyFloat_AsDouble(args[3]));
    if (PyErr_Occurred()) return nullptr;

    const at::Tensor* const residual = args[2] == Py_None ? nullptr : tensor_of(args[2]);
    at::Tensor residual_out, normed;
    if (args[2] != Py_None) {
        if (residual == nullptr || !is_float(*residual) || !is_rows(*residual, tokens, hidden, device))
            return refuse("residual must be bfloat16 or float32 [%lld, %lld] on the device of x, contiguous in its last dimension",
                          (long long)tokens, (long long)hidden);
        if (args[5] == Py_None) {
            residual_out = new_rows(tokens, hidden, residual->scalar_type(), *residual);
        } else {
            const at::Tensor* const given = tensor_of(args[5]);
            if (given == nullptr || given->scalar_type() != residual->scalar_type() || !is_rows(*given, tokens, hidden, device))
                return refuse("residual_out must have the type of residual and be [%lld, %lld] on the device of x, contiguous in "
                              "its last dimension", (long long)tokens, (long long)hidden);
            residual_out = *given;
        }
        a.residual = address(*residual); a.residual_stride = row_stride(*residual);
        a.residual_out = address(residual_out); a.residual_out_stride = row_stride(residual_out);
        a.residual_f32 = residual->scalar_type() == at::kFloat;
    } else if (args[5] != Py_None) {
        return refuse("residual_out needs a residual");
    }
    if (args[4] == Py_True) {
        normed = new_rows(tokens, hidden, at::kBFloat16, *x);
    } else if (args[4] != Py_False && args[4] != Py_None) {
        const at::Tensor* const given = tensor_of(args[4]);
        if (given == nullptr || given->scalar_type() != at::kBFloat16 || !is_rows(*given, tokens, hidden, device))
            return refuse("normed must be a truth value or bfloat16 [%lld, %lld] on the device of x, contiguous in its last dimension",
                          (long long)tokens, (long long)hidden);
        normed = *given;
    }
    if (normed.defined()) { a.normed = address(normed); a.normed_stride = row_stride(normed); }

    const int64_t words = (hidden + 127) / 128;
    at::Tensor x_q, x_sf;
    if (args[6] == Py_None) {
        x_q = new_rows(tokens, hidden, at::kFloat8_e4m3fn, *x);
        x_sf = new_rows(tokens, words, at::kInt, *x);
    } else {
        const at::Tensor* const q = tensor_of(args[6]);
        const at::Tensor* const sf = tensor_of(args[7]);
        if (q == nullptr || sf == nullptr || q->scalar_type() != at::kFloat8_e4m3fn || sf->scalar_type() != at::kInt ||
            !is_rows(*q, tokens, hidden, device) || !is_rows(*sf, tokens, words, device) || !q->is_contiguous() ||
            !sf->is_contiguous())
            return refuse("the workspace's rows do not fit x, or are on another device");
        x_q = *q;
        x_sf = *sf;
    }
    if (args[8] != Py_None) {
        const at::Tensor* const shared = tensor_of(args[8]);
        if (shared == nullptr || shared->scalar_type() != at::kInt || shared->dim() != 2 || !on_device(*shared, device))
            return refuse("the workspace's shared scale view is not on the device of x");
        a.shared_sf = address(*shared);
        a.shared_sf_rows = static_cast<uint32_t>(shared->size(0));
        a.block_m = static_cast<uint32_t>(PyLong_AsUnsignedLong(args[9]));
        if (PyErr_Occurred()) return nullptr;
    }
    a.x = address(*x); a.x_stride = row_stride(*x);
    a.weight = address(*weight); a.weight_f32 = weight->scalar_type() == at::kFloat;
    a.x_q = address(x_q); a.x_sf = address(x_sf);
    a.num_tokens = static_cast<uint32_t>(tokens); a.hidden = static_cast<uint32_t>(hidden);
    a.device = device;
    if (const int code = rms_norm_fn(&a, stream_of(device))) return raise_for(code);
    return Py_BuildValue("(NNNN)", wrap(x_q), wrap(x_sf), normed.defined() ? wrap(normed) : none(),
                         residual_out.defined() ? wrap(residual_out) : none());
    END_HANDLE_TH_ERRORS
}

// router_logits(x, router_weight, out)
PyObject* router_logits(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 3) return refuse("router_logits takes 3 arguments, got %zd", count);
    const at::Tensor* const x = tensor_of(args[0]);
    if (x == nullptr || x->dim() != 2 || x->scalar_type() != at::kBFloat16 || !x->is_cuda()) return refuse(kXMessage);
    const int64_t tokens = x->size(0), hidden = x->size(1);
    const int device = x->get_device();
    if (!is_rows(*x, tokens, hidden, device)) return refuse(kXMessage);
    const at::Tensor* const w = tensor_of(args[1]);
    if (w == nullptr || w->dim() != 3 || w->scalar_type() != at::kBFloat16 || (w->size(0) != 1 && w->size(0) != 3) ||
        w->size(1) < 1 || w->size(1) > 2048 || w->size(2) != hidden || !on_device(*w, device) || !w->is_contiguous())
        return refuse("router_weight must be contiguous bfloat16 [1 or 3, E <= 2048, %lld] on the device of x; call "
                      "transform_router_weight_for_gc_moe first", (long long)hidden);
    if (hidden > kMaxCount) return refuse("hidden %lld is too large", (long long)hidden);
    if (tokens > kMaxCount) return refuse_tokens(tokens);
    const int64_t experts = w->size(1);
    at::Tensor out;
    if (args[2] == Py_None) {
        out = new_rows(tokens, experts, at::kFloat, *x);
    } else {
        const at::Tensor* const given = tensor_of(args[2]);
        if (given == nullptr || given->scalar_type() != at::kFloat || !is_rows(*given, tokens, experts, device) ||
            !given->is_contiguous())
            return refuse("out must be contiguous float32 [%lld, %lld] on the device of x", (long long)tokens, (long long)experts);
        out = *given;
    }
    gcmoe_logits_args a = {};
    a.x = address(*x); a.x_stride = row_stride(*x);
    a.weight = address(*w);
    a.out = address(out);
    a.num_tokens = static_cast<uint32_t>(tokens); a.hidden = static_cast<uint32_t>(hidden);
    a.num_experts = static_cast<uint32_t>(experts); a.planes = static_cast<uint32_t>(w->size(0));
    a.device = device;
    if (const int code = router_logits_fn(&a, stream_of(device))) return raise_for(code);
    return wrap(out);
    END_HANDLE_TH_ERRORS
}

// route(logits, topk, sigmoid, bias, num_groups, topk_groups, group_by_max, renormalize, scale, topk_idx, topk_weights)
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    if (count != 11) return refuse("route takes 11 arguments, got %zd", count);
    const at::Tensor* const logits = tensor_of(args[0]);
    gcmoe_route_args a = {};
    const bool f32 = logits != nullptr && logits->scalar_type() == at::kFloat;
    const bool bf16 = logits != nullptr && logits->scalar_type() == at::kBFloat16;
    if (logits == nullptr || !(f32 || bf16 || logits->scalar_type() == at::kHalf) || logits->dim() != 2 || !logits->is_cuda() ||
        !is_rows(*logits, logits->size(0), logits->size(1), logits->get_device()))
        return refuse("logits must be a 2-D CUDA float32, bfloat16 or float16 tensor, contiguous in its last dimension");
    const int64_t tokens = logits->size(0), experts = logits->size(1);
    const int device = logits->get_device();
    if (tokens > kMaxCount) return refuse_tokens(tokens);
    const long topk = PyLong_AsLong(args[1]), groups = PyLong_AsLong(args[4]), topk_groups = PyLong_AsLong(args[5]);
    a.scale = static_cast<float>(PyFloat_AsDouble(args[8]));
    if (PyErr_Occurred()) return nullptr;
    if (topk < 1 || topk > 32 || groups < 1 || groups > 32 || topk_groups < 1 || topk_groups > groups || experts > 2048)
        return refuse("invalid routing: top %ld of %lld experts in %ld of %ld groups", topk, (long long)experts, topk_groups, groups);
    if (args[3] != Py_None) {
        const at::Tensor* const bias = tensor_of(args[3]);
        if (bias == nullptr || bias->scalar_type() != at::kFloat || bias->dim() != 1 || bias->size(0) != experts ||
            !on_device(*bias, device) || !bias->is_contiguous())
            return refuse("bias must be contiguous float32 [%lld] on the device of the logits", (long long)experts);
        a.bias = address(*bias);
    }
    at::Tensor idx, weights;
    if (args[9] == Py_None && args[10] == Py_None) {
        idx = new_rows(tokens, topk, at::kLong, *logits);
        weights = new_rows(tokens, topk, at::kFloat, *logits);
    } else {
        const at::Tensor* const i = tensor_of(args[9]);
        const at::Tensor* const w = tensor_of(args[10]);
        if (i == nullptr || w == nullptr || i->scalar_type() != at::kLong || w->scalar_type() != at::kFloat ||
            !is_rows(*i, tokens, topk, device) || !is_rows(*w, tokens, topk, device) || !i->is_contiguous() || !w->is_contiguous())
            return refuse("out must be contiguous int64 and float32 [%lld, %ld] on the device of logits", (long long)tokens, topk);
        idx = *i;
        weights = *w;
    }
    a.logits = address(*logits); a.logits_stride = row_stride(*logits);
    a.topk_idx = address(idx); a.topk_weights = address(weights);
    a.num_tokens = static_cast<uint32_t>(tokens); a.num_experts = static_cast<uint32_t>(experts);
    a.topk = static_cast<uint32_t>(topk);
    a.num_groups = static_cast<uint32_t>(groups); a.topk_groups = static_cast<uint32_t>(topk_groups);
    a.logit_type = f32 ? 0 : bf16 ? 1 : 2;
    a.sigmoid = args[2] == Py_True; a.group_by_max = args[6] == Py_True; a.renormalize = args[7] == Py_True;
    a.device = device;
    if (const int code = route_fn(&a, stream_of(device))) return raise_for(code);
    return Py_BuildValue("(NN)", wrap(idx), wrap(weights));
    END_HANDLE_TH_ERRORS
}

// bind(rms_norm, router_logits, route, last_error): addresses of the C functions
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long norm, logits, route_at, error;
    if (!PyArg_ParseTuple(args, "KKKK", &norm, &logits, &route_at, &error)) return nullptr;
    rms_norm_fn = reinterpret_cast<decltype(rms_norm_fn)>(norm);
    router_logits_fn = reinterpret_cast<decltype(router_logits_fn)>(logits);
    route_fn = reinterpret_cast<decltype(route_fn)>(route_at);
    last_error_fn = reinterpret_cast<decltype(last_error_fn)>(error);
    Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(rms_norm)), METH_FASTCALL, nullptr},
    {"router_logits", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(router_logits)), METH_FASTCALL, nullptr},
    {"route", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(route)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding() { return PyModule_Create(&module); }
