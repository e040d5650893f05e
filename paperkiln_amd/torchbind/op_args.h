// What the native sides of the operators past the block's share (post_ops.cpp, student_ops.cpp): allocation, refusals, autograd nodes' guards, arguments.
#pragma once
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>

#include <cstdint>
#include <limits>

#include "torch_args.h"

namespace pk_torch {

// As torch_args.h's empty_of, past the dispatcher: a call on a few tokens is host time, and these are half of it.
inline Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType t, const Tensor& like) { return at::detail::empty_cuda(sizes, t, like.device(), c10::nullopt); }

[[noreturn]] inline void refuse(const char* who, const std::string& what) { throw std::runtime_error(std::string(who) + ": " + what); }

inline void on_gpu(const char* who, const Tensor& t) {
    if (!t.is_cuda()) refuse(who, "paperkiln_amd has no CPU path: tensors must live on the GPU");
}
// a vector of one value for each row, dense
inline void vector_of(const char* who, const char* what, const Tensor& t, at::ScalarType type, int64_t n, const Tensor& like) {
    if (t.device() != like.device()) refuse(who, std::string(what) + " must live on the device of the other tensors");
    if (t.scalar_type() != type) refuse(who, std::string(what) + " must be " + (type == at::kInt ? "int32" : "float32"));
    if (t.numel() != n) refuse(who, std::string("shape mismatch: ") + what + " has " + std::to_string(t.numel()) + " values, expected " + std::to_string(n));
    if (!t.is_contiguous()) refuse(who, std::string(what) + " must be contiguous");
}
inline int32_t narrow(const char* who, int64_t n) {
    if (n < 0 || n > std::numeric_limits<int32_t>::max()) refuse(who, "shape mismatch: a dimension is out of range");
    return static_cast<int32_t>(n);
}
inline void no_tangent(const char* who, const Tensor& t) {
    if (t._fw_grad(0).defined()) refuse(who, "forward-mode differentiation is not implemented");
}
inline void first_order(const char* who) {
    if (at::GradMode::is_enabled()) refuse(who, "its gradient is not differentiable");
}
// A backward pass that is being recorded into a graph while gradients of this node's inputs belong to a stream outside of the recording (a graph of the same
// leaves that was built before and lives on keeps their accumulation there): the engine would have that stream wait for the recording, which ends the process.
inline void recordable(const char* who, Node& node) {
    using Stream = c10::hip::HIPStreamMasqueradingAsCUDA;
    const auto recording = [](hipStream_t s) {  // the null stream never is, and must not be asked
        hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
        return s && hipStreamIsCapturing(s, &status) == hipSuccess && status != hipStreamCaptureStatusNone;
    };
    const Stream now = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA();
    if (!recording(now.stream())) return;
    for (size_t i = 0; i < node.num_outputs(); ++i) {
        const auto& next = node.next_edge(i);
        if (!next.is_valid() || !node.task_should_compute_output(i)) continue;
        const auto other = next.function->stream();
        if (other && *other != now.unwrap() && !recording(Stream(*other).stream()))
            refuse(who, "a backward pass is being recorded whose inputs' gradients belong to a stream outside of the recording: drop the graphs of the same leaves first");
    }
}

inline void changed(const Tensor& t) {  // what was saved of it for a backward pass is no longer what it was
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

struct Logits {
    int64_t rows, vocab, ld;
    int dtype;
};
inline Logits matrix(const char* who, const char* what, const Tensor& x) {
    on_gpu(who, x);
    if (x.dim() != 2 || x.size(1) < 1) refuse(who, std::string("shape mismatch: ") + what + " is a [rows, vocab] matrix");
    if (x.stride(1) != 1 && x.size(1) > 1) refuse(who, std::string(what) + ": the vocabulary must be contiguous");
    return Logits{x.size(0), x.size(1), x.size(0) > 1 ? x.stride(0) : x.size(1), dtype_code(x.scalar_type())};
}
inline Tensor gradient_of(const char* who, const Tensor& logits, const Tensor& out) {
    if (!out.defined()) return new_tensor(logits.sizes(), logits.scalar_type(), logits);
    if (out.sizes() != logits.sizes() || out.scalar_type() != logits.scalar_type() || out.device() != logits.device()) refuse(who, "shape mismatch: out");
    return out;
}

inline PyObject* tuple_of(std::vector<Tensor>&& v) {
    PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(v.size()));
    if (!t) throw python_error();
    for (size_t i = 0; i < v.size(); ++i) PyTuple_SET_ITEM(t, static_cast<Py_ssize_t>(i), THPVariable_Wrap(std::move(v[i])));
    return t;
}

inline Tensor optional_arg(PyObject* o, const char* what) { return o == Py_None ? Tensor() : tensor_arg(o, what); }
inline float number_arg(PyObject* o) { return static_cast<float>(float_arg(o)); }
inline int whole_arg(PyObject* o, const char* what) {  // int() of it, refused past 32 bits
    PyObject* i = PyNumber_Long(o);
    if (!i) throw python_error();
    const long long x = PyLong_AsLongLong(i);
    Py_DECREF(i);
    if (x == -1 && PyErr_Occurred()) throw python_error();
    if (x < std::numeric_limits<int>::min() || x > std::numeric_limits<int>::max()) throw std::runtime_error(std::string(what) + " is out of range");
    return static_cast<int>(x);
}

}  // namespace pk_torch
