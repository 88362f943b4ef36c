// What the native host paths share: the devices' status words, error types, and tensors as the kernels take them.
#pragma once

#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <optional>
#include <string>

#include "../../include/kda_b200.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace kda_host {

constexpr int CHUNK = KDA_CHUNK;

// ---- per-device status word and its pinned host mirror (owned by ops._DeviceStatus) -------------------------
constexpr int MAX_DEVICES = 64;
struct StatusWord {
    std::atomic<int32_t*> dev{nullptr};  // set after host: calls of other threads look without the interpreter lock
    const volatile int32_t* host = nullptr;
};
inline StatusWord g_status[MAX_DEVICES];
// Python callables: status_of(device_index) creates the words; report(device_index) raises and clears;
// guard_span() reads the mutable span of the guard contract
inline py::object* g_status_of = nullptr;
inline py::object* g_report = nullptr;
inline py::object* g_guard_span = nullptr;

inline void set_status(int device, int64_t dev_ptr, int64_t host_ptr) {
    TORCH_CHECK(device >= 0 && device < MAX_DEVICES, "device index out of range");
    g_status[device].host = reinterpret_cast<const volatile int32_t*>(host_ptr);
    g_status[device].dev.store(reinterpret_cast<int32_t*>(dev_ptr), std::memory_order_release);
}

inline void set_callbacks(py::object status_of, py::object report, py::object guard_span) {
    g_status_of = new py::object(std::move(status_of));  // (never destroyed: they outlive the interpreter's modules)
    g_report = new py::object(std::move(report));
    g_guard_span = new py::object(std::move(guard_span));
}

inline const StatusWord& status_word(int device) {
    TORCH_CHECK(device >= 0 && device < MAX_DEVICES, "device index out of range");
    const StatusWord& st = g_status[device];
    if (!st.dev.load(std::memory_order_acquire) || *st.host) {
        py::gil_scoped_acquire gil;
        if (!st.dev.load(std::memory_order_relaxed)) (*g_status_of)(device);
        if (*st.host) (*g_report)(device);  // a wait that gave up in an earlier call surfaces here
    }
    return st;
}

// the guard contract's span is a module attribute that callers may change between calls; it is read at every call
inline float guard_span() {
    py::gil_scoped_acquire gil;
    return (*g_guard_span)().cast<float>();
}

// debugging / A-B switches of the environment (ops.chunk_kda documents them), read at every call
inline int64_t env_flags() {
    auto is_one = [](const char* n) { const char* v = std::getenv(n); return v && v[0] == '1' && !v[1]; };
    int64_t f = 0;
    if (is_one("OPENKIMI_B200_FP32_MATH")) f |= KDA_FLAG_FORCE_SIMT;
    if (is_one("OPENKIMI_B200_ROW_COPIES")) f |= KDA_FLAG_ROW_COPIES;
    if (const char* v = std::getenv("OPENKIMI_B200_FP32_STAGES")) f |= (std::strtol(v, nullptr, 10) & 31) << 5;
    return f;
}

inline void check_rc(int rc, const char* what) {
    if (rc == KDA_OK) return;
    std::string msg = std::string(what) + " failed: " + kda_status_string(rc);
    const std::string extra = kda_last_cuda_error();
    if (rc == KDA_ERR_LAUNCH && !extra.empty()) msg += " (" + extra + ")";
    throw std::runtime_error(msg);
}

inline std::string shape_of(const Tensor& t) {
    std::string s = "(";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + (t.dim() == 1 ? ",)" : ")");
}
[[noreturn]] inline void value_error(const std::string& m) { throw py::value_error(m); }
[[noreturn]] inline void type_error(const std::string& m) { throw py::type_error(m); }

inline void require_cuda(const Tensor& t) {
    if (!t.is_cuda()) throw std::runtime_error("chunk_kda runs only on a CUDA device (sm_100a); there is no CPU fallback");
}

// the kernels follow raw pointers: every tensor of a call has to be where q is
inline void require_device(const Tensor& q, const char* name, const Tensor& t) {
    if (t.defined() && t.device() != q.device())
        throw std::runtime_error(std::string("expected ") + name + " on " + q.device().str() + ", the device of q, but it is on " +
                                 t.device().str());
}

// A call that nobody differentiates backward does not pass through its autograd node, which refuses forward-mode inputs.
template <class Tensors>
inline void refuse_tangents(const Tensors& inputs) {
    for (const Tensor* t : inputs)
        if (t->defined() && t->_fw_grad(0).defined())
            throw std::runtime_error("the KDA kernels have no forward-mode derivative (an input carries a tangent)");
}

inline int dtype_code(const Tensor& t) {
    if (t.scalar_type() == at::kBFloat16) return KDA_DTYPE_BF16;
    if (t.scalar_type() == at::kFloat) return KDA_DTYPE_F32;
    type_error(std::string("q/k/v must be float32 or bfloat16, got ") + c10::toString(t.scalar_type()));
}

// contiguous, in dtype dt, starting on a 16-byte boundary (a view into the middle of a buffer is copied)
inline Tensor ready(const Tensor& t, at::ScalarType dt) {
    Tensor r = t.scalar_type() == dt ? t : t.to(dt);
    if (!r.is_contiguous()) r = r.contiguous();
    return (reinterpret_cast<uintptr_t>(r.data_ptr()) & 15) == 0 ? r : r.clone();
}
// the same without a new reference where t is that already or undefined; copy holds what else it becomes
inline const Tensor& ready(const Tensor& t, at::ScalarType dt, Tensor& copy) {
    if (!t.defined() || (t.scalar_type() == dt && t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0)) return t;
    return copy = ready(t, dt);
}
// a new tensor without the dispatcher's detour (half of what at::empty costs)
inline Tensor fresh(at::IntArrayRef sizes, at::ScalarType dt, const Tensor& like) {
    return Tensor(at::detail::empty_cuda(sizes, dt, like.device(), std::nullopt));
}
inline const Tensor& val(const OptTensor& t) {
    static const Tensor none;
    return t ? *t : none;
}
template <class T>
T* ptr(const Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }

inline void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// A kernel has written t: what autograd has saved of it is no longer what it was.  (A tensor made in inference mode has no version.)
inline void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A cached table belongs to the stream that made it: the current one reads it too, so that its memory waits for both when the cache drops it.
inline const Tensor& read_here(const Tensor& t) {
    c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), at::cuda::getCurrentCUDAStream(t.device().index()));
    return t;
}

inline Tensor bytes(size_t n, const Tensor& like) { return fresh({(int64_t)n}, at::kByte, like); }
inline Tensor fresh_like(const Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }
inline OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }  // (a node's inputs must be defined tensors)

}  // namespace kda_host
