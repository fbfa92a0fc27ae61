// tms_py.h -- what the calls' Python sides over torch tensors share: checks, and
// tensors as the C ABI has them.
#pragma once

#include <ATen/MemoryOverlap.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/tmcache_hip.h"

namespace py = pybind11;
using at::Tensor;
typedef std::optional<Tensor> MaybeTensor;

inline void want(bool ok, const char* what) {
    if (!ok) throw py::value_error(what);
}

inline void check(int rc, const char* call) {
    if (rc != TMS_OK)
        throw std::runtime_error(std::string(call) + " failed: " + tms_status_string(rc) + " (" + std::to_string(rc) + ")");
}

inline int gpu_of(const Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }

// The device of a call's tensors as the current one: a launch into the null stream, torch's default, goes
// to the current device, wherever the tensors are.
struct OnDeviceOf {
    c10::OptionalDeviceGuard guard;
    explicit OnDeviceOf(const Tensor& t) {
        if (t.is_cuda()) guard.reset_device(t.device());
    }
};

inline const Tensor* of(const MaybeTensor& t) { return t ? &*t : nullptr; }

// No call has a derivative: a gradient or a forward-mode tangent that would have to go through one is
// refused.  (Tangents are on without the gradient mode too.)
inline void want_no_gradient(std::initializer_list<const Tensor*> tensors) {
    const bool gradients = at::GradMode::is_enabled(), tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const Tensor* t : tensors) {
        if (!t) continue;
        want(!gradients || !t->requires_grad(), "no gradient goes through this call: detach its tensors, or call it under torch.no_grad()");
        want(!tangents || !t->_fw_grad(0).defined(), "no tangent goes through this call: unpack its dual tensors");   // (0: the only level)
    }
}

// Autograd finds by its version that a tensor it kept has been written (inference tensors have none).
inline void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
inline void written(const MaybeTensor& t) {
    if (t) written(*t);
}

// An output is the input's own tensor or shares no memory with it, as far as their strides tell.
inline void want_apart(const Tensor& out, const Tensor& in) {
    want(at::has_internal_overlap(out) != at::MemOverlap::Yes && at::get_overlap_status(out, in) != at::MemOverlapStatus::Partial,
         "out: overlaps itself or, in part, the input");
}

// A number of Python's as 32 bits, for the library to judge; none is a smaller one by wrapping.
inline int32_t i32(int64_t n) { return (int32_t)std::clamp<int64_t>(n, INT32_MIN, INT32_MAX); }

inline const int32_t* ints(const Tensor& t, std::initializer_list<int64_t> shape, const char* what, int device) {
    const bool ok = t.scalar_type() == at::kInt && t.sizes().equals(at::IntArrayRef(shape.begin(), shape.size())) &&
                    t.is_contiguous() && gpu_of(t) == device;
    if (!ok) {
        std::string s = std::string(what) + ": a contiguous int32 tensor [";
        for (int64_t n : shape) s += std::to_string(n) + ", ";
        s.replace(s.size() - 2, 2, "] on cuda:" + std::to_string(device));
        throw py::value_error(s);
    }
    return t.const_data_ptr<int32_t>();
}

// A pool's page, head and slot strides; that of a single page or head does not matter.
inline void pool(const Tensor& t, int64_t* stride, const char* what) {
    want(t.stride(3) == 1, what);
    for (int i = 0; i < 3; ++i) stride[i] = t.size(i) == 1 && i < 2 ? 0 : t.stride(i);
}

inline tms_cache cache_of(const Tensor& k, const Tensor* v, const Tensor* scores, const Tensor& tables, const Tensor& kv_len,
                          const Tensor* q_start, int64_t tokens, int64_t max_q, int64_t max_kv) {
    tms_cache c{};
    want(k.dim() == 4 && k.size(0) >= 1, "k_cache: [pages, kv_heads, page_size, head_dim]");
    want(k.scalar_type() == at::kBFloat16 || k.scalar_type() == at::kHalf, "k_cache: bfloat16 or float16");
    want(k.is_cuda(), "k_cache: a device tensor");
    const int device = gpu_of(k);
    c.k = k.data_ptr();
    pool(k, c.k_stride, "k_cache: the last stride must be 1");
    c.dtype = k.scalar_type() == at::kBFloat16 ? TMS_DTYPE_BF16 : TMS_DTYPE_F16;
    c.pages = i32(k.size(0));
    c.kv_heads = i32(k.size(1));
    c.page_size = i32(k.size(2));
    c.head_dim = i32(k.size(3));
    if (v) {
        want(v->sizes() == k.sizes() && v->scalar_type() == k.scalar_type() && gpu_of(*v) == device, "v_cache: like k_cache");
        c.v = v->data_ptr();
        pool(*v, c.v_stride, "v_cache: the last stride must be 1");
    }
    if (scores) {
        want(scores->scalar_type() == at::kFloat && scores->sizes() == k.sizes().slice(0, 3) && scores->is_contiguous() &&
                 gpu_of(*scores) == device,
             "scores: contiguous float32 [pages, kv_heads, page_size]");
        c.scores = scores->data_ptr<float>();
    }
    want(tables.dim() == 2 && tables.scalar_type() == at::kInt && gpu_of(tables) == device && tables.is_contiguous() &&
             tables.size(1) >= 1,
         "tables: contiguous int32 [batch, entries]");
    c.batch = i32(tables.size(0));
    c.tables = tables.const_data_ptr<int32_t>();
    c.table_stride = tables.size(1);
    c.kv_len = ints(kv_len, {tables.size(0)}, "kv_len", device);
    if (q_start) c.q_start = ints(*q_start, {tables.size(0) + 1}, "q_start", device);
    c.tokens = i32(tokens);
    c.max_q = i32(max_q);
    c.max_kv = i32(max_kv);
    return c;
}

// [tokens, heads, head_dim] rows of the cache's type; the stride of a single token or head does not matter.
inline void rows(const Tensor& t, const Tensor& k, int64_t* stride, const char* what) {
    want(t.dim() == 3 && k.dim() == 4 && t.scalar_type() == k.scalar_type() && gpu_of(t) == gpu_of(k) &&
             t.size(2) == k.size(3) && t.stride(2) == 1,
         what);
    for (int i = 0; i < 2; ++i) stride[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

inline float* f32_rows(const Tensor& t, const Tensor& q, const char* what) {
    want(t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == q.size(0) && t.size(1) == q.size(1) && t.is_contiguous() &&
             gpu_of(t) == gpu_of(q),
         what);
    return t.data_ptr<float>();
}

inline float scale_of(std::optional<double> scale, const Tensor& q) {
    return scale ? (float)*scale : (float)(1.0 / std::sqrt((double)q.size(2)));
}

inline hipStream_t stream_of(int64_t stream) { return reinterpret_cast<hipStream_t>(stream); }

inline int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return TMS_DTYPE_F32;
        case at::kHalf: return TMS_DTYPE_F16;
        case at::kBFloat16: return TMS_DTYPE_BF16;
        default: return -1;
    }
}

inline bool row_contiguous(const Tensor& t) { return t.stride(1) == 1 || t.size(1) <= 1; }
