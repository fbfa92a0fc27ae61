// tms_cache_py.cpp -- the Python side of tmcache_hip.h over torch tensors: what
// tensormark_amd/cache.py's functions check, allocate and call.  In C++ for the
// host's time alone: a decode step's call takes the GPU some 3 to 15 us, and the
// same checks in Python with ctypes took 7 to 12 us of the host besides the launch;
// a call is 4.5 to 9 us of the host with this (a token of each of 64 sequences into
// the cache: 11.0 us with ctypes, 4.3 with this; one session's attention: 15.0 and 11.6).
#include <ATen/MemoryOverlap.h>
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

static void want(bool ok, const char* what) {
    if (!ok) throw py::value_error(what);
}

static void check(int rc, const char* call) {
    if (rc != TMS_OK)
        throw std::runtime_error(std::string(call) + " failed: " + tms_status_string(rc) + " (" + std::to_string(rc) + ")");
}

static int gpu_of(const Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }

// The device of a call's tensors as the current one: a launch into the null stream, torch's default, goes
// to the current device, wherever the tensors are.
struct OnDeviceOf {
    c10::OptionalDeviceGuard guard;
    explicit OnDeviceOf(const Tensor& t) {
        if (t.is_cuda()) guard.reset_device(t.device());
    }
};

static const Tensor* of(const MaybeTensor& t) { return t ? &*t : nullptr; }

// No call has a backward: a gradient that would have to go through one is refused.
static void want_no_gradient(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return;
    for (const Tensor* t : tensors)
        want(!t || !t->requires_grad(), "no gradient goes through this call: detach its tensors, or call it under torch.no_grad()");
}

// Autograd finds by its version that a tensor it kept has been written (inference tensors have none).
static void written(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
static void written(const MaybeTensor& t) {
    if (t) written(*t);
}

// An output is the input's own tensor or shares no memory with it, as far as their strides tell.
static void want_apart(const Tensor& out, const Tensor& in) {
    want(at::has_internal_overlap(out) != at::MemOverlap::Yes && at::get_overlap_status(out, in) != at::MemOverlapStatus::Partial,
         "out: overlaps itself or, in part, the input");
}

// A number of Python's as 32 bits, for the library to judge; none is a smaller one by wrapping.
static int32_t i32(int64_t n) { return (int32_t)std::clamp<int64_t>(n, INT32_MIN, INT32_MAX); }

static const int32_t* ints(const Tensor& t, std::initializer_list<int64_t> shape, const char* what, int device) {
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
static void pool(const Tensor& t, int64_t* stride, const char* what) {
    want(t.stride(3) == 1, what);
    for (int i = 0; i < 3; ++i) stride[i] = t.size(i) == 1 && i < 2 ? 0 : t.stride(i);
}

static tms_cache cache_of(const Tensor& k, const Tensor* v, const Tensor* scores, const Tensor& tables, const Tensor& kv_len,
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
static void rows(const Tensor& t, const Tensor& k, int64_t* stride, const char* what) {
    want(t.dim() == 3 && k.dim() == 4 && t.scalar_type() == k.scalar_type() && gpu_of(t) == gpu_of(k) &&
             t.size(2) == k.size(3) && t.stride(2) == 1,
         what);
    for (int i = 0; i < 2; ++i) stride[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

static float* f32_rows(const Tensor& t, const Tensor& q, const char* what) {
    want(t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(0) == q.size(0) && t.size(1) == q.size(1) && t.is_contiguous() &&
             gpu_of(t) == gpu_of(q),
         what);
    return t.data_ptr<float>();
}

static float scale_of(std::optional<double> scale, const Tensor& q) {
    return scale ? (float)*scale : (float)(1.0 / std::sqrt((double)q.size(2)));
}

static hipStream_t stream_of(int64_t stream) { return reinterpret_cast<hipStream_t>(stream); }

static void kv_append(const Tensor& k_new, const Tensor& v_new, const Tensor& k, const Tensor& v, const Tensor& tables,
                      const Tensor& kv_len, const Tensor& q_start, int64_t max_q, const MaybeTensor& scores, int64_t stream) {
    want_no_gradient({&k_new, &v_new, &k, &v, of(scores)});
    const OnDeviceOf on(k);
    const tms_cache c = cache_of(k, &v, of(scores), tables, kv_len, &q_start, k_new.dim() ? k_new.size(0) : 0, max_q, 0);
    tms_append_args a{};
    rows(k_new, k, a.k_new_stride, "k_new: [tokens, heads, head_dim] like k_cache, last stride 1");
    rows(v_new, k, a.v_new_stride, "v_new: [tokens, heads, head_dim] like k_cache, last stride 1");
    want(k_new.sizes() == v_new.sizes() && k_new.size(1) == k.size(1), "k_new, v_new: one row a key head");
    a.k_new = k_new.data_ptr();
    a.v_new = v_new.data_ptr();
    check(tms_kv_append(&c, &a, stream_of(stream)), "tms_kv_append");
    written(k);
    written(v);
    written(scores);
}

static std::tuple<Tensor, Tensor> paged_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& tables,
                                                  const Tensor& kv_len, const Tensor& q_start, int64_t max_q, int64_t max_kv,
                                                  int64_t window, int64_t sinks, std::optional<double> scale,
                                                  const MaybeTensor& out_, const MaybeTensor& lse_, int64_t stream) {
    want_no_gradient({&q, &k, &v, of(out_), of(lse_)});
    const OnDeviceOf on(k);
    const tms_cache c = cache_of(k, &v, nullptr, tables, kv_len, &q_start, q.dim() ? q.size(0) : 0, max_q, max_kv);
    tms_attention_args a{};
    rows(q, k, a.q_stride, "q: [tokens, heads, head_dim] like k_cache, last stride 1");
    const Tensor out = out_ ? *out_ : at::empty(q.sizes(), q.options());
    const Tensor lse = lse_ ? *lse_ : at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
    want(out.sizes() == q.sizes(), "out: like q");
    rows(out, k, a.out_stride, "out: like q");
    if (out_) want_apart(out, q);
    a.q = q.data_ptr();
    a.out = out.data_ptr();
    a.lse = f32_rows(lse, q, "lse: contiguous float32 [tokens, q_heads]");
    a.q_heads = i32(q.size(1));
    a.window = std::max(i32(window), 0);
    a.sinks = i32(sinks);
    a.scale = scale_of(scale, q);
    const int64_t need = tms_paged_attention_workspace(&c, &a);
    if (need < 0) check((int)need, "tms_paged_attention");
    Tensor workspace;
    if (need > 0) {
        workspace = at::empty({need}, q.options().dtype(at::kByte));
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = (size_t)need;
    }
    check(tms_paged_attention(&c, &a, stream_of(stream)), "tms_paged_attention");
    written(out_);
    written(lse_);
    return {out, lse};
}

static Tensor kv_add_scores(const Tensor& q, const Tensor& lse, const Tensor& k, const MaybeTensor& scores, const Tensor& tables,
                            const Tensor& kv_len, const Tensor& q_start, int64_t max_q, int64_t max_kv, int64_t window, int64_t sinks,
                            std::optional<double> scale, const MaybeTensor& out_, int64_t stream) {
    want_no_gradient({&q, &lse, &k, of(scores), of(out_)});
    const OnDeviceOf on(k);
    want(scores.has_value(), "scores: needed");
    const tms_cache c = cache_of(k, nullptr, &*scores, tables, kv_len, &q_start, q.dim() ? q.size(0) : 0, max_q, max_kv);
    tms_score_args a{};
    rows(q, k, a.q_stride, "q: [tokens, heads, head_dim] like k_cache, last stride 1");
    const Tensor out = out_ ? *out_ : *scores;
    want(out.scalar_type() == at::kFloat && out.sizes() == scores->sizes() && out.is_contiguous() && gpu_of(out) == gpu_of(k),
         "out: like scores");
    if (out_) want_apart(out, *scores);
    a.q = q.data_ptr();
    a.lse = f32_rows(lse, q, "lse: contiguous float32 [tokens, q_heads]");
    a.out = out.data_ptr<float>();
    a.q_heads = i32(q.size(1));
    a.window = std::max(i32(window), 0);
    a.sinks = i32(sinks);
    a.scale = scale_of(scale, q);
    check(tms_kv_add_scores(&c, &a, stream_of(stream)), "tms_kv_add_scores");
    written(out);
    return out;
}

static std::tuple<Tensor, Tensor> kv_evict(const Tensor& k, const Tensor& v, const MaybeTensor& scores, const Tensor& tables,
                                           const Tensor& kv_len, const Tensor& dst_tables, int64_t budget, int64_t max_kv, int64_t sinks,
                                           int64_t recent, const MaybeTensor& new_len_, const MaybeTensor& kept_, int64_t stream) {
    want_no_gradient({&k, &v, of(scores)});
    const OnDeviceOf on(k);
    want(scores.has_value(), "scores: needed");
    const tms_cache c = cache_of(k, &v, &*scores, tables, kv_len, nullptr, 0, 0, max_kv);
    const int device = gpu_of(k);
    const int64_t B = tables.size(0), H = k.size(1);
    want(dst_tables.dim() == 2 && dst_tables.size(0) == B, "dst_tables: int32 [batch, entries]");
    want(budget >= 1 && budget <= INT32_MAX, "budget: at least 1");
    tms_evict_args a{};
    a.dst_tables = ints(dst_tables, {B, dst_tables.size(1)}, "dst_tables", device);
    a.dst_table_stride = dst_tables.size(1);
    a.budget = i32(budget);
    a.sinks = i32(sinks);
    a.recent = i32(recent);
    const Tensor new_len = new_len_ ? *new_len_ : at::empty({B}, tables.options());
    const Tensor kept = kept_ ? *kept_ : at::empty({B, H, budget}, tables.options());
    a.new_len = const_cast<int32_t*>(ints(new_len, {B}, "new_len", device));
    a.kept = const_cast<int32_t*>(ints(kept, {B, H, budget}, "kept", device));
    check(tms_kv_evict(&c, &a, stream_of(stream)), "tms_kv_evict");
    written(k);
    written(v);
    written(*scores);
    written(new_len_);
    written(kept_);
    return {new_len, kept};
}

static int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return TMS_DTYPE_F32;
        case at::kHalf: return TMS_DTYPE_F16;
        case at::kBFloat16: return TMS_DTYPE_BF16;
        default: return -1;
    }
}

static bool row_contiguous(const Tensor& t) { return t.stride(1) == 1 || t.size(1) <= 1; }

static Tensor adjust_logits(const Tensor& logits, const MaybeTensor& params, const MaybeTensor& recent, const MaybeTensor& n_recent,
                            const MaybeTensor& drafts, int64_t steps, const MaybeTensor& bias_ids, const MaybeTensor& bias_values,
                            const MaybeTensor& mask, const MaybeTensor& out_, int64_t stream) {
    want_no_gradient({&logits, of(bias_values), of(out_)});
    const OnDeviceOf on(logits);
    want(logits.dim() == 2 && dtype_code(logits) >= 0 && logits.is_cuda() && row_contiguous(logits),
         "logits: device [rows, vocab] of float32, float16 or bfloat16, last stride 1");
    const int device = gpu_of(logits);
    const int64_t R = logits.size(0), V = logits.size(1);
    want(steps >= 1 && R % steps == 0, "logits: a multiple of `steps` rows");
    const int64_t S = R / steps;
    tms_adjust_args a{};
    a.dtype = dtype_code(logits);
    a.seqs = i32(S);
    a.steps = i32(steps);
    a.vocab = i32(V);
    a.row_stride = R > 1 ? logits.stride(0) : V;
    if (params) {
        want(params->scalar_type() == at::kByte && params->is_contiguous() && params->numel() == S * (int64_t)sizeof(tms_row_params) &&
                 gpu_of(*params) == device,
             "params: uint8 ROW_DTYPE records, one a sequence");
        a.params = (const tms_row_params*)params->data_ptr();
    }
    if (recent) {
        want(recent->dim() == 2 && recent->size(0) == S && recent->scalar_type() == at::kInt && gpu_of(*recent) == device &&
                 row_contiguous(*recent) && (S <= 1 || recent->stride(0) >= recent->size(1)),
             "recent: int32 [seqs, n] on the logits' device, rows contiguous");
        a.recent = recent->const_data_ptr<int32_t>();
        a.recent_stride = S > 1 ? recent->stride(0) : recent->size(1);
        a.n_history = i32(recent->size(1));
        if (n_recent) a.n_recent = ints(*n_recent, {S}, "n_recent", device);
    }
    if (drafts && steps > 1) a.drafts = ints(*drafts, {S, steps - 1}, "drafts", device);
    want(bias_ids.has_value() == bias_values.has_value(), "bias_ids and bias_values go together");
    if (bias_ids && bias_ids->numel()) {
        const int64_t n = bias_ids->size(-1);
        a.n_bias = i32(n);
        a.bias_ids = ints(*bias_ids, {S, n}, "bias_ids", device);
        want(bias_values->scalar_type() == at::kFloat && bias_values->sizes() == bias_ids->sizes() && bias_values->is_contiguous() &&
                 gpu_of(*bias_values) == device,
             "bias_values: contiguous float32, like bias_ids");
        a.bias_values = bias_values->const_data_ptr<float>();
    }
    if (mask) {
        want(mask->dim() == 2 && mask->size(0) == R && mask->element_size() == 4 && !mask->is_floating_point() && row_contiguous(*mask) &&
                 gpu_of(*mask) == device && mask->size(1) >= (V + 31) / 32,
             "mask: 32-bit words [rows, ceil(vocab / 32)]");
        a.mask = (const uint32_t*)mask->const_data_ptr();
        a.mask_stride = R > 1 ? mask->stride(0) : mask->size(1);
    }
    const Tensor out = out_ ? *out_ : at::empty(logits.sizes(), logits.options());
    want(out.sizes() == logits.sizes() && (out.scalar_type() == logits.scalar_type() || out.scalar_type() == at::kFloat) &&
             gpu_of(out) == device && row_contiguous(out),
         "out: like logits, of its type or float32");
    if (out_) want_apart(out, logits);
    a.out_dtype = dtype_code(out);
    a.out_stride = R > 1 ? out.stride(0) : V;
    a.logits = logits.data_ptr();
    a.out = out.data_ptr();
    check(tms_adjust_logits(&a, stream_of(stream)), "tms_adjust_logits");
    written(out_);
    return out;
}

PYBIND11_MODULE(_cache_ops, m) {
    m.def("kv_append", &kv_append);
    m.def("paged_attention", &paged_attention);
    m.def("kv_add_scores", &kv_add_scores);
    m.def("kv_evict", &kv_evict);
    m.def("adjust_logits", &adjust_logits);
}
