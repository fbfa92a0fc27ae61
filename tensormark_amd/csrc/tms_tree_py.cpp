// tms_tree_py.cpp -- the Python side of tmtree_hip.h over torch tensors: what
// tensormark_amd/tree.py's functions check, allocate and call.  In C++ for the host's
// time alone, as tms_cache_py.cpp.
#include "tms_py.h"

#include "../../include/tmtree_hip.h"

static const float* freqs_of(const Tensor& freqs, int device) {
    want(freqs.dim() == 1 && freqs.scalar_type() == at::kFloat && freqs.is_contiguous() && gpu_of(freqs) == device,
         "freqs: contiguous float32 [rotary_dim / 2] on the tensors' device");
    return freqs.const_data_ptr<float>();
}

// Heads' strides of a [tokens, heads, head_dim] tensor; that of a single token or head does not matter.
static void head_strides(const Tensor& t, int64_t* stride) {
    for (int i = 0; i < 2; ++i) stride[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

// What a call writes shares no memory with what it reads, as far as their strides tell.
static void want_separate(const Tensor& out, std::initializer_list<const Tensor*> others, const char* what) {
    for (const Tensor* t : others)
        if (t && t->numel() && out.numel()) {
            const at::MemOverlapStatus s = at::get_overlap_status(out, *t);
            want(s != at::MemOverlapStatus::Partial && s != at::MemOverlapStatus::Full, what);
        }
}

static Tensor rotary(const Tensor& x, const Tensor& positions, const Tensor& freqs, bool interleaved, double scale, const MaybeTensor& out_,
                     int64_t stream) {
    want_no_gradient({&x, &freqs, of(out_)});
    const OnDeviceOf on(x);
    want(x.dim() == 3 && dtype_code(x) >= 0 && x.is_cuda() && x.stride(2) == 1,
         "x: device [tokens, heads, head_dim] of float32, float16 or bfloat16, last stride 1");
    const int device = gpu_of(x);
    tms_rotary_args a{};
    head_strides(x, a.x_stride);
    a.positions = ints(positions, {x.size(0)}, "positions", device);
    a.freqs = freqs_of(freqs, device);
    const Tensor out = out_ ? *out_ : at::empty(x.sizes(), x.options());
    want(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && gpu_of(out) == device && out.stride(2) == 1, "out: like x");
    if (out_) want_apart(out, x);
    head_strides(out, a.out_stride);
    a.x = x.const_data_ptr();
    a.out = out.data_ptr();
    a.dtype = dtype_code(x);
    a.tokens = i32(x.size(0));
    a.heads = i32(x.size(1));
    a.head_dim = i32(x.size(2));
    a.rotary_dim = i32(2 * freqs.size(0));
    a.interleaved = interleaved;
    a.scale = (float)scale;
    check(tms_rotary(&a, stream_of(stream)), "tms_rotary");
    written(out_);
    return out;
}

static MaybeTensor kv_append_rotary(const MaybeTensor& q, const Tensor& k_new, const Tensor& v_new, const Tensor& k, const Tensor& v,
                                    const Tensor& tables, const Tensor& kv_len, const Tensor& q_start, const MaybeTensor& positions,
                                    const Tensor& freqs, int64_t max_q, bool interleaved, double scale, const MaybeTensor& scores,
                                    const MaybeTensor& out_, int64_t stream) {
    want_no_gradient({of(q), &k_new, &v_new, &k, &v, &freqs, of(scores), of(out_)});
    const OnDeviceOf on(k);
    const tms_cache c = cache_of(k, &v, of(scores), tables, kv_len, &q_start, k_new.dim() ? k_new.size(0) : 0, max_q, 0);
    const int device = gpu_of(k);
    tms_append_rotary_args a{};
    rows(k_new, k, a.k_new_stride, "k_new: [tokens, heads, head_dim] like k_cache, last stride 1");
    rows(v_new, k, a.v_new_stride, "v_new: [tokens, heads, head_dim] like k_cache, last stride 1");
    want(k_new.sizes() == v_new.sizes() && k_new.size(1) == k.size(1), "k_new, v_new: one row a key head");
    a.k_new = k_new.const_data_ptr();
    a.v_new = v_new.const_data_ptr();
    if (positions) a.positions = ints(*positions, {k_new.size(0)}, "positions", device);
    a.freqs = freqs_of(freqs, device);
    want(q || !out_, "out: needs q");
    MaybeTensor out;
    if (q) {
        rows(*q, k, a.q_stride, "q: [tokens, heads, head_dim] like k_cache, last stride 1");
        want(q->size(0) == k_new.size(0), "q: a row a new token");
        out = out_ ? *out_ : at::empty(q->sizes(), q->options());
        want(out->sizes() == q->sizes(), "out: like q");
        rows(*out, k, a.out_stride, "out: like q");
        if (out_) {
            want_apart(*out, *q);
            want_separate(*out, {&k_new, &v_new}, "out: shares memory with k_new or v_new");
        }
        a.q = q->const_data_ptr();
        a.out = out->data_ptr();
        a.q_heads = i32(q->size(1));
    }
    a.rotary_dim = i32(2 * freqs.size(0));
    a.interleaved = interleaved;
    a.scale = (float)scale;
    check(tms_kv_append_rotary(&c, &a, stream_of(stream)), "tms_kv_append_rotary");
    written(k);
    written(v);
    written(scores);
    written(out_);
    return out;
}

static std::tuple<Tensor, Tensor> tree_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& tables,
                                                 const Tensor& kv_len, const Tensor& q_start, const Tensor& parents, int64_t max_q,
                                                 int64_t max_kv, int64_t window, int64_t sinks, std::optional<double> scale,
                                                 const MaybeTensor& out_, const MaybeTensor& lse_, int64_t stream) {
    want_no_gradient({&q, &k, &v, of(out_), of(lse_)});
    const OnDeviceOf on(k);
    const tms_cache c = cache_of(k, &v, nullptr, tables, kv_len, &q_start, q.dim() ? q.size(0) : 0, max_q, max_kv);
    tms_attention_args a{};
    rows(q, k, a.q_stride, "q: [tokens, heads, head_dim] like k_cache, last stride 1");
    const int32_t* up = ints(parents, {q.size(0)}, "parents", gpu_of(k));
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
    const int64_t need = tms_tree_attention_workspace(&c, &a);
    if (need < 0) check((int)need, "tms_tree_attention");
    Tensor workspace;
    if (need > 0) {
        workspace = at::empty({need}, q.options().dtype(at::kByte));
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = (size_t)need;
    }
    check(tms_tree_attention(&c, &a, up, stream_of(stream)), "tms_tree_attention");
    written(out_);
    written(lse_);
    return {out, lse};
}

// Rows of probabilities; returns their stride.
static int64_t probabilities(const Tensor& t, const char* what) {
    want(t.dim() == 2 && dtype_code(t) >= 0 && t.is_cuda() && row_contiguous(t), what);
    return t.size(0) > 1 ? t.stride(0) : t.size(1);
}

static std::tuple<Tensor, Tensor, Tensor> verify_tree(const Tensor& target, const Tensor& tokens, const Tensor& parents,
                                                      const Tensor& q_start, const Tensor& uniforms, int64_t max_q, const MaybeTensor& draft,
                                                      const MaybeTensor& path_, const MaybeTensor& kept_, const MaybeTensor& token_,
                                                      int64_t stream) {
    want_no_gradient({&target, &uniforms, of(draft)});
    const OnDeviceOf on(target);
    tms_verify_tree_args a{};
    a.target_stride = probabilities(target, "target: device [tokens, vocab] of float32, float16 or bfloat16, last stride 1");
    const int device = gpu_of(target);
    const int64_t T = target.size(0);
    a.target = target.const_data_ptr();
    a.dtype = dtype_code(target);
    a.vocab = i32(target.size(1));
    a.tokens = i32(T);
    if (draft) {
        want(draft->sizes() == target.sizes() && draft->scalar_type() == target.scalar_type() && gpu_of(*draft) == device, "draft: like target");
        a.draft_stride = probabilities(*draft, "draft: like target");
        a.draft = draft->const_data_ptr();
        if (T == 0) a.draft = nullptr;
    }
    a.draft_tokens = ints(tokens, {T}, "tokens", device);
    a.parents = ints(parents, {T}, "parents", device);
    want(q_start.dim() == 1 && q_start.size(0) >= 1, "q_start: int32 [batch + 1]");
    const int64_t B = q_start.size(0) - 1;
    a.batch = i32(B);
    a.q_start = ints(q_start, {B + 1}, "q_start", device);
    want(uniforms.scalar_type() == at::kDouble && uniforms.dim() == 1 && uniforms.size(0) == T && uniforms.is_contiguous() &&
             gpu_of(uniforms) == device,
         "uniforms: contiguous float64 [tokens]");
    a.uniforms = uniforms.const_data_ptr<double>();
    want(max_q >= 0, "max_q: not below 0");
    if (max_q > TMS_TREE_MAX_NODES) check(TMS_ERR_CAPACITY, "tms_verify_tree");
    a.max_q = i32(max_q);
    const Tensor path = path_ ? *path_ : at::empty({B, max_q}, tokens.options());
    const Tensor kept = kept_ ? *kept_ : at::empty({B}, tokens.options());
    const Tensor token = token_ ? *token_ : at::empty({B}, tokens.options());
    a.path = const_cast<int32_t*>(ints(path, {B, max_q}, "path", device));
    a.kept = const_cast<int32_t*>(ints(kept, {B}, "kept", device));
    a.token = const_cast<int32_t*>(ints(token, {B}, "token", device));
    for (const MaybeTensor* t : {&path_, &kept_, &token_})
        if (*t) want_separate(**t, {&target, &tokens, &parents, &q_start, &uniforms, of(draft)}, "path, kept, token: share memory with what the call reads");
    const char* apart = "path, kept, token: share memory";
    if (path_) want_separate(path, {&kept, &token}, apart);
    if (kept_) want_separate(kept, {&token}, apart);
    const int64_t need = tms_verify_tree_workspace(&a);
    if (need < 0) check((int)need, "tms_verify_tree");
    Tensor workspace;
    if (need > 0) {
        workspace = at::empty({need}, tokens.options().dtype(at::kByte));
        a.workspace = workspace.data_ptr();
        a.workspace_bytes = (size_t)need;
    }
    check(tms_verify_tree(&a, stream_of(stream)), "tms_verify_tree");
    written(path_);
    written(kept_);
    written(token_);
    return {path, kept, token};
}

static Tensor kv_compact(const Tensor& k, const Tensor& v, const Tensor& tables, const Tensor& kv_len, const Tensor& kept,
                         const Tensor& n_kept, const MaybeTensor& q_start, const MaybeTensor& dst_tables, const MaybeTensor& scores,
                         const MaybeTensor& new_len_, int64_t stream) {
    want_no_gradient({&k, &v, of(scores)});
    const OnDeviceOf on(k);
    const tms_cache c = cache_of(k, &v, of(scores), tables, kv_len, of(q_start), 0, 0, 0);
    const int device = gpu_of(k);
    const int64_t B = tables.size(0);
    tms_compact_args a{};
    want(kept.dim() == 2 && kept.size(0) == B && kept.scalar_type() == at::kInt && gpu_of(kept) == device && row_contiguous(kept) &&
             (B <= 1 || kept.stride(0) >= kept.size(1)),
         "kept: int32 [batch, n] on the cache's device, rows contiguous");
    a.kept = kept.const_data_ptr<int32_t>();
    a.kept_stride = B > 1 ? kept.stride(0) : kept.size(1);
    a.max_kept = i32(kept.size(1));
    a.n_kept = ints(n_kept, {B}, "n_kept", device);
    if (dst_tables) {
        want(dst_tables->dim() == 2 && dst_tables->size(1) >= 1, "dst_tables: int32 [batch, entries]");
        a.dst_tables = ints(*dst_tables, {B, dst_tables->size(1)}, "dst_tables", device);
        a.dst_table_stride = dst_tables->size(1);
    }
    const Tensor new_len = new_len_ ? *new_len_ : at::empty({B}, tables.options());
    a.new_len = const_cast<int32_t*>(ints(new_len, {B}, "new_len", device));
    if (new_len_)
        want_separate(new_len, {&kv_len, &n_kept, &kept, &tables, of(q_start), of(dst_tables)}, "new_len: shares memory with what the call reads");
    check(tms_kv_compact(&c, &a, stream_of(stream)), "tms_kv_compact");
    written(k);
    written(v);
    written(scores);
    written(new_len_);
    return new_len;
}

PYBIND11_MODULE(_tree_ops, m) {
    m.def("rotary", &rotary);
    m.def("kv_append_rotary", &kv_append_rotary);
    m.def("tree_attention", &tree_attention);
    m.def("verify_tree", &verify_tree);
    m.def("kv_compact", &kv_compact);
}
