// Which device is current when the cache calls' Python side calls the library:
// tms_cache_py.cpp itself over a library that only notes it, and over tensors
// that say they are on cuda:1 while cuda:0 is current.  No GPU is touched.
#include <torch/extension.h>

#undef PYBIND11_MODULE
#define PYBIND11_MODULE(name, m) [[maybe_unused]] static void module_##name(py::module_& m)
#include "../../tensormark_amd/csrc/tms_cache_py.cpp"

#include <c10/core/impl/FakeGuardImpl.h>

typedef c10::impl::FakeGuardImpl<c10::DeviceType::CUDA> Fake;
static int launched_on;

static int note() {
    launched_on = Fake::getDeviceIndex();
    return TMS_OK;
}

extern "C" {
const char* tms_status_string(int) { return ""; }
int tms_kv_append(const tms_cache*, const tms_append_args*, hipStream_t) { return note(); }
int64_t tms_paged_attention_workspace(const tms_cache*, const tms_attention_args*) { return 0; }
int tms_paged_attention(const tms_cache*, const tms_attention_args*, hipStream_t) { return note(); }
int tms_kv_add_scores(const tms_cache*, const tms_score_args*, hipStream_t) { return note(); }
int tms_kv_evict(const tms_cache*, const tms_evict_args*, hipStream_t) { return note(); }
int tms_adjust_logits(const tms_adjust_args*, hipStream_t) { return note(); }
}

static Tensor there(at::IntArrayRef sizes, at::ScalarType type) {
    static char memory[1 << 16];
    const c10::Device device(c10::DeviceType::CUDA, 1);
    return at::for_blob(memory, sizes).options(at::device(device).dtype(type)).target_device(device).make_tensor();
}

// The device that each of the five calls launched on, and the one that was current after it.
extern "C" void cache_devices(int* launched, int* after) {
    static const Fake fake;
    c10::impl::device_guard_impl_registry[(size_t)c10::DeviceType::CUDA].store(&fake);
    const Tensor k = there({2, 1, 16, 64}, at::kHalf), q = there({1, 2, 64}, at::kHalf), kn = there({1, 1, 64}, at::kHalf);
    const Tensor scores = there({2, 1, 16}, at::kFloat), lse = there({1, 2}, at::kFloat), tables = there({1, 2}, at::kInt);
    const Tensor len = there({1}, at::kInt), starts = there({2}, at::kInt), kept = there({1, 1, 8}, at::kInt);
    const Tensor logits = there({1, 100}, at::kFloat);
    for (int call = 0; call < 5; ++call) {
        launched_on = -1;
        Fake::setDeviceIndex(0);
        if (call == 0) kv_append(kn, kn, k, k, tables, len, starts, 1, scores, 0);
        if (call == 1) paged_attention(q, k, k, tables, len, starts, 1, 16, 0, 0, {}, q, lse, 0);
        if (call == 2) kv_add_scores(q, lse, k, scores, tables, len, starts, 1, 16, 0, 0, {}, {}, 0);
        if (call == 3) kv_evict(k, k, scores, tables, len, tables, 8, 16, 0, 0, len, kept, 0);
        if (call == 4) adjust_logits(logits, {}, {}, {}, {}, 1, {}, {}, {}, logits, 0);
        launched[call] = launched_on;
        after[call] = Fake::getDeviceIndex();
    }
}
