// Which device is current when the tree calls' Python side calls the library:
// tms_tree_py.cpp itself over a library that only notes it, and over tensors
// that say they are on cuda:1 while cuda:0 is current.  No GPU is touched.
#include <torch/extension.h>

#undef PYBIND11_MODULE
#define PYBIND11_MODULE(name, m) [[maybe_unused]] static void module_##name(py::module_& m)
#include "../../tensormark_amd/csrc/tms_tree_py.cpp"

#include <c10/core/impl/FakeGuardImpl.h>

typedef c10::impl::FakeGuardImpl<c10::DeviceType::CUDA> Fake;
static int launched_on;

static int note() {
    launched_on = Fake::getDeviceIndex();
    return TMS_OK;
}

extern "C" {
const char* tms_status_string(int) { return ""; }
int tms_rotary(const tms_rotary_args*, hipStream_t) { return note(); }
int tms_kv_append_rotary(const tms_cache*, const tms_append_rotary_args*, hipStream_t) { return note(); }
int64_t tms_tree_attention_workspace(const tms_cache*, const tms_attention_args*) { return 0; }
int tms_tree_attention(const tms_cache*, const tms_attention_args*, const int32_t*, hipStream_t) { return note(); }
int64_t tms_verify_tree_workspace(const tms_verify_tree_args*) { return 0; }
int tms_verify_tree(const tms_verify_tree_args*, hipStream_t) { return note(); }
int tms_kv_compact(const tms_cache*, const tms_compact_args*, hipStream_t) { return note(); }
}

// A tensor of memory of its own.
static Tensor there(at::IntArrayRef sizes, at::ScalarType type) {
    static char memory[1 << 20];
    static size_t used;
    char* at = memory + used;
    used += 1 << 14;
    const c10::Device device(c10::DeviceType::CUDA, 1);
    return at::for_blob(at, sizes).options(at::device(device).dtype(type)).target_device(device).make_tensor();
}

// The device that each of the five calls launched on, and the one that was current after it.
extern "C" void tree_devices(int* launched, int* after) {
    static const Fake fake;
    c10::impl::device_guard_impl_registry[(size_t)c10::DeviceType::CUDA].store(&fake);
    const Tensor k = there({2, 1, 16, 64}, at::kHalf), v = there({2, 1, 16, 64}, at::kHalf), q = there({1, 2, 64}, at::kHalf);
    const Tensor kn = there({1, 1, 64}, at::kHalf), lse = there({1, 2}, at::kFloat), tables = there({1, 2}, at::kInt);
    const Tensor len = there({1}, at::kInt), starts = there({2}, at::kInt), one = there({1}, at::kInt), kept = there({1, 1}, at::kInt);
    const Tensor freqs = there({32}, at::kFloat), target = there({1, 100}, at::kFloat), u = there({1}, at::kDouble);
    const Tensor n1 = there({1}, at::kInt), n2 = there({1}, at::kInt), n3 = there({1}, at::kInt);
    for (int call = 0; call < 5; ++call) {
        launched_on = -1;
        Fake::setDeviceIndex(0);
        if (call == 0) rotary(q, one, freqs, false, 1.0, q, 0);
        if (call == 1) kv_append_rotary(q, kn, kn, k, v, tables, len, starts, {}, freqs, 1, false, 1.0, {}, q, 0);
        if (call == 2) tree_attention(q, k, v, tables, len, starts, one, 1, 16, 0, 0, {}, q, lse, 0);
        if (call == 3) verify_tree(target, one, one, starts, u, 1, {}, kept, n1, n2, 0);
        if (call == 4) kv_compact(k, v, tables, len, kept, n1, {}, {}, {}, n3, 0);
        launched[call] = launched_on;
        after[call] = Fake::getDeviceIndex();
    }
}
