// Argument checks of the C++ entries of the experts' products (no GPU needed):
// prints "case: message" for each refused call.  No pointer passed here is ever
// dereferenced: each call fails a check, and a product that passed them all
// would ask this file for the number of SMs before its launch.
#include <cstdint>
#include <cstdio>
#include <functional>
#include <string>

#include "kiwi/common.hpp"
#include "kiwi/gemm/fp8_gemm.hpp"
#include "kiwi/gemm/grouped_gemm.hpp"
#include "kiwi/gemm/grouped_linear.hpp"
#include "kiwi/ops/swiglu.hpp"

namespace kiwi::gemm {
int num_sms() { throw kiwi::error("accepted"); }
}  // namespace kiwi::gemm

namespace {

template <typename T>
T* at(uintptr_t address) {
    return reinterpret_cast<T*>(address);
}

constexpr uintptr_t kBase = 1 << 20;  // 16-byte aligned, never dereferenced

kiwi::gemm::Fp8GemmArgs fp8_args() {
    kiwi::gemm::Fp8GemmArgs a{};
    a.a = at<uint8_t>(kBase);
    a.lda = 256;
    a.b = at<uint8_t>(kBase);
    a.ldb = 256;
    a.a_scale = at<float>(kBase);
    a.a_scale_stride = 2;
    a.b_scale = at<float>(kBase);
    a.counts = at<int32_t>(kBase);
    a.num_groups = 2;
    a.n = 256;
    a.k = 256;
    a.rows = 8;
    a.c = at<__nv_bfloat16>(kBase);
    a.ldc = 256;
    return a;
}

void report(const char* name, const std::function<void()>& call) {
    try {
        call();
        std::printf("%s: returned\n", name);
    } catch (const std::exception& e) {
        std::printf("%s: %s\n", name, e.what());
    }
}

void fp8(const char* name, const std::function<void(kiwi::gemm::Fp8GemmArgs&)>& change) {
    kiwi::gemm::Fp8GemmArgs a = fp8_args();
    change(a);
    report(name, [&] { kiwi::gemm::fp8_gemm(a, nullptr); });
}

void linear(const char* name, void (*entry)(const kiwi::gemm::GroupedLinearArgs&, cudaStream_t),
            const std::function<void(kiwi::gemm::GroupedLinearArgs&)>& change) {
    kiwi::gemm::GroupedLinearArgs a{};
    a.x = a.w = a.dy = at<__nv_bfloat16>(kBase);
    a.ldx = a.ldw = a.lddy = a.ldo = 256;
    a.out = at<void>(kBase);
    a.counts = at<int32_t>(kBase);
    a.num_groups = 2;
    a.n = 256;
    a.k = 256;
    a.rows = 8;
    change(a);
    report(name, [&] { entry(a, nullptr); });
}

/// Both directions of SwiGLU; the backward's dh has y's base and a row stride to match.
void swiglu(const char* name, uintptr_t y, int64_t ldy, uintptr_t out, int ffn) {
    report(name, [&] {
        kiwi::ops::swiglu_forward(at<__nv_bfloat16>(y), ldy, nullptr, at<__nv_bfloat16>(out), 8, ffn, nullptr);
    });
    report((std::string(name) + " backward").c_str(), [&] {
        kiwi::ops::swiglu_backward(at<__nv_bfloat16>(y), ldy, at<__nv_bfloat16>(y), ldy, nullptr,
                                   at<__nv_bfloat16>(out), nullptr, 8, ffn, nullptr);
    });
}

}  // namespace

int main() {
    fp8("fp8 groups without counts", [](auto& a) { a.counts = nullptr; });
    fp8("fp8 no groups", [](auto& a) { a.num_groups = 0; });
    fp8("fp8 no output", [](auto& a) { a.c = nullptr; });
    fp8("fp8 k", [](auto& a) { a.k = 250; });
    fp8("fp8 large k", [](auto& a) { a.k = INT32_MAX - 15; });
    linear("forward large k", kiwi::gemm::grouped_linear_forward, [](auto& a) { a.k = INT32_MAX - 63; });
    linear("dgrad large k", kiwi::gemm::grouped_linear_dgrad, [](auto& a) { a.k = INT32_MAX - 63; });
    linear("forward unaligned rows", kiwi::gemm::grouped_linear_forward, [](auto& a) {
        a.out_fp32 = true;  // of no effect: y is bf16
        a.ldo = 260;
    });
    linear("wgrad unaligned rows", kiwi::gemm::grouped_linear_wgrad, [](auto& a) { a.ldo = 260; });
    linear("wgrad large k", kiwi::gemm::grouped_linear_wgrad, [](auto& a) { a.k = INT32_MAX - 63; });
    swiglu("swiglu columns", kBase, 512, kBase, 192);
    swiglu("swiglu no columns", kBase, 512, kBase, 0);
    swiglu("swiglu row stride", kBase, 516, kBase, 256);
    swiglu("swiglu short rows", kBase, 504, kBase, 256);
    swiglu("swiglu input base", kBase + 8, 512, kBase, 256);
    swiglu("swiglu output base", kBase, 512, kBase + 2, 256);
    swiglu("swiglu missing input", 0, 512, kBase, 256);
    swiglu("swiglu missing output", kBase, 512, 0, 256);
    return 0;
}
