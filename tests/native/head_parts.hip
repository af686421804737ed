// Reads "type rows classes width" lines and prints after each, for the gradients of a cross entropy of that
// size, its launches in order: "dx+8" writes eight partial sums of dX (0: the result itself), "dx=8" adds up
// eight; "dw" likewise; and how many arrays reach out of the workspace. Host code only: nothing is launched.
#include <hip/hip_runtime.h>
#include <stdio.h>

#include <vector>

namespace note {
void launch(...);
}
#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) ::note::launch(__VA_ARGS__)
#define hipGetLastError() hipSuccess
#undef __global__
#undef __launch_bounds__
#define __launch_bounds__(...)
#define __global__ __device__  // kernels are not registered: there is no device code

#include "mg/device/common.h"
namespace mg {
namespace dev {
struct HeadArgs;
struct HeadScales;
struct AmaxArgs;
struct PrepareArgs;
struct PrepareScales;
struct SmallArgs;
}  // namespace dev
}  // namespace mg
namespace note {
void launch(const mg::dev::HeadArgs&);
void launch(const mg::dev::AmaxArgs&, const mg::dev::AmaxArgs&, const mg::dev::AmaxArgs&);
void launch(const mg::dev::PrepareArgs&, const mg::dev::PrepareArgs&, const mg::dev::PrepareScales&);
void launch(const mg::dev::SmallArgs&);
template <class... A>
void launch(const float*, const float*, const int32_t*, A...) {}  // the forward pass's join
template <class T>
void launch(const float* parts, uint32_t count, uint32_t rows, uint32_t cols, uint32_t ld, T*, uint64_t,
            const mg::dev::HeadScales*, uint32_t which);
template <class T>
void launch(std::nullptr_t, uint32_t, uint32_t, uint32_t, uint32_t, T*, uint64_t, std::nullptr_t, uint32_t) {}
template <class T>
void launch(const float* parts, uint32_t count, uint32_t rows, uint32_t cols, uint32_t ld, T* out, uint64_t out_ld,
            std::nullptr_t, uint32_t which) {
    launch(parts, count, rows, cols, ld, out, out_ld, (const mg::dev::HeadScales*)nullptr, which);
}
}  // namespace note

#include "../../metalgym_amd/csrc/cross_entropy.hip"

namespace mg {
int set_error(int code, const char*, ...) { return code; }
}  // namespace mg

namespace {
uint64_t space_bytes;
uint32_t outside;
void touched(const void* p, uint64_t bytes) {
    if (p && (uint64_t)(uintptr_t)p - 4096 + bytes > space_bytes) ++outside;
}
void part(uint32_t which, uint32_t launched, const float* parts, uint64_t floats) {
    printf(" %s+%u", which ? "dw" : "dx", parts ? launched : 0);
    touched(parts, 4 * floats);
}
}  // namespace

namespace note {
void launch(const mg::dev::HeadArgs& a) {
    for (const auto& p : a.p) {
        if (!p.out || p.b.base != a.g) continue;
        if (&p == &a.p[1] && a.p[0].which) continue;  // one product alone
        const uint32_t sums = p.low ? 2 * p.splits : p.splits;
        part(p.which, sums, p.parts, (uint64_t)sums * (p.low ? a.rows : p.n) * p.parts_ld);
    }
    touched(a.g, 2ull * a.rows_ld * a.g_ld);
}
void launch(const mg::dev::AmaxArgs&, const mg::dev::AmaxArgs&, const mg::dev::AmaxArgs&) {}
void launch(const mg::dev::PrepareArgs& x, const mg::dev::PrepareArgs& w, const mg::dev::PrepareScales&) {
    const uint32_t size = x.to_even ? 4 : 2;
    touched(x.to, (uint64_t)size * x.rows * x.wide), touched(w.to, (uint64_t)size * w.rows * w.wide);
}
void launch(const mg::dev::SmallArgs& a) {  // the logits' launch, then the gradients', of the same arguments
    part(0, (a.classes + a.range - 1) / a.range, a.parts_x,
         (uint64_t)((a.classes + a.range - 1) / a.range) * a.rows * a.parts_ld);
    part(1, (a.rows + a.range - 1) / a.range, a.parts_w,
         (uint64_t)((a.rows + a.range - 1) / a.range) * a.classes * a.parts_ld);
}
template <class T>
void launch(const float* parts, uint32_t count, uint32_t rows, uint32_t, uint32_t ld, T*, uint64_t,
            const mg::dev::HeadScales*, uint32_t which) {
    printf(" %s=%u", which ? "dw" : "dx", count);
    touched(parts, 4ull * count * rows * ld);
}
}  // namespace note

int main() {
    uint32_t type, rows, classes, width;
    while (scanf("%u %u %u %u", &type, &rows, &classes, &width) == 4) {
        mg_cross_entropy_backward_args p{};
        char* const some = reinterpret_cast<char*>(uintptr_t(1) << 50);  // never read
        p.x = p.w = p.dx = p.dw = some;
        p.targets = reinterpret_cast<int32_t*>(some);
        p.lse = p.dloss = reinterpret_cast<float*>(some);
        p.x_ld = p.w_ld = p.dx_ld = p.dw_ld = width;
        p.rows = rows, p.classes = classes, p.width = width, p.type = type;
        p.workspace = reinterpret_cast<void*>(4096);
        if (mg_cross_entropy_backward_workspace(rows, classes, width, type, &space_bytes)) return 1;
        outside = 0;
        printf("%u %u %u %u:", type, rows, classes, width);
        const int rc = type == MG_TYPE_FP32   ? mg::cross_entropy_backward<float>(nullptr, p)
                       : type == MG_TYPE_BF16 ? mg::cross_entropy_backward<__bf16>(nullptr, p)
                                              : mg::cross_entropy_backward<_Float16>(nullptr, p);
        if (rc) return 1;
        printf(" outside %u\n", outside);
    }
    return 0;
}
