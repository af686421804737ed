// Reads "steps seqs channels states groups backward" lines and prints how the selective scan goes about each:
// "channels of a quad (0: no quads), workgroups of a group, splits". Host code only.
#include <hip/hip_runtime.h>
#include <stdio.h>

#undef hipLaunchKernelGGL
#define hipLaunchKernelGGL(...) ((void)0)
#define hipGetLastError() hipSuccess
#undef __global__
#undef __launch_bounds__
#define __launch_bounds__(...)
#define __global__ __device__  // kernels are not registered: there is no device code

#include "../../metalgym_amd/csrc/selective_scan.hip"

namespace mg {
int set_error(int code, const char*, ...) { return code; }
}  // namespace mg

int main() {
    uint32_t steps, seqs, channels, states, groups, backward;
    while (scanf("%u %u %u %u %u %u", &steps, &seqs, &channels, &states, &groups, &backward) == 6) {
        const mg::ScanShape s = mg::scan_shape(steps, seqs, channels, states, groups, false, backward);
        printf("%u %u %u\n", s.wide, s.apiece, s.splits);
    }
    return 0;
}
