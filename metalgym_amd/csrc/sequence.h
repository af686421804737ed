// What the operators over rollouts share (causal convolution, selective scan): rows of
// (step, sequence), their checks, and sums of partial results.
#pragma once
#include "operator_types.h"

namespace mg {
namespace dev {

// Rows of steps x seqs: step t of sequence n is row t step_rows + n seq_rows. A sequence
// is as long as lengths says, at most steps; reset holds a byte a row.
struct Rollout {
    const uint8_t* reset;
    const uint32_t* lengths;
    uint64_t step_rows, seq_rows;
    uint32_t steps, seqs;

    __device__ __forceinline__ uint64_t row(uint32_t t, uint32_t n) const { return t * step_rows + n * seq_rows; }
    __device__ __forceinline__ uint32_t length(uint32_t n) const {
        if (!lengths) return steps;
        const uint32_t l = ((const __attribute__((address_space(4))) uint32_t*)lengths)[n];  // nobody writes it meanwhile
        return l < steps ? l : steps;
    }
};

// 1 / (1 + e^-v) and 1 minus it, neither as a difference of nearly equal numbers.
__device__ __forceinline__ void sigmoid_of(float v, float& s, float& rest) {
    const float t = __builtin_amdgcn_exp2f(-1.44269504f * __builtin_fabsf(v));
    const float r = __builtin_amdgcn_rcpf(1.0f + t), tr = t * r;
    s = v >= 0.0f ? r : tr;
    rest = v >= 0.0f ? tr : r;
}
// v / (1 + e^-v): 0 where the exponential leaves fp32's range.
__device__ __forceinline__ float silu(float v) {
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * v));
}
__device__ __forceinline__ float silu_slope(float v) {
    float s, rest;
    sigmoid_of(v, s, rest);
    return s * (1.0f + v * rest);
}

// log(1 + e^v) = max(v, 0) + log(1 + t), t = e^-|v|. A small t is the whole of the result for
// negative v: e^-|v| takes its argument's rounding along, and the logarithm what 1 + t lost of t.
__device__ __forceinline__ float softplus(float v) {
    const float u = __builtin_fmaxf(-__builtin_fabsf(v), -200.0f);
    const float hi = u * 1.44269504f;
    const float lo = __builtin_fmaf(u, 1.92596299e-8f, __builtin_fmaf(u, 1.44269504f, -hi));
    float t = __builtin_amdgcn_exp2f(hi);
    t = __builtin_fmaf(t, lo * 0.693147181f, t);
    const float w = 1.0f + t;
    const float l = __builtin_fmaf(__builtin_amdgcn_logf(w), 0.693147181f, t - (w - 1.0f));
    const float r = __builtin_fmaxf(v, 0.0f) + l;
    return v != v ? v : r;
}

// Where the sums of partial rows go: columns [0, end[0]) to to[0], up to end[1] to to[1],
// and so on; a null array takes none.
struct SumTargets {
    float* to[3];
    uint64_t end[3];
};

// Adds `parts` partial rows of `width` columns: 32 columns a workgroup, 32 slices of the
// rows, each added in order, then the slices in order. Without parts the sums are 0.
static __global__ void __launch_bounds__(1024) sum_parts_kernel(const float* __restrict__ partial, uint32_t parts,
                                                               uint64_t width, const SumTargets out) {
    __shared__ float lds[32][33];
    const uint32_t lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    for (uint64_t c0 = (uint64_t)blockIdx.x * 32; c0 < width; c0 += (uint64_t)gridDim.x * 32) {
        const uint64_t c = c0 + lane;
        float s = 0.0f;
        if (c < width) {
#pragma unroll 8
            for (uint32_t p = slice; p < parts; p += 32) s += partial[p * width + c];
        }
        __syncthreads();
        lds[slice][lane] = s;
        __syncthreads();
        if (slice == 0 && c < width) {
            s = lds[0][lane];
#pragma unroll
            for (int k = 1; k < 32; ++k) s += lds[k][lane];
            const int k = c < out.end[0] ? 0 : c < out.end[1] ? 1 : 2;
            float* const to = k == 0 ? out.to[0] : k == 1 ? out.to[1] : out.to[2];
            if (to) to[c - (k == 0 ? 0 : out.end[k - 1])] = s;
        }
    }
}

}  // namespace dev

constexpr uint32_t kCus = 256;

// The checks that every call over a rollout makes; step_rows and seq_rows 0 stand for
// [steps][seqs] rows and are filled in.
inline int check_rollout(const char* what, uint32_t steps, uint32_t seqs, uint32_t channels, uint32_t type,
                         uint64_t* step_rows, uint64_t* seq_rows, const void* lengths) {
    MG_CHECK(type_known(type), MG_ERR_INVALID, "%s: unknown type %u", what, type);
    MG_CHECK(channels >= 1 && channels <= 65536, MG_ERR_INVALID, "%s: channels %u must be in [1, 65536]", what,
             channels);
    MG_CHECK(steps <= (1u << 30) && seqs <= (1u << 30), MG_ERR_INVALID, "%s: steps and seqs must be at most 2^30",
             what);
    if (!*step_rows && !*seq_rows) *step_rows = seqs, *seq_rows = 1;
    MG_CHECK(*step_rows <= (1ull << 32) && *seq_rows <= (1ull << 32), MG_ERR_INVALID,
             "%s: step_rows and seq_rows must be at most 2^32", what);
    // rows are apart where one of the two strides passes over all rows of the other
    const bool steps_inside = steps <= 1 || (*step_rows >= 1 && (seqs <= 1 || *seq_rows > *step_rows * (steps - 1)));
    const bool seqs_inside = seqs <= 1 || (*seq_rows >= 1 && (steps <= 1 || *step_rows > *seq_rows * (seqs - 1)));
    MG_CHECK(steps_inside || seqs_inside, MG_ERR_INVALID, "%s: rows of step_rows %llu and seq_rows %llu overlap", what,
             (unsigned long long)*step_rows, (unsigned long long)*seq_rows);
    MG_CHECK(aligned(lengths, 4), MG_ERR_INVALID, "%s: lengths is not aligned to its type", what);
    return MG_OK;
}

// One operand of `cols` elements a row: its pointer, alignment and row stride (0: cols).
inline int check_operand(const char* what, const char* name, const void* p, uint64_t* ld, uint64_t cols, uint32_t type,
                         bool any) {
    if (!*ld) *ld = cols;
    MG_CHECK(p || !any, MG_ERR_INVALID, "%s: %s is NULL", what, name);
    MG_CHECK(aligned(p, type_bytes(type)), MG_ERR_INVALID, "%s: %s is not aligned to its type", what, name);
    MG_CHECK(*ld >= cols && *ld <= (1ull << 24), MG_ERR_INVALID, "%s: %s_ld %llu must be in [%llu, 2^24]", what, name,
             (unsigned long long)*ld, (unsigned long long)cols);
    return MG_OK;
}
inline int check_vector(const char* what, const char* name, const void* p, uint32_t type, bool required) {
    MG_CHECK(p || !required, MG_ERR_INVALID, "%s: %s is NULL", what, name);
    MG_CHECK(aligned(p, type_bytes(type)), MG_ERR_INVALID, "%s: %s is not aligned to its type", what, name);
    return MG_OK;
}
inline int check_workspace(const char* what, const void* p, uint64_t bytes, uint64_t need) {
    MG_CHECK(bytes >= need && (p || !need), MG_ERR_INVALID, "%s: the workspace needs %llu bytes", what,
             (unsigned long long)need);
    MG_CHECK(!need || aligned(p, 256), MG_ERR_INVALID, "%s: the workspace is not 256-byte aligned", what);
    return MG_OK;
}

inline int sum_parts(hipStream_t st, const float* partial, uint32_t parts, uint64_t width, const dev::SumTargets& out,
                     const char* what) {
    const uint64_t blocks = (width + 31) / 32;
    hipLaunchKernelGGL(dev::sum_parts_kernel, dim3((uint32_t)(blocks < 65536 ? blocks : 65536)), dim3(1024), 0, st,
                       partial, parts, width, out);
    MG_HIP(hipGetLastError(), what);
    return MG_OK;
}

}  // namespace mg
