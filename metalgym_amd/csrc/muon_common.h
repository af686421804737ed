// What both Newton-Schulz paths (muon.hip, muon_short.h) share: batches of matrices
// of any type, the matrix that is orthogonalised, and the operands' pairs.
#pragma once
#include <math.h>

#include <type_traits>

#include "kernels.h"
#include "mg/device/common.h"
#include "operator_types.h"

namespace mg {
namespace dev {

typedef _Float16 f16;
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Exponents of the operands' pairs: X and A at most 2 and 4 in size, P at most
// 64, so that 2^13 and 2^9 keep them under 2^15, half of binary16's range.
constexpr float kUnitX = 8192.0f, kUnitA = 8192.0f, kUnitP = 512.0f;

// X's pairs hold 2^extra_exp more where its singular values are known to be small, so
// that a matrix whose norm is far under eps keeps its bits: most = share x growth, share =
// |U| / (|U| + eps), which X starts at, and growth what its steps so far may have made of
// that, the product of their largest |a + b s^2 + c s^4| (an odd polynomial of degree 5
// that takes [-r, r] to [-r', r'] has p(s) / s at most 5 r' / r, so it is at most 2 5^32,
// well inside fp32). Where most is not under a half nothing changes. At a fixed exponent, the result was
// off by 1e-4 of itself at a share of 1e-5, and nothing was left of it at 1e-13.
__device__ __forceinline__ int extra_exp(float most) {
    if (!(most > 0.0f && most < 0.5f)) return 0;
    const int e = -1 - ilogbf(most);
    return e < 100 ? e : 100;
}

// x f = hi + lo to 22 bits. The product is made one value first: the compiler otherwise
// rounds it to binary16 in one step for hi (v_fma_mixlo_f16) and to fp32 for lo, and where
// the two roundings fall on different sides of a tie, hi and lo are off by a step of hi.
__device__ __forceinline__ void split4(const float (&x)[4], float f, f16x4& hi, f16x4& lo) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float y = x[e] * f;
        asm("" : "+v"(y));
        v[e] = y;
    }
    hi = __builtin_convertvector(v, f16x4);
    lo = __builtin_convertvector(v - __builtin_convertvector(hi, f32x4), f16x4);
}

// A batch of matrices of any type as a kernel reads or writes it.
struct Batch {
    void* data;
    size_t stride;
    uint32_t ld;
    uint32_t type;
    __device__ __forceinline__ size_t at(uint32_t k, uint32_t i, uint32_t j) const {
        return k * stride + (uint64_t)i * ld + j;
    }
};
// f(a value of the type's T)
template <class F>
__device__ __forceinline__ void with_type(uint32_t type, F&& f) {
    switch (type) {
        case MG_TYPE_FP32: return f(float{});
        case MG_TYPE_BF16: return f(__bf16{});
        default: return f(f16{});
    }
}
// A lane's N = 16 elements of a 32 x 32 tile as the matrix instructions leave them, or
// 8 of 16 rows:
// element e lies 8 (e / 4) + e % 4 rows under y0, in column x, if the matrix (rows x
// cols) reaches there.
template <int N>
__device__ __forceinline__ void tile_read(const Batch& b, uint32_t rows, uint32_t cols, uint32_t k, uint32_t y0,
                                          uint32_t x, float (&w)[N]) {
    with_type(b.type, [&](auto t) {
        const auto* from = static_cast<const decltype(t)*>(b.data) + b.at(k, 0, x < cols ? x : 0);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t y = y0 + 2 * (e & ~3) + (e & 3);
            w[e] = (float)from[(uint64_t)(y < rows ? y : rows - 1) * b.ld];
        }
    });
}
template <int N>
__device__ __forceinline__ void tile_write(const Batch& b, uint32_t rows, uint32_t cols, uint32_t k, uint32_t y0,
                                           uint32_t x, const float (&w)[N]) {
    if (x >= cols) return;
    with_type(b.type, [&](auto t) {
        using T = decltype(t);
        T* const to = static_cast<T*>(b.data) + b.at(k, 0, x);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t y = y0 + 2 * (e & ~3) + (e & 3);
            if (y < rows) to[(uint64_t)y * b.ld] = (T)w[e];
        }
    });
}

// What is orthogonalised: `in`, or with a momentum batch the Muon update's U from
// the gradient `in`.
struct SourceArgs {
    Batch in, momentum;  // momentum.data NULL: in alone
    uint32_t rows, cols;
    float beta;
    uint32_t nesterov;
    // a policy's block matrices (short path): contiguous, the odd ones cols x rows, the
    // gradient clipped to max_norm by the partial squared norms (NULL: not clipped)
    uint32_t blocks;
    const float* normpart;
    float max_norm;
};
// model/optimizer.metal:49 from the partial norms, added as Adam adds them; every
// wave must be whole.
__device__ __forceinline__ float source_clip(const SourceArgs& a) {
    if (!a.normpart || !(a.max_norm > 0.0f)) return 1.0f;
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kReduceBlocks / 64; ++k) sum += a.normpart[(threadIdx.x & 63) + 64 * k];
    const float norm = sqrtf(group_sum<64>(sum));
    return norm > a.max_norm ? a.max_norm / (norm + 1e-6f) : 1.0f;
}
__device__ __forceinline__ float moved_momentum(const SourceArgs& a, float m, float g) {
    return m + (1.0f - a.beta) * (g - m);
}
__device__ __forceinline__ float update_of(const SourceArgs& a, float m, float g) {
    return a.nesterov ? g + a.beta * (m - g) : m;
}
}  // namespace dev
}  // namespace mg
