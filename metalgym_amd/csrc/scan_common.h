// What the selective scan's kernels share: their arguments, a lane's four states, sums over
// a wave's channels.
#pragma once
#include "mg/device/common.h"
#include "sequence.h"

namespace mg {
namespace dev {

constexpr int kSteps = 8;   // of a round between barriers
constexpr int kChunk = 64;  // steps between the kept states
constexpr int kSubs = kChunk / kSteps;
constexpr float kLog2e = 1.44269504f;

struct ScanArgs {
    Rollout at;
    const void* x;
    const void* dt;
    const void* b;
    const void* c;
    const void* z;
    void* y;
    const float* a;
    const float* d;
    const float* dt_bias;
    const float* initial;
    float* final;
    float* checkpoints;
    // the backward pass's
    const void* dy;
    const float* kept;
    const float* dfinal;
    void* dx;
    void* ddt;
    void* db;
    void* dc;
    void* dz;
    float* dinitial;
    float* sums;     // [parts][channels (states + 2)]: dA, dD, ddt_bias
    float* shared;   // [blocks of a group][steps seqs][groups][2][states]: parts of dB and dC
    // of each split but the last (the first, backwards), from a state of zero
    float* ends;     // [splits][seqs][channels][states]
    float* decays;   // [splits][seqs][channels]: the sum of delta, or -1 where an episode begins
    float* saved;    // the initial state, as the final one may take its place
    uint64_t x_ld, dt_ld, b_ld, c_ld, z_ld, y_ld, dy_ld, dx_ld, ddt_ld, db_ld, dc_ld, dz_ld;
    uint32_t channels, states, groups;
    uint32_t per;     // channels of a group
    uint32_t apiece;  // blocks of a group
    uint32_t blocks;  // of all channels
    uint32_t splits, split_steps;
};

// An element on its way, in a register of its own. Two of 16 bits that share one wait for their loads as
// they are put together, and a round's then do not come under the round before: 32 steps of 4096 x 256
// with 16 states, bf16, took 167 us for 161, the gradients 725 for 611.
template <class T>
struct Raw {
    uint32_t bits;
    __device__ __forceinline__ operator float() const {
        if constexpr (sizeof(T) == 2)
            return (float)__builtin_bit_cast(T, (uint16_t)bits);
        else
            return __builtin_bit_cast(T, bits);
    }
};
template <class T>
__device__ __forceinline__ Raw<T> raw_at(const T* p) {
    if constexpr (sizeof(T) == 2)
        return Raw<T>{__builtin_bit_cast(uint16_t, *p)};
    else
        return Raw<T>{__builtin_bit_cast(uint32_t, *p)};
}
// Keeps the conversions of a round's elements behind this point.
template <class T, int R>
__device__ __forceinline__ void arrive(Raw<T> (&v)[R]) {
#pragma unroll
    for (int j = 0; j < R; ++j) asm volatile("" : "+v"(v[j].bits));
}

// Four consecutive states of a channel; past `count` 0, or not written.
__device__ __forceinline__ f32x4 load_states(const float* p, int count) {
    typedef float near __attribute__((ext_vector_type(4), aligned(4)));
    if (count >= 4) return *reinterpret_cast<const near*>(p);
    f32x4 v = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < count) v[i] = p[i];
    return v;
}
__device__ __forceinline__ void store_states(float* p, int count, f32x4 v) {
    typedef float near __attribute__((ext_vector_type(4), aligned(4)));
    if (count >= 4) {
        *reinterpret_cast<near*>(p) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < count) p[i] = v[i];
}

// A in base 2. A rate of -infinity is fp32's lowest value: a step of delta 0 (past the end, or a split that is empty)
// then leaves the state as it is, and not NaN.
__device__ __forceinline__ f32x4 base2_of(f32x4 a) {
    f32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = a[i] * kLog2e;
        r[i] = r[i] < -3.402823466e38f ? -3.402823466e38f : r[i];
    }
    return r;
}
__device__ __forceinline__ f32x4 decay_of(f32x4 a2, float delta) {
    f32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_exp2f(a2[i] * delta);
    return r;
}

// States to 0, in a branch of its own: as selects that every step makes it would be an
// eighth of the instructions.
__device__ __forceinline__ void clear_states(f32x4& h) {
    asm volatile("");
    h = f32x4{};
}
template <int C>
__device__ __forceinline__ void clear_states(f32x4 (&h)[C]) {
    asm volatile("");
#pragma unroll
    for (int c = 0; c < C; ++c) h[c] = f32x4{};
}

// The items of a launch: (split, sequence, block of channels), the last fastest.
struct ScanItem {
    uint32_t block, n, split;
    __device__ __forceinline__ ScanItem(const ScanArgs& p, uint64_t item) {
        const uint64_t rest = item / p.blocks;
        block = (uint32_t)(item - rest * p.blocks);
        split = (uint32_t)(rest / p.at.seqs);
        n = (uint32_t)(rest - (uint64_t)split * p.at.seqs);
    }
};

// Of each pair (v[2 q], v[2 q + 1]), of which lanes l and l ^ X hold one part each: the lower
// lanes' sum of the first, the upper lanes' of the second. One wait for all N swaps.
template <int X, int N>
__device__ __forceinline__ void swap_add(const float (&v)[2 * N], float (&w)[N]) {
    static_assert((X == 16 && N == 2) || (X == 32 && N == 4), "the two steps of sum_channels");
    float a[N], b[N];
#pragma unroll
    for (int q = 0; q < N; ++q) a[q] = v[2 * q], b[q] = v[2 * q + 1];
    if constexpr (X == 16)
        asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %2\n\tv_permlane16_swap_b32 %1, %3"
            : "+v"(a[0]), "+v"(a[1]), "+v"(b[0]), "+v"(b[1]));
    else
        asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %4\n\tv_permlane32_swap_b32 %1, %5\n\t"
            "v_permlane32_swap_b32 %2, %6\n\tv_permlane32_swap_b32 %3, %7"
            : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(b[0]), "+v"(b[1]), "+v"(b[2]), "+v"(b[3]));
#pragma unroll
    for (int q = 0; q < N; ++q) w[q] = a[q] + b[q];
}

// Sums of eight values (four states of dB, then of dC) over a wave's channels: each pair
// of values shares a register from the swaps on. Writes them to LDS, [2][SP].
template <int L, int SP = 4 * L>
__device__ __forceinline__ void sum_channels(const float (&v)[8], float* to) {
    const int lane = threadIdx.x & 63, s = 4 * (lane % L);
    if constexpr (L == 64) {
#pragma unroll
        for (int q = 0; q < 8; ++q) to[(q >> 2) * SP + s + (q & 3)] = v[q];
        return;
    }
    float w[4];
    swap_add<32>(v, w);
    const int upper = lane >> 5;
    if constexpr (L == 32) {
#pragma unroll
        for (int q = 0; q < 4; ++q) to[(q >> 1) * SP + s + 2 * (q & 1) + upper] = w[q];
        return;
    }
    float r[2];
    swap_add<16>(w, r);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        if constexpr (L <= 8) r[q] += dpp_lane<0x128>(r[q]);  // row_ror 8, 4, 2, 1
        if constexpr (L <= 4) r[q] += dpp_lane<0x124>(r[q]);
        if constexpr (L <= 2) r[q] += dpp_lane<0x122>(r[q]);
        if constexpr (L <= 1) r[q] += dpp_lane<0x121>(r[q]);
    }
    if ((lane & 15) < L) {
        const int i = s + 2 * (lane >> 4 & 1) + upper;
        to[i] = r[0], to[SP + i] = r[1];
    }
}

}  // namespace dev
}  // namespace mg
