// The selective scan of 9 to 16 states, and of 17 to 64: four lanes a channel.
//
// A quad of lanes holds C channels, NS times four states of each a lane. What a step needs of a
// channel (delta, delta x, dy) is worked out by one lane of the quad, which does so for every
// 4 / C th step of one channel, and the others take it by a DPP move; sums over states come
// back to that lane by two more. B and C lie in LDS as fp32 for a workgroup's four waves, which
// otherwise run on their own.
#pragma once
#include "scan_common.h"

namespace mg {
namespace dev {

constexpr int kWindow = 32;  // steps of B and C in LDS

// Lane n's value in every lane of each quad; n is a constant once loops are unrolled.
__device__ __forceinline__ float quad_take(int n, float v) {
    return n == 0 ? dpp_lane<0x00>(v) : n == 1 ? dpp_lane<0x55>(v) : n == 2 ? dpp_lane<0xAA>(v) : dpp_lane<0xFF>(v);
}
// Lane n of a quad gets the quad's sum of v[n].
__device__ __forceinline__ float quad_sums(const float (&v)[4]) {
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
    const float a = (odd ? v[1] : v[0]) + dpp_lane<0xB1>(odd ? v[0] : v[1]);
    const float b = (odd ? v[3] : v[2]) + dpp_lane<0xB1>(odd ? v[2] : v[3]);
    return (high ? b : a) + dpp_lane<0x4E>(high ? a : b);
}

// How a quad's lanes share out C channels' elements.
template <int C>
struct QuadMap {
    static constexpr int P = 4 / C;       // steps that a quad's lanes take at once
    static constexpr int R = kSteps / P;  // times that they do in a round of kSteps
    // which of a round's steps the lane's element j is of
    static __device__ __forceinline__ uint32_t step(int j) { return j * P + (threadIdx.x & 3) / C; }
    // and which lane of the quad, at which j, has step k of channel c
    static __device__ __forceinline__ int lane(int k, int c) { return k % P * C + c; }
};

// A workgroup's channels, a lane's states of C of them, and the one it works for. Vector c NS + q
// of a lane holds states 16 q + 4 lane ... of channel c.
template <int C, int NS>
struct QuadLane : QuadMap<C> {
    static constexpr int CH = 64 * C;  // channels of a workgroup
    static constexpr int U = C * NS;   // vectors of a lane
    static constexpr int SP = 16 * NS;  // states, with padding
    uint32_t group, first, own;  // the quad's first channel, and this lane's
    bool in;                     // whether that is one
    int state, held[U];          // the first of the lane's states, and how many each vector has
    f32x4 a2[U];                 // A log2(e)

    __device__ __forceinline__ QuadLane(const ScanArgs& p, uint32_t block) {
        group = block / p.apiece;
        const uint32_t limit = (group + 1) * p.per;
        first = group * p.per + (block - group * p.apiece) * CH + (threadIdx.x >> 2) * C;
        own = first + threadIdx.x % C;
        in = own < limit;
        own = in ? own : limit - 1;
        state = 4 * (threadIdx.x & 3);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            held[u] = first + u / NS < limit ? (int)p.states - state - 16 * (u % NS) : 0;
            a2[u] = load_states(p.a + (size_t)(first + u / NS) * p.states + state + 16 * (u % NS), held[u]);
        }
    }
    // a2 as it is meant: apart from its loads, which the others need not wait for
    __device__ __forceinline__ void ready() {
#pragma unroll
        for (int u = 0; u < U; ++u) a2[u] = base2_of(a2[u]);
    }
    __device__ __forceinline__ size_t at(const ScanArgs& p, uint32_t n, int u) const {
        return ((size_t)n * p.channels + first + u / NS) * p.states + state + 16 * (u % NS);
    }
    __device__ __forceinline__ void load(const ScanArgs& p, const float* from, uint32_t n, f32x4 (&h)[U]) const {
#pragma unroll
        for (int u = 0; u < U; ++u) h[u] = load_states(from + at(p, n, u), held[u]);
    }
    __device__ __forceinline__ void store(const ScanArgs& p, float* to, uint32_t n, const f32x4 (&h)[U]) const {
#pragma unroll
        for (int u = 0; u < U; ++u) store_states(to + at(p, n, u), held[u], h[u]);
    }
};

// A kernel's arguments, read anew: a round's addresses are worked out from them in scalar
// registers, which held through a kernel would be twice what there are, and be spilled to vector
// registers' lanes (the gradient's round then moves a hundred of them).
typedef const __attribute__((address_space(4))) ScanArgs* ArgsAgain;
__device__ __forceinline__ ArgsAgain args_again() {
    ArgsAgain p = (ArgsAgain)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

// A lane's elements of a row array of one sequence, by buffer loads: the round's address, a
// step's distance and the lane's own bytes (the host has made sure that eight steps fit 31
// bits). As pointers each array took two registers a lane, and the backward pass kept its own
// in scratch. What is past the end or of no channel lies nowhere: it reads 0, and is not written.
template <class T, int C>
struct QuadRows {
    static constexpr uint32_t kNone = 0x80000000u;
    const char* base;
    uint32_t by;    // bytes from step to step
    uint32_t mine;  // the lane's first step and its channel
    template <int NS>
    __device__ __forceinline__ QuadRows(const ArgsAgain p, const QuadLane<C, NS>& at, const void* array, uint64_t ld,
                                        uint32_t n)
        : base(static_cast<const char*>(array) + n * p->at.seq_rows * ld * sizeof(T)),
          by((uint32_t)(p->at.step_rows * ld * sizeof(T))),
          mine(at.in ? QuadMap<C>::step(0) * by + at.own * (uint32_t)sizeof(T) : kNone) {}
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(uint32_t t) const {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + (uint64_t)t * by), (short)0, 0x7fffffff,
                                                 0x00020000);
    }
    __device__ __forceinline__ int place(uint32_t t, uint32_t end, int j) const {
        return (int)(t + QuadMap<C>::step(j) < end ? mine : kNone);
    }
    // the lane's elements of the round at t, as they lie: a conversion here would wait for each
    __device__ __forceinline__ void load(uint32_t t, uint32_t end, Raw<T> (&v)[QuadMap<C>::R]) const {
        const __amdgpu_buffer_rsrc_t r = at(t);
#pragma unroll
        for (int j = 0; j < QuadMap<C>::R; ++j) {
            const int s = j * QuadMap<C>::P * (int)by;
            if constexpr (sizeof(T) == 2)
                v[j].bits = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(r, place(t, end, j), s, 0);
            else
                v[j].bits = __builtin_amdgcn_raw_buffer_load_b32(r, place(t, end, j), s, 0);
        }
    }
    __device__ __forceinline__ void store(uint32_t t, uint32_t end, const float (&v)[QuadMap<C>::R]) const {
        const __amdgpu_buffer_rsrc_t r = at(t);
#pragma unroll
        for (int j = 0; j < QuadMap<C>::R; ++j) {
            const int s = j * QuadMap<C>::P * (int)by;
            if constexpr (sizeof(T) == 2)
                __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (T)v[j]), r, place(t, end, j),
                                                      s, 0);
            else
                __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, (T)v[j]), r, place(t, end, j), s, 0);
        }
    }
};

// B and C of a window's steps, [steps][SP] each; a thread's share on its way.
template <int STEPS, class T, int SP>
struct QuadShared {
    static constexpr int N = STEPS * SP / 256;
    Raw<T> b[N], c[N];
    uint8_t reset;
    __device__ __forceinline__ void load(uint32_t group, uint32_t n, uint32_t t, uint32_t end) {
        const ArgsAgain p = args_again();
        const uint32_t states = p->states;
        const uint64_t row0 = n * p->at.seq_rows, by = p->at.step_rows;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t e = threadIdx.x + i * 256, s = t + e / SP, k = e % SP;
            b[i] = c[i] = Raw<T>{0};
            if (s >= end || k >= states) continue;
            const uint64_t row = row0 + s * by;
            b[i] = raw_at(static_cast<const T*>(p->b) + row * p->b_ld + (size_t)group * states + k);
            c[i] = raw_at(static_cast<const T*>(p->c) + row * p->c_ld + (size_t)group * states + k);
        }
        const uint32_t lane = threadIdx.x & 63;
        const uint8_t* const resets = p->at.reset;
        reset = 0;
        if (resets && lane < STEPS && t + lane < end) reset = resets[row0 + (t + lane) * by];
    }
    __device__ __forceinline__ void put(float* tb, float* tc) const {
#pragma unroll
        for (int i = 0; i < N; ++i) tb[threadIdx.x + i * 256] = (float)b[i], tc[threadIdx.x + i * 256] = (float)c[i];
    }
    __device__ __forceinline__ uint64_t resets() const { return __ballot(reset != 0); }
};

template <int NS>
__device__ __forceinline__ void quad_row(const float* row, f32x4 (&v)[NS]) {
#pragma unroll
    for (int q = 0; q < NS; ++q) v[q] = *reinterpret_cast<const f32x4*>(row + 16 * q);
}

// The state (or, backwards, the gradient) that the splits up to one leave, each a decay and an end.
template <int C, int NS>
__device__ __forceinline__ void quad_join(const ScanArgs& p, const QuadLane<C, NS>& at, uint32_t n, uint32_t split,
                                          f32x4 (&h)[C * NS]) {
    const size_t cells = (size_t)p.at.seqs * p.channels;
    f32x4 behind[C * NS];
    at.load(p, p.ends + split * cells * p.states, n, behind);
#pragma unroll
    for (int u = 0; u < C * NS; ++u) {
        const float sum = at.held[u] > 0 ? p.decays[split * cells + (size_t)n * p.channels + at.first + u / NS] : 0.0f;
        const f32x4 decay = decay_of(at.a2[u], sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[u][i] = sum < 0.0f ? behind[u][i] : __builtin_fmaf(decay[i], h[u][i], behind[u][i]);
    }
}

// The rates of a lane's elements; steps past the end have delta 0, which leaves a state as
// it is, and so have lanes without a channel.
template <int C, class T>
__device__ __forceinline__ void quad_rates(bool in, uint32_t t, uint32_t end, float bias,
                                           const Raw<T> (&dt)[QuadMap<C>::R], const Raw<T> (&x)[QuadMap<C>::R],
                                           float (&delta)[QuadMap<C>::R], float (&u)[QuadMap<C>::R]) {
#pragma unroll
    for (int j = 0; j < QuadMap<C>::R; ++j) {
        const bool live = in && t + QuadMap<C>::step(j) < end;
        delta[j] = live ? softplus((float)dt[j] + bias) : 0.0f;
        u[j] = live ? delta[j] * (float)x[j] : 0.0f;
    }
}

// As scan_kernel. A state's step is a product, an exponential at half rate and three multiply-adds,
// six issues of a wave: 32 steps of 4096 x 256 with 16 states, bf16 take 163 us, of which those issues
// are 89 and the 479 MB would be 94, only partly under each other. Four waves a SIMD (two where a lane
// has 16 states: three spill 54 registers, 32 x 4096 x 128 of 64 states, fp16 384 us for 291): five spill,
// 201 us.
template <class T, int C, int NS, bool FULL, bool Z>
__global__ void __launch_bounds__(256, NS > 2 ? 2 : 4) scan_quad_kernel(const ScanArgs p, uint64_t items) {
    using Lane = QuadLane<C, NS>;
    constexpr int R = Lane::R;
    constexpr int SP = Lane::SP;
    __shared__ __align__(16) float sb[2][kWindow * SP], sc[2][kWindow * SP];
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const ScanItem it(p, item);
        Lane at(p, it.block);
        const uint32_t n = it.n, length = p.at.length(n), begin = it.split * p.split_steps;
        uint32_t end = begin + p.split_steps;
        end = end < length ? end : length;
        f32x4 h[Lane::U] = {};
        if constexpr (FULL) {
            if (p.initial) at.load(p, p.splits > 1 ? p.saved : p.initial, n, h);
        } else if (it.split == 0 && p.initial) {
            f32x4 first[Lane::U];
            at.load(p, p.initial, n, first);
            at.store(p, p.saved, n, first);
        }
        const float bias = p.dt_bias ? p.dt_bias[at.own] : 0.0f, skip = FULL && p.d ? p.d[at.own] : 0.0f;
        float sum[C] = {};
        bool begun = false;
        Raw<T> x[R], dt[R], z[R];
        auto fetch = [&](uint32_t t) {
            const ArgsAgain q = args_again();
            QuadRows<T, C>(q, at, q->x, q->x_ld, n).load(t, end, x);
            QuadRows<T, C>(q, at, q->dt, q->dt_ld, n).load(t, end, dt);
            if constexpr (FULL && Z) QuadRows<T, C>(q, at, q->z, q->z_ld, n).load(t, end, z);
        };
        QuadShared<kWindow, T, SP> shared;
        if (begin < end) {
            shared.load(at.group, n, begin, end);
            fetch(begin);
        }
        at.ready();
        if constexpr (FULL) {
#pragma unroll 2
            for (uint32_t k = 0; k < it.split; ++k) quad_join(p, at, n, k, h);
        }
        __syncthreads();  // the item before is done with LDS
        if (begin < end) shared.put(sb[0], sc[0]);
        __syncthreads();
        int turn = 0;
        for (uint32_t w = begin; w < end; w += kWindow, turn ^= 1) {
            uint32_t resets = (uint32_t)shared.resets();
            if (!FULL) begun |= resets != 0;
            const bool more = w + kWindow < end;
            if (more) shared.load(at.group, n, w + kWindow, end);
            const uint32_t until = more ? w + kWindow : end;
            const float* b_at = sb[turn] + at.state;
            const float* c_at = sc[turn] + at.state;
            for (uint32_t t = w; t < until; t += kSteps, resets >>= kSteps) {
                float delta[R], u[R];
                Raw<T> was[R], gate[R];
                arrive(x), arrive(dt);
                quad_rates<C>(at.in, t, end, bias, dt, x, delta, u);
#pragma unroll
                for (int j = 0; j < R; ++j) was[j] = x[j], gate[j] = FULL && Z ? z[j] : Raw<T>{0};
                if (t + kSteps < end) fetch(t + kSteps);
                if (FULL && p.checkpoints && t % kChunk == 0)
                    at.store(p, p.checkpoints + (size_t)(t / kChunk) * p.at.seqs * p.channels * p.states, n, h);
                float out[R];
                {
                    float part[4];
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        if (resets >> k & 1) clear_states(h);
                        f32x4 b[NS], cc[NS];
                        quad_row(b_at + k * SP, b);
                        if constexpr (FULL) quad_row(c_at + k * SP, cc);
#pragma unroll
                        for (int c = 0; c < C; ++c) {
                            const int from = Lane::lane(k, c), j = k / Lane::P;
                            const float d = quad_take(from, delta[j]), uu = quad_take(from, u[j]);
                            float y = 0.0f;
#pragma unroll
                            for (int q = 0; q < NS; ++q) {
                                f32x4& s = h[c * NS + q];
                                const f32x4 decay = decay_of(at.a2[c * NS + q], d);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    s[i] = __builtin_fmaf(decay[i], s[i], uu * b[q][i]);
                                    if constexpr (FULL) y = q + i ? __builtin_fmaf(s[i], cc[q][i], y) : s[i] * cc[q][i];
                                }
                            }
                            if constexpr (FULL)
                                part[from] = y;
                            else
                                sum[c] += d;
                        }
                        if constexpr (FULL)
                            if (k % Lane::P == Lane::P - 1) out[k / Lane::P] = quad_sums(part);
                    }
                }
                if constexpr (FULL) {
#pragma unroll
                    for (int j = 0; j < R; ++j) {
                        float y = __builtin_fmaf(skip, (float)was[j], out[j]);
                        if (Z) y *= silu((float)gate[j]);
                        out[j] = y;
                    }
                    const ArgsAgain q = args_again();
                    QuadRows<T, C>(q, at, q->y, q->y_ld, n).store(t, end, out);
                }
                b_at += kSteps * SP, c_at += kSteps * SP;
            }
            if (more) shared.put(sb[turn ^ 1], sc[turn ^ 1]);
            __syncthreads();
        }
        if constexpr (FULL) {
            if (p.final && it.split == p.splits - 1) at.store(p, p.final, n, h);
        } else {
            const size_t row = ((size_t)it.split * p.at.seqs + n) * p.channels;
            at.store(p, p.ends + (size_t)it.split * p.at.seqs * p.channels * p.states, n, h);
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (at.held[c * NS] > 0 && at.state == 0) p.decays[row + at.first + c] = begun ? -1.0f : sum[c];
        }
    }
}

// As scan_ends_backward_kernel.
template <class T, int C, int NS>
__global__ void __launch_bounds__(256) scan_quad_ends_backward_kernel(const ScanArgs p, uint64_t items) {
    using Lane = QuadLane<C, NS>;
    constexpr int R = Lane::R;
    constexpr int SP = Lane::SP;
    __shared__ __align__(16) float sb[kWindow * SP], sc[kWindow * SP];
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const ScanItem it(p, item);
        Lane at(p, it.block);
        at.ready();
        const uint32_t n = it.n, length = p.at.length(n), split = it.split + 1, begin = split * p.split_steps;
        uint32_t end = begin + p.split_steps;
        end = end < length ? end : length;
        const float bias = p.dt_bias ? p.dt_bias[at.own] : 0.0f;
        f32x4 g[Lane::U] = {};
        float sum[C] = {};
        bool begun = false;
        for (uint32_t window = begin < end ? (end - begin + kWindow - 1) / kWindow : 0; window--;) {
            const uint32_t from = begin + window * kWindow, to = end - from < (uint32_t)kWindow ? end : from + kWindow;
            QuadShared<kWindow, T, SP> shared;
            shared.load(at.group, n, from, to);
            __syncthreads();
            shared.put(sb, sc);
            __syncthreads();
            const uint32_t resets = (uint32_t)shared.resets();
            begun |= resets != 0;
            for (int r = (int)((to - from + kSteps - 1) / kSteps); r--;) {
                const uint32_t t = from + r * kSteps;
                Raw<T> dt[R], z[R], dy[R];
                float delta[R], none[R], into[R];
                const ArgsAgain q = args_again();
                QuadRows<T, C>(q, at, q->dt, q->dt_ld, n).load(t, to, dt);
                QuadRows<T, C>(q, at, q->dy, q->dy_ld, n).load(t, to, dy);
                if (q->z) QuadRows<T, C>(q, at, q->z, q->z_ld, n).load(t, to, z);
                quad_rates<C>(at.in, t, to, bias, dt, dt, delta, none);
#pragma unroll
                for (int j = 0; j < R; ++j) into[j] = p.z ? (float)dy[j] * silu((float)z[j]) : (float)dy[j];
                const uint32_t bits = resets >> (r * kSteps);
#pragma unroll
                for (int k = kSteps - 1; k >= 0; --k) {
                    f32x4 cc[NS];
                    quad_row(sc + (r * kSteps + k) * SP + at.state, cc);
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        const int lane = Lane::lane(k, c), j = k / Lane::P;
                        const float d = quad_take(lane, delta[j]), dyk = quad_take(lane, into[j]);
                        sum[c] += d;
#pragma unroll
                        for (int q = 0; q < NS; ++q) {
                            const f32x4 decay = decay_of(at.a2[c * NS + q], d);
                            f32x4& s = g[c * NS + q];
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(cc[q][i], dyk, s[i]) * decay[i];
                        }
                    }
                    if (bits >> k & 1) clear_states(g);
                }
            }
        }
        const size_t row = ((size_t)split * p.at.seqs + n) * p.channels;
        at.store(p, p.ends + (size_t)split * p.at.seqs * p.channels * p.states, n, g);
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (at.held[c * NS] > 0 && at.state == 0) p.decays[row + at.first + c] = begun ? -1.0f : sum[c];
    }
}

// Step k of a round: the states on, from delta and delta x in the lanes that have them.
template <int C, int NS>
__device__ __forceinline__ void quad_step(const QuadLane<C, NS>& at, const float* b_row, int k,
                                          const float (&delta)[QuadMap<C>::R], const float (&u)[QuadMap<C>::R],
                                          f32x4 (&h)[C * NS]) {
    f32x4 b[NS];
    quad_row(b_row + at.state, b);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int lane = QuadMap<C>::lane(k, c), j = k / QuadMap<C>::P;
        const float d = quad_take(lane, delta[j]), uu = quad_take(lane, u[j]);
#pragma unroll
        for (int q = 0; q < NS; ++q) {
            const f32x4 decay = decay_of(at.a2[c * NS + q], d);
            f32x4& s = h[c * NS + q];
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(decay[i], s[i], uu * b[q][i]);
        }
    }
}

// As scan_backward_kernel, 32 steps at a time: their states every kSteps steps wait in LDS,
// each lane's own. The second half of a chunk walks over the first to its own first state.
// The decays are worked out twice: to keep them beside the states would take the registers of
// a wave a SIMD. 32 steps of 4096 x 256 with 16 states, bf16: 611 us, where 688 MB are 135; the vector
// units issue most of the time, about 21 times a state's step (three walks over its decay, ten
// products of the gradient itself) and for the sums over channels, from two waves a SIMD, as many as
// 241 registers leave. Elements asked for half a round sooner changed nothing.
template <class T, int C, int NS, bool Z>
__global__ void __launch_bounds__(256, 2) scan_quad_backward_kernel(const ScanArgs p, uint32_t parts) {
    using Lane = QuadLane<C, NS>;
    constexpr int R = Lane::R, U = Lane::U, SP = Lane::SP, kRounds = kWindow / kSteps;
    __shared__ __align__(16) float sb[kWindow * SP], sc[kWindow * SP];
    __shared__ f32x4 starts[kRounds - 1][U][256];
    __shared__ float rates[kRounds - 1][R][256];           // delta of the rounds that are walked over
    __shared__ float sums[2][kSteps][4][2 * SP];  // each wave's for dB and dC
    const uint32_t block = blockIdx.x % p.blocks, part = blockIdx.x / p.blocks;
    const int wave = threadIdx.x >> 6;
    Lane at(p, block);
    at.ready();
    const float skip = p.d ? p.d[at.own] : 0.0f, bias = p.dt_bias ? p.dt_bias[at.own] : 0.0f;
    f32x4 da[U] = {};
    float dd = 0.0f, dbias = 0.0f;
    int turn = 0;
    const uint64_t items = (uint64_t)p.at.seqs * p.splits;
    for (uint64_t item = part; item < items; item += parts) {
        const uint32_t split = (uint32_t)(item / p.at.seqs), n = (uint32_t)(item - (uint64_t)split * p.at.seqs);
        const uint32_t length = p.at.length(n), begin = split * p.split_steps;
        uint32_t end = begin + p.split_steps;
        end = end < length ? end : length;
        f32x4 g[U] = {};
        if (p.dfinal) at.load(p, p.dfinal, n, g);
        const size_t cells = (size_t)p.at.seqs * p.channels;
#pragma unroll 2
        for (uint32_t k = p.splits - 1; k > split; --k) quad_join(p, at, n, k, g);
        for (uint32_t window = begin < end ? (end - begin + kWindow - 1) / kWindow : 0; window--;) {
            const uint32_t from = begin + window * kWindow, to = end - from < (uint32_t)kWindow ? end : from + kWindow;
            const uint32_t chunk = from / kChunk * kChunk;
            const int rounds = (int)((to - from + kSteps - 1) / kSteps);
            f32x4 h[U] = {};
            if (chunk && p.kept)
                at.load(p, p.kept + chunk / kChunk * cells * p.states, n, h);
            else if (!chunk && p.initial)
                at.load(p, p.initial, n, h);
            Raw<T> x[R], dt[R], dy[R], z[R];
            auto fetch = [&](uint32_t t, uint32_t last, bool all) {
                const ArgsAgain q = args_again();
                QuadRows<T, C>(q, at, q->x, q->x_ld, n).load(t, last, x);
                QuadRows<T, C>(q, at, q->dt, q->dt_ld, n).load(t, last, dt);
                if (!all) return;
                QuadRows<T, C>(q, at, q->dy, q->dy_ld, n).load(t, last, dy);
                if constexpr (Z) QuadRows<T, C>(q, at, q->z, q->z_ld, n).load(t, last, z);
            };
            uint32_t resets = 0;
            for (uint32_t w = chunk; w <= from; w += kWindow) {
                const uint32_t last = w == from ? to : w + kWindow;
                const int walk = w == from ? rounds - 1 : kRounds;
                QuadShared<kWindow, T, SP> shared;
                shared.load(at.group, n, w, last);
                fetch(w, last, walk == 0);
                __syncthreads();  // every wave is done with B and C
                shared.put(sb, sc);
                __syncthreads();
                resets = (uint32_t)shared.resets();
                for (int r = 0; r < walk; ++r) {
                    const uint32_t t = w + r * kSteps;
                    float delta[R], u[R];
                    arrive(x), arrive(dt);
                    quad_rates<C>(at.in, t, last, bias, dt, x, delta, u);
                    if (t + kSteps < last) fetch(t + kSteps, last, w == from && r + 1 == walk);
                    if (w == from) {
#pragma unroll
                        for (int u = 0; u < U; ++u) starts[r][u][threadIdx.x] = h[u];
#pragma unroll
                        for (int j = 0; j < R; ++j) rates[r][j][threadIdx.x] = delta[j];
                    }
                    const uint32_t bits = resets >> (r * kSteps);
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        if (bits >> k & 1) clear_states(h);
                        quad_step(at, sb + (r * kSteps + k) * SP, k, delta, u, h);
                    }
                }
            }
            for (int r = rounds; r--; turn ^= 1) {
                const uint32_t t = from + r * kSteps;
                float delta[R], u[R], into[R];  // dy before the gate
                arrive(x), arrive(dt), arrive(dy);
                if constexpr (Z) arrive(z);
                if (r + 1 < rounds) {
#pragma unroll
                    for (int j = 0; j < R; ++j) delta[j] = rates[r][j][threadIdx.x], u[j] = delta[j] * (float)x[j];
                } else {
                    quad_rates<C>(at.in, t, to, bias, dt, x, delta, u);
                }
#pragma unroll
                for (int j = 0; j < R; ++j) {
                    into[j] = Z ? (float)dy[j] * silu((float)z[j]) : (float)dy[j];
                    // a lane without a channel, or past the end, adds nothing
                    into[j] = at.in && t + Lane::step(j) < to ? into[j] : 0.0f;
                }
                if (r + 1 < rounds) {
#pragma unroll
                    for (int u = 0; u < U; ++u) h[u] = starts[r][u][threadIdx.x];
                }
                const uint32_t bits = resets >> (r * kSteps);
                float gb[R], ga[R], y[R];
                f32x4 first[U], states[kSteps][U];
#pragma unroll
                for (int w = 0; w < U; ++w) first[w] = h[w];
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    if (bits >> k & 1) clear_states(h);
                    quad_step(at, sb + (r * kSteps + k) * SP, k, delta, u, h);
#pragma unroll
                    for (int w = 0; w < U; ++w) states[k][w] = h[w];
                }
                // or the compiler keeps what it knows of the decays, B and the moved values
#pragma unroll
                for (int j = 0; j < R; ++j) asm volatile("" : "+v"(delta[j]), "+v"(u[j])::"memory");
                float part_b[4], part_a[4], part_y[4];
#pragma unroll
                for (int k = kSteps - 1; k >= 0; --k) {
                    f32x4 b[NS], cc[NS];
                    quad_row(sb + (r * kSteps + k) * SP + at.state, b);
                    quad_row(sc + (r * kSteps + k) * SP + at.state, cc);
                    float v[NS][8] = {};
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        const int lane = Lane::lane(k, c), j = k / Lane::P;
                        const float dyk = quad_take(lane, into[j]), uu = quad_take(lane, u[j]);
                        float sum_b = 0.0f, sum_y = 0.0f;
#pragma unroll
                        for (int q = 0; q < NS; ++q) {
                            const int w = c * NS + q;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                g[w][i] = __builtin_fmaf(cc[q][i], dyk, g[w][i]);
                                v[q][i] = __builtin_fmaf(g[w][i], uu, v[q][i]);
                                v[q][4 + i] = __builtin_fmaf(states[k][w][i], dyk, v[q][4 + i]);
                                if (Z) sum_y = __builtin_fmaf(cc[q][i], states[k][w][i], sum_y);
                                sum_b = __builtin_fmaf(g[w][i], b[q][i], sum_b);
                            }
                        }
                        part_b[lane] = sum_b, part_y[lane] = sum_y;
                    }
                    // where an episode begins nothing goes further back
                    if (bits >> k & 1) {
                        clear_states(g);
#pragma unroll
                        for (int c = 0; c < C; ++c) part_a[Lane::lane(k, c)] = 0.0f;
                    } else {
#pragma unroll
                        for (int c = 0; c < C; ++c) {
                            const int lane = Lane::lane(k, c), j = k / Lane::P;
                            const float d = quad_take(lane, delta[j]);
                            float sum_a = 0.0f;
#pragma unroll
                            for (int q = 0; q < NS; ++q) {
                                const int w = c * NS + q;
                                const f32x4 decay = decay_of(at.a2[w], d);
                                const f32x4 before = k ? states[k ? k - 1 : 0][w] : first[w];
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    g[w][i] *= decay[i];
                                    const float via = g[w][i] * before[i];
                                    sum_a = __builtin_fmaf(via, at.a2[w][i], sum_a);
                                    da[w][i] = __builtin_fmaf(via, d, da[w][i]);
                                }
                            }
                            part_a[lane] = sum_a;
                        }
                    }
#pragma unroll
                    for (int q = 0; q < NS; ++q) sum_channels<4, SP>(v[q], sums[turn][k][wave] + 16 * q);
                    if (k % Lane::P == 0) {
                        const int j = k / Lane::P;
                        gb[j] = quad_sums(part_b), ga[j] = quad_sums(part_a);
                        if (Z) y[j] = quad_sums(part_y);
                    }
                }
                Raw<T> x0[R], dt0[R], dy0[R], z0[R];
#pragma unroll
                for (int j = 0; j < R; ++j) x0[j] = x[j], dt0[j] = dt[j], dy0[j] = dy[j], z0[j] = Z ? z[j] : Raw<T>{0};
                if (r) fetch(t - kSteps, to, true);
#pragma unroll
                for (int j = 0; j < R; ++j) {
                    if (Z) y[j] = (float)dy0[j] * __builtin_fmaf(skip, (float)x0[j], y[j]) * silu_slope((float)z0[j]);
                    float slope, rest;
                    sigmoid_of((float)dt0[j] + bias, slope, rest);
                    ga[j] = __builtin_fmaf((float)x0[j], gb[j], ga[j] * 0.693147181f) * slope;
                    gb[j] = __builtin_fmaf(into[j], skip, delta[j] * gb[j]);
                    if (at.in && t + Lane::step(j) < to) {
                        dd = __builtin_fmaf(into[j], (float)x0[j], dd);
                        dbias += ga[j];
                    }
                }
                {
                    const ArgsAgain q = args_again();
                    QuadRows<T, C>(q, at, q->dx, q->dx_ld, n).store(t, to, gb);
                    QuadRows<T, C>(q, at, q->ddt, q->ddt_ld, n).store(t, to, ga);
                    if (Z && q->dz) QuadRows<T, C>(q, at, q->dz, q->dz_ld, n).store(t, to, y);
                }
                __syncthreads();
#pragma unroll
                for (int e = threadIdx.x; e < kSteps * 2 * SP; e += 256) {
                    const int k = e / (2 * SP), w = e % (2 * SP), i = w % SP;
                    if (t + k >= to || i >= (int)p.states) continue;
                    const float sum = (sums[turn][k][0][w] + sums[turn][k][1][w]) +
                                      (sums[turn][k][2][w] + sums[turn][k][3][w]);
                    const uint32_t which = w / SP;
                    const ArgsAgain q = args_again();
                    if (q->apiece == 1) {
                        const uint64_t row = (t + k) * q->at.step_rows + n * q->at.seq_rows;
                        const uint64_t place = row * (which ? q->dc_ld : q->db_ld) + (size_t)at.group * q->states + i;
                        static_cast<T*>(which ? q->dc : q->db)[place] = (T)sum;
                    } else {
                        const size_t row = ((size_t)(block % q->apiece) * q->at.steps + t + k) * q->at.seqs + n;
                        q->shared[((row * q->groups + at.group) * 2 + which) * q->states + i] = sum;
                    }
                }
            }
        }
        if (p.dinitial && split == 0) at.store(p, p.dinitial, n, g);
    }
    if (!p.sums) return;
    float* const out = p.sums + (size_t)part * p.channels * (p.states + 2);
    at.store(p, out, 0, da);
    // a channel's lanes of the quad
    if constexpr (C == 1) dd += dpp_lane<0xB1>(dd), dbias += dpp_lane<0xB1>(dbias);
    dd += dpp_lane<0x4E>(dd), dbias += dpp_lane<0x4E>(dbias);
    if (at.in && (threadIdx.x & 3) < C) {
        out[(size_t)p.channels * p.states + at.own] = dd;
        out[(size_t)p.channels * (p.states + 1) + at.own] = dbias;
    }
}

// One step of every sequence, four sequences at a time: no LDS, every load at once, the
// states to memory and back. A quad's lanes each work for one of the four. 65536 x 128 of 16 states,
// bf16: 243 us, 4.7 TB/s where a large copy reaches 5.1.
template <class T, int NS, bool Z>
__global__ void __launch_bounds__(256) scan_quad_step_kernel(const ScanArgs p, uint64_t items) {
    using Lane = QuadLane<1, NS>;
    typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t n0 = (uint32_t)(item / p.blocks) * 4;
        Lane at(p, (uint32_t)(item % p.blocks));
        at.ready();
        const uint32_t last = p.at.seqs - 1;
        const float skip = p.d ? p.d[at.own] : 0.0f, bias = p.dt_bias ? p.dt_bias[at.own] : 0.0f;
        f32x4 h[4][NS], b[4][NS], c[4][NS];
        bool fresh[4], live[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint32_t n = n0 + s < last ? n0 + s : last;
            const uint64_t row = p.at.row(0, n);
            live[s] = p.at.length(n) != 0;
            fresh[s] = live[s] && p.at.reset && p.at.reset[row];
#pragma unroll
            for (int q = 0; q < NS; ++q) {
                h[s][q] = p.initial ? load_states(p.initial + at.at(p, n, q), at.held[q]) : f32x4{};
                b[s][q] = c[s][q] = f32x4{};
                if (!live[s]) continue;
                const size_t from = (size_t)at.group * p.states + at.state + 16 * q;
                const T* const bs = static_cast<const T*>(p.b) + row * p.b_ld + from;
                const T* const cs = static_cast<const T*>(p.c) + row * p.c_ld + from;
                if (p.states == Lane::SP) {
                    const four vb = *reinterpret_cast<const four*>(bs), vc = *reinterpret_cast<const four*>(cs);
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[s][q][i] = (float)vb[i], c[s][q][i] = (float)vc[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (at.state + 16 * q + i < (int)p.states) b[s][q][i] = (float)bs[i], c[s][q][i] = (float)cs[i];
                }
            }
        }
        const uint32_t mine = n0 + (threadIdx.x & 3), n = mine < last ? mine : last;
        const bool works = mine <= last && p.at.length(n) != 0;
        float x = 0.0f, dt = 0.0f, z = 0.0f;
        const uint64_t row = p.at.row(0, n);
        if (works) {
            x = (float)static_cast<const T*>(p.x)[row * p.x_ld + at.own];
            dt = (float)static_cast<const T*>(p.dt)[row * p.dt_ld + at.own];
            if (Z) z = (float)static_cast<const T*>(p.z)[row * p.z_ld + at.own];
        }
        const float delta = works ? softplus(dt + bias) : 0.0f, u = works ? delta * x : 0.0f;
        float part[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const float d = quad_take(s, delta), uu = quad_take(s, u);
            part[s] = 0.0f;
#pragma unroll
            for (int q = 0; q < NS; ++q) {
                f32x4& v = h[s][q];
                if (fresh[s]) v = f32x4{};
                const f32x4 decay = decay_of(at.a2[q], d);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float moved = __builtin_fmaf(decay[i], v[i], uu * b[s][q][i]);
                    v[i] = live[s] ? moved : v[i];
                    part[s] = __builtin_fmaf(v[i], c[s][q][i], part[s]);
                }
                if (p.final && n0 + s <= last) store_states(p.final + at.at(p, n0 + s, q), at.held[q], v);
            }
        }
        float y = quad_sums(part);
        if (works && at.in) {
            y = __builtin_fmaf(skip, x, y);
            if (Z) y *= silu(z);
            static_cast<T*>(p.y)[row * p.y_ld + at.own] = (T)y;
        }
    }
}

}  // namespace dev
}  // namespace mg
