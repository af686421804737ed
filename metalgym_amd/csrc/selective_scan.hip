// Selective state space scan over a rollout, and its gradients (mg_selective_scan,
// mg_selective_scan_backward).
//
// Each channel has `states` states: h = exp(delta A) h + delta B x, y = sum_s C h + D x,
// with delta = softplus(dt + bias) of the channel and step, and B, C of the step, shared by
// a group's channels. A lane holds four states of a channel and L lanes the channel, so a
// workgroup takes 256 / L channels of one sequence. It walks over the steps eight at a time:
// the rows' elements come in along the channels, delta, delta x, B and C go to LDS as fp32
// once, and the eight steps then run from LDS and registers.
//
// What it costs is a v_exp (half the rate) and four products for each state and step: 16001 steps of
// 512 channels with 64 states take 285 us, 95 of them for the splits' ends (see below), where the
// bytes would take 10. Where there are few sequences the steps are split over workgroups: a first
// launch takes each split from a state of zero to its end, a second joins the splits before
// its own (a split's decay is exp(A sum of delta)) and walks over its steps again.
//
// The gradient needs every state again. It starts from the states that the forward pass
// kept every 64 steps (kChunk), walks over those 64 once to have the states every 8 steps in
// LDS, and takes the 8 steps back to front with their states and decays in registers.
#include <type_traits>

#include "scan_common.h"
#include "scan_quad.h"

namespace mg {
namespace dev {

// A workgroup's channels of one group, and a lane's four states among them.
template <int L>
struct ScanLane {
    static constexpr int CH = 256 / L;  // channels of a workgroup
    static constexpr int SP = 4 * L;    // states, with padding
    uint32_t group, first, limit;       // the workgroup's channels: [first, limit), CH at most
    uint32_t channel;
    int state, count;  // the first of the lane's states, and how many there are from it
    f32x4 a2;          // A log2(e)

    __device__ __forceinline__ ScanLane(const ScanArgs& p, uint32_t block) {
        group = block / p.apiece;
        first = group * p.per + (block - group * p.apiece) * CH;
        limit = (group + 1) * p.per;
        channel = first + threadIdx.x / L;
        state = 4 * (threadIdx.x % L);
        count = channel < limit ? (int)p.states - state : 0;
        a2 = base2_of(load_states(p.a + (size_t)channel * p.states + state, count));
    }
    __device__ __forceinline__ size_t at(const ScanArgs& p, uint32_t n) const {
        return ((size_t)n * p.channels + channel) * p.states + state;
    }
};

// What a round of steps needs, in LDS.
template <int L>
struct ScanRound {
    float delta[kSteps * ScanLane<L>::CH];
    float u[kSteps * ScanLane<L>::CH];  // delta x
    float b[kSteps * ScanLane<L>::SP];
    float c[kSteps * ScanLane<L>::SP];
    uint32_t resets;  // a bit a step
};

// A thread's elements of a round: the same channel of every few steps. They stay as they
// lie until they are used: a conversion waits for its load. RAW: in registers of their own, for the
// gradients of 16-bit types (32 x 4096 x 256 with 4 states, bf16 959 us without, so 824); the forward
// pass has more waves from fewer registers (the same shape 136 us, and 151 with them).
template <class T, int L, bool RAW>
struct ScanFetch {
    using E = std::conditional_t<RAW, Raw<T>, T>;
    using Lane = ScanLane<L>;
    static constexpr int N = (kSteps * Lane::CH + 255) / 256;
    static constexpr int NB = (kSteps * Lane::SP + 255) / 256;
    E x[N], dt[N], z[N], dy[N], b[NB], c[NB];
    uint8_t reset;

    static __device__ __forceinline__ E take(const T* p) {
        if constexpr (RAW)
            return raw_at(p);
        else
            return *p;
    }
    static __device__ __forceinline__ int step(int i) { return (threadIdx.x + i * 256) / Lane::CH; }
    static __device__ __forceinline__ int slot(int i) { return threadIdx.x + i * 256; }
    static __device__ __forceinline__ uint32_t channel(const Lane& at) {
        return at.first + threadIdx.x % Lane::CH;
    }
    // whether element i is one of the round that begins at step t
    static __device__ __forceinline__ bool in(const Lane& at, int i, uint32_t t, uint32_t end) {
        return slot(i) < kSteps * Lane::CH && t + step(i) < end && channel(at) < at.limit;
    }

    template <bool DY>
    __device__ __forceinline__ void load(const ScanArgs& p, const Lane& at, uint32_t n, uint32_t t, uint32_t end) {
        const uint32_t ch = channel(at);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = dt[i] = z[i] = dy[i] = E{};
            if (!in(at, i, t, end)) continue;
            const uint64_t row = p.at.row(t + step(i), n);
            x[i] = take(static_cast<const T*>(p.x) + row * p.x_ld + ch);
            dt[i] = take(static_cast<const T*>(p.dt) + row * p.dt_ld + ch);
            if (p.z) z[i] = take(static_cast<const T*>(p.z) + row * p.z_ld + ch);
            if (DY) dy[i] = take(static_cast<const T*>(p.dy) + row * p.dy_ld + ch);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int e = threadIdx.x + i * 256, k = e / Lane::SP, s = e % Lane::SP;
            b[i] = c[i] = E{};
            if (e >= kSteps * Lane::SP || t + k >= end || s >= (int)p.states) continue;
            const uint64_t row = p.at.row(t + k, n);
            b[i] = take(static_cast<const T*>(p.b) + row * p.b_ld + (size_t)at.group * p.states + s);
            c[i] = take(static_cast<const T*>(p.c) + row * p.c_ld + (size_t)at.group * p.states + s);
        }
        reset = 0;
        if (p.at.reset && threadIdx.x < kSteps && t + threadIdx.x < end) reset = p.at.reset[p.at.row(t + threadIdx.x, n)];
    }
    // Steps past the end have delta 0: they leave the state as it is.
    __device__ __forceinline__ void put(const ScanArgs& p, const Lane& at, uint32_t t, uint32_t end,
                                        ScanRound<L>& to) {
        if constexpr (RAW) arrive(x), arrive(dt), arrive(b), arrive(c);
        const uint32_t ch = channel(at);
        const float bias = p.dt_bias && ch < at.limit ? p.dt_bias[ch] : 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (slot(i) >= kSteps * Lane::CH) continue;
            const float delta = in(at, i, t, end) ? softplus((float)dt[i] + bias) : 0.0f;
            to.delta[slot(i)] = delta;
            to.u[slot(i)] = delta * (float)x[i];
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int e = threadIdx.x + i * 256;
            if (e >= kSteps * Lane::SP) continue;
            to.b[e] = (float)b[i], to.c[e] = (float)c[i];
        }
        if (threadIdx.x < 64) {
            const uint32_t bits = (uint32_t)__ballot(reset != 0);
            if (threadIdx.x == 0) to.resets = bits;
        }
    }
};

// The state that a split of sequence n begins with: the splits before it, joined.
template <int L>
__device__ __forceinline__ f32x4 join_before(const ScanArgs& p, const ScanLane<L>& at, uint32_t n, uint32_t split) {
    const float* first = p.splits > 1 ? p.saved : p.initial;
    f32x4 h = {};
    if (p.initial && at.count > 0) h = load_states(first + at.at(p, n), at.count);
    if (at.count <= 0) return h;
    const size_t step = (size_t)p.at.seqs * p.channels;
#pragma unroll 8
    for (uint32_t k = 0; k < split; ++k) {
        const f32x4 end = load_states(p.ends + k * step * p.states + at.at(p, n), at.count);
        const float sum = p.decays[k * step + (size_t)n * p.channels + at.channel];
        const f32x4 decay = decay_of(at.a2, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = sum < 0.0f ? end[i] : __builtin_fmaf(decay[i], h[i], end[i]);
    }
    return h;
}

// FULL: y, the final state and the kept ones. Else each split but the last from a state of
// zero to its end.
template <class T, int L, bool FULL>
__global__ void __launch_bounds__(256) scan_kernel(const ScanArgs p, uint64_t items) {
    using Lane = ScanLane<L>;
    using Fetch = ScanFetch<T, L, false>;
    __shared__ ScanRound<L> rounds[2];
    __shared__ float out[2][kSteps * Lane::CH];
    const int mine = threadIdx.x / L, sub = threadIdx.x % L;
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const ScanItem it(p, item);
        const Lane at(p, it.block);
        const uint32_t n = it.n, length = p.at.length(n), begin = it.split * p.split_steps;
        uint32_t end = begin + p.split_steps;
        end = end < length ? end : length;
        f32x4 h = {};
        if (FULL)
            h = join_before<L>(p, at, n, it.split);
        else if (it.split == 0 && p.initial && at.count > 0)
            store_states(p.saved + at.at(p, n), at.count, load_states(p.initial + at.at(p, n), at.count));
        float sum = 0.0f;
        bool begun = false;
        const uint32_t ch = Fetch::channel(at);
        const float skip = FULL && p.d && ch < at.limit ? p.d[ch] : 0.0f;
        Fetch now;
        now.template load<false>(p, at, n, begin, end);
        __syncthreads();  // the item before is done with LDS
        now.put(p, at, begin, end, rounds[0]);
        __syncthreads();
        int turn = 0;
        for (uint32_t t = begin; t < end; t += kSteps, turn ^= 1) {
            Fetch next;
            const bool more = t + kSteps < end;
            if (more) next.template load<false>(p, at, n, t + kSteps, end);
            if (FULL && p.checkpoints && t % kChunk == 0 && at.count > 0)
                store_states(p.checkpoints + (size_t)(t / kChunk) * p.at.seqs * p.channels * p.states + at.at(p, n),
                             at.count, h);
            const ScanRound<L>& r = rounds[turn];
            const uint32_t resets = __builtin_amdgcn_readfirstlane(r.resets);
            if (!FULL) begun |= resets != 0;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                if (resets >> k & 1) clear_states(h);
                const float delta = r.delta[k * Lane::CH + mine], u = r.u[k * Lane::CH + mine];
                const f32x4 b = *reinterpret_cast<const f32x4*>(&r.b[k * Lane::SP + 4 * sub]);
                const f32x4 decay = decay_of(at.a2, delta);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = __builtin_fmaf(decay[i], h[i], u * b[i]);
                if (!FULL) {
                    sum += delta;
                    continue;
                }
                const f32x4 c = *reinterpret_cast<const f32x4*>(&r.c[k * Lane::SP + 4 * sub]);
                float y = h[0] * c[0];
#pragma unroll
                for (int i = 1; i < 4; ++i) y = __builtin_fmaf(h[i], c[i], y);
                y = group_sum<L>(y);
                if (sub == k % L) out[turn][k * Lane::CH + mine] = y;
            }
            if (more) next.put(p, at, t + kSteps, end, rounds[turn ^ 1]);
            __syncthreads();
            if (FULL) {
#pragma unroll
                for (int i = 0; i < Fetch::N; ++i) {
                    if (!Fetch::in(at, i, t, end)) continue;
                    float y = __builtin_fmaf(skip, (float)now.x[i], out[turn][Fetch::slot(i)]);
                    if (p.z) y *= silu((float)now.z[i]);
                    static_cast<T*>(p.y)[p.at.row(t + Fetch::step(i), n) * p.y_ld + ch] = (T)y;
                }
            }
            now = next;
        }
        if (at.count <= 0) continue;
        if (FULL) {
            if (p.final && it.split == p.splits - 1) store_states(p.final + at.at(p, n), at.count, h);
        } else {
            const size_t row = ((size_t)it.split * p.at.seqs + n) * p.channels + at.channel;
            store_states(p.ends + row * p.states + at.state, at.count, h);
            if (sub == 0) p.decays[row] = begun ? -1.0f : sum;
        }
    }
}

// One step of every sequence: no LDS, every load at once, the states to memory and back.
template <class T, int L>
__global__ void __launch_bounds__(256) scan_step_kernel(const ScanArgs p, uint64_t items) {
    using Lane = ScanLane<L>;
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const ScanItem it(p, item);
        const Lane at(p, it.block);
        const uint32_t n = it.n;
        const bool in = at.channel < at.limit;
        f32x4 h = {};
        if (p.initial && at.count > 0) h = load_states(p.initial + at.at(p, n), at.count);
        const bool live = p.at.length(n) != 0;
        const uint64_t row = p.at.row(0, n);
        float y = 0.0f;
        if (live) {
            float x = 0.0f, dt = 0.0f, z = 0.0f;
            f32x4 b = {}, c = {};
            if (in) {
                x = (float)static_cast<const T*>(p.x)[row * p.x_ld + at.channel];
                dt = (float)static_cast<const T*>(p.dt)[row * p.dt_ld + at.channel];
                if (p.z) z = (float)static_cast<const T*>(p.z)[row * p.z_ld + at.channel];
                if (p.dt_bias) dt += p.dt_bias[at.channel];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < at.count) {
                    const size_t s = (size_t)at.group * p.states + at.state + i;
                    b[i] = static_cast<const T*>(p.b)[row * p.b_ld + s];
                    c[i] = static_cast<const T*>(p.c)[row * p.c_ld + s];
                }
            if (p.at.reset && p.at.reset[row]) h = f32x4{};
            const float delta = softplus(dt), u = delta * x;
            const f32x4 decay = decay_of(at.a2, delta);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[i] = __builtin_fmaf(decay[i], h[i], u * b[i]);
                y = __builtin_fmaf(h[i], c[i], y);
            }
            y = group_sum<L>(y);
            if (in && threadIdx.x % L == 0) {
                if (p.d) y = __builtin_fmaf(p.d[at.channel], x, y);
                if (p.z) y *= silu(z);
                static_cast<T*>(p.y)[row * p.y_ld + at.channel] = (T)y;
            }
        }
        if (p.final && at.count > 0) store_states(p.final + at.at(p, n), at.count, h);
    }
}

// Each split but the first, back to front with nothing from behind it.
template <class T, int L>
__global__ void __launch_bounds__(256) scan_ends_backward_kernel(const ScanArgs p, uint64_t items) {
    using Lane = ScanLane<L>;
    using Fetch = ScanFetch<T, L, false>;
    __shared__ ScanRound<L> r;
    const int mine = threadIdx.x / L, sub = threadIdx.x % L;
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        ScanItem it(p, item);
        const Lane at(p, it.block);
        const uint32_t n = it.n, length = p.at.length(n), begin = (it.split + 1) * p.split_steps;
        uint32_t end = begin + p.split_steps;
        end = end < length ? end : length;
        f32x4 g = {};
        float sum = 0.0f;
        bool begun = false;
        for (uint32_t left = begin < end ? (end - begin + kSteps - 1) / kSteps : 0; left--;) {
            const uint32_t t = begin + left * kSteps;
            Fetch f;
            f.template load<true>(p, at, n, t, end);
            __syncthreads();
            f.put(p, at, t, end, r);
#pragma unroll
            for (int i = 0; i < Fetch::N; ++i)  // u's place takes the gradient before the gate
                if (Fetch::slot(i) < kSteps * Lane::CH) r.u[Fetch::slot(i)] = p.z ? (float)f.dy[i] * silu((float)f.z[i]) : (float)f.dy[i];
            __syncthreads();
            const uint32_t resets = __builtin_amdgcn_readfirstlane(r.resets);
            begun |= resets != 0;
#pragma unroll
            for (int k = kSteps - 1; k >= 0; --k) {
                const float delta = r.delta[k * Lane::CH + mine], dy = r.u[k * Lane::CH + mine];
                const f32x4 c = *reinterpret_cast<const f32x4*>(&r.c[k * Lane::SP + 4 * sub]);
                const f32x4 decay = decay_of(at.a2, delta);
                sum += delta;
#pragma unroll
                for (int i = 0; i < 4; ++i) g[i] = __builtin_fmaf(c[i], dy, g[i]) * decay[i];
                if (resets >> k & 1) clear_states(g);
            }
        }
        if (at.count <= 0) continue;
        const size_t row = ((size_t)(it.split + 1) * p.at.seqs + n) * p.channels + at.channel;
        store_states(p.ends + row * p.states + at.state, at.count, g);
        if (sub == 0) p.decays[row] = begun ? -1.0f : sum;
    }
}

template <int L>
struct BackwardShared {
    using Lane = ScanLane<L>;
    ScanRound<L> r;
    float dy[kSteps * Lane::CH];
    float gb[kSteps * Lane::CH];  // sum over states of g B
    float ga[kSteps * Lane::CH];  // of g a h' A
    float y[kSteps * Lane::CH];   // of C h
    float bc[kSteps][4][2 * Lane::SP];  // each wave's sums for dB and dC
    f32x4 starts[kSubs][256];
};

// One (part, block): items part, part + parts, ... of (split, sequence).
template <class T, int L>
__global__ void __launch_bounds__(256) scan_backward_kernel(const ScanArgs p, uint32_t parts) {
    using Lane = ScanLane<L>;
    using Fetch = ScanFetch<T, L, sizeof(T) == 2>;
    __shared__ BackwardShared<L> s;
    const int mine = threadIdx.x / L, sub = threadIdx.x % L, wave = threadIdx.x >> 6;
    const uint32_t block = blockIdx.x % p.blocks, part = blockIdx.x / p.blocks;
    const Lane at(p, block);
    const uint32_t ch = Fetch::channel(at);
    const bool in = ch < at.limit;
    const float skip = in && p.d ? p.d[ch] : 0.0f, bias = in && p.dt_bias ? p.dt_bias[ch] : 0.0f;
    f32x4 da = {};
    float dd = 0.0f, dbias = 0.0f;
    const uint64_t items = (uint64_t)p.at.seqs * p.splits;
    for (uint64_t item = part; item < items; item += parts) {
        const uint32_t split = (uint32_t)(item / p.at.seqs), n = (uint32_t)(item - (uint64_t)split * p.at.seqs);
        const uint32_t length = p.at.length(n), begin = split * p.split_steps;
        uint32_t end = begin + p.split_steps;
        end = end < length ? end : length;
        f32x4 g = {};
        if (at.count > 0) {
            if (p.dfinal) g = load_states(p.dfinal + at.at(p, n), at.count);
            const size_t step = (size_t)p.at.seqs * p.channels;
#pragma unroll 8
            for (uint32_t k = p.splits - 1; k > split; --k) {
                const f32x4 behind = load_states(p.ends + k * step * p.states + at.at(p, n), at.count);
                const float sum = p.decays[k * step + (size_t)n * p.channels + at.channel];
                const f32x4 decay = decay_of(at.a2, sum);
#pragma unroll
                for (int i = 0; i < 4; ++i) g[i] = sum < 0.0f ? behind[i] : __builtin_fmaf(decay[i], g[i], behind[i]);
            }
        }
        const uint32_t chunks = begin < end ? (end - begin + kChunk - 1) / kChunk : 0;
        for (uint32_t chunk = chunks; chunk--;) {
            const uint32_t from = begin + chunk * kChunk;
            const uint32_t to = end - from < (uint32_t)kChunk ? end : from + kChunk;
            const int subs = (int)((to - from + kSteps - 1) / kSteps);
            // the states every kSteps steps
            f32x4 h = {};
            if (at.count > 0) {
                if (from && p.kept)
                    h = load_states(p.kept + (size_t)(from / kChunk) * p.at.seqs * p.channels * p.states + at.at(p, n),
                                    at.count);
                else if (!from && p.initial)
                    h = load_states(p.initial + at.at(p, n), at.count);
            }
            for (int j = 0; j + 1 < subs; ++j) {
                s.starts[j][threadIdx.x] = h;
                Fetch f;
                f.template load<false>(p, at, n, from + j * kSteps, to);
                __syncthreads();
                f.put(p, at, from + j * kSteps, to, s.r);
                __syncthreads();
                const uint32_t resets = __builtin_amdgcn_readfirstlane(s.r.resets);
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    if (resets >> k & 1) clear_states(h);
                    const float delta = s.r.delta[k * Lane::CH + mine], u = s.r.u[k * Lane::CH + mine];
                    const f32x4 b = *reinterpret_cast<const f32x4*>(&s.r.b[k * Lane::SP + 4 * sub]);
                    const f32x4 decay = decay_of(at.a2, delta);
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[i] = __builtin_fmaf(decay[i], h[i], u * b[i]);
                }
            }
            s.starts[subs - 1][threadIdx.x] = h;
            for (int j = subs; j--;) {
                const uint32_t t = from + j * kSteps;
                Fetch f;
                f.template load<true>(p, at, n, t, to);
                __syncthreads();
                f.put(p, at, t, to, s.r);
#pragma unroll
                for (int i = 0; i < Fetch::N; ++i)
                    if (Fetch::slot(i) < kSteps * Lane::CH)
                        s.dy[Fetch::slot(i)] = p.z ? (float)f.dy[i] * silu((float)f.z[i]) : (float)f.dy[i];
                __syncthreads();
                const uint32_t resets = __builtin_amdgcn_readfirstlane(s.r.resets);
                f32x4 before[kSteps], decay[kSteps];
                h = s.starts[j][threadIdx.x];
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    const float delta = s.r.delta[k * Lane::CH + mine], u = s.r.u[k * Lane::CH + mine];
                    const f32x4 b = *reinterpret_cast<const f32x4*>(&s.r.b[k * Lane::SP + 4 * sub]);
                    decay[k] = decay_of(at.a2, delta);
                    if (resets >> k & 1) clear_states(h);
                    before[k] = h;
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[i] = __builtin_fmaf(decay[k][i], h[i], u * b[i]);
                }
#pragma unroll
                for (int k = kSteps - 1; k >= 0; --k) {
                    const float delta = s.r.delta[k * Lane::CH + mine], u = s.r.u[k * Lane::CH + mine];
                    const float dy = s.dy[k * Lane::CH + mine];
                    const f32x4 b = *reinterpret_cast<const f32x4*>(&s.r.b[k * Lane::SP + 4 * sub]);
                    const f32x4 c = *reinterpret_cast<const f32x4*>(&s.r.c[k * Lane::SP + 4 * sub]);
                    float gb = 0.0f, ga = 0.0f, y = 0.0f, v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        g[i] = __builtin_fmaf(c[i], dy, g[i]);
                        v[i] = g[i] * u;
                        v[4 + i] = h[i] * dy;
                        y = __builtin_fmaf(c[i], h[i], y);
                        gb = __builtin_fmaf(g[i], b[i], gb);
                        g[i] *= decay[k][i];
                        const float via = g[i] * before[k][i];
                        ga = __builtin_fmaf(via, at.a2[i], ga);
                        da[i] = __builtin_fmaf(via, delta, da[i]);
                        h[i] = before[k][i];
                    }
                    // the state before an episode's first step is not h but 0
                    if (resets >> k & 1) clear_states(g);
                    sum_channels<L>(v, s.bc[k][wave]);
                    float three[3] = {gb, ga, y};
                    group_sum_n<L>(three);
                    if (sub == k % L) {
                        s.gb[k * Lane::CH + mine] = three[0];
                        s.ga[k * Lane::CH + mine] = three[1];
                        s.y[k * Lane::CH + mine] = three[2];
                    }
                    if (k) {
                        // h is the state after step k - 1, also where an episode began at k
                        if (resets >> k & 1) {
                            const float d1 = s.r.u[(k - 1) * Lane::CH + mine];
                            const f32x4 b1 = *reinterpret_cast<const f32x4*>(&s.r.b[(k - 1) * Lane::SP + 4 * sub]);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                h[i] = __builtin_fmaf(decay[k - 1][i], before[k - 1][i], d1 * b1[i]);
                        }
                    }
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < Fetch::N; ++i) {
                    if (!Fetch::in(at, i, t, to)) continue;
                    const int e = Fetch::slot(i);
                    const uint64_t row = p.at.row(t + Fetch::step(i), n);
                    const float x = (float)f.x[i], raw = (float)f.dt[i] + bias, delta = s.r.delta[e], dy = s.dy[e];
                    if (p.z && p.dz) {
                        const float y = __builtin_fmaf(skip, x, s.y[e]);
                        static_cast<T*>(p.dz)[row * p.dz_ld + ch] = (T)((float)f.dy[i] * y * silu_slope((float)f.z[i]));
                    }
                    static_cast<T*>(p.dx)[row * p.dx_ld + ch] = (T)__builtin_fmaf(dy, skip, delta * s.gb[e]);
                    float slope, rest;
                    sigmoid_of(raw, slope, rest);
                    const float ddt = __builtin_fmaf(x, s.gb[e], s.ga[e] * 0.693147181f) * slope;
                    static_cast<T*>(p.ddt)[row * p.ddt_ld + ch] = (T)ddt;
                    dd = __builtin_fmaf(dy, x, dd);
                    dbias += ddt;
                }
                for (int e = threadIdx.x; e < kSteps * 2 * Lane::SP; e += 256) {
                    const int k = e / (2 * Lane::SP), w = e % (2 * Lane::SP), i = w % Lane::SP;
                    if (t + k >= to || i >= (int)p.states) continue;
                    const float v = (s.bc[k][0][w] + s.bc[k][1][w]) + (s.bc[k][2][w] + s.bc[k][3][w]);
                    const uint32_t which = w / Lane::SP;
                    if (p.apiece == 1) {
                        const uint64_t row = p.at.row(t + k, n) * (which ? p.dc_ld : p.db_ld);
                        static_cast<T*>(which ? p.dc : p.db)[row + (size_t)at.group * p.states + i] = (T)v;
                    } else {
                        const size_t row = ((size_t)(block % p.apiece) * p.at.steps + t + k) * p.at.seqs + n;
                        p.shared[((row * p.groups + at.group) * 2 + which) * p.states + i] = v;
                    }
                }
            }
        }
        if (p.dinitial && split == 0 && at.count > 0) store_states(p.dinitial + at.at(p, n), at.count, g);
    }
    if (!p.sums) return;
    float* const out = p.sums + (size_t)part * p.channels * (p.states + 2);
    if (at.count > 0) store_states(out + (size_t)at.channel * p.states + at.state, at.count, da);
    // the channel's threads, in order
    float* const trade = reinterpret_cast<float*>(s.starts);
    __syncthreads();
    trade[threadIdx.x] = dd, trade[256 + threadIdx.x] = dbias;
    __syncthreads();
    if (threadIdx.x < Lane::CH && in) {
        for (int k = 1; k < L; ++k) {
            dd += trade[threadIdx.x + k * Lane::CH];
            dbias += trade[256 + threadIdx.x + k * Lane::CH];
        }
        out[(size_t)p.channels * p.states + ch] = dd;
        out[(size_t)p.channels * (p.states + 1) + ch] = dbias;
    }
}

// dB and dC from their blocks' parts, in order.
template <class T>
__global__ void __launch_bounds__(256) scan_shared_kernel(const ScanArgs p) {
    const uint64_t width = (uint64_t)p.groups * 2 * p.states, rows = (uint64_t)p.at.steps * p.at.seqs;
    for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < rows * width; e += (uint64_t)gridDim.x * 256) {
        const uint64_t row = e / width;
        const uint32_t w = (uint32_t)(e - row * width), t = (uint32_t)(row / p.at.seqs);
        const uint32_t n = (uint32_t)(row - (uint64_t)t * p.at.seqs);
        if (t >= p.at.length(n)) continue;
        float v = p.shared[e];
        for (uint32_t k = 1; k < p.apiece; ++k) v += p.shared[k * rows * width + e];
        const uint32_t group = w / (2 * p.states), which = w / p.states & 1, i = w % p.states;
        const uint64_t at = p.at.row(t, n) * (which ? p.dc_ld : p.db_ld) + (size_t)group * p.states + i;
        static_cast<T*>(which ? p.dc : p.db)[at] = (T)v;
    }
}

}  // namespace dev

namespace {

constexpr uint32_t kMostStates = 256;
static_assert(dev::kChunk == MG_SCAN_CHUNK, "the states that callers keep room for");
constexpr uint64_t kMostGroups = 1u << 20;  // workgroups of a launch

uint32_t lanes_of(uint32_t states) {
    uint32_t l = 1;
    while (4 * l < states) l *= 2;
    return l;
}

struct ScanShape {
    uint32_t lanes, per, apiece, blocks, splits, split_steps;
    uint32_t wide;  // channels of a quad, 0 where it is not quads that scan
};
// The steps are split where the channels and sequences alone give fewer than two workgroups
// a CU: each split's steps are walked over twice, which pays once the chip is half idle (1024 steps
// of 256 channels with 16 states, bf16, split and not, us: 16 sequences 55 and 215, 64 160 and 214, 100
// 239 and 256, 128, which are 512 workgroups, 294 and 280; backwards 150 and 731, 529 and 792, 913
// and 964, 1074 and 965). Quads take
// 9 to 64 states (32 steps of 4096 x 256 with 16, bf16: 251 us without them, so 165; the gradient
// 983 and 611), but not rows whose steps lie too far apart for 31 bits, nor the gradient of more than
// 32 (a lane's registers). Two channels each where 16 states leave four workgroups a CU without a split (the
// same with one: 198 and 791), but not where that leaves more lanes without a channel, backwards a third more: us
// of 32 x 4096 bf16 with one and two, 64 channels 46 and 76, 256 in four groups 164 and 260, 160 in one 108 and
// 135; backwards 193 and 279, 768 and 1109, 598 and 573.
ScanShape scan_shape(uint32_t steps, uint32_t seqs, uint32_t channels, uint32_t states, uint32_t groups, bool far,
                     bool backward) {
    ScanShape s;
    s.lanes = lanes_of(states);
    s.wide = !far && s.lanes >= 4 && s.lanes <= (backward ? 8 : 16);
    s.per = channels / groups;
    const uint32_t ch = s.wide ? 64 : 256 / s.lanes;
    s.apiece = (s.per + ch - 1) / ch;
    s.blocks = s.apiece * groups;
    const uint64_t have = (uint64_t)s.blocks * seqs;
    const uint32_t units = (steps + dev::kChunk - 1) / dev::kChunk;
    uint64_t splits = 1;
    if (have && have < 2 * kCus) splits = (4 * kCus + have - 1) / have;
    if (splits > units) splits = units;
    if (splits < 1) splits = 1;
    const uint32_t each = units ? (uint32_t)((units + splits - 1) / splits) : 1;
    s.splits = units ? (units + each - 1) / each : 1;
    s.split_steps = each * dev::kChunk;
    const uint32_t pairs = (s.per + 127) / 128;
    const bool filled = 6 * pairs <= (backward ? 4 : 3) * s.apiece;
    if (s.wide && s.lanes == 4 && filled && s.splits == 1 && (uint64_t)pairs * groups * seqs >= 4 * kCus)
        s.wide = 2, s.apiece = pairs, s.blocks = pairs * groups;
    return s;
}
// Whether eight steps of an array of rows pass 31 bits.
bool lies_far(uint64_t step_rows, uint64_t ld, uint32_t type) {
    return step_rows * ld > (1ull << 27) / type_bytes(type);
}

uint64_t padded(uint64_t bytes) { return (bytes + 255) & ~(uint64_t)255; }
// ends, decays and the saved state of split steps
uint64_t split_bytes(const ScanShape& s, uint64_t seqs, uint64_t channels, uint64_t states) {
    if (s.splits <= 1) return 0;
    return padded(s.splits * seqs * channels * states * 4) + padded(s.splits * seqs * channels * 4) +
           padded(seqs * channels * states * 4);
}
char* place_splits(char* at, const ScanShape& s, dev::ScanArgs& a) {
    if (s.splits <= 1) return at;
    const uint64_t cells = (uint64_t)a.at.seqs * a.channels;
    a.ends = reinterpret_cast<float*>(at), at += padded(s.splits * cells * a.states * 4);
    a.decays = reinterpret_cast<float*>(at), at += padded(s.splits * cells * 4);
    a.saved = reinterpret_cast<float*>(at), at += padded(cells * a.states * 4);
    return at;
}

// Each block's part of dB and dC, where a group has several.
uint64_t shared_bytes(const ScanShape& s, uint64_t steps, uint64_t seqs, uint64_t groups, uint64_t states) {
    return s.apiece > 1 ? padded(s.apiece * steps * seqs * groups * 2 * states * 4) : 0;
}
uint32_t backward_parts(const ScanShape& s, uint32_t seqs) {
    const uint64_t items = (uint64_t)seqs * s.splits, want = (8 * kCus + s.blocks - 1) / s.blocks;
    return (uint32_t)(items < want ? items : want);
}

template <class Fn>
void with_lanes(uint32_t lanes, Fn&& f) {
    switch (lanes) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        case 16: return f(std::integral_constant<int, 16>{});
        case 32: return f(std::integral_constant<int, 32>{});
        default: return f(std::integral_constant<int, 64>{});
    }
}
dim3 grid_of(uint64_t items) { return dim3((uint32_t)(items < kMostGroups ? items : kMostGroups)); }

// f(channels of a quad, vectors of a lane for each) for a shape whose quads scan.
template <class Fn>
void with_quads(const ScanShape& s, Fn&& f) {
    if (s.wide == 2) return f(std::integral_constant<int, 2>{}, std::integral_constant<int, 1>{});
    if (s.lanes == 4) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
    if (s.lanes == 8) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
    f(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
}
template <class Fn>
void with_gate(const void* z, Fn&& f) {
    if (z) return f(std::true_type{});
    f(std::false_type{});
}

template <class T>
int scan(hipStream_t st, const dev::ScanArgs& given, const ScanShape& s) {
    dev::ScanArgs a = given;
    if (a.at.steps <= 1 && !a.checkpoints) {
        if (s.wide) {
            a.apiece = (s.per + 63) / 64, a.blocks = a.apiece * a.groups;
            const uint64_t items = (uint64_t)a.blocks * ((a.at.seqs + 3) / 4);
            with_quads(s, [&](auto, auto ns) {
                with_gate(a.z, [&](auto z) {
                    hipLaunchKernelGGL((dev::scan_quad_step_kernel<T, decltype(ns)::value, decltype(z)::value>),
                                       grid_of(items), dim3(256), 0, st, a, items);
                });
            });
        } else {
            const uint64_t items = (uint64_t)s.blocks * a.at.seqs;
            with_lanes(s.lanes, [&](auto l) {
                hipLaunchKernelGGL((dev::scan_step_kernel<T, decltype(l)::value>), grid_of(items), dim3(256), 0, st, a,
                                   items);
            });
        }
        MG_HIP(hipGetLastError(), "selective scan step launch");
        return MG_OK;
    }
    const uint64_t each = (uint64_t)s.blocks * a.at.seqs, ends = each * (s.splits - 1), all = each * s.splits;
    if (s.wide) {
        with_quads(s, [&](auto c, auto ns) {
            constexpr int C = decltype(c)::value, NS = decltype(ns)::value;
            if constexpr (C == 1)  // pairs of channels have no splits
                if (ends)
                    hipLaunchKernelGGL((dev::scan_quad_kernel<T, C, NS, false, false>), grid_of(ends), dim3(256), 0, st,
                                       a, ends);
            with_gate(a.z, [&](auto z) {
                hipLaunchKernelGGL((dev::scan_quad_kernel<T, C, NS, true, decltype(z)::value>), grid_of(all), dim3(256),
                                   0, st, a, all);
            });
        });
    } else {
        with_lanes(s.lanes, [&](auto l) {
            constexpr int L = decltype(l)::value;
            if (ends) hipLaunchKernelGGL((dev::scan_kernel<T, L, false>), grid_of(ends), dim3(256), 0, st, a, ends);
            hipLaunchKernelGGL((dev::scan_kernel<T, L, true>), grid_of(all), dim3(256), 0, st, a, all);
        });
    }
    MG_HIP(hipGetLastError(), "selective scan launch");
    return MG_OK;
}

template <class T>
int scan_backward(hipStream_t st, const dev::ScanArgs& a, const ScanShape& s, float* da, float* dd, float* dbias) {
    const uint32_t parts = backward_parts(s, a.at.seqs);
    if (parts) {
        const uint64_t ends = (uint64_t)s.blocks * a.at.seqs * (s.splits - 1);
        if (s.wide)
            with_quads(s, [&](auto c, auto ns) {
                constexpr int C = decltype(c)::value, NS = decltype(ns)::value <= 2 ? decltype(ns)::value : 2;
                if constexpr (C == 1)
                    if (ends)
                        hipLaunchKernelGGL((dev::scan_quad_ends_backward_kernel<T, C, NS>), grid_of(ends), dim3(256), 0,
                                           st, a, ends);
                with_gate(a.z, [&](auto z) {
                    hipLaunchKernelGGL((dev::scan_quad_backward_kernel<T, C, NS, decltype(z)::value>),
                                       dim3(s.blocks * parts), dim3(256), 0, st, a, parts);
                });
            });
        else
            with_lanes(s.lanes, [&](auto l) {
                constexpr int L = decltype(l)::value;
                if (ends)
                    hipLaunchKernelGGL((dev::scan_ends_backward_kernel<T, L>), grid_of(ends), dim3(256), 0, st, a, ends);
                hipLaunchKernelGGL((dev::scan_backward_kernel<T, L>), dim3(s.blocks * parts), dim3(256), 0, st, a,
                                   parts);
            });
        MG_HIP(hipGetLastError(), "selective scan backward launch");
        if (s.apiece > 1 && a.at.steps) {
            const uint64_t cells = (uint64_t)a.at.steps * a.at.seqs * a.groups * 2 * a.states;
            const uint64_t blocks = (cells + 255) / 256;
            hipLaunchKernelGGL(dev::scan_shared_kernel<T>, dim3((uint32_t)(blocks < 16 * kCus ? blocks : 16 * kCus)),
                               dim3(256), 0, st, a);
            MG_HIP(hipGetLastError(), "selective scan shared sums launch");
        }
    }
    if (!a.sums) return MG_OK;
    const uint64_t cs = (uint64_t)a.channels * a.states, c = a.channels;
    return sum_parts(st, a.sums, parts, cs + 2 * c, dev::SumTargets{{da, dd, dbias}, {cs, cs + c, cs + 2 * c}},
                     "selective scan sums launch");
}

int check_states(const char* what, uint32_t channels, uint32_t states, uint32_t groups) {
    MG_CHECK(states >= 1 && states <= kMostStates, MG_ERR_INVALID, "%s: states %u must be in [1, %u]", what, states,
             kMostStates);
    MG_CHECK(groups >= 1 && channels % groups == 0, MG_ERR_INVALID, "%s: groups %u must divide channels %u", what,
             groups, channels);
    return MG_OK;
}

// The parts of dB and dC are one for each row of `steps` x `seqs`, of which lengths may leave most out: what no memory
// holds must not wrap around to what some does.
int check_shared(const char* what, const ScanShape& s, uint64_t steps, uint64_t seqs, uint64_t states) {
    const uint64_t row = (uint64_t)s.blocks * 2 * states * 4;
    MG_CHECK(s.apiece <= 1 || steps * seqs <= (1ull << 48) / row, MG_ERR_INVALID,
             "%s: the workspace of %llu steps of %llu seqs would pass 2^48 bytes", what, (unsigned long long)steps,
             (unsigned long long)seqs);
    return MG_OK;
}

// What both directions take alike.
template <class Args>
int check_inputs(const char* what, Args& p, bool any) {
    const uint64_t wide = (uint64_t)p.groups * p.states;
    int rc;
    if ((rc = check_operand(what, "x", p.x, &p.x_ld, p.channels, p.type, any)) ||
        (rc = check_operand(what, "dt", p.dt, &p.dt_ld, p.channels, p.type, any)) ||
        (rc = check_operand(what, "b", p.b, &p.b_ld, wide, p.type, any)) ||
        (rc = check_operand(what, "c", p.c, &p.c_ld, wide, p.type, any)) ||
        (p.z && (rc = check_operand(what, "z", p.z, &p.z_ld, p.channels, p.type, any))) ||
        (rc = check_vector(what, "a", p.a, MG_TYPE_FP32, p.seqs != 0)) ||
        (rc = check_vector(what, "d", p.d, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "dt_bias", p.dt_bias, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "initial", p.initial, MG_TYPE_FP32, false)))
        return rc;
    return MG_OK;
}
template <class Args>
bool inputs_far(const Args& p) {
    return lies_far(p.step_rows, p.x_ld, p.type) || lies_far(p.step_rows, p.dt_ld, p.type) ||
           lies_far(p.step_rows, p.z_ld, p.type);
}
template <class Args>
dev::ScanArgs inputs_of(const Args& p, const ScanShape& s) {
    dev::ScanArgs a{};
    a.at = {p.reset, p.lengths, p.step_rows, p.seq_rows, p.steps, p.seqs};
    a.x = p.x, a.dt = p.dt, a.b = p.b, a.c = p.c, a.z = p.z, a.a = p.a, a.d = p.d, a.dt_bias = p.dt_bias;
    a.initial = p.initial;
    a.x_ld = p.x_ld, a.dt_ld = p.dt_ld, a.b_ld = p.b_ld, a.c_ld = p.c_ld, a.z_ld = p.z_ld;
    a.channels = p.channels, a.states = p.states, a.groups = p.groups;
    a.per = s.per, a.apiece = s.apiece, a.blocks = s.blocks, a.splits = s.splits, a.split_steps = s.split_steps;
    return a;
}

}  // namespace
}  // namespace mg

using namespace mg;

extern "C" {

int mg_selective_scan_workspace(uint32_t steps, uint32_t seqs, uint32_t channels, uint32_t states, uint64_t* bytes) {
    const char* what = "selective scan workspace";
    MG_CHECK(bytes, MG_ERR_INVALID, "%s: null argument", what);
    uint64_t a = 0, b = 0;
    int rc;
    if ((rc = check_rollout(what, steps, seqs, channels, MG_TYPE_FP32, &a, &b, nullptr)) ||
        (rc = check_states(what, channels, states, 1)))
        return rc;
    // more groups make more blocks, and those at most as many splits
    *bytes = 0;
    for (bool far : {false, true}) {
        const uint64_t need = split_bytes(scan_shape(steps, seqs, channels, states, 1, far, false), seqs, channels, states);
        *bytes = need > *bytes ? need : *bytes;
    }
    return MG_OK;
}

int mg_selective_scan(void* stream, const mg_selective_scan_args* args) {
    const char* what = "selective scan";
    MG_CHECK(args, MG_ERR_INVALID, "selective scan: null argument");
    mg_selective_scan_args p = *args;
    int rc;
    if ((rc = check_rollout(what, p.steps, p.seqs, p.channels, p.type, &p.step_rows, &p.seq_rows, p.lengths)) ||
        (rc = check_states(what, p.channels, p.states, p.groups)))
        return rc;
    const bool any = p.steps && p.seqs;
    if ((rc = check_inputs(what, p, any)) ||
        (rc = check_operand(what, "y", p.y, &p.y_ld, p.channels, p.type, any)) ||
        (rc = check_vector(what, "final", p.final, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "checkpoints", p.checkpoints, MG_TYPE_FP32, false)))
        return rc;
    if (!p.seqs || (!p.steps && !p.final)) return MG_OK;
    const ScanShape s = scan_shape(p.steps, p.seqs, p.channels, p.states, p.groups,
                                   inputs_far(p) || lies_far(p.step_rows, p.y_ld, p.type), false);
    if ((rc = check_workspace(what, p.workspace, p.workspace_bytes, split_bytes(s, p.seqs, p.channels, p.states))))
        return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice on;
    if ((rc = on.enter(st, "selective scan: stream device"))) return rc;
    dev::ScanArgs a = inputs_of(p, s);
    a.y = p.y, a.y_ld = p.y_ld, a.final = p.final, a.checkpoints = p.checkpoints;
    place_splits(static_cast<char*>(p.workspace), s, a);
    return p.type == MG_TYPE_FP32   ? scan<float>(st, a, s)
           : p.type == MG_TYPE_BF16 ? scan<__bf16>(st, a, s)
                                    : scan<_Float16>(st, a, s);
}

int mg_selective_scan_backward_workspace(uint32_t steps, uint32_t seqs, uint32_t channels, uint32_t states,
                                         uint32_t groups, uint64_t* bytes) {
    const char* what = "selective scan backward workspace";
    MG_CHECK(bytes, MG_ERR_INVALID, "%s: null argument", what);
    uint64_t a = 0, b = 0;
    int rc;
    if ((rc = check_rollout(what, steps, seqs, channels, MG_TYPE_FP32, &a, &b, nullptr)) ||
        (rc = check_states(what, channels, states, groups)))
        return rc;
    *bytes = 0;
    for (bool far : {false, true}) {
        const ScanShape s = scan_shape(steps, seqs, channels, states, groups, far, true);
        if ((rc = check_shared(what, s, steps, seqs, states))) return rc;
        const uint64_t need = split_bytes(s, seqs, channels, states) + shared_bytes(s, steps, seqs, groups, states) +
                              padded((uint64_t)backward_parts(s, seqs) * channels * (states + 2) * 4);
        *bytes = need > *bytes ? need : *bytes;
    }
    return MG_OK;
}

int mg_selective_scan_backward(void* stream, const mg_selective_scan_backward_args* args) {
    const char* what = "selective scan backward";
    MG_CHECK(args, MG_ERR_INVALID, "selective scan backward: null argument");
    mg_selective_scan_backward_args p = *args;
    int rc;
    if ((rc = check_rollout(what, p.steps, p.seqs, p.channels, p.type, &p.step_rows, &p.seq_rows, p.lengths)) ||
        (rc = check_states(what, p.channels, p.states, p.groups)))
        return rc;
    const bool any = p.steps && p.seqs;
    const uint64_t wide = (uint64_t)p.groups * p.states;
    if ((rc = check_inputs(what, p, any)) ||
        (rc = check_operand(what, "dy", p.dy, &p.dy_ld, p.channels, p.type, any)) ||
        (rc = check_operand(what, "dx", p.dx, &p.dx_ld, p.channels, p.type, any)) ||
        (rc = check_operand(what, "ddt", p.ddt, &p.ddt_ld, p.channels, p.type, any)) ||
        (rc = check_operand(what, "db", p.db, &p.db_ld, wide, p.type, any)) ||
        (rc = check_operand(what, "dc", p.dc, &p.dc_ld, wide, p.type, any)) ||
        (p.z && (rc = check_operand(what, "dz", p.dz, &p.dz_ld, p.channels, p.type, any))) ||
        (rc = check_vector(what, "checkpoints", p.checkpoints, MG_TYPE_FP32, any && p.steps > dev::kChunk)) ||
        (rc = check_vector(what, "dfinal", p.dfinal, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "da", p.da, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "dd", p.dd, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "ddt_bias", p.ddt_bias, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "dinitial", p.dinitial, MG_TYPE_FP32, false)))
        return rc;
    MG_CHECK(p.z || !p.dz, MG_ERR_INVALID, "selective scan backward: dz without z");
    const bool sums = p.da || p.dd || p.ddt_bias;
    if (!sums && (!p.seqs || (!p.steps && !p.dinitial))) return MG_OK;
    const ScanShape s = scan_shape(p.steps, p.seqs, p.channels, p.states, p.groups,
                                   inputs_far(p) || lies_far(p.step_rows, p.dy_ld, p.type) ||
                                       lies_far(p.step_rows, p.dx_ld, p.type) ||
                                       lies_far(p.step_rows, p.ddt_ld, p.type) ||
                                       lies_far(p.step_rows, p.dz_ld, p.type),
                                   true);
    uint64_t need = 0;
    if ((rc = mg_selective_scan_backward_workspace(p.steps, p.seqs, p.channels, p.states, p.groups, &need)) ||
        (rc = check_workspace(what, p.workspace, p.workspace_bytes, need)))
        return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice on;
    if ((rc = on.enter(st, "selective scan backward: stream device"))) return rc;
    dev::ScanArgs a = inputs_of(p, s);
    a.dy = p.dy, a.kept = p.checkpoints, a.dfinal = p.dfinal, a.dx = p.dx, a.ddt = p.ddt, a.db = p.db, a.dc = p.dc;
    a.dz = p.dz, a.dinitial = p.dinitial;
    a.dy_ld = p.dy_ld, a.dx_ld = p.dx_ld, a.ddt_ld = p.ddt_ld, a.db_ld = p.db_ld, a.dc_ld = p.dc_ld, a.dz_ld = p.dz_ld;
    char* at = place_splits(static_cast<char*>(p.workspace), s, a);
    a.shared = reinterpret_cast<float*>(at);
    at += shared_bytes(s, p.steps, p.seqs, p.groups, p.states);
    a.sums = sums ? reinterpret_cast<float*>(at) : nullptr;
    return p.type == MG_TYPE_FP32   ? scan_backward<float>(st, a, s, p.da, p.dd, p.ddt_bias)
           : p.type == MG_TYPE_BF16 ? scan_backward<__bf16>(st, a, s, p.da, p.dd, p.ddt_bias)
                                    : scan_backward<_Float16>(st, a, s, p.da, p.dd, p.ddt_bias);
}

}  // extern "C"
