// Short causal convolution of each channel over a rollout's steps, and its gradients
// (mg_causal_conv, mg_causal_conv_backward).
//
// A thread holds one 16-byte vector of channels and walks over a tile of steps with the
// last taps - 1 inputs in registers, so an input is read once but for the tile's first
// taps - 1 (and, backwards, those past its end). Both are bound by HBM: backwards 32 steps of
// 4096 x 256 fp32 take 89 us, 4.8 TB/s where a large copy reaches 5.1. One step of 4096 x 512 bf16
// takes 11 us, twice its bytes' time: the launch, and the weights that come before the first sum.
#include <type_traits>

#include "sequence.h"

namespace mg {
namespace dev {

struct ConvArgs {
    Rollout at;
    const void* x;
    const float* weight;
    const float* bias;
    void* y;
    const void* initial;
    void* final;
    const void* dy;
    const void* dfinal;
    void* dx;
    void* dinitial;
    float* partial;  // [gridDim.y][channels (taps + 1)]: dweight, then dbias
    uint64_t x_ld, y_ld, dy_ld, dx_ld;
    uint32_t channels, vectors, silu;
    uint32_t lanes;  // threads of a workgroup that lie side by side over vectors: a power of two
    uint32_t tile;   // steps
    uint32_t tiles;
};

template <int E>
__device__ __forceinline__ void clear(float (&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.0f;
}

// The weights and the bias of a thread's channels. Those of a whole vector lie one after the
// other: read one by one they cost a step of 4096 x 512 bf16 9 of its 19 us.
template <int W, int E>
__device__ __forceinline__ void load_taps(const ConvArgs& a, uint32_t v, float (&w)[W][E], float (&bias)[E]) {
    typedef float four __attribute__((ext_vector_type(4), aligned(4)));
    if (v * E + E <= a.channels) {
        const float* const from = a.weight + (size_t)v * E * W;
        float all[E * W];
#pragma unroll
        for (int i = 0; i < E * W; i += 4) {
            const four r = *reinterpret_cast<const four*>(from + i);
#pragma unroll
            for (int q = 0; q < 4; ++q) all[i + q] = r[q];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            bias[e] = 0.0f;
#pragma unroll
            for (int k = 0; k < W; ++k) w[k][e] = all[e * W + k];
        }
        if (!a.bias) return;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const four r = *reinterpret_cast<const four*>(a.bias + (size_t)v * E + e);
#pragma unroll
            for (int q = 0; q < 4; ++q) bias[e + q] = r[q];
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint32_t c = v * E + e;
        const bool in = c < a.channels;
        bias[e] = in && a.bias ? a.bias[c] : 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) w[k][e] = in ? a.weight[(size_t)c * W + k] : 0.0f;
    }
}

// What a thread walks over: sequence n, of `length` steps, its rows of one vector.
template <class T, int W, int FIT>
struct ConvWalk {
    static constexpr int E = 16 / sizeof(T);
    const ConvArgs& a;
    uint32_t v, n, length;

    __device__ __forceinline__ bool reset(uint32_t t) const { return a.at.reset && a.at.reset[a.at.row(t, n)]; }
    __device__ __forceinline__ void row(const void* p, uint64_t ld, uint32_t t, float (&x)[E]) const {
        load_vec<FIT, T, E>(static_cast<const T*>(p) + a.at.row(t, n) * ld, v, a.channels, x);
    }
    // place k of a window of [seqs][taps - 1][channels]
    template <class P>
    __device__ __forceinline__ P* place(P* p, int k) const {
        return p + ((size_t)n * (W - 1) + k) * a.channels;
    }
    // The inputs of the steps before t, zeros before their episode's first. Returns how many
    // of them are of t - 1's episode.
    __device__ __forceinline__ int window(uint32_t t, float (&win)[W - 1][E]) const {
        int live = W - 1;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            const int64_t s = (int64_t)t - (W - 1) + k;
            if (s >= 0)
                row(a.x, a.x_ld, (uint32_t)s, win[k]);
            else if (a.initial)
                load_vec<FIT, T, E>(place(static_cast<const T*>(a.initial), (int)(s + W - 1)), v, a.channels, win[k]);
            else
                clear(win[k]);
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            const int64_t s = (int64_t)t - (W - 1) + k;
            if (s < 0 || !reset((uint32_t)s)) continue;
#pragma unroll
            for (int j = 0; j < k; ++j) clear(win[j]);
            live = W - 1 - k;
        }
        return live;
    }
};

// U: steps whose inputs are read ahead: four for a tile, while a single step would only repeat its
// own reads (4096 x 512 bf16 13.5 us for 12.7, 65536 x 512 182 for 173).
template <class T, int W, int FIT, int U>
__global__ void __launch_bounds__(256) conv_kernel(const ConvArgs a) {
    constexpr int E = 16 / sizeof(T);
    const uint32_t v = blockIdx.x * a.lanes + (threadIdx.x & (a.lanes - 1));
    if (v >= a.vectors) return;
    const uint32_t rows = 256 / a.lanes;
    float w[W][E], bias[E];
    load_taps(a, v, w, bias);
    const uint64_t items = (uint64_t)a.at.seqs * a.tiles;
    for (uint64_t item = (uint64_t)blockIdx.y * rows + threadIdx.x / a.lanes; item < items;
         item += (uint64_t)gridDim.y * rows) {
        const uint32_t tile = (uint32_t)(item / a.at.seqs), n = (uint32_t)(item - (uint64_t)tile * a.at.seqs);
        const ConvWalk<T, W, FIT> walk{a, v, n, a.at.length(n)};
        const uint32_t t0 = tile * a.tile, end = walk.length < t0 + a.tile ? walk.length : t0 + a.tile;
        if (t0 < end) {
            float win[W - 1][E];
            walk.window(t0, win);
            for (uint32_t t = t0; t < end; t += U) {
                float x[U][E];
                bool fresh[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t s = t + u < end ? t + u : end - 1;
                    walk.row(a.x, a.x_ld, s, x[u]);
                    fresh[u] = walk.reset(s);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (t + u >= end) break;
                    if (fresh[u]) {
#pragma unroll
                        for (int k = 0; k < W - 1; ++k) clear(win[k]);
                    }
                    float y[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float s = bias[e];
#pragma unroll
                        for (int k = 0; k < W - 1; ++k) s = __builtin_fmaf(w[k][e], win[k][e], s);
                        s = __builtin_fmaf(w[W - 1][e], x[u][e], s);
                        y[e] = a.silu ? silu(s) : s;
#pragma unroll
                        for (int k = 0; k + 1 < W - 1; ++k) win[k][e] = win[k + 1][e];
                        win[W - 2][e] = x[u][e];
                    }
                    store_vec<FIT, T, E>(static_cast<T*>(a.y) + a.at.row(t + u, n) * a.y_ld, v, a.channels, y);
                }
            }
        }
        // The tile that reads the initial window writes the final one, which may be the
        // same.
        if (tile == 0 && a.final) {
            float last[W - 1][E];
            walk.window(walk.length, last);
#pragma unroll
            for (int k = 0; k < W - 1; ++k)
                store_vec<FIT, T, E>(walk.place(static_cast<T*>(a.final), k), v, a.channels, last[k]);
        }
    }
}

// dpre = dy silu'(pre); dx[s] = sum of w[k] dpre[t] over the steps t that see s at place k.
// A tile takes the steps past its end that see its inputs too, so that each dx is one
// thread's sum; the weights' gradients are of the tile's own steps. `pending` holds the
// sums that later steps still add to.
template <class T, int W, int FIT>
__global__ void __launch_bounds__(256) conv_backward_kernel(const ConvArgs a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float lds[256 * (E + 1)];
    const uint32_t v = blockIdx.x * a.lanes + (threadIdx.x & (a.lanes - 1));
    const bool mine = v < a.vectors;
    const uint32_t rows = 256 / a.lanes;
    float w[W][E], bias[E], dw[W][E], db[E];
    if (mine) load_taps(a, v, w, bias);
#pragma unroll
    for (int k = 0; k < W; ++k) clear(dw[k]);
    clear(db);
    const uint64_t items = mine ? (uint64_t)a.at.seqs * a.tiles : 0;
    for (uint64_t item = (uint64_t)blockIdx.y * rows + threadIdx.x / a.lanes; item < items;
         item += (uint64_t)gridDim.y * rows) {
        const uint32_t tile = (uint32_t)(item / a.at.seqs), n = (uint32_t)(item - (uint64_t)tile * a.at.seqs);
        const ConvWalk<T, W, FIT> walk{a, v, n, a.at.length(n)};
        const uint32_t t0 = tile * a.tile, end = walk.length < t0 + a.tile ? walk.length : t0 + a.tile;
        if (t0 >= end && tile) continue;
        const uint32_t past = walk.length - end < (uint32_t)(W - 1) ? walk.length : end + W - 1;
        float win[W - 1][E], pending[W - 1][E];  // of the places of the window
        int live = walk.window(t0, win);
#pragma unroll
        for (int k = 0; k < W - 1; ++k) clear(pending[k]);
        // what a place holds leaves it complete: step t - (W - 1)
        auto leave = [&](uint32_t t, const float (&d)[E]) {
            const int64_t s = (int64_t)t - (W - 1);
            if (s >= (int64_t)t0 && s < (int64_t)end)
                store_vec<FIT, T, E>(static_cast<T*>(a.dx) + a.at.row((uint32_t)s, n) * a.dx_ld, v, a.channels, d);
            else if (s < 0 && a.dinitial)
                store_vec<FIT, T, E>(walk.place(static_cast<T*>(a.dinitial), (int)(s + W - 1)), v, a.channels, d);
        };
        for (uint32_t t = t0; t < past; t += 2) {
            float xs[2][E], ds[2][E];
            bool fresh[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t s = t + u < past ? t + u : past - 1;
                walk.row(a.x, a.x_ld, s, xs[u]);
                walk.row(a.dy, a.dy_ld, s, ds[u]);
                fresh[u] = walk.reset(s);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (t + u >= past) break;
                if (fresh[u]) {
                    live = 0;
#pragma unroll
                    for (int k = 0; k < W - 1; ++k) clear(win[k]);
                }
                float d[E], gone[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float s = bias[e];
#pragma unroll
                    for (int k = 0; k < W - 1; ++k) s = __builtin_fmaf(w[k][e], win[k][e], s);
                    s = __builtin_fmaf(w[W - 1][e], xs[u][e], s);
                    d[e] = a.silu ? ds[u][e] * silu_slope(s) : ds[u][e];
                }
                if (t + u < end) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
#pragma unroll
                        for (int k = 0; k < W - 1; ++k) dw[k][e] = __builtin_fmaf(d[e], win[k][e], dw[k][e]);
                        dw[W - 1][e] = __builtin_fmaf(d[e], xs[u][e], dw[W - 1][e]);
                        db[e] += d[e];
                    }
                }
#pragma unroll
                for (int k = 0; k < W - 1; ++k)
                    if (W - 1 - k <= live) {
#pragma unroll
                        for (int e = 0; e < E; ++e) pending[k][e] = __builtin_fmaf(w[k][e], d[e], pending[k][e]);
                    }
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    gone[e] = pending[0][e];
#pragma unroll
                    for (int k = 0; k + 1 < W - 1; ++k) pending[k][e] = pending[k + 1][e], win[k][e] = win[k + 1][e];
                    pending[W - 2][e] = w[W - 1][e] * d[e], win[W - 2][e] = xs[u][e];
                }
                live = live < W - 1 ? live + 1 : live;
                leave(t + u, gone);
            }
        }
        // the places that are left: at the sequence's end the final window's own gradient
        // reaches those of the last episode
        const bool ends = past == walk.length && a.dfinal;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            if (ends && W - 1 - k <= live) {
                float d[E];
                load_vec<FIT, T, E>(walk.place(static_cast<const T*>(a.dfinal), k), v, a.channels, d);
#pragma unroll
                for (int e = 0; e < E; ++e) pending[k][e] += d[e];
            }
            leave(past + k, pending[k]);
        }
    }
    if (!a.partial) return;
    // the workgroup's sums, thread row after thread row
    float* const out = a.partial + (size_t)blockIdx.y * a.channels * (W + 1);
#pragma unroll
    for (int k = 0; k <= W; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) lds[threadIdx.x * (E + 1) + e] = k < W ? dw[k][e] : db[e];
        __syncthreads();
        if (threadIdx.x >= a.lanes || !mine) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float s = lds[threadIdx.x * (E + 1) + e];
            for (uint32_t r = 1; r < rows; ++r) s += lds[(r * a.lanes + threadIdx.x) * (E + 1) + e];
            const uint32_t c = v * E + e;
            if (c < a.channels) out[k < W ? (size_t)c * W + k : (size_t)a.channels * W + c] = s;
        }
    }
}

}  // namespace dev

namespace {

constexpr uint32_t kConvParts = 4 * kCus;  // most workgroups that leave a partial row of a channel

struct ConvShape {
    uint32_t vectors, lanes, columns, tile, tiles;
    uint64_t groups;  // of thread rows over (sequence, tile)
};
ConvShape conv_shape(uint32_t steps, uint32_t seqs, uint32_t channels, uint32_t type, bool backward) {
    ConvShape s;
    const uint32_t e = 16 / type_bytes(type);
    s.vectors = (channels + e - 1) / e;
    for (s.lanes = 1; s.lanes < 256 && s.lanes < s.vectors;) s.lanes *= 2;
    s.columns = (s.vectors + s.lanes - 1) / s.lanes;
    s.tile = 32;
    // A tile of 8 steps reads 3 inputs more than it needs (and, backwards, their gradients), one of 32
    // as many; the shorter gives four times the threads where those of 32 steps would leave the chip
    // idle. us, 8 first: forward bf16 1000 x 64 x 256 20 and 29, 32 x 4096 x 256 35 and 34; backward 32 x
    // 512 x 256 34 and 53, 1000 x 64 x 256 74 and 65, 32 x 4096 x 256 102 and 73.
    if ((uint64_t)seqs * s.vectors * ((steps + 31) / 32) < kCus * (backward ? 256 : 512)) s.tile = 8;
    s.tiles = steps ? (steps + s.tile - 1) / s.tile : 1;
    const uint64_t items = (uint64_t)seqs * s.tiles, rows = 256 / s.lanes;
    s.groups = (items + rows - 1) / rows;
    return s;
}

template <class T, class Fn>
void with_fit(uint32_t channels, Fn&& f) {
    constexpr uint32_t E = 16 / sizeof(T);
    if (channels % E == 0) return f(std::integral_constant<int, dev::kFull>{});
    if (channels < E) return f(std::integral_constant<int, dev::kTiny>{});
    f(std::integral_constant<int, dev::kTail>{});
}
template <class Fn>
void with_taps(uint32_t taps, Fn&& f) {
    if (taps == 2) return f(std::integral_constant<int, 2>{});
    if (taps == 3) return f(std::integral_constant<int, 3>{});
    f(std::integral_constant<int, 4>{});
}

template <class T>
int conv(hipStream_t st, const dev::ConvArgs& a, uint32_t taps, const ConvShape& s) {
    const dim3 grid(s.columns, (uint32_t)(s.groups < 65535 ? s.groups : 65535));
    with_fit<T>(a.channels, [&](auto fit) {
        with_taps(taps, [&](auto w) {
            constexpr int W = decltype(w)::value, F = decltype(fit)::value;
            if (a.at.steps <= 1)
                hipLaunchKernelGGL((dev::conv_kernel<T, W, F, 1>), grid, dim3(256), 0, st, a);
            else
                hipLaunchKernelGGL((dev::conv_kernel<T, W, F, 4>), grid, dim3(256), 0, st, a);
        });
    });
    MG_HIP(hipGetLastError(), "causal conv launch");
    return MG_OK;
}

uint32_t conv_parts(const ConvShape& s) { return (uint32_t)(s.groups < kConvParts ? s.groups : kConvParts); }

template <class T>
int conv_backward(hipStream_t st, const dev::ConvArgs& a, uint32_t taps, const ConvShape& s, float* dweight,
                  float* dbias) {
    const uint32_t parts = conv_parts(s);
    if (parts) {
        with_fit<T>(a.channels, [&](auto fit) {
            with_taps(taps, [&](auto w) {
                hipLaunchKernelGGL((dev::conv_backward_kernel<T, decltype(w)::value, decltype(fit)::value>),
                                   dim3(s.columns, parts), dim3(256), 0, st, a);
            });
        });
        MG_HIP(hipGetLastError(), "causal conv backward launch");
    }
    if (!dweight && !dbias) return MG_OK;
    const uint64_t cw = (uint64_t)a.channels * taps, width = cw + a.channels;
    return sum_parts(st, a.partial, parts, width, dev::SumTargets{{dweight, dbias, nullptr}, {cw, width, width}},
                     "causal conv sums launch");
}

int check_taps(const char* what, uint32_t taps) {
    MG_CHECK(taps >= 2 && taps <= 4, MG_ERR_INVALID, "%s: taps %u must be 2, 3 or 4", what, taps);
    return MG_OK;
}

}  // namespace
}  // namespace mg

using namespace mg;

extern "C" {

int mg_causal_conv(void* stream, const mg_causal_conv_args* args) {
    const char* what = "causal conv";
    MG_CHECK(args, MG_ERR_INVALID, "causal conv: null argument");
    mg_causal_conv_args p = *args;
    int rc;
    if ((rc = check_rollout(what, p.steps, p.seqs, p.channels, p.type, &p.step_rows, &p.seq_rows, p.lengths)) ||
        (rc = check_taps(what, p.taps)))
        return rc;
    const bool any = p.steps && p.seqs;
    if ((rc = check_operand(what, "x", p.x, &p.x_ld, p.channels, p.type, any)) ||
        (rc = check_operand(what, "y", p.y, &p.y_ld, p.channels, p.type, any)) ||
        (rc = check_vector(what, "weight", p.weight, MG_TYPE_FP32, any)) ||
        (rc = check_vector(what, "bias", p.bias, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "initial", p.initial, p.type, false)) ||
        (rc = check_vector(what, "final", p.final, p.type, false)))
        return rc;
    if (!p.seqs || (!p.steps && !p.final)) return MG_OK;
    MG_CHECK(p.weight, MG_ERR_INVALID, "causal conv: weight is NULL");
    hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice on;
    if ((rc = on.enter(st, "causal conv: stream device"))) return rc;
    const ConvShape s = conv_shape(p.steps, p.seqs, p.channels, p.type, false);
    dev::ConvArgs a{};
    a.at = {p.reset, p.lengths, p.step_rows, p.seq_rows, p.steps, p.seqs};
    a.x = p.x, a.weight = p.weight, a.bias = p.bias, a.y = p.y, a.initial = p.initial, a.final = p.final;
    a.x_ld = p.x_ld, a.y_ld = p.y_ld, a.channels = p.channels, a.silu = p.silu;
    a.vectors = s.vectors, a.lanes = s.lanes, a.tile = s.tile, a.tiles = s.tiles;
    return p.type == MG_TYPE_FP32   ? conv<float>(st, a, p.taps, s)
           : p.type == MG_TYPE_BF16 ? conv<__bf16>(st, a, p.taps, s)
                                    : conv<_Float16>(st, a, p.taps, s);
}

int mg_causal_conv_backward_workspace(uint32_t steps, uint32_t seqs, uint32_t channels, uint32_t taps,
                                      uint64_t* bytes) {
    const char* what = "causal conv backward workspace";
    MG_CHECK(bytes, MG_ERR_INVALID, "%s: null argument", what);
    uint64_t a = 0, b = 0;
    int rc;
    if ((rc = check_rollout(what, steps, seqs, channels, MG_TYPE_FP32, &a, &b, nullptr)) ||
        (rc = check_taps(what, taps)))
        return rc;
    // the partial rows of whichever type has more
    const uint32_t wide = conv_parts(conv_shape(steps, seqs, channels, MG_TYPE_FP32, true));
    const uint32_t narrow = conv_parts(conv_shape(steps, seqs, channels, MG_TYPE_BF16, true));
    *bytes = (uint64_t)(wide > narrow ? wide : narrow) * channels * (taps + 1) * 4;
    return MG_OK;
}

int mg_causal_conv_backward(void* stream, const mg_causal_conv_backward_args* args) {
    const char* what = "causal conv backward";
    MG_CHECK(args, MG_ERR_INVALID, "causal conv backward: null argument");
    mg_causal_conv_backward_args p = *args;
    int rc;
    if ((rc = check_rollout(what, p.steps, p.seqs, p.channels, p.type, &p.step_rows, &p.seq_rows, p.lengths)) ||
        (rc = check_taps(what, p.taps)))
        return rc;
    const bool any = p.steps && p.seqs;
    if ((rc = check_operand(what, "x", p.x, &p.x_ld, p.channels, p.type, any)) ||
        (rc = check_operand(what, "dy", p.dy, &p.dy_ld, p.channels, p.type, any)) ||
        (rc = check_operand(what, "dx", p.dx, &p.dx_ld, p.channels, p.type, any)) ||
        (rc = check_vector(what, "weight", p.weight, MG_TYPE_FP32, p.seqs != 0)) ||
        (rc = check_vector(what, "bias", p.bias, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "initial", p.initial, p.type, false)) ||
        (rc = check_vector(what, "dfinal", p.dfinal, p.type, false)) ||
        (rc = check_vector(what, "dinitial", p.dinitial, p.type, false)) ||
        (rc = check_vector(what, "dweight", p.dweight, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "dbias", p.dbias, MG_TYPE_FP32, false)))
        return rc;
    const ConvShape s = conv_shape(p.steps, p.seqs, p.channels, p.type, true);
    const bool sums = p.dweight || p.dbias;
    if (sums) {
        uint64_t need = 0;
        mg_causal_conv_backward_workspace(p.steps, p.seqs, p.channels, p.taps, &need);
        if ((rc = check_workspace(what, p.workspace, p.workspace_bytes, need))) return rc;
    } else if (!p.seqs || (!p.steps && !p.dinitial)) {
        return MG_OK;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice on;
    if ((rc = on.enter(st, "causal conv backward: stream device"))) return rc;
    dev::ConvArgs a{};
    a.at = {p.reset, p.lengths, p.step_rows, p.seq_rows, p.steps, p.seqs};
    a.x = p.x, a.weight = p.weight, a.bias = p.bias, a.initial = p.initial;
    a.dy = p.dy, a.dfinal = p.dfinal, a.dx = p.dx, a.dinitial = p.dinitial;
    a.partial = sums ? static_cast<float*>(p.workspace) : nullptr;
    a.x_ld = p.x_ld, a.dy_ld = p.dy_ld, a.dx_ld = p.dx_ld, a.channels = p.channels, a.silu = p.silu;
    a.vectors = s.vectors, a.lanes = s.lanes, a.tile = s.tile, a.tiles = s.tiles;
    return p.type == MG_TYPE_FP32   ? conv_backward<float>(st, a, p.taps, s, p.dweight, p.dbias)
           : p.type == MG_TYPE_BF16 ? conv_backward<__bf16>(st, a, p.taps, s, p.dweight, p.dbias)
                                    : conv_backward<_Float16>(st, a, p.taps, s, p.dweight, p.dbias);
}

}  // extern "C"
