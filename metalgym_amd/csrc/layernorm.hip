// LayerNorm forward and backward for rows of any width (mg_layernorm,
// mg_layernorm_backward).
//
// Both read each row once into registers: a group of G lanes holds a row as V
// 16-byte vectors a lane, so the mean, the centred second moment and the output
// come from one pass over memory. Rows of up to 1024 columns take a group inside
// a wave (its sums are lane exchanges, no barrier), up to 16384 a workgroup; a
// group walks over rows with gamma (and beta, or the gradient's sums) in its
// registers; the backward of 8193 to 16384 columns, and of 513 to 1023 in fp32, has more
// values a lane than registers and keeps some in scratch (28 to 172 bytes a lane, 12 at
// 513 to 1023). Wider rows are read again from L2 for each pass. The kernels are
// bound by HBM: 131072 x 128 fp32 with a residual 42 us (6.4 TB/s, where a copy of
// 1 GiB reaches 5.0), 4095 x 8192 bf16 44, the backward of 262144 x 128 100 us (5.4).
// Small calls are launches: 64 x 128 2.4 us, the backward of 4096 x 128 4.6 + 3.3.
//
// The backward's dgamma and dbeta are sums over all rows. Each lane adds its
// rows' terms for the columns it holds; a workgroup adds its groups' sums and
// writes one partial row, and a second launch adds the partial rows in fixed
// order: chains of rows / (groups of the grid) terms, 32 slices of up to 32 partial
// rows, then the slices, with no atomics.
#include <type_traits>

#include "kernels.h"
#include "mg/device/common.h"
#include "operator_types.h"

namespace mg {
namespace dev {

struct NormArgs {
    const void* x;
    const void* residual;
    void* sum;
    const float* gamma;
    const float* beta;
    void* y;
    float* mean;
    float* rstd;
    size_t x_ld, residual_ld, sum_ld, y_ld;
    uint32_t rows, cols;
    float eps;
};

struct NormGradArgs {
    const void* x;
    const void* dy;
    const void* dsum;
    const float* gamma;
    const float* mean;
    const float* rstd;
    void* dx;
    float* dgamma;  // where the grid is one workgroup, else NULL
    float* dbeta;
    float* partial;  // [gridDim.x][2][cols], or NULL
    size_t x_ld, dy_ld, dsum_ld, dx_ld;
    uint32_t rows, cols;
};

// Sums of N values over a group of G lanes, or over the workgroup (G = NT): the
// waves' sums meet in LDS, added in order by every thread. red holds two sets, so
// that one barrier a sum is enough: `turn` alternates.
template <int G, int NT, int N>
__device__ __forceinline__ void norm_sum(float (&v)[N], float (*red)[N][NT / 64], int turn) {
    if constexpr (G <= 64) {
        group_sum_n<G>(v);
    } else {
        group_sum_n<64>(v);
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red[turn][i][wave] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = red[turn][i][0];
#pragma unroll
            for (int w = 1; w < NT / 64; ++w) s += red[turn][i][w];
            v[i] = s;
        }
    }
}

template <int FIT, int V, int E>
__device__ __forceinline__ void load_vector_param(const float* p, float fill, uint32_t v0, uint32_t stride,
                                                  uint32_t cols, float (&out)[V][E]) {
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const uint32_t c = (v0 + k * stride) * E + e;
            float q[4] = {fill, fill, fill, fill};
            if (p) load_vec<FIT>(p, c / 4, cols, q);
#pragma unroll
            for (int u = 0; u < 4; ++u) out[k][e + u] = q[u];
        }
}

// E consecutive floats from column c.
template <int FIT, int E>
__device__ __forceinline__ void store_floats(float* out, uint32_t c, uint32_t cols, const float (&x)[E]) {
#pragma unroll
    for (int e = 0; e < E; e += 4) {
        const float q[4] = {x[e], x[e + 1], x[e + 2], x[e + 3]};
        store_vec<FIT>(out, (c + e) / 4, cols, q);
    }
}

// FIT: kFull where cols = G V E.
template <class T, int G, int V, int NT, int FIT>
__global__ void __launch_bounds__(NT) layernorm_kernel(const NormArgs a) {
    constexpr int E = 16 / sizeof(T), RP = NT / G;  // rows of a workgroup's pass
    __shared__ float red[2][1][NT / 64];
    const uint32_t t = threadIdx.x % G, cols = a.cols;
    const float n = (float)cols;
    float gamma[V][E], beta[V][E];
    load_vector_param<FIT>(a.gamma, 1.0f, t, G, cols, gamma);
    load_vector_param<FIT>(a.beta, 0.0f, t, G, cols, beta);
    for (uint64_t base = (uint64_t)blockIdx.x * RP; base < a.rows; base += (uint64_t)gridDim.x * RP) {
        // groups past the last row repeat it without a store: lane exchanges need every lane
        const uint64_t want = base + threadIdx.x / G;
        const bool live = want < a.rows;
        const uint64_t r = live ? want : a.rows - 1;
        const T* x = static_cast<const T*>(a.x) + r * a.x_ld;
        float v[V][E];
#pragma unroll
        for (int k = 0; k < V; ++k) load_vec<FIT>(x, t + k * G, cols, v[k]);
        if (a.residual) {
            const T* res = static_cast<const T*>(a.residual) + r * a.residual_ld;
            T* sum = static_cast<T*>(a.sum) + r * a.sum_ld;
            float w[V][E];
#pragma unroll
            for (int k = 0; k < V; ++k) load_vec<FIT>(res, t + k * G, cols, w[k]);
#pragma unroll
            for (int k = 0; k < V; ++k) {
#pragma unroll
                for (int e = 0; e < E; ++e) v[k][e] = (float)(T)(v[k][e] + w[k][e]);  // normalised as stored
                if (live) store_vec<FIT>(sum, t + k * G, cols, v[k]);
            }
        }
        float s[1] = {};
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) s[0] += v[k][e];
        norm_sum<G, NT>(s, red, 0);
        const float mean = s[0] / n;
        float q[1] = {};
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                v[k][e] -= mean;
                if (FIT == kFull || (t + k * G) * E + e < cols) q[0] += v[k][e] * v[k][e];
            }
        norm_sum<G, NT>(q, red, 1);
        const float rstd = 1.0f / sqrtf(q[0] / n + a.eps);
        if (!live) continue;
        T* y = static_cast<T*>(a.y) + r * a.y_ld;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = v[k][e] * rstd * gamma[k][e] + beta[k][e];
            store_vec<FIT>(y, t + k * G, cols, o);
        }
        if (t == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// Rows of more columns than a workgroup's registers hold: one workgroup a row,
// the row read once from HBM and again from L2 for the second moment and the
// output (with a residual, from the sum that the first pass wrote: each thread
// reads what it wrote itself).
template <class T, int NT>
__global__ void __launch_bounds__(NT) layernorm_wide_kernel(const NormArgs a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float red[2][1][NT / 64];
    const uint32_t cols = a.cols, nv = (cols + E - 1) / E;
    const float n = (float)cols;
    for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + r * a.x_ld;
        float s[1] = {};
        for (uint32_t v = threadIdx.x; v < nv; v += NT) {
            float u[E];
            load_vec<kTail>(x, v, cols, u);
            if (a.residual) {
                float w[E];
                load_vec<kTail>(static_cast<const T*>(a.residual) + r * a.residual_ld, v, cols, w);
#pragma unroll
                for (int e = 0; e < E; ++e) u[e] = (float)(T)(u[e] + w[e]);
                store_vec<kTail>(static_cast<T*>(a.sum) + r * a.sum_ld, v, cols, u);
            }
            float p = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) p += u[e];
            s[0] += p;
        }
        if (a.residual) x = static_cast<const T*>(a.sum) + r * a.sum_ld;
        norm_sum<NT, NT>(s, red, 0);
        const float mean = s[0] / n;
        float q[1] = {};
        for (uint32_t v = threadIdx.x; v < nv; v += NT) {
            float u[E], p = 0.0f;
            load_vec<kTail>(x, v, cols, u);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (v * E + e < cols) p += (u[e] - mean) * (u[e] - mean);
            q[0] += p;
        }
        norm_sum<NT, NT>(q, red, 1);
        const float rstd = 1.0f / sqrtf(q[0] / n + a.eps);
        for (uint32_t v = threadIdx.x; v < nv; v += NT) {
            float u[E], gamma[1][E], beta[1][E];
            load_vec<kTail>(x, v, cols, u);
            load_vector_param<kTail>(a.gamma, 1.0f, v, 0, cols, gamma);
            load_vector_param<kTail>(a.beta, 0.0f, v, 0, cols, beta);
#pragma unroll
            for (int e = 0; e < E; ++e) u[e] = (u[e] - mean) * rstd * gamma[0][e] + beta[0][e];
            store_vec<kTail>(static_cast<T*>(a.y) + r * a.y_ld, v, cols, u);
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// At 16 floats a lane and a short vector, gamma is read again for each row, from L1:
// held, it takes the kernel past 128 registers, with which two workgroups fit a CU
// (10007 x 1001 binary16: 22.9 us, so 20.0). Without short vectors the second workgroup
// gains less than the reads cost (100000 x 1024: 117 us, so 121).
template <class T, int G, int V, int NT, int FIT>
__global__ void __launch_bounds__(NT, G <= 64 && FIT == kTail ? 4 : 1) layernorm_backward_kernel(const NormGradArgs a) {
    constexpr int E = 16 / sizeof(T), RP = NT / G, W = NT / 64;
    // the workgroup's sums of its waves (groups inside a wave), or norm_sum's sets
    constexpr int LDS = G <= 64 ? W * 2 * G * V * E : 2 * 2 * W;
    __shared__ float lds[LDS];
    auto* red = reinterpret_cast<float(*)[2][W]>(lds);
    const uint32_t t = threadIdx.x % G, cols = a.cols;
    const float inv_n = 1.0f / (float)cols;
    float gamma[V][E], sg[V][E] = {}, sb[V][E] = {};
    constexpr bool HOLD = G > 64 || V * E <= 8 || FIT == kFull;
    if (HOLD) load_vector_param<FIT>(a.gamma, 1.0f, t, G, cols, gamma);
    int turn = 0;
    for (uint64_t base = (uint64_t)blockIdx.x * RP; base < a.rows; base += (uint64_t)gridDim.x * RP) {
        const uint64_t want = base + threadIdx.x / G;
        const bool live = want < a.rows;
        const uint64_t r = live ? want : a.rows - 1;
        const T* xr = static_cast<const T*>(a.x) + r * a.x_ld;
        const T* dyr = static_cast<const T*>(a.dy) + r * a.dy_ld;
        float x[V][E], d[V][E];
#pragma unroll
        for (int k = 0; k < V; ++k) load_vec<FIT>(xr, t + k * G, cols, x[k]);
#pragma unroll
        for (int k = 0; k < V; ++k) load_vec<FIT>(dyr, t + k * G, cols, d[k]);
        if (!HOLD) load_vector_param<FIT>(a.gamma, 1.0f, t, G, cols, gamma);
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s[2] = {};
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                // a repeated row may be read while its dx is written over it: it adds nothing.
                // Nor does what lies past the row's end: -mean rstd may be infinite where no
                // element's xn is, and infinity times its d = 0 is NaN.
                const bool in = live && (FIT == kFull || (t + k * G) * E + e < cols);
                const float xn = in ? (x[k][e] - mean) * rstd : 0.0f, dy = live ? d[k][e] : 0.0f;
                sg[k][e] += dy * xn;
                sb[k][e] += dy;
                x[k][e] = xn;
                d[k][e] = dy * gamma[k][e];
                s[0] += d[k][e];
                s[1] += d[k][e] * xn;
            }
        norm_sum<G, NT>(s, red, turn);
        turn ^= 1;
        if (!live) continue;
        const float m0 = s[0] * inv_n, m1 = s[1] * inv_n;
        T* dx = static_cast<T*>(a.dx) + r * a.dx_ld;
        const T* dsum = a.dsum ? static_cast<const T*>(a.dsum) + r * a.dsum_ld : nullptr;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float o[E] = {};
            if (dsum) load_vec<FIT>(dsum, t + k * G, cols, o);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += rstd * (d[k][e] - m0 - x[k][e] * m1);
            store_vec<FIT>(dx, t + k * G, cols, o);
        }
    }
    float* out_g = a.partial ? a.partial + (size_t)blockIdx.x * 2 * cols : a.dgamma;
    float* out_b = a.partial ? out_g + cols : a.dbeta;
    if (!out_g && !out_b) return;
    if constexpr (G <= 64) {
        // the groups of a wave by lane exchanges, the waves through LDS
#pragma unroll
        for (int step = G; step < 64; step *= 2)
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    sg[k][e] += __shfl_xor(sg[k][e], step);
                    sb[k][e] += __shfl_xor(sb[k][e], step);
                }
        float* mine = lds + (threadIdx.x >> 6) * 2 * G * V * E;
        if ((threadIdx.x & 63) < G)
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    mine[(t + k * G) * E + e] = sg[k][e];
                    mine[G * V * E + (t + k * G) * E + e] = sb[k][e];
                }
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < 2 * G * V * E; c += NT) {
            float sum = lds[c];
#pragma unroll
            for (int w = 1; w < W; ++w) sum += lds[w * 2 * G * V * E + c];
            const uint32_t col = c % (G * V * E);
            float* out = c < G * V * E ? out_g : out_b;
            if (out && col < cols) out[col] = sum;
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            if (out_g) store_floats<FIT>(out_g, (t + k * G) * E, cols, sg[k]);
            if (out_b) store_floats<FIT>(out_b, (t + k * G) * E, cols, sb[k]);
        }
    }
}

// dx of rows wider than a workgroup's registers: the row's two sums, then dx with
// x, dy from L2. dgamma and dbeta come from layernorm_columns_kernel.
template <class T, int NT>
__global__ void __launch_bounds__(NT) layernorm_backward_wide_kernel(const NormGradArgs a) {
    constexpr int E = 16 / sizeof(T);
    __shared__ float red[2][2][NT / 64];
    const uint32_t cols = a.cols, nv = (cols + E - 1) / E;
    const float inv_n = 1.0f / (float)cols;
    int turn = 0;
    for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* xr = static_cast<const T*>(a.x) + r * a.x_ld;
        const T* dyr = static_cast<const T*>(a.dy) + r * a.dy_ld;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s[2] = {};
        for (uint32_t v = threadIdx.x; v < nv; v += NT) {
            float x[E], d[E], gamma[1][E], p0 = 0.0f, p1 = 0.0f;
            load_vec<kTail>(xr, v, cols, x);
            load_vec<kTail>(dyr, v, cols, d);
            load_vector_param<kTail>(a.gamma, 1.0f, v, 0, cols, gamma);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float g = gamma[0][e] * d[e];  // 0 past the row's end, where -mean rstd may be infinite
                p0 += g;
                p1 += g * (v * E + e < cols ? (x[e] - mean) * rstd : 0.0f);
            }
            s[0] += p0;
            s[1] += p1;
        }
        norm_sum<NT, NT>(s, red, turn);
        turn ^= 1;
        const float m0 = s[0] * inv_n, m1 = s[1] * inv_n;
        for (uint32_t v = threadIdx.x; v < nv; v += NT) {
            float x[E], d[E], gamma[1][E], o[E] = {};
            load_vec<kTail>(xr, v, cols, x);
            load_vec<kTail>(dyr, v, cols, d);
            load_vector_param<kTail>(a.gamma, 1.0f, v, 0, cols, gamma);
            if (a.dsum) load_vec<kTail>(static_cast<const T*>(a.dsum) + r * a.dsum_ld, v, cols, o);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float g = gamma[0][e] * d[e];
                o[e] += rstd * (g - m0 - (x[e] - mean) * rstd * m1);
            }
            store_vec<kTail>(static_cast<T*>(a.dx) + r * a.dx_ld, v, cols, o);
        }
    }
}

// Partial sums of dgamma and dbeta by columns: a thread holds one vector of
// columns and adds the rows blockIdx.y, blockIdx.y + gridDim.y, ... It runs
// before the wide dx kernel, whose dx may lie over x or dy.
template <class T>
__global__ void __launch_bounds__(256) layernorm_columns_kernel(const NormGradArgs a) {
    constexpr int E = 16 / sizeof(T);
    const uint32_t v = blockIdx.x * 256 + threadIdx.x, cols = a.cols;
    if (v * E >= cols) return;
    float sg[E] = {}, sb[E] = {};
#pragma unroll 4
    for (uint64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        float x[E], dy[E];
        load_vec<kTail>(static_cast<const T*>(a.x) + r * a.x_ld, v, cols, x);
        load_vec<kTail>(static_cast<const T*>(a.dy) + r * a.dy_ld, v, cols, dy);
        const float mean = a.mean[r], rstd = a.rstd[r];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            sg[e] += dy[e] * ((x[e] - mean) * rstd);
            sb[e] += dy[e];
        }
    }
    float* out = a.partial + (size_t)blockIdx.y * 2 * cols;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (v * E + e < cols) out[v * E + e] = sg[e], out[cols + v * E + e] = sb[e];
}

// Adds the partial rows: 32 columns a workgroup, 32 slices of the partial rows,
// each added in order, then the slices in order.
__global__ void __launch_bounds__(1024) layernorm_reduce_kernel(const float* __restrict__ partial, uint32_t parts,
                                                                uint32_t cols, float* dgamma, float* dbeta) {
    __shared__ float lds[32][33];
    const uint32_t lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const uint64_t c = (uint64_t)blockIdx.x * 32 + lane, width = 2 * (uint64_t)cols;
    float s = 0.0f;
    if (c < width) {
#pragma unroll 8
        for (uint32_t p = slice; p < parts; p += 32) s += partial[p * width + c];
    }
    lds[slice][lane] = s;
    __syncthreads();
    if (slice == 0 && c < width) {
        s = lds[0][lane];
#pragma unroll
        for (int k = 1; k < 32; ++k) s += lds[k][lane];
        float* out = c < cols ? dgamma : dbeta;
        if (out) out[c < cols ? c : c - cols] = s;
    }
}

}  // namespace dev

namespace {

constexpr uint32_t kCus = 256;
constexpr uint32_t kNormCols = 16384;  // the widest row in a workgroup's registers
constexpr uint32_t kBackwardWaveNT = 512;  // threads of a backward workgroup whose groups lie inside waves
constexpr uint32_t kBackwardWaveParts = 2 * kCus;
constexpr uint32_t kWideParts = 64;  // row slices of layernorm_columns_kernel

// Lanes of a row's group: 8 floats a lane, so that a group reaches 512 columns
// inside a wave, and 16 where that keeps a row in one wave (1024) or one
// workgroup (16384). Both types hold the same columns a lane.
struct NormShape {
    uint32_t group, floats;
};
NormShape norm_shape(uint32_t cols) {
    for (uint32_t g = 4; g <= 64; g *= 2)
        if (cols <= g * 8) return {g, 8};
    if (cols <= 1024) return {64, 16};
    for (uint32_t g = 256; g <= 1024; g *= 2)
        if (cols <= g * 8) return {g, 8};
    return {1024, 16};
}

// Workgroups of the backward pass, each of which writes a partial row: two a CU
// where a workgroup holds many rows; one a CU (of up to 1024 threads) for wide
// rows, whose partial rows are traffic. Workgroups of 256 threads (1025 to 2048 columns)
// are two waves a SIMD at two a CU; they go four a CU where each then has eight rows:
// 22369 x 1500 fp32 120 us with two a CU, 87 with four; 4000 x 1500 bf16 17.9 and 18.9.
uint32_t backward_parts(uint32_t rows, uint32_t cols) {
    if (!rows) return 0;
    if (cols > kNormCols) return rows < kWideParts ? rows : kWideParts;
    const NormShape s = norm_shape(cols);
    const uint32_t per = s.group <= 64 ? kBackwardWaveNT / s.group : 1;
    const uint32_t most = s.group <= 64                             ? kBackwardWaveParts
                          : s.group == 1024                         ? kCus
                          : s.group == 256 && rows >= 8 * 4 * kCus ? 4 * kCus
                                                                    : 2 * kCus;
    const uint64_t need = ((uint64_t)rows + per - 1) / per;
    return need < most ? (uint32_t)need : most;
}

// f(how rows of cols lie in groups of G lanes and F floats a lane, in vectors of E)
template <int G, int F, int E, class Fn>
void with_fit(uint32_t cols, Fn&& f) {
    if (cols == (uint32_t)(G * F)) return f(std::integral_constant<int, dev::kFull>{});
    if constexpr (G == 4)
        if (cols < (uint32_t)E) return f(std::integral_constant<int, dev::kTiny>{});
    f(std::integral_constant<int, dev::kTail>{});
}

template <class T, int G, int F>
void launch_norm(hipStream_t st, const dev::NormArgs& a) {
    constexpr int E = 16 / sizeof(T), V = F / E, NT = G <= 64 ? 256 : G;
    const uint64_t need = ((uint64_t)a.rows + NT / G - 1) / (NT / G), most = kCus * 2048 / NT;
    const dim3 grid((uint32_t)(need < most ? need : most)), block(NT);
    with_fit<G, F, E>(a.cols, [&](auto fit) {
        hipLaunchKernelGGL((dev::layernorm_kernel<T, G, V, NT, decltype(fit)::value>), grid, block, 0, st, a);
    });
}

template <class T, int G, int F>
void launch_norm_backward(hipStream_t st, const dev::NormGradArgs& a, uint32_t parts) {
    constexpr int E = 16 / sizeof(T), V = F / E, NT = G <= 64 ? (int)kBackwardWaveNT : G;
    with_fit<G, F, E>(a.cols, [&](auto fit) {
        hipLaunchKernelGGL((dev::layernorm_backward_kernel<T, G, V, NT, decltype(fit)::value>), dim3(parts), dim3(NT), 0,
                           st, a);
    });
}

// Calls f.template operator()<G, F>() for the shape's constants.
template <class F>
void with_shape(NormShape s, F&& f) {
    switch (s.group) {
        case 4: return f.template operator()<4, 8>();
        case 8: return f.template operator()<8, 8>();
        case 16: return f.template operator()<16, 8>();
        case 32: return f.template operator()<32, 8>();
        case 64: return s.floats == 8 ? f.template operator()<64, 8>() : f.template operator()<64, 16>();
        case 256: return f.template operator()<256, 8>();
        case 512: return f.template operator()<512, 8>();
        default: return s.floats == 8 ? f.template operator()<1024, 8>() : f.template operator()<1024, 16>();
    }
}

template <class T>
struct NormLauncher {
    hipStream_t st;
    const dev::NormArgs& a;
    template <int G, int F>
    void operator()() const {
        launch_norm<T, G, F>(st, a);
    }
};
template <class T>
struct NormBackwardLauncher {
    hipStream_t st;
    const dev::NormGradArgs& a;
    uint32_t parts;
    template <int G, int F>
    void operator()() const {
        launch_norm_backward<T, G, F>(st, a, parts);
    }
};

template <class T>
int layernorm(hipStream_t st, const dev::NormArgs& a) {
    if (a.cols > kNormCols)
        hipLaunchKernelGGL((dev::layernorm_wide_kernel<T, 1024>), dim3(a.rows < 2 * kCus ? a.rows : 2 * kCus),
                           dim3(1024), 0, st, a);
    else
        with_shape(norm_shape(a.cols), NormLauncher<T>{st, a});
    MG_HIP(hipGetLastError(), "layernorm launch");
    return MG_OK;
}

template <class T>
int layernorm_backward(hipStream_t st, dev::NormGradArgs a, float* workspace) {
    const bool sums = a.dgamma || a.dbeta;
    float *dgamma = a.dgamma, *dbeta = a.dbeta;
    const uint32_t parts = backward_parts(a.rows, a.cols);
    const bool wide = a.cols > kNormCols;
    const bool direct = !sums || (parts == 1 && !wide);  // one workgroup's sums are the result
    if (!direct) a.partial = workspace, a.dgamma = a.dbeta = nullptr;
    if (a.rows && wide) {
        constexpr uint32_t E = 16 / sizeof(T);
        if (sums) {
            const uint32_t nv = (a.cols + E - 1) / E;
            hipLaunchKernelGGL((dev::layernorm_columns_kernel<T>), dim3((nv + 255) / 256, parts), dim3(256), 0, st, a);
            MG_HIP(hipGetLastError(), "layernorm columns launch");
        }
        hipLaunchKernelGGL((dev::layernorm_backward_wide_kernel<T, 1024>),
                           dim3(a.rows < 2 * kCus ? a.rows : 2 * kCus), dim3(1024), 0, st, a);
    } else if (a.rows) {
        with_shape(norm_shape(a.cols), NormBackwardLauncher<T>{st, a, parts});
    }
    MG_HIP(hipGetLastError(), "layernorm backward launch");
    if (!direct) {
        hipLaunchKernelGGL(dev::layernorm_reduce_kernel, dim3((2 * a.cols + 31) / 32), dim3(1024), 0, st, a.partial,
                           parts, a.cols, dgamma, dbeta);
        MG_HIP(hipGetLastError(), "layernorm reduce launch");
    }
    return MG_OK;
}

// The checks of one [rows][cols] operand: its pointer, its alignment to its type
// and its row stride (0 stands for cols, and is filled in).
int check_rows(const char* what, const char* name, const void* p, uint64_t* ld, uint32_t rows, uint32_t cols,
               uint32_t type) {
    if (!*ld) *ld = cols;
    MG_CHECK(p || !rows, MG_ERR_INVALID, "%s: %s is NULL", what, name);
    MG_CHECK(aligned(p, type_bytes(type)), MG_ERR_INVALID, "%s: %s is not aligned to its type", what, name);
    MG_CHECK(*ld >= cols, MG_ERR_INVALID, "%s: %s_ld %llu is less than cols %u", what, name, (unsigned long long)*ld,
             cols);
    MG_CHECK(*ld <= (1ull << 40), MG_ERR_INVALID, "%s: %s_ld %llu is out of range", what, name,
             (unsigned long long)*ld);
    return MG_OK;
}

int check_shape(const char* what, uint32_t cols, uint32_t type) {
    MG_CHECK(type_known(type), MG_ERR_INVALID, "%s: unknown type %u", what, type);
    MG_CHECK(cols >= 1 && cols <= (1u << 24), MG_ERR_INVALID, "%s: cols %u must be in [1, 2^24]", what, cols);
    return MG_OK;
}

int check_floats(const char* what, const char* name, const void* p) {
    MG_CHECK(aligned(p, 4), MG_ERR_INVALID, "%s: %s is not aligned to its type", what, name);
    return MG_OK;
}

}  // namespace
}  // namespace mg

using namespace mg;

extern "C" {

int mg_layernorm(void* stream, const mg_layernorm_args* args) {
    const char* what = "layernorm";
    MG_CHECK(args, MG_ERR_INVALID, "layernorm: null argument");
    mg_layernorm_args p = *args;
    int rc;
    if ((rc = check_shape(what, p.cols, p.type))) return rc;
    MG_CHECK(p.eps >= 0.0f && p.eps < __builtin_huge_valf(), MG_ERR_INVALID,
             "layernorm: eps must be finite and not negative");
    MG_CHECK(!p.residual == !p.sum, MG_ERR_INVALID, "layernorm: residual and sum go together");
    if ((rc = check_rows(what, "x", p.x, &p.x_ld, p.rows, p.cols, p.type)) ||
        (rc = check_rows(what, "y", p.y, &p.y_ld, p.rows, p.cols, p.type)) ||
        (rc = check_floats(what, "gamma", p.gamma)) || (rc = check_floats(what, "beta", p.beta)) ||
        (rc = check_floats(what, "mean", p.mean)) || (rc = check_floats(what, "rstd", p.rstd)))
        return rc;
    if (p.residual && ((rc = check_rows(what, "residual", p.residual, &p.residual_ld, p.rows, p.cols, p.type)) ||
                       (rc = check_rows(what, "sum", p.sum, &p.sum_ld, p.rows, p.cols, p.type))))
        return rc;
    if (!p.rows) return MG_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice on;
    if ((rc = on.enter(st, "layernorm: stream device"))) return rc;
    const dev::NormArgs a{p.x,    p.residual, p.sum,         p.gamma,  p.beta, p.y,    p.mean, p.rstd,
                          p.x_ld, p.residual_ld, p.sum_ld, p.y_ld, p.rows, p.cols, p.eps};
    return p.type == MG_TYPE_FP32   ? layernorm<float>(st, a)
           : p.type == MG_TYPE_BF16 ? layernorm<__bf16>(st, a)
                                    : layernorm<_Float16>(st, a);
}

int mg_layernorm_backward_workspace(uint32_t rows, uint32_t cols, uint64_t* bytes) {
    MG_CHECK(bytes, MG_ERR_INVALID, "layernorm backward workspace: null argument");
    int rc = check_shape("layernorm backward workspace", cols, MG_TYPE_FP32);
    if (rc) return rc;
    const uint32_t parts = backward_parts(rows, cols);
    *bytes = parts == 1 && cols <= kNormCols ? 0 : (uint64_t)parts * 2 * cols * 4;
    return MG_OK;
}

int mg_layernorm_backward(void* stream, const mg_layernorm_backward_args* args) {
    const char* what = "layernorm backward";
    MG_CHECK(args, MG_ERR_INVALID, "layernorm backward: null argument");
    mg_layernorm_backward_args p = *args;
    int rc;
    if ((rc = check_shape(what, p.cols, p.type))) return rc;
    if ((rc = check_rows(what, "x", p.x, &p.x_ld, p.rows, p.cols, p.type)) ||
        (rc = check_rows(what, "dy", p.dy, &p.dy_ld, p.rows, p.cols, p.type)) ||
        (rc = check_rows(what, "dx", p.dx, &p.dx_ld, p.rows, p.cols, p.type)) ||
        (p.dsum && (rc = check_rows(what, "dsum", p.dsum, &p.dsum_ld, p.rows, p.cols, p.type))) ||
        (rc = check_floats(what, "gamma", p.gamma)) || (rc = check_floats(what, "mean", p.mean)) ||
        (rc = check_floats(what, "rstd", p.rstd)) || (rc = check_floats(what, "dgamma", p.dgamma)) ||
        (rc = check_floats(what, "dbeta", p.dbeta)))
        return rc;
    MG_CHECK((p.mean && p.rstd) || !p.rows, MG_ERR_INVALID, "layernorm backward: mean and rstd are required");
    MG_CHECK(!p.reserved, MG_ERR_INVALID, "layernorm backward: reserved must be 0");
    if (p.dgamma || p.dbeta) {
        uint64_t need = 0;
        mg_layernorm_backward_workspace(p.rows, p.cols, &need);
        MG_CHECK(p.workspace_bytes >= need && (p.workspace || !need), MG_ERR_INVALID,
                 "layernorm backward: the workspace needs %llu bytes", (unsigned long long)need);
        MG_CHECK(aligned(p.workspace, 16), MG_ERR_INVALID, "layernorm backward: the workspace is not 16-byte aligned");
    } else if (!p.rows) {
        return MG_OK;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice on;
    if ((rc = on.enter(st, "layernorm backward: stream device"))) return rc;
    const dev::NormGradArgs a{p.x,     p.dy,    p.dsum,  p.gamma,   p.mean,  p.rstd, p.dx,  p.dgamma,
                              p.dbeta, nullptr, p.x_ld, p.dy_ld, p.dsum_ld, p.dx_ld, p.rows, p.cols};
    float* ws = static_cast<float*>(p.workspace);
    return p.type == MG_TYPE_FP32   ? layernorm_backward<float>(st, a, ws)
           : p.type == MG_TYPE_BF16 ? layernorm_backward<__bf16>(st, a, ws)
                                    : layernorm_backward<_Float16>(st, a, ws);
}

}  // extern "C"
