// Newton-Schulz steps of matrices whose short side m is at most 128, which the
// policy's block matrices are (128 x hidden): their symmetric m x m matrices fit
// one workgroup's LDS, and a launch for each product would be all latency.
//
// Launches of a batch: `first` once, then for each segment of one or two steps
// `square` and `update`. X is cut into slabs of 128 columns.
//  first:  X's slabs from the source (with the momentum's update) as pairs, each
//          workgroup at its own exponent, and the slabs' part of X X'.
//  square: one workgroup a matrix adds the parts to A (the first time its trace is
//          the squared norm, so no pass over X is spent on that), and takes the
//          segment's steps to Q in LDS.
//  update: X <- Q X slab by slab, and the slabs' part of the new X X', or at the
//          end the result.
// With m = 128 and n = 512 a segment of two steps is five m x m products (2 us
// each on one CU, of which 1.3 us matrix instructions) between launches of a few
// microseconds.
#pragma once
#include "muon_common.h"

namespace mg {
namespace dev {

constexpr int kSlab = 128;      // columns of a slab
constexpr int kShortParts = 16;  // most workgroups that share a matrix's slabs
constexpr int kMostExp = 120;    // exponent of a slab of zeros, or of next to nothing

// A matrix of MP x C pairs in LDS: two planes of rows of 2 C bytes, cut into
// 16-byte chunks; chunk c of row r sits at c ^ turn(r), so that 32 rows' reads of
// one chunk, and a fragment's, fall on all banks.
template <int R, int C>
struct PairTile {
    static constexpr int kRow = 2 * C, kPlane = R * kRow, kBytes = 2 * kPlane;
    static __device__ __forceinline__ int turn(int r) { return (r / (128 / C)) & (C / 8 - 1); }
    // eight elements from column 8 chunk
    static __device__ __forceinline__ f16x8 chunk(const char* t, int plane, int r, int c) {
        return *reinterpret_cast<const f16x8*>(t + plane * kPlane + r * kRow + ((c ^ turn(r)) << 4));
    }
    // four elements from column c, a multiple of 4
    static __device__ __forceinline__ char* quad(char* t, int plane, int r, int c) {
        return t + plane * kPlane + r * kRow + (((c >> 3) ^ turn(r)) << 4) + ((c & 4) << 1);
    }
    static __device__ __forceinline__ void put(char* t, int r, int c, f16x4 hi, f16x4 lo) {
        *reinterpret_cast<f16x4*>(quad(t, 0, r, c)) = hi;
        *reinterpret_cast<f16x4*>(quad(t, 1, r, c)) = lo;
    }
};

// Lane q of each four lanes holds four values of column 4 a + q; gives it value q
// of the four columns 4 a .. 4 a + 3.
__device__ __forceinline__ f16x4 quad_transpose(f16x4 v) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const int q = threadIdx.x & 3;
    u32x2 w = __builtin_bit_cast(u32x2, v);  // values (0, 1), (2, 3)
    // lanes q and q ^ 1 trade halves: even lanes get value 0 of both columns, then 2
    const uint32_t n0 = __builtin_amdgcn_mov_dpp(w[0], 0xB1, 0xF, 0xF, true);
    const uint32_t n1 = __builtin_amdgcn_mov_dpp(w[1], 0xB1, 0xF, 0xF, true);
    const uint32_t p0 = q & 1 ? (n0 >> 16) | (w[0] & 0xFFFF0000u) : (w[0] & 0xFFFFu) | (n0 << 16);
    const uint32_t p1 = q & 1 ? (n1 >> 16) | (w[1] & 0xFFFF0000u) : (w[1] & 0xFFFFu) | (n1 << 16);
    // lanes q and q ^ 2 trade words: the lower two lanes keep values 0 and 1
    const uint32_t give = q & 2 ? p0 : p1;
    const uint32_t got = __builtin_amdgcn_mov_dpp(give, 0x4E, 0xF, 0xF, true);
    const u32x2 out = q & 2 ? u32x2{got, p1} : u32x2{p0, got};
    return __builtin_bit_cast(f16x4, out);
}

__device__ __forceinline__ f32x16 pair_mfma(const f16x8 (&a)[2], const f16x8 (&b)[2], f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], c, 0, 0, 0);
}

// Exponents and scale of a matrix's X while it is the source's own.
struct ShortState {
    int exp[kShortParts];  // of each workgroup's slabs: pairs hold U 2^exp
    int least;             // the least of them: A's unit before the norm is known
    float scale;           // 2^-least / (|U| + eps)
};

struct ShortArgs {
    SourceArgs src;
    uint32_t slabs, parts;
    f16* xt;        // [count][2][slabs 128][MP] X transposed, planes hi and lo
    float* partial;  // [count][parts][tiles][16][64] X X' on and under the diagonal, in register order
    f16* q;         // [count][2][MP][MP]
    ShortState* state;  // [count]
    float eps;
    // square
    uint32_t start;  // the first segment
    uint32_t steps;  // 1 or 2
    float a, b, c;
    float unit_q;
    // update
    Batch dst;
    uint32_t step;
    float keep, rate;
};

// Tile t of the lower triangle in rows: (0,0) (1,0) (1,1) (2,0) ...
__device__ __forceinline__ void short_tile(int t, int& bi, int& bj) {
    bi = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3;
    bj = t - bi * (bi + 1) / 2;
}
template <int MP>
struct ShortShape {
    static constexpr int NB = MP / 32, TILES = NB * (NB + 1) / 2, PER = (TILES + 3) / 4;  // tiles a wave, four waves
    using Sq = PairTile<MP, MP>;
    using Rows = PairTile<MP, kSlab>;  // a slab of X
};

// Adds the slab's part of X X' (rows in LDS as pairs) to each wave's tiles, in
// chains of 32 contraction elements.
template <int MP>
__device__ __forceinline__ void short_gram(const char* rows, f32x16 (&gram)[ShortShape<MP>::PER]) {
    using S = ShortShape<MP>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int u = 0; u < S::PER; ++u) {
        const int t = wave + 4 * u;
        if (t >= S::TILES) break;
        int bi, bj;
        short_tile(t, bi, bj);
#pragma unroll
        for (int kk = 0; kk < kSlab / 16; kk += 2) {
            f32x16 s = {};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                f16x8 a[2], b[2];
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    a[p] = S::Rows::chunk(rows, p, 32 * bi + r, 2 * (kk + e) + h);
                    b[p] = S::Rows::chunk(rows, p, 32 * bj + r, 2 * (kk + e) + h);
                }
                s = pair_mfma(a, b, s);
            }
            gram[u] += s;
        }
    }
}
template <int MP>
__device__ __forceinline__ void short_gram_store(const ShortArgs& a, uint32_t mat,
                                                 const f32x16 (&gram)[ShortShape<MP>::PER]) {
    using S = ShortShape<MP>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float* out = a.partial + ((size_t)mat * a.parts + blockIdx.x) * S::TILES * 1024;
#pragma unroll
    for (int u = 0; u < S::PER; ++u) {
        const int t = wave + 4 * u;
        if (t >= S::TILES) break;
#pragma unroll
        for (int r = 0; r < 16; ++r) out[(size_t)t * 1024 + r * 64 + lane] = gram[u][r];
    }
}

__device__ __forceinline__ float magnitude(float x) {
    return fabsf(x) < __builtin_huge_valf() ? fabsf(x) : __builtin_huge_valf();
}

// Grid (parts, count). A slab goes through LDS as fp32 (rows i of X, padded), from
// there as pairs to the Gram product's rows and, transposed, to xt.
template <int MP>
__global__ void __launch_bounds__(256) short_first_kernel(const ShortArgs a) {
    using S = ShortShape<MP>;
    constexpr int LD = kSlab + 1;
    __shared__ __align__(16) char rows[S::Rows::kBytes];
    __shared__ float stage[MP * LD];
    __shared__ float wmax[4];
    const uint32_t mat = blockIdx.y;
    const int t = threadIdx.x;
    const uint32_t n_rows = a.src.rows, n_cols = a.src.cols;
    const bool tall = n_rows > n_cols;
    // slab s into the stage, as X(i, j); returns the thread's largest magnitude,
    // infinite where one is not finite
    auto fill = [&](uint32_t s, auto update) {
        float most = 0.0f;
        const uint32_t j0 = s * kSlab;
        if (tall) {  // source rows are X's columns
            constexpr int RP = 256 / MP;
            const int i = t % MP;
#pragma unroll 8
            for (int j = t / MP; j < kSlab; j += RP) {
                const bool in = j0 + j < n_rows && (uint32_t)i < n_cols;
                const float u = in ? source_value<decltype(update)::value>(a.src, mat, j0 + j, i) : 0.0f;
                stage[i * LD + j] = u;
                most = fmaxf(most, magnitude(u));
            }
        } else {
            const int j = t & (kSlab - 1);
#pragma unroll 8
            for (int i = t / kSlab; i < MP; i += 256 / kSlab) {
                const bool in = j0 + j < n_cols && (uint32_t)i < n_rows;
                const float u = in ? source_value<decltype(update)::value>(a.src, mat, i, j0 + j) : 0.0f;
                stage[i * LD + j] = u;
                most = fmaxf(most, magnitude(u));
            }
        }
        return most;
    };
    float most = 0.0f;
    for (uint32_t s = blockIdx.x; s < a.slabs; s += a.parts) most = fmaxf(most, fill(s, std::true_type{}));
    most = group_max<64>(most);
    if ((t & 63) == 0) wmax[t >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    // 2^12 <= most 2^exp < 2^13; without a finite size the products carry the NaN
    int e = 0;
    if (most < __builtin_huge_valf()) {
        e = most > 0.0f ? 12 - ilogbf(most) : kMostExp;
        e = e > kMostExp ? kMostExp : e;
    }
    const float unit = ldexpf(1.0f, e);
    if (t == 0) a.state[mat].exp[blockIdx.x] = e;
    f32x16 gram[S::PER] = {};
    const bool one = a.slabs <= a.parts;  // the stage still holds the only slab
    for (uint32_t s = blockIdx.x; s < a.slabs; s += a.parts) {
        if (!one) {
            __syncthreads();
            fill(s, std::false_type{});
        }
        __syncthreads();
        for (int q = t; q < MP * (kSlab / 4); q += 256) {
            const int i = q / (kSlab / 4), j = 4 * (q % (kSlab / 4));
            f16x4 hi, lo;
            for (int k = 0; k < 4; ++k) {
                f16 h, l;
                split(stage[i * LD + j + k] * unit, h, l);
                hi[k] = h, lo[k] = l;
            }
            S::Rows::put(rows, i, j, hi, lo);
        }
        f16* xt = a.xt + (size_t)mat * 2 * a.slabs * kSlab * MP + (size_t)s * kSlab * MP;
        const size_t plane = (size_t)a.slabs * kSlab * MP;
        for (int q = t; q < kSlab * (MP / 8); q += 256) {
            const int j = q / (MP / 8), i = 8 * (q % (MP / 8));
            f16x8 hi, lo;
            for (int k = 0; k < 8; ++k) {
                f16 h, l;
                split(stage[(i + k) * LD + j] * unit, h, l);
                hi[k] = h, lo[k] = l;
            }
            *reinterpret_cast<f16x8*>(xt + (size_t)j * MP + i) = hi;
            *reinterpret_cast<f16x8*>(xt + plane + (size_t)j * MP + i) = lo;
        }
        __syncthreads();
        short_gram<MP>(rows, gram);
    }
    short_gram_store<MP>(a, mat, gram);
}

// out = x y of two symmetric matrices in LDS, the wave's tiles in registers: wave
// w holds the tiles (bi, bj) with bi in {w / 2 NB / 2 ..}, 2 x 2 of them at MP = 128
// and one at 64; at 32 the first wave holds the only one.
template <int MP>
struct ShortProduct {
    using Sq = PairTile<MP, MP>;
    static constexpr int W = MP == 128 ? 2 : 1;  // tile rows and columns of a wave
    f32x16 v[W][W];
    int bi, bj;
    bool on;
    __device__ __forceinline__ ShortProduct() {
        const int wave = threadIdx.x >> 6;
        bi = MP == 32 ? 0 : (wave >> 1) * W, bj = MP == 32 ? 0 : (wave & 1) * W;
        on = MP > 32 || wave == 0;
    }
    __device__ __forceinline__ void run(const char* x, const char* y) {
        if (!on) return;
        const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] = f32x16{};
#pragma unroll
        for (int kk = 0; kk < MP / 16; kk += 2) {
            f32x16 s[W][W] = {};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                f16x8 fa[W][2], fb[W][2];
#pragma unroll
                for (int i = 0; i < W; ++i)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        fa[i][p] = Sq::chunk(x, p, 32 * (bi + i) + r, 2 * (kk + e) + h);
                        fb[i][p] = Sq::chunk(y, p, 32 * (bj + i) + r, 2 * (kk + e) + h);
                    }
#pragma unroll
                for (int i = 0; i < W; ++i)
#pragma unroll
                    for (int j = 0; j < W; ++j) s[i][j] = pair_mfma(fa[i], fb[j], s[i][j]);
            }
#pragma unroll
            for (int i = 0; i < W; ++i)
#pragma unroll
                for (int j = 0; j < W; ++j) v[i][j] += s[i][j];
        }
    }
    // f(value x 4, row i of the first, column j): four rows i .. i + 3 of one column
    template <class F>
    __device__ __forceinline__ void each(F&& f) const {
        if (!on) return;
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int x = 0; x < W; ++x)
#pragma unroll
            for (int y = 0; y < W; ++y)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const float q[4] = {v[x][y][r], v[x][y][r + 1], v[x][y][r + 2], v[x][y][r + 3]};
                    f(q, 32 * (bi + x) + 2 * r + 4 * (lane >> 5), 32 * (bj + y) + (lane & 31));
                }
    }
    // The result times f as pairs into `out` after every wave has read what it overwrites.
    __device__ __forceinline__ void put(char* out, float f) const {
        __syncthreads();
        each([&](const float (&q)[4], int i, int j) {
            f16x4 hi, lo;
            split4(q, f, hi, lo);
            Sq::put(out, j, i, hi, lo);
        });
        __syncthreads();
    }
};

// One workgroup a matrix: A from the partial products, then the segment's steps. Two
// matrices in LDS are enough for two steps: A and P, then B = P A over A, A' = P B
// over B, P' over A', and Q = P' P.
template <int MP>
__global__ void __launch_bounds__(256) short_square_kernel(const ShortArgs a) {
    using S = ShortShape<MP>;
    using Sq = typename S::Sq;
    __shared__ __align__(16) char gram[Sq::kBytes], poly[Sq::kBytes];
    __shared__ float wtrace[4];
    const uint32_t mat = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    ShortState& state = a.state[mat];
    int least = kMostExp;
    if (a.start)
        for (uint32_t p = 0; p < a.parts; ++p) least = state.exp[p] < least ? state.exp[p] : least;
    f32x16 sum[S::PER] = {};
    const float* in = a.partial + (size_t)mat * a.parts * S::TILES * 1024 + lane;
    for (uint32_t p = 0; p < a.parts; ++p, in += S::TILES * 1024) {
        const float f = a.start ? ldexpf(1.0f, 2 * (least - state.exp[p])) : 1.0f;
#pragma unroll
        for (int u = 0; u < S::PER; ++u) {
            const int t = wave + 4 * u;
            if (t >= S::TILES) break;
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[u][r] += f * in[(size_t)t * 1024 + r * 64];
        }
    }
    float to_unit = kUnitA / (kUnitX * kUnitX);
    if (a.start) {
        float trace = 0.0f;
#pragma unroll
        for (int u = 0; u < S::PER; ++u) {
            int bi, bj;
            short_tile(wave + 4 * u, bi, bj);
            if (wave + 4 * u >= S::TILES || bi != bj) continue;
#pragma unroll
            for (int r = 0; r < 16; ++r) trace += c32_row(r, lane) == (lane & 31) ? sum[u][r] : 0.0f;
        }
        trace = group_sum<64>(trace);
        if (lane == 0) wtrace[wave] = trace;
        __syncthreads();
        trace = wtrace[0] + wtrace[1] + wtrace[2] + wtrace[3];
        const float scale = 1.0f / (sqrtf(trace) + a.eps * ldexpf(1.0f, least));
        if (threadIdx.x == 0) state.least = least, state.scale = scale;
        to_unit = scale * scale * kUnitA;
    }
#pragma unroll
    for (int u = 0; u < S::PER; ++u) {
        const int t = wave + 4 * u;
        if (t >= S::TILES) break;
        int bi, bj;
        short_tile(t, bi, bj);
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const float q[4] = {sum[u][r], sum[u][r + 1], sum[u][r + 2], sum[u][r + 3]};
            const int i = 32 * bi + 2 * r + 4 * (lane >> 5), j = 32 * bj + (lane & 31);
            f16x4 hi, lo;
            split4(q, to_unit, hi, lo);
            Sq::put(gram, j, i, hi, lo);
            if (bi != bj) Sq::put(gram, i + (lane & 3), j & ~3, quad_transpose(hi), quad_transpose(lo));
        }
    }
    __syncthreads();
    ShortProduct<MP> prod;
    // a I + b A + c (A A) in registers, times kUnitP
    auto polynomial = [&](const char* A) {
        prod.run(A, A);
        const float cc = a.c * (kUnitP / (kUnitA * kUnitA)), cb = a.b * (kUnitP / kUnitA), ca = a.a * kUnitP;
        if (!prod.on) return;
#pragma unroll
        for (int x = 0; x < prod.W; ++x)
#pragma unroll
            for (int y = 0; y < prod.W; ++y)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const int i = 32 * (prod.bi + x) + 2 * r + 4 * (lane >> 5), j = 32 * (prod.bj + y) + (lane & 31);
                    const f16x4 hi = *reinterpret_cast<const f16x4*>(Sq::quad(const_cast<char*>(A), 0, j, i));
                    const f16x4 lo = *reinterpret_cast<const f16x4*>(Sq::quad(const_cast<char*>(A), 1, j, i));
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        prod.v[x][y][r + e] = cc * prod.v[x][y][r + e] + cb * ((float)hi[e] + (float)lo[e]) +
                                              (i + e == j ? ca : 0.0f);
                }
    };
    float to_q = a.unit_q / kUnitP;
    polynomial(gram);
    if (a.steps == 2) {
        prod.put(poly, 1.0f);
        prod.run(poly, gram);
        prod.put(gram, 1.0f / kUnitP);
        prod.run(poly, gram);
        prod.put(gram, 1.0f / kUnitP);
        polynomial(gram);
        prod.put(gram, 1.0f);
        prod.run(gram, poly);
        to_q = a.unit_q / (kUnitP * kUnitP);
    }
    f16* q = a.q + (size_t)mat * 2 * MP * MP;
    prod.each([&](const float (&w)[4], int i, int j) {
        f16x4 hi, lo;
        split4(w, to_q, hi, lo);
        *reinterpret_cast<f16x4*>(q + j * MP + i) = hi;
        *reinterpret_cast<f16x4*>(q + MP * MP + j * MP + i) = lo;
    });
}

// Grid (parts, count). X' X = Q X as X' rows: a wave holds 32 columns of X, its
// fragments straight from xt, Q in LDS. FINAL writes the result; otherwise the new
// pairs replace the old in xt (each workgroup's own slabs) and go to LDS in rows
// for the Gram product.
template <int MP, bool FINAL>
__global__ void __launch_bounds__(256) short_update_kernel(const ShortArgs a) {
    using S = ShortShape<MP>;
    using Sq = typename S::Sq;
    constexpr int LD = kSlab + 1, LDT = MP + 1;
    constexpr int kStage = FINAL ? (MP * LD > kSlab * LDT ? MP * LD : kSlab * LDT) * 4 : S::Rows::kBytes;
    __shared__ __align__(16) char q[Sq::kBytes];
    __shared__ __align__(16) char stage[kStage];
    const uint32_t mat = blockIdx.y;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, r = lane & 31, h = lane >> 5;
    const f16* qin = a.q + (size_t)mat * 2 * MP * MP;
    for (int c = t; c < 2 * MP * (MP / 8); c += 256) {
        const int p = c / (MP * (MP / 8)), row = c / (MP / 8) % MP, ch = c % (MP / 8);
        *reinterpret_cast<f16x8*>(q + p * Sq::kPlane + row * Sq::kRow + ((ch ^ Sq::turn(row)) << 4)) =
            *reinterpret_cast<const f16x8*>(qin + (size_t)c * 8);
    }
    // takes the exponents out of X Q, and puts X's own in
    const ShortState& state = a.state[mat];
    float f = 1.0f / (a.unit_q * kUnitX);
    if (a.start) f = state.scale * ldexpf(1.0f, state.least - state.exp[blockIdx.x]) / a.unit_q;
    if (!FINAL) f *= kUnitX;
    const size_t plane = (size_t)a.slabs * kSlab * MP;
    const uint32_t n_rows = a.src.rows, n_cols = a.src.cols;
    const bool tall = n_rows > n_cols;
    f32x16 gram[FINAL ? 1 : S::PER] = {};
    for (uint32_t s = blockIdx.x; s < a.slabs; s += a.parts) {
        f16* const xt = a.xt + (size_t)mat * 2 * plane + ((size_t)s * kSlab + 32 * wave) * MP;
        f16x8 x[MP / 16][2];
#pragma unroll
        for (int kk = 0; kk < MP / 16; ++kk)
#pragma unroll
            for (int p = 0; p < 2; ++p)
                x[kk][p] = *reinterpret_cast<const f16x8*>(xt + p * plane + (size_t)r * MP + 16 * kk + 8 * h);
        __syncthreads();  // Q is in place, and the slab before has left the stage
#pragma unroll
        for (int b = 0; b < S::NB; ++b) {
            f32x16 acc = {};
#pragma unroll
            for (int kk = 0; kk < MP / 16; kk += 2) {
                f32x16 c = {};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f16x8 y[2];
#pragma unroll
                    for (int p = 0; p < 2; ++p) y[p] = Sq::chunk(q, p, 32 * b + r, 2 * (kk + e) + h);
                    c = pair_mfma(x[kk + e], y, c);
                }
                acc += c;
            }
            // X'(i, j .. j + 3) with i = 32 b + r
#pragma unroll
            for (int g = 0; g < 16; g += 4) {
                const float w[4] = {acc[g], acc[g + 1], acc[g + 2], acc[g + 3]};
                const int i = 32 * b + r, j = 2 * g + 4 * h;
                if constexpr (FINAL) {
                    float* o = reinterpret_cast<float*>(stage);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (tall)
                            o[(32 * wave + j + e) * LDT + i] = w[e] * f;
                        else
                            o[i * LD + 32 * wave + j + e] = w[e] * f;
                    }
                } else {
                    f16x4 hi, lo;
                    split4(w, f, hi, lo);
                    S::Rows::put(stage, i, 32 * wave + j, hi, lo);
                    f16* at = xt + (size_t)(j + (lane & 3)) * MP + (i & ~3);
                    *reinterpret_cast<f16x4*>(at) = quad_transpose(hi);
                    *reinterpret_cast<f16x4*>(at + plane) = quad_transpose(lo);
                }
            }
        }
        __syncthreads();
        if constexpr (FINAL) {
            const float* o = reinterpret_cast<const float*>(stage);
            const uint32_t j0 = s * kSlab;
            auto write = [&](uint32_t y, uint32_t c, float value) {
                const size_t at = mat * a.dst.stride + y * a.dst.ld + c;
                batch_store(a.dst, at, a.step ? a.keep * batch_load(a.dst, at) - a.rate * value : value);
            };
            if (tall) {
#pragma unroll 4
                for (int j = t / MP; j < kSlab; j += 256 / MP)
                    if (j0 + j < n_rows && (uint32_t)(t % MP) < n_cols) write(j0 + j, t % MP, o[j * LDT + t % MP]);
            } else {
                const int j = t & (kSlab - 1);
#pragma unroll 4
                for (int i = t / kSlab; i < MP; i += 256 / kSlab)
                    if ((uint32_t)i < n_rows && j0 + j < n_cols) write(i, j0 + j, o[i * LD + j]);
            }
        } else {
            short_gram<MP>(stage, gram);
        }
    }
    if constexpr (!FINAL) short_gram_store<MP>(a, mat, gram);
}

}  // namespace dev
}  // namespace mg
