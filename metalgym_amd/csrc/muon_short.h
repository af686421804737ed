// Newton-Schulz steps of matrices whose short side m is at most 128, which the
// policy's block matrices are (128 x hidden): their symmetric m x m matrices fit
// one workgroup's LDS, and a launch for each product would be all latency.
//
// Launches of a batch: `first` once, then one `step` for each segment of one or two
// steps. X is cut into slabs of 64 columns, shared by up to eight workgroups.
//  first: X's slabs from the source (with the momentum's update) as pairs, each
//         workgroup at its own exponent, and the slabs' part of X X'.
//  step:  every workgroup of a matrix adds the parts to A (the first time its trace is
//         the squared norm, so no pass over X is spent on that) and takes the segment's
//         steps to Q in LDS, all of them the same; then X <- Q X on its slabs, and
//         their part of the new X X', or at the end the result. The repeated work is on
//         CUs that would be idle: with one workgroup a matrix doing it, in launches of
//         its own, Q went through memory (two of 512 x 128 in three segments: 74.6 us, so 67.4;
//         1000 of 128 x 512: 1262, so 721).
// Each kernel runs its code once or a few times, so what it costs is latencies: loads
// are issued in batches, one wave holds one 32 x 32 tile, and code is kept in loops
// (unrolled four waves' worth of tiles each, the same kernels spent 13 to 25 us
// fetching 20 to 50 KB of instructions).
#pragma once
#include "muon_common.h"

namespace mg {
namespace dev {

constexpr int kSlab = 64;       // columns of a slab
constexpr int kShortParts = 8;  // most workgroups that share a matrix's slabs
constexpr int kMostExp = 120;   // exponent of a slab of zeros, or of next to nothing

// Pairs in the order of the matrix instructions' operands, in LDS and in memory: a
// matrix of K columns (the contraction) is cut into 32 rows x 16 columns, each two
// planes of 64 lanes x 8 elements: lane 32 h + r holds row r and columns 8 h ... A
// fragment is then 1 KB in a row, and a wave's stores of results (four columns of
// eight rows at a time) run along 128 bytes.
template <int K>
struct Frags {
    static constexpr int kBlock = K / 16 * 2 * 512;  // elements of 32 rows
    // columns c ... of row r: c a multiple of 4
    static __device__ __forceinline__ int at(int plane, int r, int c) {
        return (r >> 5) * kBlock + ((c >> 4) * 2 + plane) * 512 + ((c & 8) << 5) + ((r & 31) << 3) + (c & 4);
    }
    // the fragment of rows 32 b ... and columns 16 k ... for this lane
    static __device__ __forceinline__ f16x8 frag(const f16* m, int plane, int b, int k) {
        return *reinterpret_cast<const f16x8*>(m + b * kBlock + (k * 2 + plane) * 512 + (threadIdx.x & 63) * 8);
    }
    static __device__ __forceinline__ void put(f16* m, int r, int c, f16x4 hi, f16x4 lo) {
        f16* const to = m + at(0, r, c);
        *reinterpret_cast<f16x4*>(to) = hi;
        *reinterpret_cast<f16x4*>(to + 512) = lo;
    }
};

// Lane q of each four lanes holds four values of column 4 a + q; gives it value q
// of the four columns 4 a .. 4 a + 3. Byte permutes with a lane's own selectors:
// selects become branches here.
__device__ __forceinline__ f16x4 quad_transpose(f16x4 v) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const uint32_t q = threadIdx.x & 3;
    const uint32_t halves = q & 1 ? 0x03020706u : 0x05040100u;  // (partner's high, own high) or (own low, partner's low)
    const uint32_t first = q & 2 ? 0x07060504u : 0x03020100u;   // the permute's first operand, or its second
    const u32x2 w = __builtin_bit_cast(u32x2, v);  // values (0, 1), (2, 3)
    // lanes q and q ^ 1 trade halves: even lanes get value 0 of both columns, then 2
    const uint32_t n0 = __builtin_amdgcn_mov_dpp(w[0], 0xB1, 0xF, 0xF, true);
    const uint32_t n1 = __builtin_amdgcn_mov_dpp(w[1], 0xB1, 0xF, 0xF, true);
    const uint32_t p0 = __builtin_amdgcn_perm(n0, w[0], halves), p1 = __builtin_amdgcn_perm(n1, w[1], halves);
    // lanes q and q ^ 2 trade words: the lower two lanes keep values 0 and 1
    const uint32_t got = __builtin_amdgcn_mov_dpp(__builtin_amdgcn_perm(p0, p1, first), 0x4E, 0xF, 0xF, true);
    const u32x2 out = {__builtin_amdgcn_perm(got, p0, first), __builtin_amdgcn_perm(p1, got, first)};
    return __builtin_bit_cast(f16x4, out);
}

// a b of pairs over 32 contraction elements (two fragments). The products of low halves
// come first, so that the sum is of full size in the last two instructions only: each
// rounds it, and cuts off what its small products have under 2^-25 of its largest, 0.1
// of a last place each (rms error of 72 x 56: 1.71e-6 with the instructions in the order
// of their elements, 1.58e-6 so). SWAP: with the bits of the product with a and b in each
// other's place. LOW: with the product of the low halves too, 2^-24 of a square.
template <bool SWAP, bool LOW>
__device__ __forceinline__ f32x16 pair_mfma(const f16x8 (&a)[2][2], const f16x8 (&b)[2][2]) {
    f32x16 c = {};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        if (LOW) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[e][1], b[e][1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[e][!SWAP], b[e][SWAP], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[e][SWAP], b[e][!SWAP], c, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[e][0], b[e][0], c, 0, 0, 0);
    return c;
}

struct ShortState {
    int exp[kShortParts];  // of each workgroup's slabs while X is the source's own: pairs hold U 2^exp
    float share;           // |U| / (|U| + eps), from the first segment on
};

struct ShortArgs {
    SourceArgs src;
    uint32_t slabs, parts;
    f16* xt;        // [count][slabs] X transposed: a slab's columns of X by MP, Frags<MP>
    // [count][parts][tiles][16][64] X X' on and under the diagonal, in register order. A
    // step's workgroups read all of a matrix's and write their own of the next: two buffers.
    const float* partial_in;
    float* partial;
    ShortState* state;  // [count]
    float eps;
    uint32_t start;  // the first segment
    float growth_in, growth;  // extra_exp's, of this segment's X and of the next one's
    uint32_t steps;  // 1 or 2
    float a, b, c;
    float unit_q;
    Batch dst;
    uint32_t step;
    float keep, rate, odd_rate;  // odd_rate: of the odd matrices of a policy's blocks
    // The arguments as they are for matrix k.
    __device__ __forceinline__ ShortArgs of(uint32_t k) const {
        ShortArgs a = *this;
        if (src.blocks && (k & 1)) {
            a.src.rows = src.cols, a.src.cols = src.rows;
            a.src.in.ld = a.src.momentum.ld = a.dst.ld = a.src.cols;
            a.rate = odd_rate;
        }
        return a;
    }
};

// Tile t of the lower triangle in rows: (0,0) (1,0) (1,1) (2,0) ...
__device__ __forceinline__ void short_tile(int t, int& bi, int& bj) {
    bi = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3;
    bj = t - bi * (bi + 1) / 2;
}
template <int MP>
struct ShortShape {
    static constexpr int NB = MP / 32, TILES = NB * (NB + 1) / 2;  // of 32 x 32, on and under the diagonal
    static constexpr int CB = kSlab / 32;               // column blocks of a slab
    static constexpr int W = CB * NB < 8 ? CB * NB : 8;  // waves over a slab's column and row blocks
    static constexpr int NT = 64 * W, PER = MP * kSlab / NT;  // elements of a slab a thread
    static constexpr int THREADS = 64 * (W > TILES ? W : TILES);  // a wave a tile of a symmetric matrix
    // sums of few products: 1 x 5 is off by 7.5e-7 (rms) without, 3.9e-7 with it
    static constexpr bool LOW = MP == 32;
    static constexpr int SQ = 2 * MP * MP, SLAB = 2 * MP * kSlab;  // elements of a pair of planes
};

// 32 x 32 of x y' over K contraction elements, rows 32 bi of x and 32 bj of y, in
// chains of 32.
template <int K, bool LOW>
__device__ __forceinline__ f32x16 short_product(const f16* x, const f16* y, int bi, int bj) {
    f32x16 v = {};
#pragma unroll 2
    for (int kk = 0; kk < K / 16; kk += 2) {
        f16x8 a[2][2], b[2][2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                a[e][p] = Frags<K>::frag(x, p, bi, kk + e);
                b[e][p] = Frags<K>::frag(y, p, bj, kk + e);
            }
        v += pair_mfma<false, LOW>(a, b);
    }
    return v;
}

// Adds the slab's part of X X' (rows in LDS as pairs) to the wave's tile of it.
template <int MP>
__device__ __forceinline__ void short_gram(const f16* rows, f32x16& gram) {
    const int t = threadIdx.x >> 6;
    if (t >= ShortShape<MP>::TILES) return;
    int bi, bj;
    short_tile(t, bi, bj);
    gram += short_product<kSlab, ShortShape<MP>::LOW>(rows, rows, bi, bj);
}
// The workgroup's partial sums, in register order.
template <int MP>
__device__ __forceinline__ void short_gram_store(const ShortArgs& a, uint32_t mat, const f32x16& gram) {
    using S = ShortShape<MP>;
    const int t = threadIdx.x >> 6;
    if (t >= S::TILES) return;
    float* out = a.partial + (((size_t)mat * a.parts + blockIdx.x) * S::TILES + t) * 1024 + (threadIdx.x & 63);
#pragma unroll
    for (int r = 0; r < 16; ++r) out[r * 64] = gram[r];
}

__device__ __forceinline__ float magnitude(float x) {
    return fabsf(x) < __builtin_huge_valf() ? fabsf(x) : __builtin_huge_valf();
}

// A thread's part of a slab of the source: PER consecutive elements across the
// source's rows at one place along them, so that threads run along the rows. Of
// tall matrices those are X(i, j .. ), of others X(i .. , j).
template <int MP>
struct ShortPart {
    using S = ShortShape<MP>;
    int i, j;
    float u[S::PER];
    __device__ __forceinline__ explicit ShortPart(bool tall) {
        const int t = threadIdx.x;
        i = tall ? t % MP : t / kSlab * S::PER, j = tall ? t / MP * S::PER : t % kSlab;
    }
    // U with zeros in the padding; UPDATE also moves the momentum. The loads are
    // issued together, from clamped places: one at a time, each would cost a latency.
    template <bool UPDATE, class T>
    __device__ __forceinline__ void load(const SourceArgs& a, uint32_t mat, uint32_t s, float clip) {
        const bool tall = a.rows > a.cols;
        const uint32_t y0 = tall ? s * kSlab + j : i, x = tall ? i : s * kSlab + j;
        const uint32_t xc = x < a.cols ? x : a.cols - 1;
        const uint32_t yc = y0 < a.rows ? y0 : a.rows - 1;
        const T* in = static_cast<const T*>(a.in.data) + a.in.at(mat, yc, xc);
#pragma unroll
        for (int e = 0; e < S::PER; ++e) {
            u[e] = (float)*in * clip;
            in += y0 + e + 1 < a.rows ? a.in.ld : 0u;
        }
        if (a.momentum.data) {
            float* const mom = static_cast<float*>(a.momentum.data) + a.momentum.at(mat, yc, xc);
            const float* from = mom;
            float b[S::PER];
#pragma unroll
            for (int e = 0; e < S::PER; ++e) {
                b[e] = *from;
                from += y0 + e + 1 < a.rows ? a.momentum.ld : 0u;
            }
            float* to = mom;
#pragma unroll
            for (int e = 0; e < S::PER; ++e) {
                if constexpr (UPDATE) {
                    b[e] = moved_momentum(a, b[e], u[e]);
                    if (x < a.cols && y0 + e < a.rows) *to = b[e];
                    to += a.momentum.ld;
                }
                u[e] = update_of(a, b[e], u[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < S::PER; ++e) u[e] = x < a.cols && y0 + e < a.rows ? u[e] : 0.0f;
    }
    template <bool UPDATE>
    __device__ __forceinline__ void load(const SourceArgs& a, uint32_t mat, uint32_t s, float clip) {
        if (threadIdx.x >= S::NT) return;  // whole waves
        switch (a.in.type) {
            case MG_TYPE_FP32: return load<UPDATE, float>(a, mat, s, clip);
            case MG_TYPE_BF16: return load<UPDATE, __bf16>(a, mat, s, clip);
            default: return load<UPDATE, f16>(a, mat, s, clip);
        }
    }
};

// Grid (parts, count). The slabs as pairs, to xt and in rows to LDS for the Gram
// product: one of the two takes a thread's four elements as they are, the other
// those of four threads.
template <int MP>
__global__ void __launch_bounds__(ShortShape<MP>::THREADS) short_first_kernel(const ShortArgs args) {
    using S = ShortShape<MP>;
    constexpr int W = S::THREADS / 64;
    __shared__ __align__(16) f16 rows[S::SLAB];
    __shared__ float wmax[W];
    const uint32_t mat = blockIdx.y;
    const ShortArgs a = args.of(mat);
    const int t = threadIdx.x;
    const bool tall = a.src.rows > a.src.cols;
    const float clip = source_clip(a.src);
    ShortPart<MP> part(tall);
    float most = 0.0f;
#pragma unroll 1
    for (uint32_t s = blockIdx.x; s < a.slabs; s += a.parts) {
        part.template load<true>(a.src, mat, s, clip);
        if (t < S::NT)
#pragma unroll
            for (int e = 0; e < S::PER; ++e) most = fmaxf(most, magnitude(part.u[e]));
    }
    most = group_max<64>(most);
    if ((t & 63) == 0) wmax[t >> 6] = most;
    __syncthreads();
    most = wmax[0];
    for (int w = 1; w < W; ++w) most = fmaxf(most, wmax[w]);
    // 2^12 <= most 2^exp < 2^13; without a finite size the products carry the NaN
    int e = 0;
    if (most < __builtin_huge_valf()) {
        e = most > 0.0f ? 12 - ilogbf(most) : kMostExp;
        e = e > kMostExp ? kMostExp : e;
    }
    const float unit = ldexpf(1.0f, e);
    if (t == 0) a.state[mat].exp[blockIdx.x] = e;
    f32x16 gram = {};
#pragma unroll 1
    for (uint32_t s = blockIdx.x; s < a.slabs; s += a.parts) {
        if (a.slabs > a.parts) {  // else the only slab is still held
            part.template load<false>(a.src, mat, s, clip);
            __syncthreads();
        }
        f16* const xt = a.xt + ((size_t)mat * a.slabs + s) * S::SLAB;
        if (t < S::NT)
#pragma unroll
            for (int k = 0; k < S::PER; k += 4) {
                const float x[4] = {part.u[k], part.u[k + 1], part.u[k + 2], part.u[k + 3]};
                f16x4 hi, lo;
                split4(x, unit, hi, lo);
                const f16x4 hi_t = quad_transpose(hi), lo_t = quad_transpose(lo);
                if (tall) {
                    Frags<kSlab>::put(rows, part.i, part.j + k, hi, lo);
                    Frags<MP>::put(xt, part.j + k + (t & 3), part.i & ~3, hi_t, lo_t);
                } else {
                    Frags<MP>::put(xt, part.j, part.i + k, hi, lo);
                    Frags<kSlab>::put(rows, part.i + k + (t & 3), part.j & ~3, hi_t, lo_t);
                }
            }
        __syncthreads();
        short_gram<MP>(rows, gram);
    }
    short_gram_store<MP>(a, mat, gram);
}

// Grid (parts, count). The segment's steps, a wave a tile. Two matrices in LDS are
// enough for two steps: A and P, then B = P A over A, A' = B P over B, P' over A', and
// Q = P P' over P'. A wave's four consecutive results lie in one column, and are kept
// as four of a row, so what is kept is the product's transpose: in this order A' = P A P
// keeps its symmetry under rounding (with P P A an error of A grows up to threefold).
// Only tiles on and under the diagonal are computed (67.0 us with all of them, 62.7 so). At m = 128 a product takes 2.3 us: 2300 to 3300 of its 5300 cycles are
// the products (ten waves: two SIMDs have three), the rest writing the result in both
// orders and two barriers. Two tiles a wave read less LDS, but their code took longer to
// fetch than that saved; reading a chain ahead gained nothing.
//
// Then X' X = Q X as X' rows: a wave takes 32 columns of X by 32 rows of Q. The first
// slab is on its way to LDS meanwhile. FINAL writes the result, in the orientation that
// runs along dst's rows. Otherwise the new pairs replace the old in xt (each
// workgroup's own slabs) and go to LDS in rows for the Gram product.
template <int MP, bool FINAL>
__global__ void __launch_bounds__(ShortShape<MP>::THREADS) short_step_kernel(const ShortArgs args) {
    using S = ShortShape<MP>;
    using F = Frags<MP>;
    __shared__ __align__(1024) f16 lds[2][S::SQ > S::SLAB ? S::SQ : S::SLAB];  // at last the slab's rows too
    __shared__ __align__(1024) f16 slab[S::SLAB];
    const uint32_t mat = blockIdx.y;
    const ShortArgs a = args.of(mat);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    auto load_slab = [&](uint32_t s) {
        constexpr int KB = S::SLAB * 2 / 1024, W = S::THREADS / 64;
        const f16* from = a.xt + ((size_t)mat * a.slabs + s) * S::SLAB + lane * 8;
#pragma unroll
        for (int k = 0; k < (KB + W - 1) / W; ++k) {
            const int c = wave + W * k;
            if (c < KB)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + c * 512),
                                                 (__attribute__((address_space(3))) void*)(slab + c * 512), 16, 0, 0);
        }
    };
    load_slab(blockIdx.x);
    ShortState& state = a.state[mat];
    float share = a.start ? 0.0f : state.share;  // on its way under the sums
    int least = kMostExp;
    if (a.start)
        for (uint32_t p = 0; p < a.parts; ++p) least = state.exp[p] < least ? state.exp[p] : least;
    const bool on = wave < S::TILES;
    int bi, bj;
    short_tile(wave, bi, bj);
    const int i0 = 32 * bi + 4 * h, j0 = 32 * bj + r;
    f32x16 v = {};
    const float* in = a.partial_in + ((size_t)mat * a.parts * S::TILES + wave) * 1024 + lane;
#pragma unroll 1
    for (uint32_t p0 = 0; p0 < (on ? a.parts : 0); p0 += 4) {  // four parts in flight
        float x[4][16];
#pragma unroll
        for (uint32_t p = 0; p < 4; ++p) {
            const float* from = in + (size_t)(p0 + p < a.parts ? p0 + p : p0) * S::TILES * 1024;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[p][e] = from[e * 64];
        }
#pragma unroll
        for (uint32_t p = 0; p < 4; ++p) {
            if (p0 + p >= a.parts) continue;
            const float f = a.start ? ldexpf(1.0f, 2 * (least - state.exp[p0 + p])) : 1.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] += f * x[p][e];
        }
    }
    float to_out = kUnitA / (kUnitX * kUnitX);
    float to_x = 1.0f / (a.unit_q * kUnitX);  // takes the exponents out of X Q
    if (a.start) {
        float* const wtrace = reinterpret_cast<float*>(lds[1]);  // nothing else is there yet
        float trace = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) trace += on && bi == bj && c32_row(e, lane) == r ? v[e] : 0.0f;
        trace = group_sum<64>(trace);
        if (lane == 0) wtrace[wave] = trace;
        __syncthreads();
        trace = 0.0f;
        for (int w = 0; w < S::THREADS / 64; ++w) trace += wtrace[w];
        __syncthreads();
        // 2^-least / (|U| + eps)
        const float scale = 1.0f / (sqrtf(trace) + a.eps * ldexpf(1.0f, least));
        to_out = scale * scale * kUnitA;
        to_x = scale * ldexpf(1.0f, least - state.exp[blockIdx.x]) / a.unit_q;
        share = sqrtf(trace) * scale;
        if (!FINAL && blockIdx.x == 0 && threadIdx.x == 0) state.share = share;
    } else {
        const int extra = extra_exp(share * a.growth_in);
        to_out = ldexpf(to_out, -2 * extra);
        to_x = ldexpf(to_x, -extra);
    }
    // op -1 stores A; then the products of a segment, each of two of the matrices in
    // LDS, over one of them; the last leaves Q
    const int last = a.steps == 2 ? 4 : 0;
#pragma unroll 1
    for (int op = -1; op <= last; ++op) {
        f16* const out = lds[op == 0];
        if (op >= 0) {
            const f16* x = lds[op == 2];
            const f16* y = lds[op == 1 || op == 4];
            if (on) v = short_product<MP, S::LOW>(x, y, bi, bj);
            to_out = op == 1 || op == 2 ? 1.0f / kUnitP : 1.0f;
            if (op == last) to_out = a.unit_q / (op == 4 ? kUnitP * kUnitP : kUnitP);
            if (on && (op == 0 || op == 3)) {  // a I + b A + c (A A), at kUnitP
                const float cc = a.c * (kUnitP / (kUnitA * kUnitA)), cb = a.b * (kUnitP / kUnitA);
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const int i = i0 + 2 * e;
                    const f16* from = lds[0] + F::at(0, j0, i);
                    const f16x4 hi = *reinterpret_cast<const f16x4*>(from);
                    const f16x4 lo = *reinterpret_cast<const f16x4*>(from + 512);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        v[e + k] = cc * v[e + k] + cb * ((float)hi[k] + (float)lo[k]) +
                                   (i + k == j0 ? a.a * kUnitP : 0.0f);
                }
            }
            __syncthreads();  // every wave has read what this goes over
        }
        if (on)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const float w[4] = {v[e], v[e + 1], v[e + 2], v[e + 3]};
                const int i = i0 + 2 * e;
                f16x4 hi, lo;
                split4(w, to_out, hi, lo);
                F::put(out, j0, i, hi, lo);
                if (bi > bj) F::put(out, i + (lane & 3), j0 & ~3, quad_transpose(hi), quad_transpose(lo));
            }
        __syncthreads();
    }
    const f16* const q = lds[last == 0];
    f16* const rows = lds[last != 0];
    if (!FINAL) to_x = ldexpf(to_x * kUnitX, extra_exp(share * a.growth));
    const bool tall = a.src.rows > a.src.cols;
    const int jb = wave % S::CB, b = wave / S::CB;  // the wave's columns of X and rows of Q
    f32x16 gram = {};
#pragma unroll 1
    for (uint32_t s = blockIdx.x; s < a.slabs; s += a.parts) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // the slab has arrived; the one before has left the rows
        // tall: a lane holds row i of X, its registers columns j, which are dst's rows
        const uint32_t along = s * kSlab + 32 * jb, across = 32 * b;
        const uint32_t y0 = (FINAL && !tall ? across : along) + 4 * h, c = (FINAL && !tall ? along : across) + r;
        float w[16];
        f32x16 acc = {};
        if (b < S::NB) {
            if (FINAL && a.step) tile_read(a.dst, a.src.rows, a.src.cols, mat, y0, c, w);
            // x y' of 32 x 32 in chains of 32, or its transpose
#pragma unroll
            for (int kk = 0; kk < MP / 16; kk += 2) {
                f16x8 x[2][2], y[2][2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int p = 0; p < 2; ++p)
                        x[e][p] = F::frag(slab, p, jb, kk + e), y[e][p] = F::frag(q, p, b, kk + e);
                acc += FINAL && !tall ? pair_mfma<true, S::LOW>(y, x) : pair_mfma<false, S::LOW>(x, y);
            }
        }
        if constexpr (FINAL) {
            if (b < S::NB) {
#pragma unroll
                for (int e = 0; e < 16; ++e) w[e] = a.step ? a.keep * w[e] - a.rate * (acc[e] * to_x) : acc[e] * to_x;
                tile_write(a.dst, a.src.rows, a.src.cols, mat, y0, c, w);
            }
            __syncthreads();
            if (s + a.parts < a.slabs) load_slab(s + a.parts);
        } else {
            if (b < S::NB) {
                f16* const xt = a.xt + ((size_t)mat * a.slabs + s) * S::SLAB;
                const int i = 32 * b + r;  // X'(i, j .. j + 3)
#pragma unroll
                for (int g = 0; g < 16; g += 4) {
                    const float u[4] = {acc[g], acc[g + 1], acc[g + 2], acc[g + 3]};
                    const int j = 32 * jb + 2 * g + 4 * h;
                    f16x4 hi, lo;
                    split4(u, to_x, hi, lo);
                    Frags<kSlab>::put(rows, i, j, hi, lo);
                    F::put(xt, j + (lane & 3), i & ~3, quad_transpose(hi), quad_transpose(lo));
                }
            }
            __syncthreads();
            if (s + a.parts < a.slabs) load_slab(s + a.parts);
            short_gram<MP>(rows, gram);
        }
    }
    if constexpr (!FINAL) short_gram_store<MP>(a, mat, gram);
}

}  // namespace dev
}  // namespace mg
