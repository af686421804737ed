// Newton-Schulz steps of matrices whose sides are both over 128: one launch a
// product of 128 x 128 tiles, or 64 x 64 where those are too few for the chip; half
// the tiles of symmetric results.
//
// Operands are pairs in the order of the matrix instructions' operands (Frags of
// muon_short.h): a tile's stage is contiguous runs of 4 KB that go to LDS as they
// lie, and LDS reads have no bank conflicts. Both sides are padded to the tile with
// zeros, so the product kernel has no bounds checks.
#pragma once
#include "muon_short.h"

namespace mg {
namespace dev {

constexpr int kPK = 32;   // contraction elements of a stage
constexpr int kRing = 4;  // stages in LDS
constexpr int kNormParts = 1024;  // most partial sums of a matrix's squares

// A thread's 16 elements of a 64 x 64 tile of the source at (i0, j0): column t % 64,
// rows 16 (t / 64) .. of it; zeros outside. UPDATE also moves the momentum.
template <bool UPDATE, class T>
__device__ __forceinline__ void tile_load(const SourceArgs& a, uint32_t k, uint32_t i0, uint32_t j0, float (&u)[16]) {
    const uint32_t j = j0 + (threadIdx.x & 63), i = i0 + (threadIdx.x >> 6) * 16;
    const uint32_t jc = j < a.cols ? j : a.cols - 1, ic = i < a.rows ? i : a.rows - 1;
    const T* in = static_cast<const T*>(a.in.data) + a.in.at(k, ic, jc);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        u[e] = (float)*in;
        in += i + e + 1 < a.rows ? a.in.ld : 0u;
    }
    if (a.momentum.data) {
        float* to = static_cast<float*>(a.momentum.data) + a.momentum.at(k, ic, jc);
        const float* from = to;
        float b[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            b[e] = *from;
            from += i + e + 1 < a.rows ? a.momentum.ld : 0u;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            if constexpr (UPDATE) {
                b[e] = moved_momentum(a, b[e], u[e]);
                if (j < a.cols && i + e < a.rows) *to = b[e];
                to += a.momentum.ld;
            }
            u[e] = update_of(a, b[e], u[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) u[e] = j < a.cols && i + e < a.rows ? u[e] : 0.0f;
}
template <bool UPDATE>
__device__ __forceinline__ void tile_load(const SourceArgs& a, uint32_t k, uint32_t i0, uint32_t j0, float (&u)[16]) {
    with_type(a.in.type, [&](auto t) { tile_load<UPDATE, decltype(t)>(a, k, i0, j0, u); });
}

// Partial sums of U^2 in 64 bits (fp32 squares leave its range), [count][gridDim.x]
// of them, and the momentum's update.
__global__ void __launch_bounds__(256) source_norm_kernel(const SourceArgs a, double* partial) {
    __shared__ double red[4];
    const uint32_t k = blockIdx.y, tiles_c = (a.cols + 63) / 64, tiles = tiles_c * ((a.rows + 63) / 64);
    double s = 0.0;
    for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        float u[16];
        tile_load<true>(a, k, t / tiles_c * 64, t % tiles_c * 64, u);
#pragma unroll
        for (int e = 0; e < 16; ++e) s += (double)u[e] * (double)u[e];
    }
    for (int step = 1; step < 64; step *= 2) s += __shfl_xor(s, step);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) partial[(size_t)k * gridDim.x + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// kUnitX 2^extra_exp / (|U| + eps) as 2^exp rest in every thread, rest in [1, 2), or NaN
// where the norm is not finite. The power is applied as an exponent: as a factor, of
// matrices near fp32's largest it would be subnormal, with few bits left.
struct SourceScale {
    int exp;
    float rest;
    float share;  // |U| / (|U| + eps)
};
struct MatrixScale {  // what the products need of it
    float rest, share;
};
__device__ __forceinline__ SourceScale source_scale(const double* partial, uint32_t parts, float eps,
                                                    SourceScale* shared) {
    if (threadIdx.x < 64) {
        double s = 0.0;
#pragma unroll 4
        for (uint32_t p = threadIdx.x; p < parts; p += 64) s += partial[p];
        for (int step = 1; step < 64; step *= 2) s += __shfl_xor(s, step);
        if (threadIdx.x == 0) {
            const double norm = sqrt(s);
            const bool finite = norm < __builtin_huge_val();
            const double scale = finite ? (double)kUnitX / (norm + (double)eps) : 1.0;
            shared->share = finite ? (float)(norm / (norm + (double)eps)) : 1.0f;
            shared->exp = ilogb(scale) + extra_exp(shared->share);
            shared->rest = finite ? (float)ldexp(scale, -ilogb(scale)) : __builtin_nanf("");
        }
    }
    __syncthreads();
    return *shared;
}

// A matrix of pairs: every 32 rows' blocks of 16 contraction elements, and 4 KB
// more. Tiles read the same stage of all their rows at once; without the extra 4 KB
// those lie a power of two apart, in the same few memory channels (the product of 2048
// x 8192 with itself: 250 us without, 203 with).
constexpr uint32_t kSkew = 2048;  // elements
__host__ __device__ __forceinline__ size_t planes_block(uint32_t k) { return (size_t)k * 64 + kSkew; }
struct Planes {
    f16* base;
    size_t stride;  // elements between matrices of the batch
    size_t block;   // and between 32 rows

    // columns c ... of row r of matrix k: c a multiple of 4; the low halves 512 further
    __device__ __forceinline__ f16* at(uint32_t k, uint32_t r, uint32_t c) const {
        return base + k * stride + (r >> 5) * block + (c >> 4) * 1024 + ((c & 8) << 5) + ((r & 31) << 3) + (c & 4);
    }
    __device__ __forceinline__ void put(uint32_t k, uint32_t r, uint32_t c, f16x4 hi, f16x4 lo) const {
        f16* const to = at(k, r, c);
        *reinterpret_cast<f16x4*>(to) = hi;
        *reinterpret_cast<f16x4*>(to + 512) = lo;
    }
};

// U / (|U| + eps) times kUnitX 2^extra_exp as pairs, X [mp][np] and its transpose XT [np][mp],
// zeros in the padding; one 64 x 64 tile of the source a workgroup. A thread's
// elements are a run along one of the two; the other takes four threads'.
// EXACT: a power of two takes the place of the factor, so that a 16-bit source fits the
// high halves (under 2^-27 of the norm to 2^-38 of it) and the low ones, which nothing
// reads, are not written; what is left of the factor goes to scales[k].
template <bool EXACT>
__global__ void __launch_bounds__(256) source_split_kernel(const SourceArgs a, const double* partial, uint32_t parts,
                                                           float eps, MatrixScale* scales, Planes X, Planes XT) {
    __shared__ SourceScale shared;
    const uint32_t k = blockIdx.z, i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
    float u[16];
    tile_load<false>(a, k, i0, j0, u);
    const SourceScale scale = source_scale(partial + (size_t)k * parts, parts, eps, &shared);
    if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) scales[k] = MatrixScale{scale.rest, scale.share};
    const float own = EXACT ? 1.0f : scale.rest;
    const bool tall = a.rows > a.cols;
    const Planes& by_column = tall ? X : XT;  // rows of it are the source's columns
    const Planes& by_row = tall ? XT : X;
    const uint32_t j = j0 + (threadIdx.x & 63), i = i0 + (threadIdx.x >> 6) * 16;
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
        float x[4];
#pragma unroll
        for (int f = 0; f < 4; ++f) x[f] = ldexpf(u[e + f], scale.exp);
        f16x4 hi, lo;
        split4(x, own, hi, lo);
        if constexpr (EXACT) {
            *reinterpret_cast<f16x4*>(by_column.at(k, j, i + e)) = hi;
            *reinterpret_cast<f16x4*>(by_row.at(k, i + e + (threadIdx.x & 3), j & ~3u)) = quad_transpose(hi);
        } else {
            by_column.put(k, j, i + e, hi, lo);
            by_row.put(k, i + e + (threadIdx.x & 3), j & ~3u, quad_transpose(hi), quad_transpose(lo));
        }
    }
}

// What becomes of a product's element v = (a b')(i, j).
enum {
    kSymmetric = 0,  // out(i, j) = out(j, i) = v
    kExactGram,      // the same of operands without low halves
    kPolynomial,     // the same with c v + b A(i, j) + a [i = j], v = (A A)(i, j)
    kUpdate,         // X' = v, both X [i][j] and XT [j][i]
    kExactUpdate,    // the same where b, the old XT, has no low halves
    kFinal,          // the result of a wide matrix: dst(i, j) = v, or keep dst(i, j) - rate v
    kFinalTall,      // and of a tall one, whose product has a and b in each other's place
};
struct ProductArgs {
    Planes a, b;       // [rows][K], [cols][K]
    uint32_t stages;   // K / kPK, a multiple of 4
    uint32_t tiles_j;  // tile columns (symmetric results: tile rows and columns)
    float unit;        // takes the operands' exponents out of the sums and puts the result's in
    const MatrixScale* scales;
    float growth, growth_out;  // extra_exp's, of X in the product, or 0 without X, and of the X that comes out
    Planes out, out_t;  // X [i][j] and XT [j][i], or a symmetric out
    // kPolynomial
    Planes gram;
    float ca, cb, cc;  // with the result's exponent; cc also takes the operands' out
    uint32_t m;        // rows that hold a matrix: no a I in the padding
    // kFinal
    Batch dst;
    uint32_t rows, cols;
    uint32_t step;  // an optimiser step
    float keep, rate;
};

// One T x T tile of a product a b' of pairs. Eight waves, T / 2 x T / 2 each as
// tiles of v_mfma_f32_32x32x16_f16: four of them take the first half of each stage's
// 32 contraction elements, four the second, and the two halves' sums meet at the end.
// So each SIMD has two waves, and one's waits are under the other's products. Stages
// (32 KB at T = 128) go from memory straight to a ring of four in LDS. The waves meet
// once a stage: the next one has then arrived (vmcnt counts in order), this one is in
// registers and its place free for the fourth one on, and the next one's fragments
// are read under this one's products. At T = 128 a stage takes 1150 cycles, of which
// 768 are matrix instructions. On 2048 x 8192, Q X takes 204 us: 1010 TFLOP/s of binary16
// products, where a large library product reaches 1168. X X' takes 160 us and a square
// 47: 680 and 580 TFLOP/s, as 136 tiles are for 256 CUs. Cutting all tiles' chains into 256
// equal runs was slower (1474 -> 1626 us in all): with every CU busy the clock falls, and
// the cut tiles' sums go through memory.
template <int T>
struct Tiling {
    static constexpr int Q = T / 64;                // 32 x 32 tiles of a wave, along each side
    static constexpr int kStage = 4 * T * kPK;      // elements: a and b, two planes each
    static constexpr int kBlocks = kStage / 512 / 8;  // of a wave and stage, 1 KB each
    static constexpr int kChain = T == 128 ? 4 : 2;  // stages; a contraction's are a multiple of it
};
template <int KIND, int T>
__global__ void __launch_bounds__(512) product_kernel(const ProductArgs p) {
    using G = Tiling<T>;
    // halves that a and b hold; of operands without low ones every second block is left alone
    constexpr int HA = KIND == kExactGram ? 1 : 2, HB = KIND == kExactGram || KIND == kExactUpdate ? 1 : 2;
    constexpr int Q = G::Q, kStage = G::kStage, B = G::kBlocks, L = KIND == kExactGram ? B / 2 : B;
    constexpr bool kResult = KIND >= kFinal, kSwap = KIND == kFinalTall, kX = KIND == kUpdate || KIND == kExactUpdate;
    __shared__ __align__(1024) f16 lds[kRing * kStage];
    const uint32_t mat = blockIdx.y, tile = xcd_run(blockIdx.x, gridDim.x);
    uint32_t ti, tj;
    if constexpr (KIND <= kPolynomial) {
        // tiles on and under the diagonal, row by row
        ti = (uint32_t)((sqrtf(8.0f * (float)tile + 1.0f) - 1.0f) * 0.5f);
        while (ti * (ti + 1) / 2 > tile) --ti;
        while ((ti + 1) * (ti + 2) / 2 <= tile) ++ti;
        tj = tile - ti * (ti + 1) / 2;
    } else {
        const uint32_t tiles_i = gridDim.x / p.tiles_j;
        ti = tile % tiles_i, tj = tile / tiles_i;
    }
    // on its way under the products
    const MatrixScale own = KIND == kPolynomial ? MatrixScale{} : p.scales[mat];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // a stage's 32-row blocks (4 KB), a's first, go to the waves in order: a block each
    // at T = 128, half of one at 64
    const int quarter = wave & 3, half = wave >> 2;
    const int block = quarter * B / 4, part = quarter * B % 4;
    const Planes& src = half ? p.b : p.a;
    const f16* from = src.base + mat * src.stride + ((half ? tj : ti) * (T / 32) + block) * src.block + part * 512 + lane * 8;
    auto load = [&](int slot, bool more) {
        f16* to = lds + slot * kStage + wave * B * 512;
#pragma unroll
        for (int c = 0; c < B; c += B / L)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + c * 512),
                                             (__attribute__((address_space(3))) void*)(to + c * 512), 16, 0, 0);
        from += more ? 2048 : 0;
    };
    const int wi = quarter >> 1, wj = quarter & 1;
    const f16* const mine = lds + half * 1024 + lane * 8;
    f16x8 fa[2][Q][2], fb[2][Q][2];  // [stages in turn][32 rows][plane]
    auto read = [&](int set, int slot) {
        const f16* at = mine + slot * kStage;
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h < HA) fa[set][q][h] = *reinterpret_cast<const f16x8*>(at + (Q * wi + q) * 2048 + h * 512);
                if (h < HB)
                    fb[set][q][h] = *reinterpret_cast<const f16x8*>(at + kStage / 2 + (Q * wj + q) * 2048 + h * 512);
            }
    };
    f32x16 acc[Q][Q] = {}, sum[Q][Q];
    const uint32_t stages = p.stages;
#pragma unroll
    for (uint32_t u = 0; u < (uint32_t)kRing; ++u) load(u, u + 1 < stages);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kRing - 1) * L) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(0, 0);
    for (uint32_t s = 0; s < stages; s += G::kChain) {
#pragma unroll
        for (int u = 0; u < G::kChain; ++u) {
            const int slot = G::kChain == kRing ? u : (s + u) & (kRing - 1);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kRing - 2) * L) : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            // past the last stage both repeat what is there, and nothing uses it
            read((u + 1) & 1, (slot + 1) & (kRing - 1));
            load(slot, s + u + kRing + 1 < stages);
#pragma unroll
            for (int term = 0; term < 3; ++term) {  // lo hi, hi lo, hi hi; kSwap: the bits of the other product
                if ((term == 0 && HA == 1) || (term == 1 && HB == 1)) continue;
#pragma unroll
                for (int i = 0; i < Q; ++i)
#pragma unroll
                    for (int j = 0; j < Q; ++j)
                        sum[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                            fa[u & 1][i][term == (kSwap ? 1 : 0)], fb[u & 1][j][term == (kSwap ? 0 : 1)],
                            u == 0 && term == (HA == 1 ? 2 : 0) ? f32x16{} : sum[i][j], 0, 0, 0);
            }
            // the reads and loads go between the products: issued before them, the
            // eight waves' reads keep LDS busy for 512 cycles in which nothing is multiplied
            if constexpr (T == 128) {
#pragma unroll
                for (int k = 0; k < 2 * (HA + HB); ++k) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
                }
#pragma unroll
                for (int k = 0; k < L; ++k) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // memory read
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < Q; ++i)
#pragma unroll
            for (int j = 0; j < Q; ++j) acc[i][j] += sum[i][j];
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last loads have left LDS alone
    // The halves' sums. A wave of two by two tiles keeps the rows of one tile and gives
    // the others to its partner; of one tile, registers 8 half .. 8 half + 7.
    __syncthreads();
    constexpr int N = Q == 2 ? 16 : 8;  // registers of a tile that a wave ends up with
    float unit = p.unit;
    if constexpr (KIND != kPolynomial) {
        if (p.growth > 0.0f) {
            const int extra = extra_exp(own.share * p.growth);
            if constexpr (KIND == kExactGram) unit *= own.rest * own.rest;
            if constexpr (KIND == kExactUpdate) unit *= own.rest;
            unit = ldexpf(unit, kX ? extra_exp(own.share * p.growth_out) - extra : kResult ? -extra : -2 * extra);
        }
    }
    float* const trade = reinterpret_cast<float*>(lds);
    float got[2][N];
    auto keep = [&](int qj, int e, bool other) -> float {
        if constexpr (Q == 2) return (half != 0) != other ? acc[1][qj][e] : acc[0][qj][e];
        return (half != 0) != other ? acc[0][0][8 + e] : acc[0][0][e];
    };
#pragma unroll
    for (int qj = 0; qj < Q; ++qj)
#pragma unroll
        for (int e = 0; e < N; ++e) trade[((wave * Q + qj) * N + e) * 64 + lane] = keep(qj, e, true);
    __syncthreads();
#pragma unroll
    for (int qj = 0; qj < Q; ++qj)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float theirs = trade[(((wave ^ 4) * Q + qj) * N + e) * 64 + lane], own = keep(qj, e, false);
            got[qj][e] = half ? theirs + own : own + theirs;
        }
#pragma unroll
    for (int qj = 0; qj < Q; ++qj) {
        // register e of got lies 8 (e / 4) + e % 4 rows under i0
        const uint32_t i0 = ti * T + wi * (T / 2) + (Q == 2 ? 32 : 16) * half + 4 * (lane >> 5);
        const uint32_t j = tj * T + wj * (T / 2) + 32 * qj + (lane & 31);
        if constexpr (kResult) {
            float w[N];
            if (p.step) tile_read(p.dst, p.rows, p.cols, mat, i0, j, w);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float o = got[qj][e] * unit;
                w[e] = p.step ? p.keep * w[e] - p.rate * o : o;
            }
            tile_write(p.dst, p.rows, p.cols, mat, i0, j, w);
            continue;
        }
#pragma unroll
        for (int r = 0; r < N; r += 4) {
            const uint32_t i = i0 + 2 * r;  // four rows from here: registers r .. r + 3
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = got[qj][r + e];
            if constexpr (KIND == kPolynomial) {
                const f16* g = p.gram.at(mat, j, i);
                const f16x4 gh = *reinterpret_cast<const f16x4*>(g), gl = *reinterpret_cast<const f16x4*>(g + 512);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = p.cc * v[e] + p.cb * ((float)gh[e] + (float)gl[e]) + (i + e == j && j < p.m ? p.ca : 0.0f);
            }
            f16x4 hi, lo;
            split4(v, KIND == kPolynomial ? 1.0f : unit, hi, lo);
            (kX ? p.out_t : p.out).put(mat, j, i, hi, lo);
            if (kX || ti != tj)
                p.out.put(mat, i + (lane & 3), j & ~3u, quad_transpose(hi), quad_transpose(lo));
        }
    }
}

}  // namespace dev
}  // namespace mg
