// Softmax cross entropy over many classes without its logits, and its gradients
// (mg_cross_entropy, mg_cross_entropy_backward).
//
// Forward: one product W X' whose tiles end in each row's maximum, sum of exponentials and
// sum weighted by the logits, and a launch that joins the tiles' results. Backward: the
// logits again, a piece of the classes at a time; each piece's gradient with respect to the
// logits, G = dloss (p - [target]) - dentropy p (log p + H), is stored in 16 bits, by rows and by
// classes, and enters two products, dX += G W and dW = G' X.
//
// All three are one kernel (head_kernel): tiles of a b' with both operands' contraction
// running along memory, 16-bit operands, fp32 sums. 16-bit arrays of a fitting shape are
// read where they lie, others are copied. fp32 operands become two binary16 halves at a power
// of two (22 bits), and their product three: low high + high low + high high, one after the other.
#include <type_traits>

#include "mg/device/common.h"
#include "sequence.h"

namespace mg {
namespace dev {

typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
template <class H>
struct Halves;
template <>
struct Halves<_Float16> {
    typedef h16x4 x4;
    typedef h16x8 x8;
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Halves<__bf16> {
    typedef b16x4 x4;
    typedef b16x8 x8;
    static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

// Powers of two that bring the operands into binary16's range, and back: of x (over
// all rows that have a target), of W, of the logits' gradient. All 1 where nothing is scaled.
struct HeadScales {
    float x, w, g;
    float x_back, w_back, g_back;
};

// An operand of `rows` rows of 16-bit elements, `ld` apart: a high plane, and where values
// are pairs a low one `plane` elements after it.
struct HeadOperand {
    const void* base;
    uint64_t plane;
    uint32_t ld;
    uint32_t rows;
};

enum { kStats = 0, kLogitGrad = 1, kGrad = 2 };

// One product's tiles: M from a, N from b, contraction K in `splits` ranges of `range`.
struct HeadProduct {
    HeadOperand a, b;
    uint32_t k, range, splits;
    uint32_t tiles_m, tiles_n;
    // kGrad: out(n, m) = sum, n down the rows of out; or fp32 parts [splits][out rows][parts_ld]
    void* out;
    float* parts;
    uint64_t out_ld;
    uint32_t parts_ld;
    uint32_t add;      // parts += sum
    uint32_t which;    // 0: dX, 1: dW (whose scale takes the product back)
};

struct HeadArgs {
    HeadProduct p[2];
    uint32_t tiles;  // of p[0], all splits
    const HeadScales* scales;
    const int* row_exp;  // fp32 x: each row's own power of two, so that no row feels another
    uint32_t rows, classes, first;  // classes from `first` on: the piece
    const int32_t* targets;
    // kStats: [tiles of classes][rows_ld][3], and the target's logit
    float* stats;
    float* of;
    uint32_t rows_ld, want_entropy;
    // kLogitGrad
    const float* lse;
    const float* dloss;
    const float* entropy;
    const float* dentropy;
    void* g;    // [rows_ld][g_ld], planes g_plane apart
    void* gt;   // [g_ld][rows_ld]
    uint32_t g_ld;
    uint64_t g_plane;
};

constexpr int kHeadK = 32;     // contraction elements of a stage
constexpr int kHeadRing = 4;   // stages in LDS
constexpr int kHeadN = 256;    // columns of a tile
constexpr uint32_t kNowhere = 0x80000000u;  // an offset past every operand's end: reads 0

// The logarithm and the exponential in base 2, by the hardware's instructions.
__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
constexpr float kLog2 = 1.44269504f, kLn2 = 0.693147181f;

// max, sum of 2^(s - max), sum of 2^(s - max) (s - max), of logits in base 2. Of
// nothing: -inf, 0, 0.
struct RowStats {
    float top, sum, weighted;
    __device__ __forceinline__ void join(const RowStats& o) {
        const float most = __builtin_fmaxf(top, o.top);
        // differences from a maximum of -inf would be NaN; there the sums are 0
        const float a = top == most ? 0.0f : top - most, b = o.top == most ? 0.0f : o.top - most;
        const float ea = exp2_of(a), eb = exp2_of(b);
        const float wa = a < -1000.0f ? 0.0f : a, wb = b < -1000.0f ? 0.0f : b;
        weighted = ea * (weighted + wa * sum) + eb * (o.weighted + wb * o.sum);
        sum = ea * sum + eb * o.sum;
        top = most;
    }
};

// One tile of MI x 64 rows of a by 256 rows of b. Eight waves, two along a and four
// along b, MI x 2 tiles of 32 x 32 each. A stage is 32 contraction elements of every row, 64
// bytes, which go from memory straight to LDS: a lane's 16 bytes lie in the order of the
// lanes, so the places of a row's four are exchanged on the way by the lane's own address
// (bits 1 and 2 of the row), and the reads of eight rows then meet no bank twice. The ring
// holds four stages; the waves meet once a stage, when the next has arrived, and read the
// next one's fragments under this one's products.
template <class H, int KIND, int MI, bool PAIRS>
__global__ void __launch_bounds__(512) head_kernel(const HeadArgs args) {
    using X = Halves<H>;
    typedef typename X::x8 x8;
    typedef typename X::x4 x4;
    constexpr int TM = MI * 64, kStage = (TM + kHeadN) * 64, LA = TM / 128, LB = kHeadN / 128, L = LA + LB;
    __shared__ __align__(1024) char lds[kHeadRing * kStage];
    const uint32_t tile_of_all = xcd_run(blockIdx.x, gridDim.x);
    const uint32_t sel = KIND == kGrad && tile_of_all >= args.tiles ? 1 : 0;
    const HeadProduct& p = args.p[sel];
    uint32_t tile = tile_of_all - (sel ? args.tiles : 0);
    const uint32_t per = p.tiles_m * p.tiles_n, split = tile / per;
    tile -= split * per;
    // tiles that share their rows of a lie side by side
    const uint32_t tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
    const uint32_t from = split * p.range, to = p.k - from < p.range ? p.k : from + p.range;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;

    // this wave's loads of a stage: 16 rows each
    const uint32_t chunk = (lane & 3) ^ (lane >> 3 & 3);  // of the row's four
    __amdgpu_buffer_rsrc_t res[2][2];                      // [a, b][high, low]
    uint32_t off[L];
    {
        const uint32_t m0 = tm * TM, n0 = tn * kHeadN;
        auto bind = [&](const HeadOperand& o, uint32_t r0, int which) {
            const uint32_t left = o.rows > r0 ? o.rows - r0 : 0;
            const uint32_t most = which ? kHeadN : TM, have = left < most ? left : most;
            const uint32_t bytes = have ? ((have - 1) * o.ld + p.k) * 2 : 0;
            H* at = const_cast<H*>(static_cast<const H*>(o.base)) + (uint64_t)r0 * o.ld;
            res[which][0] = __builtin_amdgcn_make_buffer_rsrc(at, (short)0, (int)bytes, 0x00020000);
            res[which][1] = __builtin_amdgcn_make_buffer_rsrc(at + o.plane, (short)0, (int)bytes, 0x00020000);
            const int n = which ? LB : LA;
#pragma unroll
            for (int c = 0; c < (which ? LB : LA); ++c) {
                const uint32_t r = (wave * n + c) * 16 + (lane >> 2);
                off[(which ? LA : 0) + c] = r < have ? r * o.ld * 2 + chunk * 16 : kNowhere;
            }
        };
        bind(p.a, m0, 0);
        bind(p.b, n0, 1);
    }
    uint32_t k = from;
    int seg = 0;
    const uint32_t each = (to - from + kHeadK - 1) / kHeadK;
    const uint32_t stages = (each * (PAIRS ? 3 : 1) + 1) & ~1u;  // the last may be empty
    auto load = [&](uint32_t slot) {
        char* const at = lds + slot * kStage;
        const bool in = k + chunk * 8 < to && (!PAIRS || seg < 3);
#pragma unroll
        for (int c = 0; c < L; ++c) {
            const int which = c >= LA;
            const int n = which ? LB : LA, i = which ? c - LA : c;
            char* const dst = at + (which ? TM * 64 : 0) + (wave * n + i) * 1024;
            const uint32_t o = in && off[c] != kNowhere ? off[c] + k * 2 : kNowhere;
            const bool low = PAIRS && seg == which;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(low ? res[which][1] : res[which][0],
                                                     (__attribute__((address_space(3))) void*)dst, 16, (int)o, 0, 0, 0);
        }
        k += kHeadK;
        if (PAIRS && k >= to) k = from, ++seg;
    };
    // fragments: lane l holds row l % 32 and eight elements of the 16, by l / 32
    const int row = lane & 31, twist = row >> 1 & 3;
    const int at0 = row * 64 + (((lane >> 5) ^ twist) << 4), at1 = row * 64 + ((2 + (lane >> 5) ^ twist) << 4);
    x8 fa[2][2][MI], fb[2][2][2];
    auto read = [&](int set, uint32_t slot) {
        const char* const a = lds + slot * kStage + wm * (MI * 2048);
        const char* const b = lds + slot * kStage + TM * 64 + wn * 4096;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = h ? at1 : at0;
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[set][h][i] = *reinterpret_cast<const x8*>(a + i * 2048 + at);
#pragma unroll
            for (int j = 0; j < 2; ++j) fb[set][h][j] = *reinterpret_cast<const x8*>(b + j * 2048 + at);
        }
    };
    f32x16 acc[MI][2] = {};
#pragma unroll
    for (uint32_t u = 0; u < (uint32_t)kHeadRing; ++u) load(u);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kHeadRing - 1) * L) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(0, 0);
    for (uint32_t s = 0; s < stages; s += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t slot = (s + u) & (kHeadRing - 1);
            // the next stage is there, this one is in registers
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kHeadRing - 2) * L) : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            read(u ^ 1, (slot + 1) & (kHeadRing - 1));
            load(slot);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = X::mfma(fa[u][h][i], fb[u][h][j], acc[i][j]);
#pragma unroll
            for (int q = 0; q < 2 * (MI + 2); ++q) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last loads have left LDS alone

    // register e of tile (i, j): row of a m(i, e), row of b n(j)
    const uint32_t m0 = tm * TM + wm * (MI * 32) + 4 * (lane >> 5), n0 = tn * kHeadN + wn * 64 + (lane & 31);
    const HeadScales sc = args.scales ? *args.scales : HeadScales{1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
    if constexpr (KIND == kGrad) {
        const float b0 = sc.g_back, b1 = p.which ? sc.x_back : sc.w_back;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t n = n0 + 32 * j;
            if (n >= p.b.rows) continue;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const uint32_t m = m0 + 32 * i + 2 * e;
                    if (m >= p.a.rows) continue;
                    f32x4 v = {acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
                    if (p.parts) {
                        f32x4* const at = reinterpret_cast<f32x4*>(
                            p.parts + ((uint64_t)split * p.b.rows + n) * p.parts_ld + m);
                        if (p.add) v += *at;
                        *at = v;
                        continue;
                    }
#pragma unroll
                    for (int q = 0; q < 4; ++q) v[q] = v[q] * b0 * b1;
                    const uint32_t count = p.a.rows - m;
                    auto put = [&](auto t) {
                        using T = decltype(t);
                        T* const at = static_cast<T*>(p.out) + n * p.out_ld + m;
                        if (count >= 4) {
                            typedef T vec __attribute__((ext_vector_type(4)));
                            const vec w = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
                            __builtin_memcpy(at, &w, sizeof(w));
                        } else {
#pragma unroll
                            for (int q = 0; q < 3; ++q)
                                if (q < (int)count) at[q] = (T)v[q];
                        }
                    };
                    if constexpr (PAIRS)
                        put(0.0f);
                    else
                        put(H{});
                }
        }
    } else {
        const float to2 = sc.w_back * kLog2;
        const uint32_t c0 = m0;  // of the piece
        const bool edge = (tm + 1) * TM > p.a.rows;
        if constexpr (KIND == kStats) {
            __syncthreads();  // every wave is done with the ring
            RowStats* const trade = reinterpret_cast<RowStats*>(lds);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t n = n0 + 32 * j;
                const int32_t target = n < args.rows ? args.targets[n] : -1;
                // two factors: their product may leave fp32's range
                const float back = PAIRS && n < args.rows ? ldexpf(1.0f, -args.row_exp[n]) : 1.0f;
                RowStats r{-__builtin_huge_valf(), 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const uint32_t c = c0 + 32 * i + 8 * (e >> 2) + (e & 3);
                        const float s = acc[i][j][e] * back * to2;
                        acc[i][j][e] = edge && c >= p.a.rows ? -__builtin_huge_valf() : s;
                        r.top = __builtin_fmaxf(r.top, acc[i][j][e]);
                        if (target >= 0 && (uint32_t)target == c) args.of[n] = s;
                    }
                const float zero = r.top == -__builtin_huge_valf() ? 0.0f : r.top;
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float d = acc[i][j][e] - zero, w = exp2_of(d);
                        r.sum += w;
                        r.weighted = __builtin_fmaf(w, __builtin_fmaxf(d, -1000.0f), r.weighted);
                    }
                RowStats o;
                float lo, hi;
                lane_pair<32>(r.top, lo, hi), r.top = lo, o.top = hi;
                lane_pair<32>(r.sum, lo, hi), r.sum = lo, o.sum = hi;
                lane_pair<32>(r.weighted, lo, hi), r.weighted = lo, o.weighted = hi;
                r.join(o);
                if (lane < 32) trade[wm * kHeadN + wn * 64 + 32 * j + lane] = r;
            }
            __syncthreads();
            if (threadIdx.x < kHeadN) {
                const uint32_t n = tn * kHeadN + threadIdx.x;
                RowStats r = trade[threadIdx.x];
                r.join(trade[kHeadN + threadIdx.x]);
                if (n < args.rows) {
                    float* const at = args.stats + (uint64_t)tm * 3 * args.rows_ld + n;
                    at[0] = r.top, at[args.rows_ld] = r.sum, at[2 * (uint64_t)args.rows_ld] = r.weighted;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t n = n0 + 32 * j;
                int32_t target = -1;
                float lse2 = 0.0f, dl = 0.0f, de = 0.0f, ent = 0.0f, back = 1.0f;
                if (n < args.rows) {
                    if (PAIRS) back = ldexpf(1.0f, -args.row_exp[n]);
                    target = args.targets[n];
                    lse2 = args.lse[n] * kLog2, dl = args.dloss[n] * sc.g;
                    if (args.dentropy) de = args.dentropy[n] * sc.g, ent = args.entropy[n];
                }
                const bool live = target >= 0 && (uint32_t)target < args.classes;
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const uint32_t c = c0 + 32 * i + 2 * e;
                        float v[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float d = __builtin_fmaf(acc[i][j][e + q] * back, to2, -lse2), prob = exp2_of(d);
                            float g = dl * prob;
                            if (args.dentropy)
                                g -= de * prob * __builtin_fmaf(__builtin_fmaxf(d, -1000.0f), kLn2, ent);
                            if (live && c + q == (uint32_t)target - args.first) g -= dl;
                            v[q] = live && !(edge && c + q >= p.a.rows) ? g : 0.0f;
                        }
                        x4 hi, lo;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            hi[q] = (H)v[q];
                            if constexpr (PAIRS) {
                                // what is not finite lies in the low half alone
                                const bool odd = !(__builtin_fabsf(v[q]) < 65504.0f);
                                hi[q] = odd ? (H)0.0f : hi[q];
                                lo[q] = odd ? (H)v[q] : (H)(v[q] - (float)hi[q]);
                            }
                        }
                        H* const g = static_cast<H*>(args.g) + (uint64_t)n * args.g_ld + c;
                        *reinterpret_cast<x4*>(g) = hi;
                        if constexpr (PAIRS) *reinterpret_cast<x4*>(g + args.g_plane) = lo;
                        // four rows of one class: the quad's lanes trade theirs
                        H* const gt =
                            static_cast<H*>(args.gt) + (uint64_t)(c + (lane & 3)) * args.rows_ld + (n & ~3u);
                        *reinterpret_cast<x4*>(gt) = quad_transpose(hi);
                        if constexpr (PAIRS) *reinterpret_cast<x4*>(gt + args.g_plane) = quad_transpose(lo);
                    }
            }
        }
    }
}

// Joins a row's tiles: a wave a row.
__global__ void __launch_bounds__(256) head_join_kernel(const float* stats, const float* of, const int32_t* targets,
                                                        uint32_t rows, uint32_t rows_ld, uint32_t tiles,
                                                        uint32_t classes, float* loss, float* lse, float* entropy) {
    const int lane = threadIdx.x & 63;
    for (uint32_t n = blockIdx.x * 4 + (threadIdx.x >> 6); n < rows; n += gridDim.x * 4) {
        RowStats r{-__builtin_huge_valf(), 0.0f, 0.0f};
        for (uint32_t t = lane; t < tiles; t += 64) {
            const float* const at = stats + (uint64_t)t * 3 * rows_ld + n;
            r.join(RowStats{at[0], at[rows_ld], at[2 * (uint64_t)rows_ld]});
        }
#pragma unroll
        for (int step = 1; step < 64; step *= 2)
            r.join(RowStats{__shfl_xor(r.top, step), __shfl_xor(r.sum, step), __shfl_xor(r.weighted, step)});
        if (lane) continue;
        const float log = __builtin_amdgcn_logf(r.sum), all = (r.top + log) * kLn2;
        const int32_t target = targets[n];
        if (loss)
            loss[n] = target >= 0 && (uint32_t)target < classes ? (r.top - of[n] + log) * kLn2 : 0.0f;
        if (lse) lse[n] = all;
        if (entropy) entropy[n] = (log - r.weighted / r.sum) * kLn2;
    }
}

// The exponent that brings v under 2^15.
__device__ __forceinline__ int lift(float v) {
    const int e = v > 0.0f ? 14 - ilogbf(v) : 0;
    return e < -126 ? -126 : e > 126 ? 126 : e;
}

// The largest finite |v| of a [rows][cols] array, a part a workgroup, of the rows that have
// a target where there are targets, and each row's exponent where asked for; of the rows'
// gradients (cols 0) the largest that a logit's gradient can be.
struct AmaxArgs {
    const float* v;
    uint64_t ld;
    uint32_t rows, cols;
    const float* more;
    float factor;
    const int32_t* targets;
    uint32_t classes;
    float* parts;
    int* row_exp;
};
constexpr uint32_t kAmaxParts = 256;
__global__ void __launch_bounds__(256) head_amax_kernel(const AmaxArgs a0, const AmaxArgs a1, const AmaxArgs a2) {
    __shared__ float red[4];
    const AmaxArgs a = blockIdx.y == 0 ? a0 : blockIdx.y == 1 ? a1 : a2;
    const uint32_t lane = threadIdx.x & 63;
    float most = 0.0f;
    auto larger = [](float most, float v) {
        v = __builtin_fabsf(v);
        return v < __builtin_huge_valf() ? __builtin_fmaxf(most, v) : most;
    };
    auto live = [&](uint32_t r) { return !a.targets || (a.targets[r] >= 0 && (uint32_t)a.targets[r] < a.classes); };
    if (a.cols) {
        for (uint32_t r = blockIdx.x * 4 + (threadIdx.x >> 6); r < a.rows; r += gridDim.x * 4) {
            float mine = 0.0f;
#pragma unroll 4
            for (uint32_t c = lane; c < a.cols; c += 64) mine = larger(mine, a.v[r * a.ld + c]);
            mine = group_max<64>(mine);
            if (a.row_exp && !lane) a.row_exp[r] = lift(mine);
            if (live(r)) most = __builtin_fmaxf(most, mine);
        }
    } else {
        for (uint32_t r = blockIdx.x * 256 + threadIdx.x; r < a.rows; r += gridDim.x * 256)
            if (live(r)) most = larger(most, __builtin_fabsf(a.v[r]) + (a.more ? a.factor * __builtin_fabsf(a.more[r]) : 0.0f));
        most = group_max<64>(most);
    }
    if (!lane) red[threadIdx.x >> 6] = most;
    __syncthreads();
    if (threadIdx.x == 0)
        a.parts[blockIdx.x] = __builtin_fmaxf(__builtin_fmaxf(red[0], red[1]), __builtin_fmaxf(red[2], red[3]));
}

// Powers of two that bring the largest of each under 2^15, from the three arrays'
// parts (NULL: 1).
__global__ void __launch_bounds__(256) head_scales_kernel(const float* x, const float* w, const float* g,
                                                          HeadScales* out) {
    __shared__ float red[3][4];
    const float* const from[3] = {x, w, g};
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const float v = group_max<64>(from[k] ? from[k][threadIdx.x] : 0.0f);
        if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = v;
    }
    __syncthreads();
    if (threadIdx.x) return;
    float s[3], back[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const float v = __builtin_fmaxf(__builtin_fmaxf(red[k][0], red[k][1]), __builtin_fmaxf(red[k][2], red[k][3]));
        const int e = lift(v);
        s[k] = from[k] ? ldexpf(1.0f, e) : 1.0f, back[k] = from[k] ? ldexpf(1.0f, -e) : 1.0f;
    }
    *out = HeadScales{s[0], s[1], s[2], back[0], back[1], back[2]};
}

// 16-bit copies of a [rows][cols] array: as it lies, [rows][ld], or turned, [cols][ld] with
// rows whose target is none as zeros; zeros up to `fill` in the contraction. fp32 becomes
// pairs at the scale.
struct CopyArgs {
    const void* from;
    uint64_t from_ld;
    uint32_t rows, cols;
    uint32_t fill;  // elements of a copy's row that are written
    uint32_t ld;
    void* to;
    uint64_t plane;
    const HeadScales* scales;
    const int* row_exp;  // in place of the scale
    uint32_t which;      // 0: x's scale, 1: W's
    const int32_t* targets;
    uint32_t classes;
};
template <class H>
__device__ __forceinline__ void split_half(float v, H& hi, H& lo) {
    const bool odd = !(__builtin_fabsf(v) < 65504.0f);
    hi = odd ? (H)0.0f : (H)v;
    lo = odd ? (H)v : (H)(v - (float)hi);
}
template <class T, class H>
__global__ void __launch_bounds__(256) head_copy_kernel(const CopyArgs a) {
    constexpr bool kPairs = sizeof(T) == 4;
    const uint32_t c = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (c >= a.fill) return;
    typedef typename Halves<H>::x4 x4;
    for (uint32_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float scale = !kPairs ? 1.0f : a.row_exp ? ldexpf(1.0f, a.row_exp[r]) : a.scales->w;
        const T* const from = static_cast<const T*>(a.from) + r * a.from_ld;
        x4 hi, lo;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const T v = c + q < a.cols ? from[c + q] : (T)0.0f;
            H h, l;
            if constexpr (kPairs)
                split_half<H>((float)v * scale, h, l);
            else
                h = (H)v;
            hi[q] = h;
            if constexpr (kPairs) lo[q] = l;
        }
        H* const to = static_cast<H*>(a.to) + (uint64_t)r * a.ld + c;
        *reinterpret_cast<x4*>(to) = hi;
        if constexpr (kPairs) *reinterpret_cast<x4*>(to + a.plane) = lo;
    }
}
template <class T, class H>
__global__ void __launch_bounds__(256) head_turn_kernel(const CopyArgs a) {
    constexpr bool kPairs = sizeof(T) == 4;
    __shared__ T tile[64][65];
    const float scale = kPairs ? (a.which ? a.scales->w : a.scales->x) : 1.0f;
    const uint32_t c0 = blockIdx.x * 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (uint32_t r0 = blockIdx.y * 64; r0 < a.fill; r0 += gridDim.y * 64) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const uint32_t r = r0 + wave * 16 + k;
            bool in = r < a.rows && c0 + lane < a.cols;
            if (in && a.targets) in = a.targets[r] >= 0 && (uint32_t)a.targets[r] < a.classes;
            tile[wave * 16 + k][lane] = in ? static_cast<const T*>(a.from)[r * a.from_ld + c0 + lane] : (T)0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const uint32_t c = c0 + wave * 16 + k;
            if (c >= a.cols || r0 + lane >= a.fill) continue;
            const T v = tile[lane][wave * 16 + k];
            H* const to = static_cast<H*>(a.to) + (uint64_t)c * a.ld + r0 + lane;
            if constexpr (kPairs) {
                H h, l;
                split_half<H>((float)v * scale, h, l);
                to[0] = h, to[a.plane] = l;
            } else {
                to[0] = (H)v;
            }
        }
    }
}

// out = the sum of its parts, in order, at the scale.
template <class T>
__global__ void __launch_bounds__(256) head_sum_kernel(const float* parts, uint32_t count, uint32_t rows, uint32_t cols,
                                                       uint32_t ld, T* out, uint64_t out_ld, const HeadScales* scales,
                                                       uint32_t which) {
    const float b0 = scales ? scales->g_back : 1.0f, b1 = !scales ? 1.0f : which ? scales->x_back : scales->w_back;
    const uint32_t c = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (c >= cols) return;
    for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y) {
        f32x4 v = {};
        for (uint32_t k = 0; k < count; ++k)
            v += *reinterpret_cast<const f32x4*>(parts + ((uint64_t)k * rows + r) * ld + c);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (c + q < cols) out[r * out_ld + c + q] = (T)(v[q] * b0 * b1);
    }
}

}  // namespace dev

namespace {

constexpr uint32_t kMostHeadRows = 1u << 20, kMostClasses = 1u << 20, kMostWidth = 1u << 16;
constexpr uint32_t kHeadM = 256;          // classes of a tile
constexpr uint32_t kPieceCells = 1u << 25;  // logits of a piece: 512 tiles, two rounds of the chip's CUs
constexpr uint32_t kRange = 4096;         // contraction elements of a gradient's tile

uint32_t up_to(uint64_t n, uint32_t m) { return (uint32_t)((n + m - 1) / m * m); }
uint64_t padded(uint64_t bytes) { return (bytes + 255) & ~(uint64_t)255; }

// Hands out a workspace's parts.
struct Carve {
    char* at;
    uint64_t used = 0;
    template <class T>
    T* take(uint64_t count) {
        T* const p = reinterpret_cast<T*>(at + used);
        used += padded(count * sizeof(T));
        return p;
    }
};

// What a call keeps in its workspace. 16-bit planes; pairs have two.
struct HeadSpace {
    uint32_t width8, rows_ld, piece, pieces, splits_x, splits_w, range_x, range_w, parts_ld;
    uint64_t planes;
    uint16_t *x, *w, *xt, *wt, *g, *gt;
    float *stats, *of, *parts_x, *parts_w, *amax;
    int* row_exp;
    dev::HeadScales* scales;
    uint64_t bytes;

    HeadSpace(void* base, uint32_t rows, uint32_t classes, uint32_t width, uint32_t type, bool backward) {
        Carve c{static_cast<char*>(base)};
        planes = type == MG_TYPE_FP32 ? 2 : 1;
        width8 = up_to(width, 8), rows_ld = up_to(rows, dev::kHeadN);
        scales = c.take<dev::HeadScales>(1);
        amax = c.take<float>(3 * dev::kAmaxParts);
        row_exp = c.take<int>(planes > 1 ? rows : 0);
        x = c.take<uint16_t>(planes * rows * width8);
        w = c.take<uint16_t>(planes * classes * width8);
        if (!backward) {
            stats = c.take<float>((uint64_t)up_to(classes, kHeadM) / kHeadM * 3 * rows_ld);
            of = c.take<float>(rows_ld);
            bytes = c.used;
            return;
        }
        const uint32_t all = up_to(classes, kHeadM);
        piece = rows_ld ? up_to(kPieceCells / rows_ld, kHeadM) : kHeadM;
        piece = piece < kRange ? kRange : piece > 32 * kRange ? 32 * kRange : piece;
        pieces = (all + piece - 1) / piece;
        piece = up_to((all + pieces - 1) / pieces, kHeadM);
        auto cut = [](uint32_t k, uint32_t& splits, uint32_t& range) {
            splits = (k + kRange / 2) / kRange;
            if (!splits) splits = 1;
            range = up_to((k + splits - 1) / splits, dev::kHeadK);
            if (k) splits = (k + range - 1) / range;
        };
        cut(piece, splits_x, range_x);
        cut(rows_ld, splits_w, range_w);
        parts_ld = up_to(width, 4);
        xt = c.take<uint16_t>(planes * width * rows_ld);
        wt = c.take<uint16_t>(planes * width * piece);
        g = c.take<uint16_t>(planes * rows_ld * piece);
        gt = c.take<uint16_t>(planes * rows_ld * piece);
        parts_x = c.take<float>(splits_x > 1 || pieces > 1 ? (uint64_t)splits_x * rows * parts_ld : 0);
        parts_w = c.take<float>(splits_w > 1 ? (uint64_t)splits_w * piece * parts_ld : 0);
        bytes = c.used;
    }
};

// A 16-bit array that the products read where it lies.
bool fits(const void* p, uint64_t ld, uint32_t cols, uint32_t type) {
    return type != MG_TYPE_FP32 && cols % 8 == 0 && ld % 8 == 0 && ld <= (1u << 21) && aligned(p, 16);
}

dim3 copy_grid(uint32_t cols, uint32_t rows) { return dim3((cols + 1023) / 1024, rows < 65535 ? rows : 65535); }

// x or W as an operand: where it lies, or its copy.
template <class T, class H>
dev::HeadOperand operand_of(hipStream_t st, const void* p, uint64_t ld, uint32_t rows, uint32_t cols, uint32_t type,
                            const HeadSpace& s, uint16_t* copy, uint32_t which, const dev::HeadScales* scales) {
    if (fits(p, ld, cols, type)) return {p, 0, (uint32_t)ld, rows};
    const uint64_t plane = (uint64_t)rows * s.width8;
    const dev::CopyArgs a{p,      ld,   rows,    cols, s.width8, s.width8, copy, plane, scales, which ? nullptr : s.row_exp,
                          which, nullptr, 0};
    hipLaunchKernelGGL((dev::head_copy_kernel<T, H>), copy_grid(s.width8, rows), dim3(256), 0, st, a);
    return {copy, plane, s.width8, rows};
}

template <class T>
struct HeadType {
    typedef T H;
};
template <>
struct HeadType<float> {
    typedef _Float16 H;
};

// The scales of fp32 operands and, backwards, of 16-bit floats' gradients.
template <class T>
const dev::HeadScales* scales_of(hipStream_t st, const void* x, uint64_t x_ld, const void* w, uint64_t w_ld,
                                 uint32_t rows, uint32_t classes, uint32_t width, const float* dloss,
                                 const float* dentropy, const int32_t* targets, const HeadSpace& s) {
    const bool pairs = std::is_same<T, float>::value, g = dloss && !std::is_same<T, __bf16>::value;
    if (!pairs && !g) return nullptr;
    float* const parts = s.amax;
    const dev::AmaxArgs ax{static_cast<const float*>(pairs ? x : nullptr), x_ld, pairs ? rows : 0, width, nullptr, 0,
                           targets, classes, parts, s.row_exp};
    const dev::AmaxArgs aw{static_cast<const float*>(pairs ? w : nullptr), w_ld, pairs ? classes : 0, width, nullptr, 0,
                           nullptr, 0, parts + dev::kAmaxParts, nullptr};
    // |p (log p + H)| is at most 1/e + H, and H at most log(classes)
    const dev::AmaxArgs ag{dloss,   0,       g ? rows : 0, 0, dentropy, __builtin_logf((float)classes) + 1.0f, targets,
                           classes, parts + 2 * dev::kAmaxParts, nullptr};
    hipLaunchKernelGGL(dev::head_amax_kernel, dim3(dev::kAmaxParts, 3), dim3(256), 0, st, ax, aw, ag);
    hipLaunchKernelGGL(dev::head_scales_kernel, dim3(1), dim3(256), 0, st, pairs ? parts : nullptr,
                       pairs ? parts + dev::kAmaxParts : nullptr, g ? parts + 2 * dev::kAmaxParts : nullptr, s.scales);
    return s.scales;
}

template <class T>
int cross_entropy(hipStream_t st, const mg_cross_entropy_args& p) {
    typedef typename HeadType<T>::H H;
    constexpr bool kPairs = sizeof(T) == 4;
    const HeadSpace s(p.workspace, p.rows, p.classes, p.width, p.type, false);
    dev::HeadArgs a{};
    a.scales = scales_of<T>(st, p.x, p.x_ld, p.w, p.w_ld, p.rows, p.classes, p.width, nullptr, nullptr, nullptr, s);
    dev::HeadProduct& m = a.p[0];
    m.a = operand_of<T, H>(st, p.w, p.w_ld, p.classes, p.width, p.type, s, s.w, 1, a.scales);
    m.b = operand_of<T, H>(st, p.x, p.x_ld, p.rows, p.width, p.type, s, s.x, 0, a.scales);
    m.k = m.range = s.width8, m.splits = 1;
    m.tiles_m = up_to(p.classes, kHeadM) / kHeadM, m.tiles_n = s.rows_ld / dev::kHeadN;
    a.tiles = m.tiles_m * m.tiles_n;
    a.rows = p.rows, a.classes = p.classes, a.targets = p.targets, a.row_exp = s.row_exp;
    a.stats = s.stats, a.of = s.of, a.rows_ld = s.rows_ld;
    hipLaunchKernelGGL((dev::head_kernel<H, dev::kStats, 4, kPairs>), dim3(a.tiles), dim3(512), 0, st, a);
    MG_HIP(hipGetLastError(), "cross entropy launch");
    const uint32_t blocks = (p.rows + 3) / 4;
    hipLaunchKernelGGL(dev::head_join_kernel, dim3(blocks < 16384 ? blocks : 16384), dim3(256), 0, st, s.stats, s.of,
                       p.targets, p.rows, s.rows_ld, m.tiles_m, p.classes, p.loss, p.lse, p.entropy);
    MG_HIP(hipGetLastError(), "cross entropy join launch");
    return MG_OK;
}

template <class T>
int cross_entropy_backward(hipStream_t st, const mg_cross_entropy_backward_args& p) {
    typedef typename HeadType<T>::H H;
    constexpr bool kPairs = sizeof(T) == 4;
    if (!p.rows) {
        hipLaunchKernelGGL(dev::head_sum_kernel<T>, copy_grid(p.width, p.classes), dim3(256), 0, st, nullptr, 0u,
                           p.classes, p.width, 0u, static_cast<T*>(p.dw), p.dw_ld, nullptr, 1u);
        MG_HIP(hipGetLastError(), "cross entropy zeros launch");
        return MG_OK;
    }
    const HeadSpace s(p.workspace, p.rows, p.classes, p.width, p.type, true);
    dev::HeadArgs a{};
    a.scales = scales_of<T>(st, p.x, p.x_ld, p.w, p.w_ld, p.rows, p.classes, p.width, p.dloss, p.dentropy, p.targets, s);
    const dev::HeadOperand w = operand_of<T, H>(st, p.w, p.w_ld, p.classes, p.width, p.type, s, s.w, 1, a.scales);
    const dev::HeadOperand x = operand_of<T, H>(st, p.x, p.x_ld, p.rows, p.width, p.type, s, s.x, 0, a.scales);
    a.rows = p.rows, a.classes = p.classes, a.targets = p.targets, a.row_exp = s.row_exp;
    a.lse = p.lse, a.dloss = p.dloss, a.entropy = p.entropy, a.dentropy = p.dentropy;
    a.rows_ld = s.rows_ld, a.g = s.g, a.gt = s.gt, a.g_ld = s.piece, a.g_plane = (uint64_t)s.rows_ld * s.piece;
    const uint64_t xt_plane = (uint64_t)p.width * s.rows_ld, wt_plane = (uint64_t)p.width * s.piece;
    auto turn = [&](const void* from, uint64_t ld, uint32_t rows, uint32_t fill, uint32_t to_ld, uint16_t* to,
                    uint64_t plane, uint32_t which) {
        const dev::CopyArgs c{from, ld, rows,     p.width, fill, to_ld, to, plane, a.scales, nullptr,
                              which, which ? nullptr : p.targets, p.classes};
        const uint32_t down = (fill + 63) / 64;
        hipLaunchKernelGGL((dev::head_turn_kernel<T, H>), dim3((p.width + 63) / 64, down < 4096 ? down : 4096),
                           dim3(256), 0, st, c);
    };
    if (p.dw) turn(p.x, p.x_ld, p.rows, s.rows_ld, s.rows_ld, s.xt, xt_plane, 0);
    const bool parts_x = s.splits_x > 1 || s.pieces > 1, parts_w = s.splits_w > 1;
    const uint32_t tall = p.width > 128 ? 256 : 128, tiles_m = (p.width + tall - 1) / tall;
    for (uint32_t first = 0; first < p.classes; first += s.piece) {
        const uint32_t here = p.classes - first < s.piece ? p.classes - first : s.piece, fill = up_to(here, kHeadM);
        const T* const w0 = static_cast<const T*>(p.w) + (uint64_t)first * p.w_ld;
        if (p.dx) turn(w0, p.w_ld, here, fill, s.piece, s.wt, wt_plane, 1);
        dev::HeadProduct& m = a.p[0];
        m = {};
        m.a = w, m.b = x;
        m.a.base = static_cast<const H*>(w.base) + (uint64_t)first * w.ld, m.a.rows = here;
        m.k = m.range = s.width8, m.splits = 1;
        m.tiles_m = fill / kHeadM, m.tiles_n = s.rows_ld / dev::kHeadN;
        a.tiles = m.tiles_m * m.tiles_n, a.first = first;
        hipLaunchKernelGGL((dev::head_kernel<H, dev::kLogitGrad, 4, kPairs>), dim3(a.tiles), dim3(512), 0, st, a);
        MG_HIP(hipGetLastError(), "cross entropy logits launch");
        uint32_t n = 0, tiles = 0;
        if (p.dx) {
            dev::HeadProduct& q = a.p[n++];
            q = {};
            q.a = {s.wt, wt_plane, s.piece, p.width}, q.b = {s.g, a.g_plane, s.piece, p.rows};
            q.k = fill, q.range = s.range_x, q.splits = (fill + s.range_x - 1) / s.range_x;
            q.tiles_m = tiles_m, q.tiles_n = s.rows_ld / dev::kHeadN;
            q.out = p.dx, q.out_ld = p.dx_ld, q.parts = parts_x ? s.parts_x : nullptr, q.parts_ld = s.parts_ld;
            q.add = first != 0, q.which = 0;
            a.tiles = q.tiles_m * q.tiles_n * q.splits, tiles += a.tiles;
        }
        if (p.dw) {
            dev::HeadProduct& q = a.p[n++];
            q = {};
            q.a = {s.xt, xt_plane, s.rows_ld, p.width}, q.b = {s.gt, a.g_plane, s.rows_ld, here};
            q.k = s.rows_ld, q.range = s.range_w, q.splits = s.splits_w;
            q.tiles_m = tiles_m, q.tiles_n = fill / dev::kHeadN;
            q.out = static_cast<T*>(p.dw) + (uint64_t)first * p.dw_ld, q.out_ld = p.dw_ld;
            q.parts = parts_w ? s.parts_w : nullptr, q.parts_ld = s.parts_ld, q.which = 1;
            const uint32_t more = q.tiles_m * q.tiles_n * q.splits;
            if (n == 1) a.tiles = more;
            tiles += more;
        }
        if (tall == 128)
            hipLaunchKernelGGL((dev::head_kernel<H, dev::kGrad, 2, kPairs>), dim3(tiles), dim3(512), 0, st, a);
        else
            hipLaunchKernelGGL((dev::head_kernel<H, dev::kGrad, 4, kPairs>), dim3(tiles), dim3(512), 0, st, a);
        MG_HIP(hipGetLastError(), "cross entropy gradients launch");
        if (p.dw && parts_w)
            hipLaunchKernelGGL(dev::head_sum_kernel<T>, copy_grid(p.width, here), dim3(256), 0, st, s.parts_w,
                               s.splits_w, here, p.width, s.parts_ld,
                               static_cast<T*>(p.dw) + (uint64_t)first * p.dw_ld, p.dw_ld, a.scales, 1u);
    }
    if (p.dx && parts_x)
        hipLaunchKernelGGL(dev::head_sum_kernel<T>, copy_grid(p.width, p.rows), dim3(256), 0, st, s.parts_x,
                           s.splits_x, p.rows, p.width, s.parts_ld, static_cast<T*>(p.dx), p.dx_ld, a.scales, 0u);
    MG_HIP(hipGetLastError(), "cross entropy sums launch");
    return MG_OK;
}

int check_head(const char* what, uint32_t rows, uint32_t classes, uint32_t width, uint32_t type) {
    MG_CHECK(type_known(type), MG_ERR_INVALID, "%s: unknown type %u", what, type);
    MG_CHECK(rows <= kMostHeadRows, MG_ERR_INVALID, "%s: rows %u must be at most 2^20", what, rows);
    MG_CHECK(classes >= 1 && classes <= kMostClasses, MG_ERR_INVALID, "%s: classes %u must be in [1, 2^20]", what,
             classes);
    MG_CHECK(width >= 1 && width <= kMostWidth, MG_ERR_INVALID, "%s: width %u must be in [1, 65536]", what, width);
    return MG_OK;
}

}  // namespace
}  // namespace mg

using namespace mg;

extern "C" {

int mg_cross_entropy_workspace(uint32_t rows, uint32_t classes, uint32_t width, uint32_t type, uint64_t* bytes) {
    const char* what = "cross entropy workspace";
    MG_CHECK(bytes, MG_ERR_INVALID, "%s: null argument", what);
    int rc = check_head(what, rows, classes, width, type);
    if (rc) return rc;
    *bytes = rows ? HeadSpace(nullptr, rows, classes, width, type, false).bytes : 0;
    return MG_OK;
}

int mg_cross_entropy(void* stream, const mg_cross_entropy_args* args) {
    const char* what = "cross entropy";
    MG_CHECK(args, MG_ERR_INVALID, "cross entropy: null argument");
    mg_cross_entropy_args p = *args;
    int rc;
    if ((rc = check_head(what, p.rows, p.classes, p.width, p.type)) ||
        (rc = check_operand(what, "x", p.x, &p.x_ld, p.width, p.type, p.rows != 0)) ||
        (rc = check_operand(what, "w", p.w, &p.w_ld, p.width, p.type, p.rows != 0)) ||
        (rc = check_vector(what, "targets", p.targets, MG_TYPE_FP32, p.rows != 0)) ||
        (rc = check_vector(what, "loss", p.loss, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "lse", p.lse, MG_TYPE_FP32, false)) ||
        (rc = check_vector(what, "entropy", p.entropy, MG_TYPE_FP32, false)))
        return rc;
    uint64_t need = 0;
    if ((rc = mg_cross_entropy_workspace(p.rows, p.classes, p.width, p.type, &need)) ||
        (rc = check_workspace(what, p.workspace, p.workspace_bytes, need)))
        return rc;
    if (!p.rows) return MG_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice on;
    if ((rc = on.enter(st, "cross entropy: stream device"))) return rc;
    return p.type == MG_TYPE_FP32   ? cross_entropy<float>(st, p)
           : p.type == MG_TYPE_BF16 ? cross_entropy<__bf16>(st, p)
                                    : cross_entropy<_Float16>(st, p);
}

int mg_cross_entropy_backward_workspace(uint32_t rows, uint32_t classes, uint32_t width, uint32_t type,
                                        uint64_t* bytes) {
    const char* what = "cross entropy backward workspace";
    MG_CHECK(bytes, MG_ERR_INVALID, "%s: null argument", what);
    int rc = check_head(what, rows, classes, width, type);
    if (rc) return rc;
    *bytes = HeadSpace(nullptr, rows, classes, width, type, true).bytes;
    return MG_OK;
}

int mg_cross_entropy_backward(void* stream, const mg_cross_entropy_backward_args* args) {
    const char* what = "cross entropy backward";
    MG_CHECK(args, MG_ERR_INVALID, "cross entropy backward: null argument");
    mg_cross_entropy_backward_args p = *args;
    int rc;
    const bool any = p.rows != 0;
    if ((rc = check_head(what, p.rows, p.classes, p.width, p.type)) ||
        (rc = check_operand(what, "x", p.x, &p.x_ld, p.width, p.type, any)) ||
        (rc = check_operand(what, "w", p.w, &p.w_ld, p.width, p.type, any)) ||
        (rc = check_vector(what, "targets", p.targets, MG_TYPE_FP32, any)) ||
        (rc = check_vector(what, "lse", p.lse, MG_TYPE_FP32, any)) ||
        (rc = check_vector(what, "dloss", p.dloss, MG_TYPE_FP32, any)) ||
        (rc = check_vector(what, "entropy", p.entropy, MG_TYPE_FP32, any && p.dentropy)) ||
        (rc = check_vector(what, "dentropy", p.dentropy, MG_TYPE_FP32, false)) ||
        (rc = check_operand(what, "dx", p.dx, &p.dx_ld, p.width, p.type, false)) ||
        (rc = check_operand(what, "dw", p.dw, &p.dw_ld, p.width, p.type, false)))
        return rc;
    uint64_t need = 0;
    if ((rc = mg_cross_entropy_backward_workspace(p.rows, p.classes, p.width, p.type, &need)) ||
        (rc = check_workspace(what, p.workspace, p.workspace_bytes, need)))
        return rc;
    if ((!p.dx || !any) && !p.dw) return MG_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice on;
    if ((rc = on.enter(st, "cross entropy backward: stream device"))) return rc;
    return p.type == MG_TYPE_FP32   ? cross_entropy_backward<float>(st, p)
           : p.type == MG_TYPE_BF16 ? cross_entropy_backward<__bf16>(st, p)
                                    : cross_entropy_backward<_Float16>(st, p);
}

}  // extern "C"
