// Softmax cross entropy over many classes without its logits, and its gradients, which keep a piece of
// them at a time (mg_cross_entropy, mg_cross_entropy_backward).
//
// Forward: one product W X' whose tiles end in each row's maximum, sum of exponentials and
// sum weighted by the logits, and a launch that joins the tiles' statistics. Backward: the
// logits again, a piece of the classes at a time; each piece's gradient with respect to the
// logits, G = dloss (p - [target]) - dentropy p (log p + H), is stored in 16 bits (fp32's as
// pairs) and enters two products, dX += G W and dW = G' X, in one launch. Their contractions run from
// row to row of an operand: LDS hands those out transposed. G is rounded because the matrix instructions take 16
// bits: a second half of it would double both products, which are three fifths of the time. That is the gradients'
// largest error: 4096 x 65536 x 1024 bf16 is 2.4e-3 off its 64-bit value, where rounding the results alone
// leaves 1.7e-3. Up to 128 rows have room for that half in their own tile.
//
// All three are one kernel (head_kernel): tiles of a b', 16-bit operands, fp32 sums. 16-bit arrays of a
// fitting shape are read where they lie, others are copied. fp32 operands become two binary16
// halves at a power of two (22 bits), and their product three: low high + high low + high high, one
// after the other.
//
// Matrix instructions bound it. bf16, 4095 x 50001 x 1024: forward 412 to 432 us on different cards, 970 to 1020 TFLOP/s;
// 4096 x 49152 x 4096 1190, and 8192 cubed as a library product 1387. Its gradients of 4096 x 65536 x
// 1024 take 1617 to 1652 us, 1000 to 1020 TFLOP/s: an epilogue of about 10 us follows 30 us of products for each tile
// of logits, and in the loop the products alone, without loads or LDS reads, take four fifths of the
// time. fp32 gradients of 4096 x 10007 x 128 take 153 to 165 us, 70 for logits and G, whose products are 8
// stages a tile, and 80 for the two products.
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

// Rows of 16-bit elements, `ld` of them apart. Pairs lie in blocks of 16 high halves and the 16
// low ones: element c of a row at pair_place(c), its low half 16 further.
struct HeadOperand {
    const void* base;
    uint32_t ld;
    uint32_t again = ~0u;  // rows from here on are the first ones once more
    __device__ __forceinline__ uint32_t row(uint32_t r) const { return r >= again ? r - again : r; }
};
__host__ __device__ __forceinline__ uint32_t pair_place(uint32_t c) { return (c & ~15u) * 2 + (c & 15); }

enum { kStats = 0, kLogitGrad = 1, kGrad = 2 };

// One product's tiles: M from a, N from b, contraction K in `splits` ranges of `range`.
struct HeadProduct {
    HeadOperand a, b;
    const uint32_t* live;  // dW: a bit for each row of a; the others count as 0
    uint32_t k, range, splits;
    uint32_t m, n;  // the result's sides
    uint32_t tiles_m, tiles_n;
    // kGrad: out(n, m) = sum, n down the rows of out; or fp32 parts [splits][out rows][parts_ld]
    void* out;
    float* parts;
    uint64_t out_ld;
    uint32_t parts_ld;
    uint32_t low;      // dX, not 0: of G's rows those from here on are the first ones' low halves, with parts of their own
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
    void* g;  // the piece's, g_ld between rows
    uint32_t* live;
    uint32_t g_ld;
};

constexpr int kHeadK = 32;     // contraction elements of a stage, or 16 pairs
// Stages in LDS. Tiles of MI = 4, and all of the gradients', have a CU to themselves; logits' of MI = 2
// share one by twos.
template <int KIND, int MI>
constexpr bool kByTwos = KIND != kGrad && MI == 2;
template <int KIND, int MI>
constexpr int kHeadRing = kByTwos<KIND, MI> ? 3 : 4;
constexpr int kHeadN = 256;    // columns of a tile
constexpr uint32_t kNowhere = 0x80000000u;  // an offset past every operand's end: reads 0

// The logarithm and the exponential in base 2, by the hardware's instructions.
__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
constexpr float kLog2 = 1.44269504f, kLn2 = 0.693147181f;

// The two halves of a value; what is not finite lies in the low one alone, so that its products
// with another's halves are of fp32's sign and infinity.
template <class H>
__device__ __forceinline__ void split_half(float v, H& hi, H& lo) {
    const bool odd = !(__builtin_fabsf(v) < 65504.0f);
    hi = odd ? (H)0.0f : (H)v;
    lo = odd ? (H)v : (H)(v - (float)hi);
}

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

// One operand's part in the main loop: SIDE rows of a tile, of which a stage holds 32
// contraction elements (16 pairs) in LDS. Rows go from memory straight there, a wave's 64 lanes in
// order, 16 bytes each; where they come from is each lane's own choice, which keeps reads off one
// bank.
//
// Not TURNED: the contraction runs along a row in memory, and a stage is 64 bytes of every row. The
// places of a row's four 16 bytes are exchanged by bits 2 and 3 of the row: 16 rows' parts of a
// fragment (lane l holds row l % 32 and eight elements of 16, by l / 32), which are read at once, then
// lie in 64 different banks.
//
// TURNED: it runs from row to row, and a stage is 32 rows of SIDE elements, or 16 of SIDE pairs.
// Reads of four elements by 16 lanes that hold each other's columns (ds_read_b64_tr_b16: of 4 rows
// x 16 columns a lane gets a column) make the same fragments; the places of 32 bytes are exchanged
// by the row's last two bits, so that four rows and two blocks of columns lie in different banks.
//
// A matrix instruction's result leaves a lane with four of each eight rows of its first operand. So
// that they are 16 in a row, to be stored 32 bytes and more at a time, OUTER fragments' lane 8 q + 4 h + r
// holds row 16 h + 4 q + r.
template <class H, int SIDE, bool TURNED, bool PAIRS, bool OUTER>
struct HeadSide {
    typedef typename Halves<H>::x8 x8;
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    static constexpr int L = SIDE / 128;  // loads of a wave and stage
    static constexpr int kBytes = SIDE * 64, kWide = PAIRS ? 2 : 1;
    static constexpr int kRow = SIDE * 2 * kWide;  // bytes of a TURNED row
    const H* base;
    uint32_t ld, again, off[L], row[L];

    // what exchanges a TURNED row's places: blocks of columns are their last bit, or of pairs
    // the one before it
    static __device__ __forceinline__ int spread(int row) {
        return PAIRS ? (row & 1) | (row & 2) << 1 : (row & 3) << 1;
    }

    // and a row's places that is not TURNED: of 16 rows that are read at once four have each value
    static __device__ __forceinline__ int shift(int row) {
        return OUTER ? (row >> 2 & 1) | (row >> 4 & 1) << 1 : row >> 2 & 3;
    }

    // `from`: the tile's first row (or column) of `rows`
    __device__ __forceinline__ HeadSide(const HeadOperand& o, uint32_t from, uint32_t rows, int wave, int lane) {
        ld = o.ld, again = o.again;
        base = static_cast<const H*>(o.base) + (TURNED ? (uint64_t)from * kWide : (uint64_t)from * ld);
        const uint32_t have = rows > from ? rows - from : 0;
#pragma unroll
        for (int c = 0; c < L; ++c) {
            if constexpr (TURNED) {
                constexpr uint32_t kLanes = kRow / 16;  // of a row
                row[c] = (wave * L + c) * (64 / kLanes) + lane / kLanes;
                const uint32_t at = lane % kLanes, place = (((at >> 1 ^ spread(row[c])) << 1) + (at & 1)) * 8;
                const uint32_t col = PAIRS ? (place >> 5 << 4) + (place & 15) : place;
                off[c] = col < have ? (row[c] * ld + place) * 2 : kNowhere;
            } else {
                const uint32_t r = (wave * L + c) * 16 + (lane >> 2), place = ((lane & 3) ^ shift(r)) * 8;
                const uint32_t at = o.row(r);
                row[c] = PAIRS ? place & 15 : place;  // the first of its elements
                off[c] = at < have ? (at * ld + place) * 2 : kNowhere;
            }
        }
    }
    // The stage of contraction elements k ..., up to `to`.
    __device__ __forceinline__ void load(char* at, int wave, uint32_t k, uint32_t to, uint32_t live) const {
        // a row of W or X may lie anywhere, so its stage has an address of its own
        const uint32_t first = !PAIRS && TURNED && k >= again ? k - again : k;
        const H* const p = base + (TURNED ? (uint64_t)first * ld : (uint64_t)k * kWide);
        const uint64_t address = reinterpret_cast<uint64_t>(p);
        typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
        const u32x4 r = {(uint32_t)address, (uint32_t)(address >> 32) & 0xffffu, 0x7fffffffu, 0x00020000u};
#pragma unroll
        for (int c = 0; c < L; ++c) {
            bool in = k + row[c] < to;
            if constexpr (TURNED) in = in && (live >> row[c] & 1);
            // Not the builtin: the compiler cannot tell the ring's stages apart, and would wait for all
            // loads before each stage's first read. Nothing here comes back in a register; the
            // loop's own waits are for LDS.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: it is in nobody else's use here
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(
                             (__attribute__((address_space(3))) char*)(at + (wave * L + c) * 1024)),
                         "v"(in ? off[c] : kNowhere), "s"(r)
                         : "memory", "m0");
#pragma clang diagnostic pop
        }
    }
    // the fragment of rows 32 b ... of the tile: the stage's elements 16 h ..., or of its pairs
    // the high (h = 0) or the low halves
    static __device__ __forceinline__ x8 read(const char* at, int b, int h, int lane) {
        if constexpr (TURNED) {
            const int k = (PAIRS ? 0 : 16 * h) + 8 * (lane >> 5) + (lane >> 2 & 3);
            // four columns of the 32 that a lane reads for the others
            const int lot = (lane >> 2 & 4) | (lane & 3), quad = OUTER ? (lot & 1) * 4 + (lot >> 1) : lot;
            const int block = 2 * b + (quad >> 2), chunk = PAIRS ? 2 * block + h : block;
            auto four = [&](int more) {
                const int r = k + more;  // its last two bits are k's
                const char* const p = at + r * kRow + ((chunk ^ spread(r)) << 5) + ((quad & 3) << 3);
                return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
            };
            const s16x4 lo = four(0), hi = four(4);
            return __builtin_bit_cast(x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int m = lane & 31, row = OUTER ? (m & 4) * 4 | (m >> 1 & 12) | (m & 3) : m;
            return *reinterpret_cast<const x8*>(at + b * 2048 + row * 64 + (((2 * h + (lane >> 5)) ^ shift(row)) << 4));
        }
    }
};

// One tile of MI x 64 by 256. Eight waves, two along a and four along b, MI x 2 tiles of 32 x 32
// each. The waves meet once a stage, when the next has arrived. With a ring of four stages they read
// the next one's fragments under this one's products: two of 16 elements, or of pairs low high,
// high low and high high. With three there is another workgroup on the CU, and a lane holds one
// stage's fragments.
template <class H, int RING, int MI, bool PAIRS, bool AT, bool BT>
__device__ __forceinline__ void head_product(const HeadProduct& p, uint32_t tm, uint32_t tn, uint32_t split, char* lds,
                                             f32x16 (&acc)[MI][2]) {
    using X = Halves<H>;
    typedef typename X::x8 x8;
    using A = HeadSide<H, MI * 64, AT, PAIRS, true>;
    using B = HeadSide<H, kHeadN, BT, PAIRS, false>;
    constexpr int kStage = A::kBytes + B::kBytes, L = A::L + B::L, K = PAIRS ? 16 : kHeadK;
    const uint32_t from = split * p.range, to = p.k - from < p.range ? p.k : from + p.range;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
    const A a(p.a, tm * (MI * 64), p.m, wave, lane);
    const B b(p.b, tn * kHeadN, p.n, wave, lane);
    uint32_t k = from;
    constexpr int kSets = RING == 3 ? 1 : 2, kTerms = PAIRS ? 3 : 2;  // of fragments
    const uint32_t stages = ((to - from + K - 1) / K + kSets - 1) & ~(kSets - 1u);  // the last may be empty
    // read a stage ahead, and without a branch, which would part the loop
    auto* const rows_live = (const __attribute__((address_space(4))) uint32_t*)p.live;
    auto live_of = [&](uint32_t at) {
        if constexpr (AT && BT)
            return rows_live[(at < to ? at : to - 1) / 32];
        else
            return ~0u;
    };
    uint32_t bits = live_of(k);
    auto load = [&](uint32_t slot) {
        char* const at = lds + slot * kStage;
        a.load(at, wave, k, to, bits >> (k & 31));
        b.load(at + A::kBytes, wave, k, to, ~0u);
        k += K;
        bits = live_of(k);
    };
    x8 fa[kSets][2][MI], fb[kSets][2][2];
    auto read = [&](int set, uint32_t slot) {
        const char* const at = lds + slot * kStage;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[set][h][i] = A::read(at, wm * MI + i, h, lane);
#pragma unroll
            for (int j = 0; j < 2; ++j) fb[set][h][j] = B::read(at + A::kBytes, wn * 2 + j, h, lane);
        }
    };
    auto multiply = [&](int set) {
#pragma unroll
        for (int h = 0; h < kTerms; ++h) {
            const int ha = PAIRS ? h == 0 : h, hb = PAIRS ? h == 1 : h;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = X::mfma(fa[set][ha][i], fb[set][hb][j], acc[i][j]);
        }
    };
    if constexpr (kSets == 1) {
        // the CU's other workgroup has the matrix units meanwhile
#pragma unroll
        for (uint32_t u = 0; u + 1 < (uint32_t)RING; ++u) load(u);
        for (uint32_t s = 0, slot = 0, free = RING - 1; s < stages; ++s) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((RING - 2) * L) : "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            load(free);
            read(0, slot);
            multiply(0);
            free = slot;
            slot = slot + 1 == RING ? 0 : slot + 1;
        }
    } else {
#pragma unroll
        for (uint32_t u = 0; u < (uint32_t)RING; ++u) load(u);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 1) * L) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        read(0, 0);
        for (uint32_t s = 0; s < stages; s += 2) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t slot = (s + u) & (RING - 1);
                // the next stage is there, this one is in registers
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((RING - 2) * L) : "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                load(slot);
                read(u ^ 1, (slot + 1) & (RING - 1));
                multiply(u);
                constexpr int kReads = 2 * (MI * (AT ? 2 : 1) + 2 * (BT ? 2 : 1)), kProducts = 2 * MI * kTerms;
                // the last reads have a quarter of the products' time to arrive
                constexpr int kCover = kProducts * 3 / 4;
#pragma unroll
                for (int q = 0; q < kProducts; ++q) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix
                    const int n = q < kCover ? (q + 1) * kReads / kCover - q * kReads / kCover : 0;
                    if (n == 1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
                    if (n == 2) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    if (n == 3) __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last loads have left LDS alone
}

template <class H, int KIND, int MI, bool PAIRS>
__global__ void __launch_bounds__(512, (kByTwos<KIND, MI> ? 4 : 2)) head_kernel(const HeadArgs args) {
    typedef typename Halves<H>::x8 x8;
    constexpr int TM = MI * 64;
    constexpr int kRing = kHeadRing<KIND, MI>;
    __shared__ __align__(1024) char lds[kRing * (TM + kHeadN) * 64];
    // Each XCD has its share of both products, whose tiles take different times: 512 x 50000 x 512 bf16
    // gradients 136 us, and 220 with the first XCDs' all of one product.
    const uint32_t sel = blockIdx.x >= args.tiles ? 1 : 0;
    const HeadProduct& p = args.p[sel];
    uint32_t tile = sel ? xcd_run(blockIdx.x - args.tiles, gridDim.x - args.tiles) : xcd_run(blockIdx.x, args.tiles);
    const uint32_t per = p.tiles_m * p.tiles_n, split = tile / per;
    tile -= split * per;
    // down four tiles of m, then on by one of n: an XCD's 32 tiles at a time are 4 x 8 and share their
    // operands in its L2
    const uint32_t first = tile / (4 * p.tiles_n) * 4, deep = p.tiles_m - first < 4 ? p.tiles_m - first : 4;
    tile -= first * p.tiles_n;
    const uint32_t tn = tile / deep, tm = first + tile - tn * deep;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
    f32x16 acc[MI][2] = {};
    if constexpr (KIND != kGrad)
        head_product<H, kRing, MI, PAIRS, false, false>(p, tm, tn, split, lds, acc);
    else if (p.which)
        head_product<H, kRing, MI, PAIRS, true, true>(p, tm, tn, split, lds, acc);
    else
        head_product<H, kRing, MI, PAIRS, true, false>(p, tm, tn, split, lds, acc);

    // register e of tile (i, j): row m0 + 32 i + e of a, row n0 + 32 j of b
    const uint32_t m0 = tm * TM + wm * (MI * 32) + 16 * (lane >> 5), n0 = tn * kHeadN + wn * 64 + (lane & 31);
    const HeadScales sc = args.scales ? *args.scales : HeadScales{1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
    if constexpr (KIND == kGrad) {
        const float b0 = sc.g_back, b1 = p.which ? sc.x_back : sc.w_back;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t n = n0 + 32 * j, part = split, rows = p.n;
            if (p.low) {
                part = 2 * split + (n >= p.low), rows = args.rows;
                if (n >= p.low) n -= p.low;
            }
            if (n >= rows) continue;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const uint32_t m = m0 + 32 * i;
                if (m >= p.m) continue;
                f32x16& v = acc[i][j];
                const uint32_t count = p.m - m;
                if (p.parts) {  // parts_ld is a multiple of 4
                    f32x4* const at = reinterpret_cast<f32x4*>(p.parts + ((uint64_t)part * rows + n) * p.parts_ld + m);
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        if ((uint32_t)e >= count) continue;
                        f32x4 four = {v[e], v[e + 1], v[e + 2], v[e + 3]};
                        if (p.add) four += at[e / 4];
                        at[e / 4] = four;
                    }
                    continue;
                }
                v = v * b0 * b1;
                auto put = [&](auto t) {
                    using T = decltype(t);
                    typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
                    constexpr int E = 16 / sizeof(T);
                    T* const at = static_cast<T*>(p.out) + n * p.out_ld + m;
                    if (count >= 16) {
#pragma unroll
                        for (int e = 0; e < 16; e += E) {
                            vec w;
#pragma unroll
                            for (int q = 0; q < E; ++q) w[q] = (T)v[e + q];
                            *reinterpret_cast<vec*>(at + e) = w;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 15; ++e)
                            if (e < (int)count) at[e] = (T)v[e];
                    }
                };
                if constexpr (PAIRS)
                    put(0.0f);
                else
                    put(H{});
            }
        }
    } else {
        // logits in base 2: two factors for pairs, as their product may leave fp32's range
        const float to2 = PAIRS ? sc.w_back * kLog2 : kLog2;
        const bool edge = (tm + 1) * TM > p.m;
        if constexpr (KIND == kStats) __syncthreads();  // every wave is done with the ring
        RowStats* const trade = reinterpret_cast<RowStats*>(lds);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t place = n0 + 32 * j, n = p.b.row(place);  // of G, and of x
            int32_t target = -1;
            if (n < args.rows) {
                target = args.targets[n];
                if constexpr (PAIRS) {
                    const float back = ldexpf(1.0f, -args.row_exp[n]);
#pragma unroll
                    for (int i = 0; i < MI; ++i) acc[i][j] *= back;
                }
            }
            // the target's place among the lane's classes, which are m0 - args.first + ...
            const uint32_t hit = (uint32_t)target - args.first - m0;
            const bool live = target >= 0 && (uint32_t)target < args.classes;
            const bool meets = __any(live && hit < MI * 32);
            if constexpr (KIND == kStats) {
                if (edge) {
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (m0 + 32 * i + e >= p.m) acc[i][j][e] = -__builtin_huge_valf();
                }
                if (meets) {
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (live && hit == (uint32_t)(32 * i + e)) args.of[n] = acc[i][j][e] * to2;
                }
                float top = -__builtin_huge_valf();
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = __builtin_fmaxf(top, acc[i][j][e]);
                RowStats r{top * to2, 0.0f, 0.0f};
                // also where the lowest finite logits leave fp32's range in base 2
                const float zero = r.top == -__builtin_huge_valf() ? 0.0f : r.top;
                if (args.want_entropy) {
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float d = __builtin_fmaf(acc[i][j][e], to2, -zero), w = exp2_of(d);
                            r.sum += w;
                            r.weighted = __builtin_fmaf(w, __builtin_fmaxf(d, -1000.0f), r.weighted);
                        }
                } else {
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) r.sum += exp2_of(__builtin_fmaf(acc[i][j][e], to2, -zero));
                }
                RowStats o;
                float lo, hi;
                lane_pair<32>(r.top, lo, hi), r.top = lo, o.top = hi;
                lane_pair<32>(r.sum, lo, hi), r.sum = lo, o.sum = hi;
                lane_pair<32>(r.weighted, lo, hi), r.weighted = lo, o.weighted = hi;
                r.join(o);
                if (lane < 32) trade[wm * kHeadN + wn * 64 + 32 * j + lane] = r;
            } else {
                const uint32_t bits = (uint32_t)__ballot(live);  // the upper lanes' rows are the lower ones'
                if (tm == 0 && wm == 0 && lane == 0) args.live[place / 32] = bits;
                float lse2 = 0.0f, dl = 0.0f, de = 0.0f, ent = 0.0f;
                if (live) {
                    lse2 = args.lse[n] * kLog2, dl = args.dloss[n] * sc.g;
                    if (args.dentropy) de = args.dentropy[n] * sc.g * kLn2, ent = args.entropy[n] * kLog2;
                }
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float d = __builtin_fmaf(acc[i][j][e], to2, -lse2), prob = exp2_of(d);
                        float g = dl * prob;
                        if (args.dentropy) g = __builtin_fmaf(-de * prob, __builtin_fmaxf(d, -1000.0f) + ent, g);
                        acc[i][j][e] = live ? g : 0.0f;
                    }
                if (edge) {
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (m0 + 32 * i + e >= p.m) acc[i][j][e] = 0.0f;
                }
                if (meets) {
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (live && hit == (uint32_t)(32 * i + e)) acc[i][j][e] -= dl;
                }
                if (!PAIRS && place >= p.b.again) {  // what the same row's rounding leaves, of 32 rows at once
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float rest = acc[i][j][e] - (float)(H)acc[i][j][e];
                            acc[i][j][e] = __builtin_fabsf(rest) < __builtin_huge_valf() ? rest : 0.0f;
                        }
                }
                // by way of LDS, from where a wave stores whole rows of the tile: places of 16 bytes are
                // exchanged by the row, whose own lie in the same banks
                constexpr uint32_t kChunks = TM * (PAIRS ? 4 : 2) / 16;  // of a row
                const uint32_t r = wn * 32 + (lane & 31);
                x8* const row = reinterpret_cast<x8*>(lds) + r * kChunks;
                __syncthreads();  // every wave is done with the ring, or the rows before
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    const uint32_t c = wm * (MI * 32) + 32 * i + 16 * (lane >> 5);  // of the tile: 16 pairs, or elements
#pragma unroll
                    for (int e = 0; e < 16; e += 8) {
                        x8 hi, lo;
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            if constexpr (PAIRS) {
                                H h, l;
                                split_half<H>(acc[i][j][e + q], h, l);
                                hi[q] = h, lo[q] = l;
                            } else {
                                hi[q] = (H)acc[i][j][e + q];
                            }
                        }
                        const uint32_t chunk = (PAIRS ? c / 4 : c / 8) + e / 8;
                        row[chunk ^ (r & 15)] = hi;
                        if constexpr (PAIRS) row[(chunk + 2) ^ (r & 15)] = lo;
                    }
                }
                __syncthreads();
                H* const g = static_cast<H*>(args.g) + (uint64_t)(tn * kHeadN + 32 * j) * args.g_ld + tm * TM * (PAIRS ? 2 : 1);
#pragma unroll
                for (uint32_t u = 0; u < kChunks / 4; ++u) {
                    const uint32_t at = u * 512 + threadIdx.x, r = at / kChunks, chunk = at % kChunks;
                    const x8 v = reinterpret_cast<const x8*>(lds)[r * kChunks + (chunk ^ (r & 15))];
                    *reinterpret_cast<x8*>(g + (uint64_t)((r >> 5) * 64 + (r & 31)) * args.g_ld + chunk * 8) = v;
                }
            }
        }
        if constexpr (KIND == kStats) {
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
        }
    }
}

// Joins the tiles of `across` rows (a power of two) a workgroup: thread by thread every few of them, then
// the threads' by halves.
__global__ void __launch_bounds__(1024) head_join_kernel(const float* stats, const float* of, const int32_t* targets,
                                                         uint32_t rows, uint32_t rows_ld, uint32_t tiles,
                                                         uint32_t classes, uint32_t across, float* loss, float* lse,
                                                         float* entropy) {
    __shared__ RowStats lds[1024];
    const uint32_t slice = threadIdx.x / across, slices = blockDim.x / across;
    const uint32_t n = blockIdx.x * across + (threadIdx.x & (across - 1));
    RowStats r{-__builtin_huge_valf(), 0.0f, 0.0f};
    if (n < rows) {
#pragma unroll 4
        for (uint32_t t = slice; t < tiles; t += slices) {
            const float* const at = stats + (uint64_t)t * 3 * rows_ld + n;
            r.join(RowStats{at[0], at[rows_ld], at[2 * (uint64_t)rows_ld]});
        }
    }
    lds[threadIdx.x] = r;
    for (uint32_t half = slices / 2; half; half /= 2) {
        __syncthreads();
        if (slice >= half) continue;
        r.join(lds[threadIdx.x + half * across]);
        lds[threadIdx.x] = r;
    }
    if (slice || n >= rows) return;
    const float log = __builtin_amdgcn_logf(r.sum), all = (r.top + log) * kLn2;
    const int32_t target = targets[n];
    if (loss) loss[n] = target >= 0 && (uint32_t)target < classes ? (r.top - of[n] + log) * kLn2 : 0.0f;
    if (lse) lse[n] = all;
    if (entropy) entropy[n] = (log - r.weighted / r.sum) * kLn2;
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
constexpr uint32_t kAmaxParts = 1024;
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

// 16-bit copies of x (job 0) and W (job 1), rows of `wide` elements with zeros past their
// columns, of what cannot be read as it lies. fp32 becomes pairs: W at the scale of all of it, x at each row's own
// for the logits and at that of all rows with a target for the gradient of W.
struct PrepareArgs {
    const void* from;
    uint64_t from_ld;
    uint32_t rows, cols;
    void* to;  // nullable
    void* to_even;  // of x, nullable
    uint32_t wide;
    const int* row_exp;  // of x
};
struct PrepareScales {
    const float* parts[3];  // of x, W and the gradients; NULL: 1
    HeadScales* out;
};
template <class T, class H>
__global__ void __launch_bounds__(256) head_prepare_kernel(const PrepareArgs a0, const PrepareArgs a1,
                                                           const PrepareScales s) {
    typedef typename Halves<H>::x4 x4;
    constexpr bool kPairs = sizeof(T) == 4;
    __shared__ float red[3][4];
    const uint32_t job = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const PrepareArgs& a = job ? a1 : a0;
    // the largest of the parts, and with it each array's scale, in every workgroup
    float scale[3] = {1.0f, 1.0f, 1.0f}, back[3] = {1.0f, 1.0f, 1.0f};
    if (s.out) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            f32x4 v = {};
            if (s.parts[k]) v = *reinterpret_cast<const f32x4*>(s.parts[k] + 4 * threadIdx.x);
            const float most = group_max<64>(__builtin_fmaxf(__builtin_fmaxf(v[0], v[1]), __builtin_fmaxf(v[2], v[3])));
            if (!lane) red[k][wave] = most;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            if (!s.parts[k]) continue;
            const int e = lift(__builtin_fmaxf(__builtin_fmaxf(red[k][0], red[k][1]), __builtin_fmaxf(red[k][2], red[k][3])));
            scale[k] = ldexpf(1.0f, e), back[k] = ldexpf(1.0f, -e);
        }
        if (blockIdx.x == 0 && job == 0 && threadIdx.x == 0)
            *s.out = HeadScales{scale[0], scale[1], scale[2], back[0], back[1], back[2]};
    }
    if (!a.to) return;
    const uint32_t across = a.wide / 4;
    const uint64_t all = (uint64_t)across * a.rows;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256) {
        const uint32_t r = (uint32_t)(i / across), c = (uint32_t)(i - (uint64_t)r * across) * 4;
        const T* const from = static_cast<const T*>(a.from) + r * a.from_ld + c;
        T v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = c + q < a.cols ? from[q] : (T)0.0f;
        const uint64_t at = kPairs ? (uint64_t)r * a.wide * 2 + pair_place(c) : (uint64_t)r * a.wide + c;
        auto put = [&](void* to, float by) {
            x4 hi, lo;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if constexpr (kPairs) {
                    H h, l;
                    split_half<H>((float)v[q] * by, h, l);
                    hi[q] = h, lo[q] = l;
                } else {
                    hi[q] = (H)v[q];
                }
            }
            *reinterpret_cast<x4*>(static_cast<H*>(to) + at) = hi;
            if constexpr (kPairs) *reinterpret_cast<x4*>(static_cast<H*>(to) + at + 16) = lo;
        };
        put(a.to, !kPairs ? 1.0f : job ? scale[1] : ldexpf(1.0f, a.row_exp[r]));
        if (kPairs && a.to_even) put(a.to_even, scale[0]);
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
#pragma unroll 8  // loads at once: gradients of 4 x 100000 x 128 bf16 103 us with one at a time, 58 with these
        for (uint32_t k = 0; k < count; ++k)
            v += *reinterpret_cast<const f32x4*>(parts + ((uint64_t)k * rows + r) * ld + c);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (c + q < cols) out[r * out_ld + c + q] = (T)(v[q] * b0 * b1);
    }
}

// ---- small products ----------------------------------------------------------------------------------
//
// Where the tiles above would be few, all of it is latency: of launches that scale and copy, and of a
// tile's 256 x 256. These take 32 x 32 a workgroup, straight from memory as fp32 whatever the type, on
// the fp32 matrix instruction, its four waves a quarter of the contraction each. 64 x 1000 x 128 fp32 takes
// 17 us back to back, 4.7 and 3.6 of them in the two kernels.

// Elements k .. k + 3 of a row; those from `end` on are 0, and not read, unless ALL are before it.
template <bool ALL, class T>
__device__ __forceinline__ f32x4 four_of(const T* row, uint32_t k, uint32_t end) {
    f32x4 v = {};
    if constexpr (ALL) {
        typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
        const vec w = *reinterpret_cast<const vec*>(row + k);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)w[e];
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k + e < end) v[e] = (float)row[k + e];
    }
    return v;
}
// The same of a column, ld apart.
template <bool ALL, class T>
__device__ __forceinline__ f32x4 four_down(const T* column, uint64_t ld, uint32_t k, uint32_t end) {
    f32x4 v = {};
    column += k * ld;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (ALL || k + e < end) v[e] = (float)column[e * ld];
    return v;
}

// acc += a b over the wave's share of k0 .. k1, a quarter in steps of 8: instruction e of a
// step takes element 8 j + e from lanes 0 to 31 and 8 j + 4 + e from the others. Four steps' loads go
// ahead of their products.
template <class FA, class FB>
__device__ __forceinline__ f32x16 small_product(uint32_t k0, uint32_t k1, FA&& a, FB&& b) {
    f32x16 acc = {};
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = threadIdx.x >> 5 & 1;
    const uint32_t each = (k1 - k0 + 31) / 32 * 8, from = k0 + wave * each, to = from + each < k1 ? from + each : k1;
    uint32_t k = from;
    for (; k + 32 <= to; k += 32) {
        f32x4 va[4], vb[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            va[u] = a(std::true_type{}, k + 8 * u + 4 * half, to);
            vb[u] = b(std::true_type{}, k + 8 * u + 4 * half, to);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(va[u][e], vb[u][e], acc, 0, 0, 0);
    }
    for (; k < to; k += 8) {
        const f32x4 va = a(std::false_type{}, k + 4 * half, to), vb = b(std::false_type{}, k + 4 * half, to);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(va[e], vb[e], acc, 0, 0, 0);
    }
    return acc;
}

// The waves' sums: thread (wave w, lane l) gets rows 8 w + 4 (l / 32) .. of a, row l % 32 of b.
__device__ __forceinline__ f32x4 small_sum(const f32x16& acc, float (&lds)[4][16][64]) {
    const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < 16; ++e) lds[wave][e][lane] = acc[e];
    __syncthreads();
    f32x4 v;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t e = 4 * wave + q;
        v[q] = (lds[0][e][lane] + lds[1][e][lane]) + (lds[2][e][lane] + lds[3][e][lane]);
    }
    return v;
}

struct SmallArgs {
    const void* x;
    const void* w;
    uint64_t x_ld, w_ld;
    uint32_t rows, classes, width, tiles_c;  // tiles of 32 classes
    const int32_t* targets;
    float* stats;  // [tiles_c][rows][3] as planes of rows_ld
    float* of;
    uint32_t rows_ld;
    const float* lse;
    const float* dloss;
    const float* entropy;
    const float* dentropy;
    float* g;  // [rows][g_ld]
    uint32_t g_ld;
    void* dx;
    void* dw;
    uint64_t dx_ld, dw_ld;
    uint32_t tiles_x;  // workgroups of dX: the rest are dW's
    // contractions cut into ranges: parts [splits][rows or classes][parts_ld], NULL: not cut
    uint32_t range;
    float* parts_x;
    float* parts_w;
    uint32_t parts_ld;
};

template <class T, int KIND>
__global__ void __launch_bounds__(256) small_logits_kernel(const SmallArgs a) {
    __shared__ float lds[4][16][64];
    __shared__ RowStats trade[4][32];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t tn = blockIdx.x / a.tiles_c, tc = blockIdx.x - tn * a.tiles_c;
    const uint32_t n = tn * 32 + (lane & 31), c = tc * 32 + (lane & 31);
    const T* const w = static_cast<const T*>(a.w) + (uint64_t)(c < a.classes ? c : a.classes - 1) * a.w_ld;
    const T* const x = static_cast<const T*>(a.x) + (uint64_t)(n < a.rows ? n : a.rows - 1) * a.x_ld;
    const f32x16 acc = small_product(
        0, a.width, [&](auto all, uint32_t k, uint32_t end) { return four_of<decltype(all)::value>(w, k, end); },
        [&](auto all, uint32_t k, uint32_t end) { return four_of<decltype(all)::value>(x, k, end); });
    const f32x4 s = small_sum(acc, lds);
    const uint32_t c0 = tc * 32 + 8 * wave + 4 * (lane >> 5);
    const int32_t target = n < a.rows ? a.targets[n] : -1;
    const bool live = target >= 0 && (uint32_t)target < a.classes;
    const uint32_t hit = (uint32_t)target - c0;
    if constexpr (KIND == kStats) {
        RowStats r{-__builtin_huge_valf(), 0.0f, 0.0f};
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            v[q] = c0 + q < a.classes ? s[q] * kLog2 : -__builtin_huge_valf();
            r.top = __builtin_fmaxf(r.top, v[q]);
            if (live && hit == (uint32_t)q) a.of[n] = v[q];
        }
        const float zero = r.top == -__builtin_huge_valf() ? 0.0f : r.top;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float d = v[q] - zero, e = exp2_of(d);
            r.sum += e;
            r.weighted = __builtin_fmaf(e, __builtin_fmaxf(d, -1000.0f), r.weighted);
        }
        RowStats o;
        float lo, hi;
        lane_pair<32>(r.top, lo, hi), r.top = lo, o.top = hi;
        lane_pair<32>(r.sum, lo, hi), r.sum = lo, o.sum = hi;
        lane_pair<32>(r.weighted, lo, hi), r.weighted = lo, o.weighted = hi;
        r.join(o);
        if (lane < 32) trade[wave][lane] = r;
        __syncthreads();
        if (threadIdx.x < 32 && n < a.rows) {
            r = trade[0][lane];
#pragma unroll
            for (int k = 1; k < 4; ++k) r.join(trade[k][lane]);
            float* const at = a.stats + (uint64_t)tc * 3 * a.rows_ld + n;
            at[0] = r.top, at[a.rows_ld] = r.sum, at[2 * (uint64_t)a.rows_ld] = r.weighted;
        }
    } else {
        if (n >= a.rows) return;
        f32x4 g = {};
        if (live) {
            const float lse2 = a.lse[n] * kLog2, dl = a.dloss[n];
            const float de = a.dentropy ? a.dentropy[n] * kLn2 : 0.0f, ent = a.dentropy ? a.entropy[n] * kLog2 : 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float d = __builtin_fmaf(s[q], kLog2, -lse2), p = exp2_of(d);
                g[q] = dl * p;
                if (a.dentropy) g[q] = __builtin_fmaf(-de * p, __builtin_fmaxf(d, -1000.0f) + ent, g[q]);
                if (hit == (uint32_t)q) g[q] -= dl;
                if (c0 + q >= a.classes) g[q] = 0.0f;
            }
        }
        *reinterpret_cast<f32x4*>(a.g + (uint64_t)n * a.g_ld + c0) = g;
    }
}

// dX = G W and dW = G' X: a's rows are the width's.
template <class T>
__global__ void __launch_bounds__(256) small_grad_kernel(const SmallArgs a) {
    __shared__ float lds[4][16][64];
    const bool dw = blockIdx.x >= a.tiles_x;
    const uint32_t tile = blockIdx.x - (dw ? a.tiles_x : 0), tiles_m = (a.width + 31) / 32;
    const uint32_t tiles_n = ((dw ? a.classes : a.rows) + 31) / 32, split = tile / (tiles_m * tiles_n);
    const uint32_t of = tile - split * tiles_m * tiles_n, tn = of / tiles_m, tm = of - tn * tiles_m;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t K = dw ? a.rows : a.classes, k0 = split * a.range, k1 = K - k0 < a.range ? K : k0 + a.range;
    const uint32_t m = tm * 32 + (lane & 31), n = tn * 32 + (lane & 31);
    const uint32_t mc = m < a.width ? m : a.width - 1;
    f32x16 acc;
    if (dw) {
        const T* const x = static_cast<const T*>(a.x) + mc;
        const float* const g = a.g + n;  // up to g_ld, a multiple of 32
        acc = small_product(
            k0, k1,
            [&](auto all, uint32_t k, uint32_t end) {
                f32x4 r = four_down<decltype(all)::value>(x, a.x_ld, k, end);
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // a row without a target may hold anything
                    const int32_t target = decltype(all)::value || k + e < end ? a.targets[k + e] : -1;
                    r[e] = target >= 0 && (uint32_t)target < a.classes ? r[e] : 0.0f;
                }
                return r;
            },
            [&](auto all, uint32_t k, uint32_t end) { return four_down<decltype(all)::value>(g, a.g_ld, k, end); });
    } else {
        const T* const w = static_cast<const T*>(a.w) + mc;
        const float* const g = a.g + (uint64_t)(n < a.rows ? n : a.rows - 1) * a.g_ld;
        acc = small_product(
            k0, k1,
            [&](auto all, uint32_t k, uint32_t end) { return four_down<decltype(all)::value>(w, a.w_ld, k, end); },
            [&](auto all, uint32_t k, uint32_t end) { return four_of<decltype(all)::value>(g, k, end); });
    }
    const f32x4 v = small_sum(acc, lds);
    const uint32_t m0 = tm * 32 + 8 * wave + 4 * (lane >> 5);
    if (n >= (dw ? a.classes : a.rows)) return;
    float* const parts = dw ? a.parts_w : a.parts_x;
    if (parts) {  // parts_ld is a multiple of 4
        if (m0 < a.width)
            *reinterpret_cast<f32x4*>(parts + ((uint64_t)split * (dw ? a.classes : a.rows) + n) * a.parts_ld + m0) = v;
        return;
    }
    T* const out = static_cast<T*>(dw ? a.dw : a.dx) + n * (dw ? a.dw_ld : a.dx_ld) + m0;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (m0 + q < a.width) out[q] = (T)v[q];
}

}  // namespace dev

namespace {

constexpr uint32_t kMostHeadRows = 1u << 20, kMostClasses = 1u << 20, kMostWidth = 1u << 16;
constexpr uint32_t kHeadM = 256;          // classes that a piece is filled up to
// Logits of a piece, about: 256 MB of 16-bit gradients, as much as the last cache. us with 2^25, 2^26 and
// 2^27: gradients of 4096 x 65536 x 128 bf16 569, 530 and 442, x 1024 1710, 1605 and 1617; 4096 x 32768 x
// 512 fp32 1298, 1172 and 1152.
constexpr uint32_t kPieceCells = 1u << 27;
// Elements past a row: rows a power of two apart meet in few memory channels. 16384 x 32768 x 256 bf16 1178
// us with them and 1263 without.
constexpr uint32_t kSkew = 128;
// Contraction elements of a gradient's tile: more keep fewer partial sums, 8192 x 8192 x 1024 bf16 397 us with
// 8192 and 458 with 4096; 16384 changes nothing.
constexpr uint32_t kMostRange = 8192;
constexpr uint32_t kSmallRange = 512;       // and of a small one's
constexpr uint32_t kMostTiles = 1u << 22;   // of a launch, whose threads have to stay under 2^32

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

// Where the small products take over, by the multiply-adds of one product (both ways measured,
// us, small first). fp32 saves the launches that scale and split it, and with few rows the passes over
// W that those make: forward 1024 x 4096 x 128 26 and 31, with a width of 512 71 and 53, 16 x 16384 x 2048
// 44 and 167; gradients 4096 x 512 x 128 47 and 74, 1024 x 4096 x 128 76 and 71, 256 x 1024 x 2048 68
// and 164. Of 16-bit types the gradients save launches (1024 x 1024 x 128 33 and 36, 4096 x 512 x 128 46
// and 43), and where there are few large tiles nothing waits for one tile's long contraction: forward 256
// x 1024 x 2048 25 and 46, 1024 x 4096 x 128 26 and 18; gradients of the first 61 and 71.
bool is_small(uint32_t rows, uint32_t classes, uint32_t width, uint32_t type, bool backward) {
    const uint64_t work = (uint64_t)up_to(rows, 32) * up_to(classes, 32) * up_to(width, 32);
    const uint64_t tiles = (uint64_t)((rows + 255) / 256) * ((classes + 255) / 256);
    const bool few = work <= 1u << 29 && tiles <= (backward ? 8 : 16);
    if (type == MG_TYPE_FP32) {
        // a launch has a tile of 32 x 32 for all of W, at 256 threads
        if (rows <= 32) return (uint64_t)classes * width <= 1ull << 33;
        return work <= 1u << (backward ? 28 : 29) || (backward && few);
    }
    return backward ? work <= 1u << 27 || few : few && width >= 512;
}

// What a call keeps in its workspace. 16-bit planes; pairs have two.
struct HeadSpace {
    bool small;
    float* small_g;
    uint32_t tiles, wide, rows_ld, high, g_ld, piece, pieces, tall, splits_x, splits_w, range_x, range_w, parts_ld;
    uint32_t low;  // the row of G where the low halves begin, 0: there are none
    uint64_t planes;
    uint16_t *x, *x_even, *w, *g;
    uint32_t* live;
    float *stats, *of, *parts_x, *parts_w, *amax;
    int* row_exp;
    dev::HeadScales* scales;
    uint64_t bytes;

    static uint32_t ranges(uint32_t k, uint32_t range) { return range ? (k + range - 1) / range : 0; }
    HeadSpace(void* base, uint32_t rows, uint32_t classes, uint32_t width, uint32_t type, bool backward) {
        Carve c{static_cast<char*>(base)};
        small = is_small(rows, classes, width, type, backward);
        if (small) {
            tiles = (classes + 31) / 32, rows_ld = rows, g_ld = tiles * 32;
            if (backward) {
                small_g = c.take<float>((uint64_t)rows * g_ld);
                range_x = range_w = kSmallRange, parts_ld = up_to(width, 4);
                splits_x = (classes + kSmallRange - 1) / kSmallRange, splits_w = (rows + kSmallRange - 1) / kSmallRange;
                parts_x = splits_x > 1 ? c.take<float>((uint64_t)splits_x * rows * parts_ld) : nullptr;
                parts_w = splits_w > 1 ? c.take<float>((uint64_t)splits_w * classes * parts_ld) : nullptr;
            } else {
                stats = c.take<float>((uint64_t)tiles * 3 * rows_ld);
                of = c.take<float>(rows_ld);
            }
            bytes = c.used;
            return;
        }
        planes = type == MG_TYPE_FP32 ? 2 : 1;
        wide = up_to(width, planes > 1 ? 16 : 8), rows_ld = up_to(rows, dev::kHeadN);
        // Classes of a tile of logits. One of 128 by 256 leaves half a CU to another, whose products run
        // under its epilogue; one of 256 by 256 reads less for each product. us, the first of the two first, 4096
        // rows, bf16: forward of 49152 classes, width 256 162 and 170, 512 249 and 244, 1024 479 and 440, 4096
        // 1612 and 1384; gradients of 10007 classes, 128 84 and 97, 512 221 and 233, 1024 312 and 321, of 65536
        // 1024 1733 and 1701. Pairs as fp32 the same way: forward of 10007, 128 66 and 74, 512 149 and 158.
        high = width <= (backward ? 512 : 256) ? 128 : 256;
        scales = c.take<dev::HeadScales>(1);
        amax = c.take<float>(3 * dev::kAmaxParts);
        row_exp = c.take<int>(planes > 1 ? rows : 0);
        x = c.take<uint16_t>(planes * rows * wide);
        w = c.take<uint16_t>(planes * classes * wide);
        if (!backward) {
            stats = c.take<float>((uint64_t)up_to(classes, high) / high * 3 * rows_ld);
            of = c.take<float>(rows_ld);
            bytes = c.used;
            return;
        }
        const uint32_t all = up_to(classes, kHeadM);
        pieces = (uint32_t)(((uint64_t)all * rows_ld + kPieceCells / 2) / kPieceCells);
        if (pieces > all / kMostRange) pieces = all / kMostRange;
        if (!pieces) pieces = 1;
        piece = up_to((all + pieces - 1) / pieces, kHeadM);
        g_ld = (uint32_t)planes * piece + kSkew;
        // The gradients' contractions, over a piece's classes and over all rows, are cut so that
        // their tiles are about as many as CUs, or of kMostRange elements where they are more.
        // Of their tiles' two heights the lower for narrow heads, where the other is half empty (4096 x 10007 x
        // 128 fp32 180 us, else 219); with a width of 256 it would read twice as much of G (123 us, else 142).
        tall = width > 128 ? 256 : 128;
        const uint64_t across = (width + tall - 1) / tall;
        const uint64_t work = across * (rows_ld / dev::kHeadN) * piece + across * (piece / dev::kHeadN) * rows_ld;
        const uint32_t each = up_to((work + kCus - 1) / kCus, 64);
        auto cut = [&](uint32_t k, uint32_t& splits, uint32_t& range) {
            uint32_t most = each < kMostRange ? each : kMostRange;
            if (most < 256) most = 256;
            splits = (k + most / 2) / most;
            if (!splits) splits = 1;
            range = up_to((k + splits - 1) / splits, dev::kHeadK);
        };
        cut(piece, splits_x, range_x);
        cut(rows_ld, splits_w, range_w);
        // G's rounding to 16 bits is as large as the results' own: the gradients' error is 1.4 times that of rounding
        // them alone, and with few rows, whose targets' elements are most of G, up to 1.9 times. Where they are at
        // most half of a tile's rows the others take what the rounding leaves (1.0 times). us without and with, bf16,
        // 30000 x 2048: 32 rows 120 and 121, 64 122 and 133, 128 133 and 161; more rows would take the products twice.
        low = planes == 1 && 2 * up_to(rows, 32) <= dev::kHeadN ? up_to(rows, 32) : 0;
        // What is launched, kept and summed are the ranges of what there is: the last of a filled-up piece may
        // hold nothing else. The first piece is the longest.
        splits_x = ranges(classes < piece ? classes : piece, range_x), splits_w = ranges(low ? 2 * low : rows, range_w);
        parts_ld = up_to(width, 4);
        x_even = c.take<uint16_t>(planes > 1 ? planes * rows * wide : 0);
        live = c.take<uint32_t>(rows_ld / 32);
        g = c.take<uint16_t>((uint64_t)rows_ld * g_ld);
        parts_x = c.take<float>(splits_x > 1 || pieces > 1 || low ? (uint64_t)splits_x * (low ? 2 : 1) * rows * parts_ld : 0);
        parts_w = c.take<float>(splits_w > 1 ? (uint64_t)splits_w * piece * parts_ld : 0);
        bytes = c.used;
    }
};

// A 16-bit array that the products read where it lies.
bool fits(const void* p, uint64_t ld, uint32_t cols, uint32_t type) {
    return type != MG_TYPE_FP32 && cols % 8 == 0 && ld % 8 == 0 && ld <= (1u << 21) && aligned(p, 16);
}

dim3 copy_grid(uint32_t cols, uint32_t rows) { return dim3((cols + 1023) / 1024, rows < 65535 ? rows : 65535); }

template <class T>
struct HeadType {
    typedef T H;
};
template <>
struct HeadType<float> {
    typedef _Float16 H;
};

// x and W as the products' operands, and their scales.
struct HeadInputs {
    dev::HeadOperand x, w;
    dev::HeadOperand x_even;  // x at one scale
    const dev::HeadScales* scales;
};
template <class T, class P>
HeadInputs prepare(hipStream_t st, const P& p, const HeadSpace& s, const float* dloss, const float* dentropy,
                   bool even) {
    typedef typename HeadType<T>::H H;
    const bool pairs = std::is_same<T, float>::value, g = dloss && !std::is_same<T, __bf16>::value;
    HeadInputs in{};
    in.x = {p.x, (uint32_t)p.x_ld};
    in.w = {p.w, (uint32_t)p.w_ld};
    dev::PrepareArgs ax{p.x, p.x_ld, p.rows, p.width, nullptr, nullptr, s.wide, s.row_exp};
    dev::PrepareArgs aw{p.w, p.w_ld, p.classes, p.width, nullptr, nullptr, s.wide, nullptr};
    if (!fits(p.x, p.x_ld, p.width, p.type)) ax.to = s.x, in.x = {s.x, (uint32_t)s.planes * s.wide};
    if (!fits(p.w, p.w_ld, p.width, p.type)) aw.to = s.w, in.w = {s.w, (uint32_t)s.planes * s.wide};
    in.x_even = in.x;
    if (pairs && even) ax.to_even = s.x_even, in.x_even.base = s.x_even;
    dev::PrepareScales scales{{nullptr, nullptr, nullptr}, nullptr};
    if (pairs || g) {
        float* const parts = s.amax;
        const dev::AmaxArgs mx{reinterpret_cast<const float*>(pairs ? p.x : nullptr), p.x_ld, pairs ? p.rows : 0,
                               p.width, nullptr, 0, p.targets, p.classes, parts, s.row_exp};
        const dev::AmaxArgs mw{reinterpret_cast<const float*>(pairs ? p.w : nullptr), p.w_ld, pairs ? p.classes : 0,
                               p.width, nullptr, 0, nullptr, 0, parts + dev::kAmaxParts, nullptr};
        // |p (log p + H)| is at most 1/e + H, and H at most log(classes)
        const dev::AmaxArgs mg{dloss, 0, g ? p.rows : 0, 0, dentropy, __builtin_logf((float)p.classes) + 1.0f,
                               p.targets, p.classes, parts + 2 * dev::kAmaxParts, nullptr};
        hipLaunchKernelGGL(dev::head_amax_kernel, dim3(dev::kAmaxParts, 3), dim3(256), 0, st, mx, mw, mg);
        if (pairs) scales.parts[0] = parts, scales.parts[1] = parts + dev::kAmaxParts;
        if (g) scales.parts[2] = parts + 2 * dev::kAmaxParts;
        scales.out = s.scales;
        in.scales = s.scales;
    }
    if (ax.to || aw.to || scales.out)
        hipLaunchKernelGGL((dev::head_prepare_kernel<T, H>), dim3(4 * kCus, 2), dim3(256), 0, st, ax, aw, scales);
    return in;
}

template <class P>
dev::SmallArgs small_args(const P& p, const HeadSpace& s) {
    dev::SmallArgs a{};
    a.x = p.x, a.w = p.w, a.x_ld = p.x_ld, a.w_ld = p.w_ld, a.rows = p.rows, a.classes = p.classes, a.width = p.width;
    a.tiles_c = s.tiles, a.targets = p.targets, a.rows_ld = s.rows_ld, a.g_ld = s.g_ld;
    return a;
}
int join_tiles(hipStream_t st, const mg_cross_entropy_args& p, const HeadSpace& s, uint32_t tiles) {
    // rows side by side make whole reads, and fewer of them more threads a row: 4095 x 50001 6.5 us, and 19
    // with four
    const uint32_t across = p.rows >= 1024 ? 32 : 4;
    hipLaunchKernelGGL(dev::head_join_kernel, dim3((p.rows + across - 1) / across), dim3(across * (across == 4 ? 64 : 32)),
                       0, st, s.stats, s.of, p.targets, p.rows, s.rows_ld, tiles, p.classes, across, p.loss, p.lse,
                       p.entropy);
    MG_HIP(hipGetLastError(), "cross entropy join launch");
    return MG_OK;
}

template <class H, int KIND, bool PAIRS>
void launch_logits(hipStream_t st, const dev::HeadArgs& a, const HeadSpace& s) {
    if (s.high == 128)
        hipLaunchKernelGGL((dev::head_kernel<H, KIND, 2, PAIRS>), dim3(a.tiles), dim3(512), 0, st, a);
    else
        hipLaunchKernelGGL((dev::head_kernel<H, KIND, 4, PAIRS>), dim3(a.tiles), dim3(512), 0, st, a);
}

template <class T>
int cross_entropy(hipStream_t st, const mg_cross_entropy_args& p) {
    typedef typename HeadType<T>::H H;
    constexpr bool kPairs = sizeof(T) == 4;
    const HeadSpace s(p.workspace, p.rows, p.classes, p.width, p.type, false);
    if (s.small) {
        dev::SmallArgs a = small_args(p, s);
        a.stats = s.stats, a.of = s.of;
        hipLaunchKernelGGL((dev::small_logits_kernel<T, dev::kStats>), dim3((p.rows + 31) / 32 * s.tiles), dim3(256), 0,
                           st, a);
        MG_HIP(hipGetLastError(), "cross entropy launch");
        return join_tiles(st, p, s, s.tiles);
    }
    dev::HeadArgs a{};
    const HeadInputs in = prepare<T>(st, p, s, nullptr, nullptr, false);
    a.scales = in.scales;
    dev::HeadProduct& m = a.p[0];
    m.a = in.w, m.b = in.x;
    m.k = m.range = s.wide, m.splits = 1, m.n = p.rows, m.tiles_n = s.rows_ld / dev::kHeadN;
    a.rows = p.rows, a.classes = p.classes, a.targets = p.targets, a.row_exp = s.row_exp;
    a.of = s.of, a.rows_ld = s.rows_ld, a.want_entropy = p.entropy != nullptr;
    const uint32_t tiles = up_to(p.classes, s.high) / s.high, most = kMostTiles / m.tiles_n;
    for (uint32_t first = 0; first < tiles; first += most) {
        m.tiles_m = tiles - first < most ? tiles - first : most;
        a.tiles = m.tiles_m * m.tiles_n, a.first = first * s.high, m.m = p.classes - a.first;
        m.a.base = static_cast<const H*>(in.w.base) + (uint64_t)a.first * in.w.ld;
        a.stats = s.stats + (uint64_t)first * 3 * s.rows_ld;
        launch_logits<H, dev::kStats, kPairs>(st, a, s);
    }
    MG_HIP(hipGetLastError(), "cross entropy launch");
    return join_tiles(st, p, s, tiles);
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
    if (s.small) {
        dev::SmallArgs a = small_args(p, s);
        a.lse = p.lse, a.dloss = p.dloss, a.entropy = p.entropy, a.dentropy = p.dentropy, a.g = s.small_g;
        a.dx = p.dx, a.dw = p.dw, a.dx_ld = p.dx_ld, a.dw_ld = p.dw_ld;
        const uint32_t tiles_n = (p.rows + 31) / 32, tiles_m = (p.width + 31) / 32;
        a.tiles_x = p.dx ? tiles_n * tiles_m * s.splits_x : 0;
        a.range = kSmallRange, a.parts_ld = s.parts_ld;
        a.parts_x = p.dx && s.splits_x > 1 ? s.parts_x : nullptr, a.parts_w = p.dw && s.splits_w > 1 ? s.parts_w : nullptr;
        hipLaunchKernelGGL((dev::small_logits_kernel<T, dev::kLogitGrad>), dim3(tiles_n * s.tiles), dim3(256), 0, st, a);
        MG_HIP(hipGetLastError(), "cross entropy logits launch");
        hipLaunchKernelGGL(dev::small_grad_kernel<T>, dim3(a.tiles_x + (p.dw ? s.tiles * tiles_m * s.splits_w : 0)),
                           dim3(256), 0, st, a);
        if (a.parts_x)
            hipLaunchKernelGGL(dev::head_sum_kernel<T>, copy_grid(p.width, p.rows), dim3(256), 0, st, a.parts_x,
                               s.splits_x, p.rows, p.width, s.parts_ld, static_cast<T*>(p.dx), p.dx_ld, nullptr, 0u);
        if (a.parts_w)
            hipLaunchKernelGGL(dev::head_sum_kernel<T>, copy_grid(p.width, p.classes), dim3(256), 0, st, a.parts_w,
                               s.splits_w, p.classes, p.width, s.parts_ld, static_cast<T*>(p.dw), p.dw_ld, nullptr, 1u);
        MG_HIP(hipGetLastError(), "cross entropy gradients launch");
        return MG_OK;
    }
    dev::HeadArgs a{};
    const HeadInputs in = prepare<T>(st, p, s, p.dloss, p.dentropy, p.dw != nullptr);
    a.scales = in.scales;
    a.rows = p.rows, a.classes = p.classes, a.targets = p.targets, a.row_exp = s.row_exp;
    a.lse = p.lse, a.dloss = p.dloss, a.entropy = p.entropy, a.dentropy = p.dentropy;
    a.rows_ld = s.rows_ld, a.g = s.g, a.g_ld = s.g_ld, a.live = s.live;
    const bool parts_x = s.splits_x > 1 || s.pieces > 1 || s.low, parts_w = s.splits_w > 1;
    const uint32_t tiles_m = (p.width + s.tall - 1) / s.tall;
    for (uint32_t first = 0; first < p.classes; first += s.piece) {
        const uint32_t here = p.classes - first < s.piece ? p.classes - first : s.piece, fill = up_to(here, kHeadM);
        dev::HeadProduct& m = a.p[0];
        m = {};
        m.a = in.w, m.b = in.x;
        m.a.base = static_cast<const H*>(in.w.base) + (uint64_t)first * in.w.ld;
        m.k = m.range = s.wide, m.splits = 1, m.m = here, m.n = p.rows;
        m.tiles_m = fill / s.high, m.tiles_n = s.rows_ld / dev::kHeadN;
        if (s.low) m.b.again = s.low;
        a.tiles = m.tiles_m * m.tiles_n, a.first = first;
        launch_logits<H, dev::kLogitGrad, kPairs>(st, a, s);
        MG_HIP(hipGetLastError(), "cross entropy logits launch");
        const dev::HeadOperand m_of_w = m.a;
        uint32_t n = 0, tiles = 0;
        if (p.dx) {
            dev::HeadProduct& q = a.p[n++];
            q = {};
            q.a = m_of_w, q.b = {s.g, s.g_ld}, q.m = p.width, q.n = s.low ? 2 * s.low : p.rows, q.low = s.low;
            q.k = here, q.range = s.range_x, q.splits = s.ranges(here, s.range_x);
            q.tiles_m = tiles_m, q.tiles_n = s.rows_ld / dev::kHeadN;
            q.out = p.dx, q.out_ld = p.dx_ld, q.parts = parts_x ? s.parts_x : nullptr, q.parts_ld = s.parts_ld;
            q.add = first != 0, q.which = 0;
            a.tiles = q.tiles_m * q.tiles_n * q.splits, tiles += a.tiles;
        }
        if (p.dw) {
            dev::HeadProduct& q = a.p[n++];
            q = {};
            q.a = in.x_even, q.b = {s.g, s.g_ld}, q.m = p.width, q.n = here, q.live = s.live;
            q.k = s.low ? 2 * s.low : p.rows, q.range = s.range_w, q.splits = s.splits_w;
            if (s.low) q.a.again = s.low;
            q.tiles_m = tiles_m, q.tiles_n = fill / dev::kHeadN;
            q.out = static_cast<T*>(p.dw) + (uint64_t)first * p.dw_ld, q.out_ld = p.dw_ld;
            q.parts = parts_w ? s.parts_w : nullptr, q.parts_ld = s.parts_ld, q.which = 1;
            const uint32_t more = q.tiles_m * q.tiles_n * q.splits;
            if (n == 1) a.tiles = more;
            tiles += more;
        }
        if (s.tall == 128)
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
                           s.splits_x * (s.low ? 2 : 1), p.rows, p.width, s.parts_ld, static_cast<T*>(p.dx), p.dx_ld,
                           a.scales, 0u);
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
    *bytes = rows ? HeadSpace(nullptr, rows, classes, width, type, true).bytes : 0;
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
