// Matrices orthogonalised by Newton-Schulz steps (mg_orthogonalize) and the Muon
// update built on them (mg_muon_step).
//
// X is m x n, m the short side. A step is X <- P X with P = a I + b A + c A^2 and
// A = X X'. All of A, P and their products are symmetric and commute, so steps can
// also be taken on m x m matrices alone: A <- P A P, Q <- P Q, and X <- Q X once
// for several steps (a segment). On long matrices that saves the two products with
// X of each step but the segment's first and last. An error of A grows by a^2 with
// each step of a segment, the most where the small singular values are still small,
// so segments are short: at most 2 steps (128 x 512 with few strong directions: relative
// error 2.0e-6 in segments of 1, 2 and 2, plain fp32 1.9e-6; 2 and 3 steps 6.5e-6, one
// segment 5e-5).
//
// Products run on the matrix units as pairs of binary16 halves: x 2^e = hi + lo
// with 22 bits, hi hi + hi lo + lo hi summed in fp32. The iteration's bounds are
// known before it starts (singular values at most 2, polynomials at most 64, or the
// call is refused), so every operand has a fixed exponent and nothing is measured
// on the way. One binary16 product would lose the small singular values of a
// matrix with few strong ones: 3e-2 of the result. A matrix instruction rounds its sum,
// and cuts off what its smaller products have under 2^-25 of the largest: towards zero,
// so that a large diagonal's small squares are always a little short. Chains of 32 or 64
// contraction elements, added up in fp32, keep that near the operands' own rounding
// (4.0e-6 of the result in one chain, 2.1e-6 so).
//
// muon_short.h takes matrices with a side of at most 128, muon_tiled.h the others.
#include "muon_short.h"
#include "muon_tiled.h"

namespace mg {
namespace {

constexpr mg_newton_schulz kDefaultNs = {5, 3.4445f, -4.7750f, 2.0315f, 1e-7f};
constexpr uint32_t kMostSide = 65536, kMostShort = 8192, kMostSteps = 32;
constexpr double kMostSingular = 2.0, kMostPolynomial = 64.0;
using dev::kUnitA;
using dev::kUnitP;
using dev::kUnitX;

size_t align256(size_t x) { return (x + 255) / 256 * 256; }
uint32_t pad(uint32_t x, uint32_t to) { return (x + to - 1) / to * to; }

// Edges of the product tiles, of symmetric results and of products with X: 64 where a
// CU would have at most one tile, or two of X's, else 128, of which a CU does twice as
// much. X's are 64 too where 128 would pad m by over a sixteenth, as the squares are
// padded with it. 1280 x 8192 takes 693 us with 64 throughout, 817 with 128 and 584 so;
// 900 x 2000 244 with 64 and 397 with 128; 1666 x 1570, just past the first bound, 460 and
// 473; 9 of 487 x 585, further past it, 276 and 255.
struct TileEdges {
    uint32_t square, x;
};
TileEdges tile_edges(uint32_t count, uint32_t m, uint32_t n) {
    const uint64_t tm = (m + 63) / 64, tn = (n + 63) / 64;
    if (count * tm * (tm + 1) / 2 > 256) return {128, 128};
    return {64, count * tm * tn > 512 && (pad(m, 128) - pad(m, 64)) * 16 <= m ? 128u : 64u};
}

// Steps of the next segment of the `left` that remain. One (on X) for small matrices,
// where a rounding error of A does not average out, and for polynomials that grow
// small singular values, and their errors, faster than the default's. Else two at the
// end, and before it too where the rounding of a 16-bit result or weight hides the
// difference (hidden); an fp32 weight may be 0 and its rate 1, which hide nothing. Over
// 117 random shapes with a short side of 36 to 1000 and fp32 results, the error is at most
// 1.7 times that of the plain fp32 iteration with two steps throughout, 1.2 with two at
// the end (the most where the short side is under 65; 1.3 at 512 x 2048 with few strong
// directions), and 1.0 with single steps; two matrices of 512 x 128 take 63.0, 65.8 and
// 68.6 us, 2048 x 8192 1438, 1667 and 1887.
uint32_t segment_steps(const mg_newton_schulz& ns, uint32_t m, uint32_t left, bool hidden) {
    if (m < (hidden ? 32 : 65) || fabsf(ns.a) > 4.0f) return 1;
    return left == 2 || (hidden && !(left & 1)) ? 2 : 1;
}
// The same for tiled products: on X where the sides are alike, as a segment then
// saves no products.
uint32_t segment_steps(const mg_newton_schulz& ns, uint32_t m, uint32_t n, uint32_t left, bool hidden) {
    return n < m + m / 4 ? 1 : segment_steps(ns, m, left, hidden);
}

// Takes [0, *reach] to the largest |p(s)| on it, and gives the largest
// |a + b s^2 + c s^4| there: both have their extremes at 0, at the end, or where
// the derivative in s^2 is 0.
double step_bounds(const mg_newton_schulz& ns, double* reach) {
    const double a = ns.a, b = ns.b, c = ns.c, end = *reach * *reach;
    double most = 0.0, poly = 0.0;
    auto look = [&](double t) {  // t = s^2
        if (!(t >= 0.0 && t <= end)) return;
        const double q = fabs(a + t * (b + t * c));
        poly = q > poly ? q : poly;
        most = sqrt(t) * q > most ? sqrt(t) * q : most;
    };
    look(0.0);
    look(end);
    if (c != 0.0) {
        look(-b / (2 * c));
        const double d = 9 * b * b - 20 * a * c;
        if (d >= 0.0) {
            look((-3 * b + sqrt(d)) / (10 * c));
            look((-3 * b - sqrt(d)) / (10 * c));
        }
    } else if (b != 0.0) {
        look(-a / (3 * b));
    }
    *reach = most;
    return poly;
}

// A power of two that keeps values of up to `most` under 2^15.
float unit_of(double most) { return ldexpf(1.0f, 14 - ilogb(most > 1.0 ? most : 1.0)); }

int check_ns(const char* what, const mg_newton_schulz* in, mg_newton_schulz* ns) {
    *ns = in ? *in : kDefaultNs;
    MG_CHECK(ns->steps >= 1 && ns->steps <= kMostSteps, MG_ERR_INVALID, "%s: steps %u must be in [1, %u]", what, ns->steps,
             kMostSteps);
    MG_CHECK(ns->eps > 0.0f && ns->eps < __builtin_huge_valf(), MG_ERR_INVALID, "%s: eps must be positive and finite",
             what);
    double reach = 1.0;
    for (uint32_t k = 0; k < ns->steps; ++k) {
        const double poly = step_bounds(*ns, &reach);
        MG_CHECK(isfinite(ns->a) && isfinite(ns->b) && isfinite(ns->c) && reach <= kMostSingular &&
                     poly <= kMostPolynomial,
                 MG_ERR_INVALID,
                 "%s: the polynomial (%g, %g, %g) leaves [-2, 2] in step %u, or a + b s^2 + c s^4 [-64, 64]", what,
                 (double)ns->a, (double)ns->b, (double)ns->c, k + 1);
    }
    return MG_OK;
}

int check_shape(const char* what, uint32_t count, uint32_t rows, uint32_t cols) {
    MG_CHECK(rows >= 1 && cols >= 1 && rows <= kMostSide && cols <= kMostSide, MG_ERR_INVALID,
             "%s: %u x %u: the sides must be in [1, %u]", what, rows, cols, kMostSide);
    MG_CHECK((rows < cols ? rows : cols) <= kMostShort, MG_ERR_INVALID,
             "%s: %u x %u: the smaller side must be at most %u", what, rows, cols, kMostShort);
    MG_CHECK(count <= 65535, MG_ERR_INVALID, "%s: count %u must be at most 65535", what, count);
    return MG_OK;
}

int check_batch(const char* what, const char* name, const mg_matrices* in, dev::Batch* out) {
    MG_CHECK(in, MG_ERR_INVALID, "%s: %s is NULL", what, name);
    int rc = check_shape(what, in->count, in->rows, in->cols);
    if (rc) return rc;
    MG_CHECK(type_known(in->type), MG_ERR_INVALID, "%s: %s has unknown type %u", what, name, in->type);
    MG_CHECK(in->data || !in->count, MG_ERR_INVALID, "%s: %s has no data", what, name);
    MG_CHECK(aligned(in->data, type_bytes(in->type)), MG_ERR_INVALID, "%s: %s is not aligned to its type", what, name);
    const uint64_t ld = in->ld ? in->ld : in->cols;
    MG_CHECK(ld >= in->cols && ld < (1ull << 31), MG_ERR_INVALID, "%s: %s: ld %llu must be in [cols, 2^31)", what, name,
             (unsigned long long)ld);
    const uint64_t stride = in->stride ? in->stride : in->rows * ld;
    if (in->count > 1) {
        MG_CHECK(stride <= (1ull << 44), MG_ERR_INVALID, "%s: %s: stride %llu is out of range", what, name,
                 (unsigned long long)stride);
        // one after another, or side by side: column panels of rows of ld
        const bool after = stride >= (in->rows - 1) * ld + in->cols;
        const bool beside = stride >= in->cols && (in->count - 1) * stride + in->cols <= ld;
        MG_CHECK(after || beside, MG_ERR_INVALID, "%s: %s: stride %llu: the matrices overlap", what, name,
                 (unsigned long long)stride);
    }
    *out = dev::Batch{in->data, (size_t)stride, (uint32_t)ld, in->type};
    return MG_OK;
}

int check_same(const char* what, const mg_matrices* a, const mg_matrices* b) {
    MG_CHECK(a->count == b->count && a->rows == b->rows && a->cols == b->cols, MG_ERR_INVALID,
             "%s: the batches differ in shape: %u of %u x %u and %u of %u x %u", what, a->count, a->rows, a->cols,
             b->count, b->rows, b->cols);
    return MG_OK;
}

// The workspace of a batch.
struct Workspace {
    size_t norms, scales, x, xt[2], gram, product, poly[2], both, total;  // byte offsets
    uint32_t m, n, mp, np;
    TileEdges tile;
    Workspace(uint32_t count, uint32_t rows, uint32_t cols) {
        m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
        tile = tile_edges(count, m, n);
        mp = pad(m, tile.x), np = pad(n, tile.x);  // the larger of the two
        // X by rows of np, its transpose by rows of mp
        const size_t wide = dev::planes_block(np) * (mp / 32) * 2 * count, tall = dev::planes_block(mp) * (np / 32) * 2 * count;
        const size_t square = dev::planes_block(mp) * (mp / 32) * 2 * count;
        total = 0;
        auto take = [&](size_t bytes) {
            const size_t at = total;
            total += align256(bytes);
            return at;
        };
        norms = take((size_t)count * dev::kNormParts * 8);
        scales = take((size_t)count * sizeof(dev::MatrixScale));
        x = take(wide), xt[0] = take(tall), xt[1] = take(tall);
        gram = take(square), product = take(square), poly[0] = take(square), poly[1] = take(square), both = take(square);
    }
};

// Workgroups a matrix (muon_short.h). One fills a CU, so they run in rounds of 256, each
// as long as a segment's steps, about 8 slabs' worth (17 us to 2.5), and its slabs: the
// least product of the two, with fewer workgroups among equals. 300 x 128 x 4096 takes
// 1570 us in 3 rounds with two each, 1851 in 2 rounds with one.
uint32_t short_parts(uint32_t count, uint32_t slabs) {
    uint32_t best = 1;
    uint64_t least = ~0ull;
    for (uint32_t p = 1; p <= (uint32_t)dev::kShortParts && p <= slabs; ++p) {
        const uint64_t cost = (((uint64_t)count * p + 255) / 256) * (8 + (slabs + p - 1) / p);
        if (cost < least) least = cost, best = p;
    }
    return best;
}

// The workspace of a batch whose short side is at most 128 (muon_short.h).
struct ShortWorkspace {
    size_t xt, partial[2], state, total;
    uint32_t mp, slabs, parts;
    ShortWorkspace(uint32_t count, uint32_t rows, uint32_t cols) {
        const uint32_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
        mp = m <= 32 ? 32 : m <= 64 ? 64 : 128;
        slabs = (n + dev::kSlab - 1) / dev::kSlab;
        parts = short_parts(count, slabs);
        const uint32_t tiles = mp / 32 * (mp / 32 + 1) / 2;
        xt = 0;
        const size_t sums = align256((size_t)count * parts * tiles * 4096);
        partial[0] = xt + align256((size_t)count * slabs * dev::kSlab * mp * 4);
        partial[1] = partial[0] + sums;
        state = partial[1] + sums;
        total = state + align256((size_t)count * sizeof(dev::ShortState));
    }
};
constexpr uint32_t kShortSide = 128;
bool is_short(uint32_t rows, uint32_t cols) { return rows <= kShortSide || cols <= kShortSide; }
size_t workspace_bytes_of(uint32_t count, uint32_t rows, uint32_t cols) {
    return is_short(rows, cols) ? ShortWorkspace(count, rows, cols).total : Workspace(count, rows, cols).total;
}

struct FinalArgs {
    dev::Batch dst;
    uint32_t step;
    float keep, rate, odd_rate;
};

template <int MP>
int newton_schulz_short(hipStream_t st, const mg_newton_schulz& ns, uint32_t count, dev::ShortArgs a, float* const (&partial)[2]) {
    const uint32_t m = a.src.rows < a.src.cols ? a.src.rows : a.src.cols;
    using Shape = dev::ShortShape<MP>;
    const dim3 slabs(a.parts, count);
    int to = 0;
    a.partial = partial[to];
    hipLaunchKernelGGL((dev::short_first_kernel<MP>), slabs, dim3(Shape::THREADS), 0, st, a);
    MG_HIP(hipGetLastError(), "newton-schulz first launch");
    double reach = 1.0, growth = 1.0;
    a.start = 1;
    for (uint32_t left = ns.steps; left; a.start = 0) {
        a.steps = segment_steps(ns, m, left, a.dst.type != MG_TYPE_FP32);
        double most = step_bounds(ns, &reach);
        if (a.steps == 2) most *= step_bounds(ns, &reach);
        a.unit_q = a.steps == 1 ? kUnitP : unit_of(most);
        a.growth_in = (float)growth;
        growth *= most;
        a.growth = (float)growth;
        left -= a.steps;
        a.partial_in = partial[to], a.partial = partial[to ^= 1];
        if (left)
            hipLaunchKernelGGL((dev::short_step_kernel<MP, false>), slabs, dim3(Shape::THREADS), 0, st, a);
        else
            hipLaunchKernelGGL((dev::short_step_kernel<MP, true>), slabs, dim3(Shape::THREADS), 0, st, a);
        MG_HIP(hipGetLastError(), "newton-schulz step launch");
    }
    return MG_OK;
}

template <int KIND>
int launch_product(hipStream_t st, const dev::ProductArgs& p, uint32_t tile, uint32_t tiles, uint32_t count,
                   const char* what) {
    if (tile == 128)
        hipLaunchKernelGGL((dev::product_kernel<KIND, 128>), dim3(tiles, count), dim3(512), 0, st, p);
    else
        hipLaunchKernelGGL((dev::product_kernel<KIND, 64>), dim3(tiles, count), dim3(512), 0, st, p);
    MG_HIP(hipGetLastError(), what);
    return MG_OK;
}

int newton_schulz_tiled(hipStream_t st, const mg_newton_schulz& ns, uint32_t count, const dev::SourceArgs& src,
                        const FinalArgs& fin, const Workspace& w, void* workspace) {
    char* const base = static_cast<char*>(workspace);
    auto planes = [&](size_t at, uint32_t rows, uint32_t k) {
        return dev::Planes{reinterpret_cast<dev::f16*>(base + at), dev::planes_block(k) * (rows / 32), dev::planes_block(k)};
    };
    double* const norms = reinterpret_cast<double*>(base + w.norms);
    const dev::Planes X = planes(w.x, w.mp, w.np);
    const dev::Planes XT[2] = {planes(w.xt[0], w.np, w.mp), planes(w.xt[1], w.np, w.mp)};
    const dev::Planes gram = planes(w.gram, w.mp, w.mp), prod = planes(w.product, w.mp, w.mp),
                      P = planes(w.poly[0], w.mp, w.mp), next = planes(w.poly[1], w.mp, w.mp),
                      both = planes(w.both, w.mp, w.mp);
    const uint32_t tiles = ((src.rows + 63) / 64) * ((src.cols + 63) / 64);
    const uint32_t parts = tiles < (uint32_t)dev::kNormParts ? tiles : dev::kNormParts;
    const uint32_t ts = w.tile.square, tx = w.tile.x, sq = w.mp / ts, mt = w.mp / tx, nt = w.np / tx;
    const uint32_t half = sq * (sq + 1) / 2, full = mt * nt;
    hipLaunchKernelGGL(dev::source_norm_kernel, dim3(parts, count), dim3(256), 0, st, src, norms);
    MG_HIP(hipGetLastError(), "newton-schulz norm launch");
    const bool tall = src.rows > src.cols;
    const bool hidden = fin.dst.type != MG_TYPE_FP32;
    // A 16-bit source fits the high halves: two products less for the first A, one for the
    // first X' (2048 x 8192: 1583 us without, 1457 with).
    bool exact = src.in.type != MG_TYPE_FP32 && !src.momentum.data && segment_steps(ns, w.m, w.n, ns.steps, hidden) < ns.steps;
    dev::MatrixScale* const scales = reinterpret_cast<dev::MatrixScale*>(base + w.scales);
    const dim3 tiles64((tall ? w.mp : w.np) / 64, (tall ? w.np : w.mp) / 64, count);
    if (exact)
        hipLaunchKernelGGL(dev::source_split_kernel<true>, tiles64, dim3(256), 0, st, src, norms, parts, ns.eps, scales, X, XT[0]);
    else
        hipLaunchKernelGGL(dev::source_split_kernel<false>, tiles64, dim3(256), 0, st, src, norms, parts, ns.eps, scales, X, XT[0]);
    MG_HIP(hipGetLastError(), "newton-schulz split launch");

    dev::ProductArgs p{};
    p.m = w.m, p.scales = scales;
    double growth = 1.0;  // extra_exp's
    // out = a b' of symmetric results
    auto symmetric = [&](const dev::Planes& a, const dev::Planes& b, uint32_t k, float unit_a, float unit_b,
                         const dev::Planes& out, float unit_out) -> int {
        p.a = a, p.b = b, p.stages = k / dev::kPK, p.tiles_j = sq, p.out = out;
        p.unit = unit_out / (unit_a * unit_b);
        p.growth = a.base == X.base ? (float)growth : 0.0f;
        if (a.base == X.base && exact)
            return launch_product<dev::kExactGram>(st, p, ts, half, count, "newton-schulz product launch");
        return launch_product<dev::kSymmetric>(st, p, ts, half, count, "newton-schulz product launch");
    };
    auto polynomial = [&](const dev::Planes& out) -> int {
        p.a = p.b = p.gram = gram, p.stages = w.mp / dev::kPK, p.tiles_j = sq, p.out = out;
        p.ca = ns.a * kUnitP, p.cb = ns.b * (kUnitP / kUnitA), p.cc = ns.c * (kUnitP / (kUnitA * kUnitA));
        return launch_product<dev::kPolynomial>(st, p, ts, half, count, "newton-schulz polynomial launch");
    };
    int rc, cur = 0;
    double reach = 1.0;
    for (uint32_t left = ns.steps; left;) {
        const uint32_t steps = segment_steps(ns, w.m, w.n, left, hidden);
        if ((rc = symmetric(X, X, w.np, kUnitX, kUnitX, gram, kUnitA))) return rc;
        float unit_q = kUnitP;
        double most_q = step_bounds(ns, &reach);
        if ((rc = polynomial(P))) return rc;
        if (steps == 2) {
            if ((rc = symmetric(P, gram, w.mp, kUnitP, kUnitA, prod, kUnitA)) ||
                (rc = symmetric(P, prod, w.mp, kUnitP, kUnitA, gram, kUnitA)) || (rc = polynomial(next)))
                return rc;
            most_q *= step_bounds(ns, &reach);
            unit_q = unit_of(most_q);
            if ((rc = symmetric(next, P, w.mp, kUnitP, kUnitP, both, unit_q))) return rc;
        }
        const dev::Planes& Q = steps == 2 ? both : P;
        left -= steps;
        p.a = Q, p.b = XT[cur], p.stages = w.mp / dev::kPK, p.tiles_j = nt;
        p.growth = (float)growth, growth *= most_q, p.growth_out = (float)growth;
        if (left) {
            p.out = X, p.out_t = XT[cur ^ 1], p.unit = 1.0f / unit_q;
            rc = exact ? launch_product<dev::kExactUpdate>(st, p, tx, full, count, "newton-schulz update launch")
                       : launch_product<dev::kUpdate>(st, p, tx, full, count, "newton-schulz update launch");
            if (rc) return rc;
            exact = false;  // X' is pairs
            cur ^= 1;
        } else {
            p.dst = fin.dst, p.step = fin.step, p.keep = fin.keep, p.rate = fin.rate, p.rows = src.rows, p.cols = src.cols;
            p.unit = 1.0f / (unit_q * kUnitX);
            if (tall) p.a = XT[cur], p.b = Q, p.tiles_j = mt;
            rc = tall ? launch_product<dev::kFinalTall>(st, p, tx, full, count, "newton-schulz result launch")
                      : launch_product<dev::kFinal>(st, p, tx, full, count, "newton-schulz result launch");
            if (rc) return rc;
        }
    }
    return MG_OK;
}

int newton_schulz(hipStream_t st, const mg_newton_schulz& ns, uint32_t count, const dev::SourceArgs& src,
                  const FinalArgs& fin, void* workspace) {
    if (is_short(src.rows, src.cols)) {
        const ShortWorkspace w(count, src.rows, src.cols);
        char* const base = static_cast<char*>(workspace);
        dev::ShortArgs a{};
        a.src = src, a.slabs = w.slabs, a.parts = w.parts;
        a.xt = reinterpret_cast<dev::f16*>(base + w.xt);
        float* const partial[2] = {reinterpret_cast<float*>(base + w.partial[0]), reinterpret_cast<float*>(base + w.partial[1])};
        a.state = reinterpret_cast<dev::ShortState*>(base + w.state);
        a.eps = ns.eps, a.a = ns.a, a.b = ns.b, a.c = ns.c;
        a.dst = fin.dst, a.step = fin.step, a.keep = fin.keep, a.rate = fin.rate, a.odd_rate = fin.odd_rate;
        return w.mp == 32   ? newton_schulz_short<32>(st, ns, count, a, partial)
               : w.mp == 64 ? newton_schulz_short<64>(st, ns, count, a, partial)
                            : newton_schulz_short<128>(st, ns, count, a, partial);
    }
    const Workspace w(count, src.rows, src.cols);
    return newton_schulz_tiled(st, ns, count, src, fin, w, workspace);
}

// The configuration's own checks; *ns receives the iteration.
int check_muon(const char* what, const mg_muon_config* c, mg_newton_schulz* ns) {
    MG_CHECK(c, MG_ERR_INVALID, "%s: null argument", what);
    auto fine = [](float x) { return x >= 0.0f && x < __builtin_huge_valf(); };
    MG_CHECK(fine(c->lr) && fine(c->weight_decay) && fine(c->scale), MG_ERR_INVALID,
             "%s: lr, weight_decay and scale must be finite and not negative", what);
    MG_CHECK(c->lr * c->weight_decay <= 1.0f, MG_ERR_INVALID, "%s: lr * weight_decay must be at most 1", what);
    MG_CHECK(fine(c->lr * fmaxf(c->scale, 256.0f)), MG_ERR_INVALID, "%s: lr * scale is out of range", what);  // 256: of 1 x 65536
    MG_CHECK(c->momentum >= 0.0f && c->momentum < 1.0f, MG_ERR_INVALID, "%s: momentum must be in [0, 1)", what);
    return check_ns(what, c->ns.steps ? &c->ns : nullptr, ns);
}
float muon_rate(const mg_muon_config& c, uint32_t rows, uint32_t cols) {
    return c.lr * (c.scale > 0.0f ? c.scale : cols > rows ? sqrtf((float)cols / (float)rows) : 1.0f);
}

int check_workspace(const char* what, uint32_t count, uint32_t rows, uint32_t cols, const void* workspace,
                    uint64_t bytes) {
    const uint64_t need = workspace_bytes_of(count, rows, cols);
    MG_CHECK(workspace && bytes >= need, MG_ERR_INVALID, "%s: the workspace needs %llu bytes", what,
             (unsigned long long)need);
    MG_CHECK(aligned(workspace, 256), MG_ERR_INVALID, "%s: the workspace is not 256-byte aligned", what);
    return MG_OK;
}

}  // namespace

int check_muon_config(const char* what, const mg_muon_config* config) {
    mg_newton_schulz ns;
    return check_muon(what, config, &ns);
}

size_t muon_blocks_bytes(const mg_policy_view& pv) {
    return ShortWorkspace(2 * pv.layers, MG_EMBED, pv.hidden).total;
}

float muon_blocks_reach(const mg_policy_view& pv, const mg_muon_config& c) {
    // an element of the result is at most its largest singular value; decay only shrinks
    return (float)kMostSingular * fmaxf(muon_rate(c, MG_EMBED, pv.hidden), muon_rate(c, pv.hidden, MG_EMBED));
}

int launch_muon_blocks(hipStream_t st, const mg_policy_view& pv, const mg_muon_config& c, const float* grad,
                       const float* normpart, float max_grad_norm, float* momentum, void* workspace) {
    mg_newton_schulz ns;
    if (int rc = check_muon("muon blocks", &c, &ns)) return rc;
    const uint32_t E = MG_EMBED, H = pv.hidden;
    auto batch = [&](const float* arena) {
        return dev::Batch{const_cast<float*>(arena) + pv.float_group, (size_t)E * H, H, MG_TYPE_FP32};
    };
    dev::SourceArgs src{};
    src.in = batch(grad), src.momentum = batch(momentum), src.rows = E, src.cols = H;
    src.beta = c.momentum, src.nesterov = c.nesterov != 0;
    src.blocks = 1, src.normpart = normpart, src.max_norm = max_grad_norm;
    const FinalArgs fin{batch(pv.params), 1, 1.0f - c.lr * c.weight_decay, muon_rate(c, E, H), muon_rate(c, H, E)};
    return newton_schulz(st, ns, 2 * pv.layers, src, fin, workspace);
}

}  // namespace mg

using namespace mg;

extern "C" {

int mg_orthogonalize_workspace(const mg_newton_schulz* in, uint32_t count, uint32_t rows, uint32_t cols,
                               uint64_t* bytes) {
    const char* what = "orthogonalize workspace";
    MG_CHECK(bytes, MG_ERR_INVALID, "orthogonalize workspace: null argument");
    mg_newton_schulz ns;
    int rc;
    if ((rc = check_ns(what, in, &ns)) || (rc = check_shape(what, count, rows, cols))) return rc;
    *bytes = count ? workspace_bytes_of(count, rows, cols) : 0;
    return MG_OK;
}

int mg_orthogonalize(void* stream, const mg_newton_schulz* in_ns, const mg_matrices* in, const mg_matrices* out,
                     void* workspace, uint64_t workspace_bytes) {
    const char* what = "orthogonalize";
    mg_newton_schulz ns;
    dev::SourceArgs src{};
    FinalArgs fin{};
    int rc;
    if ((rc = check_ns(what, in_ns, &ns)) || (rc = check_batch(what, "in", in, &src.in)) ||
        (rc = check_batch(what, "out", out, &fin.dst)) || (rc = check_same(what, in, out)))
        return rc;
    if (!in->count) return MG_OK;
    if ((rc = check_workspace(what, in->count, in->rows, in->cols, workspace, workspace_bytes))) return rc;
    src.rows = in->rows, src.cols = in->cols;
    hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice on;
    if ((rc = on.enter(st, "orthogonalize: stream device"))) return rc;
    return newton_schulz(st, ns, in->count, src, fin, workspace);
}

int mg_muon_step(void* stream, const mg_muon_config* c, const mg_matrices* params, const mg_matrices* momentum,
                 const mg_matrices* grad, void* workspace, uint64_t workspace_bytes) {
    const char* what = "muon step";
    mg_newton_schulz ns;
    dev::SourceArgs src{};
    FinalArgs fin{};
    int rc;
    if ((rc = check_muon(what, c, &ns)) ||
        (rc = check_batch(what, "params", params, &fin.dst)) ||
        (rc = check_batch(what, "momentum", momentum, &src.momentum)) ||
        (rc = check_batch(what, "grad", grad, &src.in)) || (rc = check_same(what, params, momentum)) ||
        (rc = check_same(what, params, grad)))
        return rc;
    MG_CHECK(momentum->type == MG_TYPE_FP32, MG_ERR_INVALID, "muon step: momentum must be fp32");
    if (!params->count) return MG_OK;
    if ((rc = check_workspace(what, params->count, params->rows, params->cols, workspace, workspace_bytes))) return rc;
    src.rows = params->rows, src.cols = params->cols;
    src.beta = c->momentum, src.nesterov = c->nesterov != 0;
    fin.step = 1;
    fin.keep = 1.0f - c->lr * c->weight_decay;
    fin.rate = muon_rate(*c, params->rows, params->cols);
    hipStream_t st = static_cast<hipStream_t>(stream);
    StreamDevice on;
    if ((rc = on.enter(st, "muon step: stream device"))) return rc;
    return newton_schulz(st, ns, params->count, src, fin, workspace);
}

}  // extern "C"
