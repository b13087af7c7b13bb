// The losses of a large vocabulary: what a call checks, its workspace and its
// launches (loss.hpp).
//
// Given logits: a row's partial sums, or, with the gradient, its whole row held
// in registers and read once.
//
// A head's product in 16-bit storage, value and gradient in one call: the logits
// in f32 in the workspace (kEpiZ), their 16-bit cotangent from whole rows, then
// dx and dw: three products of 2 rows model vocab flops.  Where those logits
// pass kKeepBytes, or a call is the value or the gradient alone: one pass of
// products over the whole vocabulary leaves the row sums (kEpiStats) and no
// logits; for the gradient one goes over it a piece at a time, the cotangent of
// a piece (kEpiP) entering dx, whose sum over the pieces stays in f32, and the
// piece's part of dw.  Together that is four products.  8192 x 4096 x 32000 in
// bf16, loss and gradients: 5.7 ms with the logits kept, 7.4 in two calls.
// The workspace of pieces: a piece's cotangent, 128 MiB or, of many rows, that of
// 256 columns; 12 bytes a row and column tile (256 columns, of few rows 128) of
// the whole vocabulary for the value's row sums; and with more than four slots a
// row 2 bytes a row and 64 columns for the lists of their blocks.  So it grows
// with the vocabulary, by an 85th to a 51st of what its f32 logits would take.
// In f32 the logits are products of gemm.hpp in the workspace, a piece at a
// time or all, and row kernels turn them into their cotangent in place.
#include "loss.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

namespace presk {

namespace {

int storage_code(const char* name) {
    const std::string t = name ? name : "";
    return t == "f32" ? kF32 : t == "bf16" ? kBF16 : t == "f16" ? kF16 : -1;
}

constexpr long long kMany = 1ll << 22;          // rows, model and a head's vocabulary stay below this
constexpr long long kPieceBytes = 128ll << 20;  // a piece's logits or their cotangent
constexpr long long kOnceBytes = 256ll << 20;   // f32 logits that are one piece: as many as the Infinity Cache holds, ...
constexpr long long kKeepBytes = 4ll << 30;     // ... and where the gradient follows the value, so that they stay for it
constexpr int kPieceCols = 256;                 // a piece is a multiple of these
// 16-bit storage: up to so many rows the cotangent enters dx and dw in two 16-bit
// parts, its rounding and what that left; past them its rounding alone, whose
// errors average (the gradients' whole error against that of f32 cotangents, whose
// outputs are rounded: 1.3 to 1.48 times it over 200 sizes of more rows; of fewer
// up to 2.1, 43 of 382 gradients over 1.5; in two parts 1.00).  The second part
// doubles two products: 8 x 4096 x 32000 in bf16, value and gradients, 205 us in
// one part and 245 in two; 65 rows 226 and 287; 8192 rows 5.33 and 8.57 ms.
constexpr int kFineRows = 64;

long long up(long long n, long long to) { return (n + to - 1) / to * to; }

// Tile and splits of a 16-bit product of M x N over K: 256 x 256 tiles where
// they come to three quarters of the CUs or more (2048 x 4096 x 32000 446 us, on
// 128 x 128 tiles 546), else 128 x 128: two workgroups a CU, or, where no CU
// has two of them anyway, one of eight waves with three blocks in flight (8 x 4096
// x 32000, 250 tiles, 58.7 -> 46.7 us with its weights partly in cache; 1024
// tiles of 4096 x 512 x 2048 76.8 us, deep 81.3).
struct Shape {
    int tile, tiles_m, tiles_n, splits;
};
Shape tiled(long long M, long long N, int tile) {
    const int n = tile == 256 ? 256 : 128;
    return Shape{tile, (int)(up(M, n) / n), (int)(up(N, n) / n), 1};
}
long long tiles_of(const Shape& s) { return (long long)s.tiles_m * s.tiles_n; }

Shape shape_of(long long M, long long N) {
    const Shape s = tiled(M, N, 256), t = tiled(M, N, 128);
    return tiles_of(s) >= 192 ? s : tiles_of(t) > 256 ? t : tiled(M, N, kDeep128);
}

// dx (Mx x Nx over Kx) and dw in one launch: their tiles are of one kind, and a K
// that is longer than a CU's share of the work is cut into shares of it, four
// 64-deep blocks at least.  The deep tiles where one round of the CUs holds
// every item (4096 x 512 x 2048 76.8 -> 69.2 us; 512 x 2048 x 8192, 1100 items,
// 98 us, deep 104); two a CU are kept to one round where fewer cuts do that
// (777 x 500 x 10007, 316 tiles of dw and 28 of dx cut 7 ways, 512 items and
// the mean, 105 us, 6 ways 89).  The few rows of a cotangent in two parts take no
// 256-row tiles (8 x 4096 x 32000, value and gradients, 264 -> 245 us).
constexpr int kBeside = 8;      // workgroups of the launch that are no item: the mean's, and dx's padding to 8
void pair_of(long long Mx, long long Nx, long long Kx, long long Mw, long long Nw, long long Kw, Shape* x, Shape* w) {
    const long long kx = up(Kx, 64) / 64, kw = up(Kw, 64) / 64;
    auto items = [&]() { return tiles_of(*x) * x->splits + tiles_of(*w) * w->splits; };
    auto both = [&](int tile, long long slots) {
        *x = tiled(Mx, Nx, tile);
        *w = tiled(Mw, Nw, tile);
        const double share = std::max((double)(tiles_of(*x) * kx + tiles_of(*w) * kw) / (double)slots, 1.0);
        auto cut = [&](long long k) {
            const long long n = (long long)((double)k / share + 0.5);
            return (int)std::max<long long>(1, std::min<long long>({n, k / 4, 64}));
        };
        x->splits = cut(kx);
        w->splits = cut(kw);
        for (Shape* s : {x, w}) {
            const long long over = items() - (slots - kBeside), t = std::max<long long>(tiles_of(*s), 1);
            const long long less = s->splits - (over + t - 1) / t;
            if (over > 0 && 2 * less > s->splits) s->splits = (int)less;
        }
        return tiles_of(*x) + tiles_of(*w);
    };
    if ((Mx == 0 || Mx > kFineRows) && both(256, 256) >= 192) return;
    both(kDeep128, 256);
    if (items() <= 256 - kBeside) return;
    both(128, 512);
}

// f32 logits: as many shares of K as leave no CU idle, their planes joined as
// they are read
Shape logits_of(long long M, long long N, long long K) {
    Shape s = shape_of(M, N);
    const long long nkb = up(K, 64) / 64;
    if (tiles_of(s) < 128) s.splits = (int)std::max<long long>(1, std::min<long long>({256 / tiles_of(s), nkb / 4, 8}));
    return s;
}

// A 16-bit piece's columns, at most `most`: the width whose tiles of the
// cotangent's product end nearest whole rounds of the CUs.
int piece_of(long long rows, long long V, long long most) {
    if (most >= V) return (int)up(V, kPieceCols);
    const long long rt = up(rows, 256) / 256, all = up(V, 256) / 256, top = most / 256;
    long long best = top;
    double cost = 1e300;
    for (long long c = top; c >= 1 && c * 2 > top; --c) {
        const long long n = all / c, rest = all - n * c;
        const double t = (double)(n * ((rt * c + 255) / 256) + (rest ? (rt * rest + 255) / 256 : 0)) + 0.25 * (double)(n + (rest > 0));
        if (t < cost) {
            cost = t;
            best = c;
        }
        if (top - c >= 255) break;
    }
    return (int)(best * 256);
}

struct Plan {
    bool head, value, grad;
    int st, esz, D, V, k, parts, slots, nblocks;
    long long rows, prows;
    float c, nat;                     // log2 e / T and 1 / T
    bool packx, packw;
    bool once, joint;                 // f32 logits of the whole vocabulary are kept; a row of them fits a workgroup's registers
    bool two;                         // the 16-bit cotangent is in two parts
    bool blocks, counted;             // the slots' blocks are listed (`start`); the rows are counted
    int Dp, piece, pieces, spiece;    // spiece: columns a pass of row sums takes at once
    long long ldz;
    Shape zs;                         // once
    size_t col, p, ent, start, count, most, lse, loss, top, sum, coef, scale, pm, ps, pa, xp, wp, P, z, acc, partx, partw, total;
};

GemmArgs product(long long M, long long N, long long K, long long sa_m, long long sa_k, long long sb_k, long long sb_n, long long sc_m) {
    GemmArgs g{};
    g.M = M;
    g.N = N;
    g.K = K;
    g.sa_m = sa_m;
    g.sa_k = sa_k;
    g.sb_k = sb_k;
    g.sb_n = sb_n;
    g.sc_m = sc_m;
    g.batch = 1;
    g.storage = kF32;
    g.a_kcontig = sa_k == 1;
    g.b_kcontig = sb_k == 1;
    gemm_plan(g);
    return g;
}
// the three products of an f32 piece of n columns
GemmArgs product_z(const Plan& q, bool tied, long long n) {
    return product(q.rows, n, q.D, q.D, 1, tied ? 1 : q.V, tied ? q.D : 1, q.ldz);
}
GemmArgs product_dx(const Plan& q, bool tied, long long n) {
    return product(q.rows, q.D, n, q.ldz, 1, tied ? q.D : 1, tied ? 1 : q.V, q.D);
}
GemmArgs product_dw(const Plan& q, bool tied, long long n) {
    return tied ? product(n, q.D, q.rows, 1, q.ldz, q.D, 1, q.D) : product(q.D, n, q.rows, 1, q.D, q.ldz, 1, q.V);
}

// the gradients' products of a 16-bit piece of n columns (one that is not
// asked for has no tiles)
void pair_shapes(const Plan& q, const presk_hip_loss& a, int n, Shape* x, Shape* w) {
    pair_of(a.dx ? q.rows : 0, q.D, up(n, 64) << q.two, !a.dw ? 0 : a.tied ? n : q.D, a.tied ? q.D : n, q.prows << q.two, x, w);
}

Plan plan_of(const presk_hip_loss& a, int what, bool head) {
    Plan q{};
    q.head = head;
    q.value = what & PRESK_HIP_LOSS_VALUE;
    q.grad = what & PRESK_HIP_LOSS_GRAD;
    q.st = storage_code(a.dtype);
    q.esz = q.st == kF32 ? 4 : 2;
    q.rows = a.rows;
    q.D = (int)a.model;
    q.V = (int)a.vocab;
    q.k = (int)std::max<int64_t>(a.top, 1);
    q.c = (float)(1.4426950408889634074 / a.temperature);
    q.nat = (float)(1.0 / a.temperature);
    // the counted rows' number is the mean's gradient's factor, their largest
    // cotangent f16's scale
    q.counted = a.top > 0 || (q.grad && (q.value || (head && q.st == kF16)));
    q.parts = q.counted ? loss_parts(q.rows, (int)a.top) : 0;
    size_t at = 0;
    auto take = [&](long long bytes) {
        const size_t was = at;
        at += (size_t)up(std::max<long long>(bytes, 0), 256);
        return was;
    };
    const bool half = head && q.st != kF32;
    q.once = half && q.rows && q.value && q.grad && 4 * q.rows * up(q.V, 4) <= kKeepBytes;
    q.prows = up(q.rows, 64);
    q.two = half && q.grad && q.rows <= kFineRows;
    q.nblocks = (int)(up(q.V, kCols) / kCols);
    q.col = take(4 * q.rows * a.top);
    q.p = take(4 * q.rows * a.top);
    q.ent = take(a.top ? 4 * q.rows : 0);
    q.blocks = half && q.k > 4 && !q.once;
    q.start = take(q.blocks ? 2 * q.rows * (q.nblocks + 1) : 0);
    q.count = take(4 * q.parts);
    q.most = take(4 * q.parts);
    q.lse = take(4 * q.rows);
    q.loss = take(4 * q.rows);
    q.top = take(q.value && q.grad ? 4 * q.rows : 0);
    q.sum = take(q.value && q.grad ? 4 * q.rows : 0);
    q.coef = take(q.grad ? 4 * q.rows : 0);
    q.scale = take(4);
    q.slots = 0;
    if (!q.rows) {
        q.total = at;
        return q;
    }
    if (head) {
        // one piece, or as wide as kPieceBytes allow (in f32 of equal width)
        const long long bytes = half ? 2 : 4;
        long long cols = kPieceBytes / (bytes * std::max<long long>(q.prows, 1)) / kPieceCols * kPieceCols;
        if (4 * q.rows * up(q.V, 4) <= (q.value && q.grad ? kKeepBytes : kOnceBytes)) cols = up(q.V, kPieceCols);
        if (q.st == kF32) cols = std::min(cols, ((1ll << 31) - 1) / std::max<long long>(q.rows, 1) / kPieceCols * kPieceCols);
        cols = std::min(std::max<long long>(cols, kPieceCols), up(q.V, kPieceCols));
        q.piece = half ? piece_of(q.rows, q.V, cols) : (int)up((q.V + up(q.V, cols) / cols - 1) / (up(q.V, cols) / cols), kPieceCols);
        q.pieces = (int)(up(q.V, q.piece) / q.piece);
    }
    if (half) {
        q.packx = q.D % 64 != 0;
        q.packw = (a.tied ? q.D : q.V) % 8 != 0;
        q.Dp = (int)up(q.D, 64);
        q.ldz = up(q.V, 4);
        if (q.once) {
            LossMatrix m{};
            m.storage = kF32;
            m.cols = q.V;
            q.joint = loss_joint_fits(m);
            if (!q.joint) q.slots = loss_chunks(q.rows, q.V);
            q.pieces = 1;
            q.piece = (int)up(q.V, kPieceCols);
        }
        q.spiece = q.packw ? q.piece : q.V;
        // (a launch stays below 2^32 threads)
        const long long rt = up(q.rows, 128) / 128;
        if (rt * (up(q.spiece, 128) / 128) > kMany)
            q.spiece = (int)std::max<long long>(kPieceCols, kMany / rt * 128 / kPieceCols * kPieceCols);
        for (long long v = 0; v < q.V && q.value && !q.once; v += q.spiece)
            q.slots += shape_of(q.rows, std::min<long long>(q.spiece, q.V - v)).tiles_n;
        q.xp = take(q.packx ? 2 * q.rows * q.Dp : 0);
        q.wp = take(!q.packw ? 0 : a.tied ? 2ll * q.piece * q.Dp : 2ll * q.D * up(q.piece, 64));
        if (q.once) {
            q.zs = q.joint ? logits_of(q.rows, q.V, q.D) : shape_of(q.rows, q.V);
            q.z = take(4ll * q.zs.splits * q.rows * q.ldz);
        }
        if (q.grad) {
            q.P = take((2 * q.prows * up(std::min<long long>(q.piece, q.V), 64)) << q.two);
            q.acc = take(a.dx && q.pieces > 1 ? 4 * q.rows * up(q.D, 4) : 0);
            long long px = 0, pw = 0;
            for (long long v = 0; v < q.V; v += q.piece) {
                Shape x, w;
                pair_shapes(q, a, (int)std::min<long long>(q.piece, q.V - v), &x, &w);
                if (a.dx && x.splits > 1) px = std::max(px, 4 * x.splits * q.rows * up(q.D, 4));
                const long long n = std::min<long long>(q.piece, q.V - v);
                if (a.dw && w.splits > 1) pw = std::max(pw, 4ll * w.splits * (a.tied ? n * up(q.D, 4) : q.D * up(n, 4)));
            }
            q.partx = take(px);
            q.partw = take(pw);
        }
    } else if (head) {
        q.ldz = up(std::min(q.piece, q.V), 4);
        q.P = take(4 * q.rows * q.ldz);
        long long part = 0;
        auto splits = [&](const GemmArgs& g) {
            if (g.splits > 1) part = std::max(part, 4ll * g.splits * g.M * g.N);
        };
        for (long long v = 0; v < q.V; v += q.piece) {
            const long long w = std::min<long long>(q.piece, q.V - v);
            splits(product_z(q, a.tied, w));
            if (q.grad && a.dx) splits(product_dx(q, a.tied, w));
            if (q.grad && a.dw) splits(product_dw(q, a.tied, w));
            if (q.value) q.slots += loss_chunks(q.rows, (int)w);
        }
        q.partx = take(part);
    } else if (q.value) {
        q.slots = loss_chunks(q.rows, q.V);
    }
    q.pm = take(4ll * q.slots * q.rows);
    q.ps = take(4ll * q.slots * q.rows);
    q.pa = take(4ll * q.slots * q.rows);
    q.total = at;
    return q;
}

#define LOSS_TRY(x)                                        \
    do {                                                   \
        if (hipError_t e_ = (x); e_ != hipSuccess) return e_; \
    } while (0)

struct Call {
    const presk_hip_loss& a;
    const Plan& q;
    hipStream_t s;
    char* w;
    LossTarget t;
    LossPrep prep;
    bool mean_done = false, beside = false;     // beside: given logits' sums are one launch with the targets

    template <typename T>
    T* at(size_t off) const { return (T*)(w + off); }

    hipError_t half_gemm(const LossGemm& g, LossEpi epi, int tile) const {
        return q.st == kBF16 ? loss_gemm_bf16(g, epi, a.tied, tile, s) : loss_gemm_f16(g, epi, a.tied, tile, s);
    }

    // What the products of columns [v0, v0 + n) take of x and w.
    struct Side {
        const unsigned short* p;
        long long stride;
        int rows, k;    // of w: columns and k that exist, as the logits' product sees them
    };
    bool x_packed = false;
    Side states() const {
        return q.packx ? Side{at<unsigned short>(q.xp), q.Dp, (int)q.rows, q.Dp}
                       : Side{(const unsigned short*)a.x, q.D, (int)q.rows, q.D};
    }
    // w's side of columns [v0, v0 + n); what has to be packed, x the first
    // time, is (w not where `held`)
    hipError_t weights(long long v0, int n, bool held, Side* o) {
        const unsigned short* const wt = (const unsigned short*)a.w + (a.tied ? v0 * q.D : v0);
        LossPack px{}, pw{};
        if (q.packx && !x_packed) px = LossPack{a.x, q.D, q.rows, q.D, at<void>(q.xp), q.Dp};
        x_packed = true;
        unsigned short* const dst = at<unsigned short>(q.wp);
        const int ld = (int)up(n, 64);
        if (!q.packw) *o = Side{wt, a.tied ? q.D : q.V, n, q.D};
        else if (a.tied) *o = Side{dst, q.Dp, n, q.Dp};
        else *o = Side{dst, ld, ld, q.D};
        if (q.packw && !held) pw = a.tied ? LossPack{wt, q.D, n, q.D, dst, q.Dp} : LossPack{wt, q.V, q.D, n, dst, ld};
        return loss_pack(px, pw, s);
    }
    LossGemm logits(const Side& x, const Side& w, long long v0, int n, const Shape& h) const {
        LossGemm g{};
        g.A = x.p;
        g.sa = x.stride;
        g.arows = (int)q.rows;
        g.ka = x.k;
        g.B = w.p;
        g.sb = w.stride;
        g.brows = w.rows;
        g.kb = w.k;
        g.M = (int)q.rows;
        g.N = n;
        g.K = q.D;
        g.tiles_m = h.tiles_m;
        g.tiles_n = h.tiles_n;
        g.splits = h.splits;
        g.c = q.c;
        g.t = t;
        g.col0 = (int)v0;
        g.cols = n;
        g.rows = q.rows;
        return g;
    }
    // dx and dw from columns [v, v + n)'s cotangent
    hipError_t pair(const Side& x, const Side& w, long long v, int n) {
        const long long pld = up(n, 64);
        Shape hx, hw;
        pair_shapes(q, a, n, &hx, &hw);
        unsigned short* const P = at<unsigned short>(q.P);
        LossGemm dx{}, dw{};
        for (LossGemm* g : {&dx, &dw}) {
            const Shape& h = g == &dx ? hx : hw;
            g->tiles_m = h.tiles_m;
            g->tiles_n = h.tiles_n;
            g->splits = h.splits;
            g->scale = at<float>(q.scale);
            g->flag = a.flag;
            g->two = q.two;
        }
        if (a.dx) {
            // dx[r][d] += sum over the piece of P[r][v] w(v, d); P is zero past the piece
            dx.A = P;
            dx.sa = pld;
            dx.arows = (int)q.rows;
            dx.ka = (int)pld;
            dx.B = w.p;
            dx.sb = w.stride;
            dx.brows = a.tied ? w.k : q.D;
            dx.kb = a.tied ? n : w.rows;
            dx.M = (int)q.rows;
            dx.N = q.D;
            dx.K = (int)pld;
            dx.acc = at<float>(q.acc);
            dx.a2 = 2 * q.prows * pld;
            dx.lda = up(q.D, 4);
            dx.acc_in = v > 0;
            dx.part = at<float>(q.partx);
            dx.C = v + n >= q.V ? a.dx : nullptr;
            dx.ldc = q.D;
        }
        if (a.dw) {
            const Side px{P, pld, (int)pld, (int)q.prows}, sx{x.p, x.stride, x.k, (int)q.rows};
            const Side& A = a.tied ? px : sx;
            const Side& B = a.tied ? sx : px;
            dw.A = A.p;
            dw.sa = A.stride;
            dw.arows = A.rows;
            dw.ka = A.k;
            dw.B = B.p;
            dw.sb = B.stride;
            dw.brows = B.rows;
            dw.kb = B.k;
            dw.M = a.tied ? n : q.D;
            dw.N = a.tied ? q.D : n;
            dw.K = (int)q.prows;
            (a.tied ? dw.a2 : dw.b2) = 2 * q.prows * pld;
            dw.lda = up(dw.N, 4);
            dw.part = at<float>(q.partw);
            dw.C = (unsigned short*)a.dw + (a.tied ? v * q.D : v);
            dw.ldc = a.tied ? q.D : q.V;
        }
        LossMean m{};
        if (q.value && a.mean && !mean_done) m = mean_args();
        mean_done = mean_done || m.loss;
        LOSS_TRY(q.st == kBF16 ? loss_pair_bf16(dx, dw, !a.tied, hx.tile, m, s) : loss_pair_f16(dx, dw, !a.tied, hx.tile, m, s));
        return loss_join(dx, dw, q.st, s);
    }

    hipError_t half(const float* lse) {
        const Side x = states();
        Side w;
        if (q.once) {
            // one piece: its logits in f32, their cotangent from whole rows
            LOSS_TRY(weights(0, q.V, false, &w));
            LossGemm g = logits(x, w, 0, q.V, q.zs);
            g.part = at<float>(q.z);
            g.lda = q.ldz;
            const LossPrep none{};
            const LossPrep& p = a.top ? none : prep;
            LOSS_TRY(q.st == kBF16 ? loss_logits_bf16(g, a.tied, q.zs.tile, p, s) : loss_logits_f16(g, a.tied, q.zs.tile, p, s));
            LossMatrix m = matrix(at<float>(q.z), q.ldz, kF32, 0, q.V);
            m.planes = q.zs.splits;
            m.plane = q.rows * q.ldz;
            const LossTo to{at<void>(q.P), q.st, up(q.V, 64), q.prows, q.two ? q.prows * up(q.V, 64) : 0};
            if (q.joint) {
                LossJoint j = joint_args(m, to);
                j.scale = at<float>(q.scale);
                j.flag = nullptr;
                LOSS_TRY(loss_joint(j, s));
            } else {
                LOSS_TRY(value_of(m, 0));
                LOSS_TRY(rows_of());
                LOSS_TRY(grad_of(m, lse, to, nullptr));
            }
            return pair(x, w, 0, q.V);
        }
        if (q.value) {
            int slot = 0;
            for (long long v = 0; v < q.V; v += q.spiece) {
                const int n = (int)std::min<long long>(q.spiece, q.V - v);
                LOSS_TRY(weights(v, n, false, &w));
                const Shape h = shape_of(q.rows, n);
                LossGemm g = logits(x, w, v, n, h);
                g.pm = at<float>(q.pm) + slot * q.rows;
                g.ps = at<float>(q.ps) + slot * q.rows;
                g.pa = at<float>(q.pa) + slot * q.rows;
                LOSS_TRY(half_gemm(g, kEpiStats, h.tile));
                slot += h.tiles_n;
            }
        }
        LOSS_TRY(rows_of());
        for (long long v = 0; v < q.V && q.grad; v += q.piece) {
            const int n = (int)std::min<long long>(q.piece, q.V - v);
            // (a vocabulary of one piece is packed already)
            LOSS_TRY(weights(v, n, q.value && q.pieces == 1 && q.spiece >= q.V, &w));
            const Shape h = shape_of(q.rows, n);
            LossGemm g = logits(x, w, v, n, h);
            g.lse = lse;
            g.coef = at<float>(q.coef);
            g.P = at<unsigned short>(q.P);
            g.pld = up(n, 64);
            g.plow = q.two ? q.prows * g.pld : 0;
            g.prows = (int)q.prows;
            LOSS_TRY(half_gemm(g, kEpiP, h.tile));
            LOSS_TRY(pair(x, w, v, n));
        }
        return hipSuccess;
    }

    hipError_t gemm(GemmArgs g, const float* A, const float* B, float* C, const float* bias) const {
        g.A = A;
        g.B = B;
        g.C = C;
        g.bias = bias;
        g.bias_kind = bias ? 2 : 0;
        g.work = at<float>(q.partx);
        gemm_align(g);
        return gemm_launch(g, s);
    }
    LossMatrix matrix(const void* z, long long ld, int storage, long long v0, int n) const {
        LossMatrix m{};
        m.z = z;
        m.ld = ld;
        m.storage = storage;
        m.rows = q.rows;
        m.col0 = (int)v0;
        m.cols = n;
        m.c = q.c;
        m.nat = q.nat;
        m.t = t;
        m.planes = 1;
        return m;
    }
    LossJoint joint_args(const LossMatrix& m, const LossTo& to) const {
        LossJoint j{};
        j.m = m;
        j.temperature = (float)a.temperature;
        j.lse = a.lse;
        j.loss = loss_out();
        j.ct = a.ct;
        j.count = at<int>(q.count);
        j.most = at<float>(q.most);
        j.parts = q.parts;
        j.to = to;
        j.flag = a.flag;
        return j;
    }
    // the value of logits in memory, as far as the rows' sums: whole where one
    // chunk has each row
    hipError_t value_of(const LossMatrix& m, int slot) const {
        const LossDone d{(float)a.temperature, lse_out(), loss_out(), top_out(), sum_out()};
        return loss_stats(m, at<float>(q.pm), at<float>(q.ps), at<float>(q.pa), slot, q.slots == 1 ? &d : nullptr, s);
    }
    // the cotangent of logits in memory, from what this call kept of their rows
    // or, of a gradient alone, from the forward's lse
    hipError_t grad_of(const LossMatrix& m, const float* lse, const LossTo& to, unsigned* flag) const {
        return loss_grad(m, top_out(), q.value ? sum_out() : lse, at<float>(q.coef), to, flag, s);
    }
    hipError_t single(const float* lse) {
        const float* const x = (const float*)a.x;
        float* const z = at<float>(q.P);
        // Splits of a product whose logits are read once are added there (256 x
        // 384 x 65: 21.4 us of four kernels, 18.2 of three).
        auto logits = [&](long long v, int n, bool planes, LossMatrix* m) {
            GemmArgs g = product_z(q, a.tied, n);
            *m = matrix(z, q.ldz, kF32, v, n);
            if (planes && g.splits > 1) {
                g.planes = true;
                m->z = at<float>(q.partx);
                m->ld = n;
                m->planes = g.splits;
                m->plane = q.rows * n;
            }
            return gemm(g, x, (const float*)a.w + (a.tied ? v * q.D : v), z, nullptr);
        };
        // a vocabulary of one piece: its logits, then their cotangent in place
        LossMatrix m = matrix(z, q.ldz, kF32, 0, q.V);
        const LossTo to{z, kF32, q.ldz, q.rows};
        const bool once = q.value && q.grad && q.pieces == 1 && loss_joint_fits(m);
        if (once) {
            LOSS_TRY(logits(0, q.V, true, &m));
            LOSS_TRY(loss_joint(joint_args(m, to), s));
        } else {
            int slot = 0;
            for (long long v = 0; v < q.V && q.value; v += q.piece) {
                const int n = (int)std::min<long long>(q.piece, q.V - v);
                LOSS_TRY(logits(v, n, !q.grad, &m));
                LOSS_TRY(value_of(m, slot));
                slot += loss_chunks(q.rows, n);
            }
            LOSS_TRY(rows_of());
        }
        for (long long v = 0; v < q.V && q.grad; v += q.piece) {
            const int n = (int)std::min<long long>(q.piece, q.V - v);
            if (!once) {
                if (!q.value || q.pieces > 1) LOSS_TRY(logits(v, n, false, &m));
                LOSS_TRY(grad_of(m, lse, to, nullptr));
            }
            float* const dx = (float*)a.dx;
            if (dx)
                LOSS_TRY(gemm(product_dx(q, a.tied, n), z, (const float*)a.w + (a.tied ? v * q.D : v), dx, v ? dx : nullptr));
            if (a.dw) {
                float* const dw = (float*)a.dw + (a.tied ? v * q.D : v);
                LOSS_TRY(gemm(product_dw(q, a.tied, n), a.tied ? z : x, a.tied ? x : z, dw, nullptr));
            }
        }
        return hipSuccess;
    }

    hipError_t given(const float* lse) {
        LossMatrix m = matrix(a.x, q.V, q.st, 0, q.V);
        const LossTo to{a.dx, q.st, q.V, q.rows};
        if (q.value && q.grad && loss_joint_fits(m)) return loss_joint(joint_args(m, to), s);
        if (beside) {
            LOSS_TRY(loss_stats_beside(m, at<float>(q.pm), at<float>(q.ps), prep, s));
            return rows_of(m);
        }
        // (the targets of a row in several chunks are looked up once those are joined)
        LossMatrix sums = m;
        if (q.slots > 1) sums.t.k = 0;
        if (q.value) LOSS_TRY(value_of(sums, 0));
        LOSS_TRY(rows_of(q.slots > 1 ? m : LossMatrix{}));
        if (!q.grad) return hipSuccess;
        return grad_of(m, lse, to, a.flag);
    }

    LossMean mean_args() const { return LossMean{loss_out(), q.rows, at<int>(q.count), q.parts, t.index, a.mean}; }
    float* lse_out() const { return a.lse ? a.lse : at<float>(q.lse); }
    float* loss_out() const { return a.loss ? a.loss : at<float>(q.loss); }
    float* top_out() const { return q.value && q.grad ? at<float>(q.top) : nullptr; }
    float* sum_out() const { return q.value && q.grad ? at<float>(q.sum) : nullptr; }
    LossRows row_args() const {
        LossRows r{};
        r.pm = at<float>(q.pm);
        r.ps = at<float>(q.ps);
        r.pa = at<float>(q.pa);
        // (one chunk of logits in memory: the rows are done)
        r.slots = q.slots == 1 && (!q.head || q.st == kF32 || q.once) ? 0 : q.slots;
        // (kEpiStats leaves its sums in log 2, the row kernels in the logits' units)
        const bool scaled = q.head && q.st != kF32 && !q.once;
        r.unit = scaled ? 1.f : q.c;
        r.nat = scaled ? kLn2 : q.nat;
        r.t = t;
        r.rows = q.rows;
        r.temperature = (float)a.temperature;
        if (q.value) {
            r.lse = lse_out();
            r.loss = loss_out();
            r.top = top_out();
            r.sum = sum_out();
            if (loss_rows_mean(q.rows)) r.mean = a.mean;
        }
        if (q.grad) {
            r.coef = at<float>(q.coef);
            r.ct = a.ct;
            r.mean_in = !a.ct && !q.value ? a.mean : nullptr;
            r.scale = q.head && q.st != kF32 ? at<float>(q.scale) : nullptr;
            r.shift = q.st == kF16;
        }
        r.count = at<int>(q.count);
        r.most = at<float>(q.most);
        r.parts = q.parts;
        return r;
    }
    // the rows' sums joined, their cotangents' factors, and of few rows the mean
    hipError_t rows_of(const LossMatrix& late = LossMatrix{}) {
        LossRows r = row_args();
        r.z = late;
        if (late.z) r.slots = q.slots;
        if (!r.slots && !r.coef && !r.mean) return hipSuccess;
        mean_done = r.mean;
        return loss_rows(r, s);
    }

    hipError_t run() {
        LossPrep& p = prep;
        p.index = (const long long*)a.index;
        p.teacher = a.teacher;
        p.ct = q.grad ? a.ct : nullptr;
        p.storage = q.st;
        p.rows = q.rows;
        p.vocab = q.V;
        p.top = (int)a.top;
        p.c = q.c;
        p.col = at<int>(q.col);
        p.p = at<float>(q.p);
        p.ent = at<float>(q.ent);
        p.start = q.blocks ? at<unsigned short>(q.start) : nullptr;
        p.nblocks = q.nblocks;
        p.count = at<int>(q.count);
        p.most = at<float>(q.most);
        p.parts = q.parts;
        t = LossTarget{a.top ? nullptr : p.index, q.V, p.col, p.p, p.ent, p.start, q.k, q.nblocks};
        if (q.rows) {
            // (counts alone are taken beside the logits where those are one launch)
            beside = !q.head && !q.grad && loss_beside(matrix(a.x, q.V, q.st, 0, q.V), p.top);
            if (q.counted && (a.top || !q.once) && !beside) LOSS_TRY(loss_prep(p, s));
            const float* const lse = lse_out();
            LOSS_TRY(!q.head ? given(lse) : q.st == kF32 ? single(lse) : half(lse));
        } else if (q.grad && q.head && a.dw) {
            LOSS_TRY(loss_zero(a.dw, (long long)q.D * q.V * q.esz, s));
        }
        if (q.value && a.mean && !mean_done) LOSS_TRY(loss_mean(mean_args(), s));
        return hipSuccess;
    }
};

}  // namespace

std::string loss_check(const presk_hip_loss& a, int what, bool head) {
    const int st = storage_code(a.dtype);
    const char* const op = head ? "head loss" : "distillation";
    auto no = [&](const std::string& why) { return std::string("E10001: ") + op + ": " + why; };
    if (st < 0) return std::string("E7005: ") + op + " in storage type `" + (a.dtype ? a.dtype : "") + "` (f32, bf16 or f16)";
    if (what < 1 || what > 3) return no("what is neither VALUE nor GRAD nor both");
    if (a.rows < 0 || a.rows >= kMany) return no("rows " + std::to_string(a.rows) + " not in [0, 2^22)");
    if (head ? a.model < 1 || a.model >= kMany : a.model != 0)
        return no("model " + std::to_string(a.model) + (head ? " not in [1, 2^22)" : ", which is 0 where the logits are given"));
    if (a.vocab < 1 || a.vocab >= (head ? kMany : 1ll << 30))
        return no("vocab " + std::to_string(a.vocab) + (head ? " not in [1, 2^22)" : " not in [1, 2^30)"));
    if (a.top < (head ? 0 : 1) || a.top > 1024) return no("top " + std::to_string(a.top) + (head ? " not in [0, 1024]" : " not in [1, 1024]"));
    if (!(a.temperature >= 1e-3 && a.temperature <= 1e3)) return no("a temperature of " + std::to_string(a.temperature) + ", not in [0.001, 1000]");
    if (a.top == 0 && a.temperature != 1.0) return no("a temperature without a teacher");
    if (head && st == kF32 && (a.rows * a.model >= 1ll << 31 || a.model * a.vocab >= 1ll << 31))
        return no("rows * model or model * vocab not below 2^31 in f32");
    return "";
}

namespace {

// The buffers of a checked call: their presence, alignment, and that no output
// meets another buffer.
std::string check_buffers(const presk_hip_loss& a, int what, bool head, size_t need) {
    const int st = storage_code(a.dtype);
    const char* const op = head ? "head loss" : "distillation";
    auto no = [&](const std::string& why) { return std::string("E10001: ") + op + ": " + why; };
    const bool value = what & PRESK_HIP_LOSS_VALUE, grad = what & PRESK_HIP_LOSS_GRAD;
    const auto spans = loss_buffers(a, what, head);
    if (!head && (a.w || a.dw)) return no("w or dw where the logits are given");
    for (const LossBuffer& s : spans) {
        if (s.need && s.bytes > 0 && !s.p) return no(std::string(s.name) + " is null");
        if ((uintptr_t)s.p % s.align) return no(std::string(s.name) + " is not aligned to " + std::to_string(s.align) + " bytes");
    }
    if (value && !grad && !a.loss && !a.lse && !a.mean) return no("a value without an output");
    if (grad && !a.dx && !a.dw) return no("a gradient without an output");
    if (head && st != kF32) {
        // operands that are read where they are, in vectors of 16 bytes
        if (a.model % 64 == 0 && (uintptr_t)a.x % 16) return no("x is not aligned to 16 bytes");
        if ((a.tied ? a.model : a.vocab) % 8 == 0 && (uintptr_t)a.w % 16) return no("w is not aligned to 16 bytes");
    }
    for (const LossBuffer& s : spans)
        for (const LossBuffer& o : spans)
            if (&s != &o && o.out && s.p && o.p && s.bytes > 0 && o.bytes > 0 && (uintptr_t)s.p < (uintptr_t)o.p + o.bytes &&
                (uintptr_t)o.p < (uintptr_t)s.p + s.bytes)
                return no(std::string(o.name) + " meets " + s.name);
    if (a.work_bytes < need) return no("a workspace of " + std::to_string(a.work_bytes) + " bytes, " + std::to_string(need) + " needed");
    return "";
}

size_t bytes_of(const Plan& q) { return std::max<size_t>(q.total, 256); }

}  // namespace

size_t loss_workspace(const presk_hip_loss& a, int what, bool head) { return bytes_of(plan_of(a, what, head)); }

std::string loss_check_all(const presk_hip_loss& a, int what, bool head) {
    std::string why = loss_check(a, what, head);
    return why.empty() ? check_buffers(a, what, head, loss_workspace(a, what, head)) : why;
}

hipError_t loss_run(const presk_hip_loss& a, int what, bool head, hipStream_t s) {
    const Plan q = plan_of(a, what, head);
    Call c{a, q, s, (char*)a.work, {}, {}};
    return c.run();
}

hipError_t loss_check_run(const presk_hip_loss& a, int what, bool head, hipStream_t s, std::string* why) {
    *why = loss_check(a, what, head);
    if (!why->empty()) return hipSuccess;
    const Plan q = plan_of(a, what, head);
    *why = check_buffers(a, what, head, bytes_of(q));
    if (!why->empty()) return hipSuccess;
    Call c{a, q, s, (char*)a.work, {}, {}};
    return c.run();
}

}  // namespace presk
