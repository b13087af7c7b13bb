// The losses of a large vocabulary: what a call checks, its workspace and its
// launches (loss.hpp).
//
// Given logits: a row's partial sums, or, with the gradient, its whole row held
// in registers and read once.
//
// A head's product in 16-bit storage: one pass of products over the whole
// vocabulary leaves the row sums (kEpiStats); for the gradient a second one goes
// over it a piece at a time, the cotangent of a piece (kEpiP, 16 bits) entering
// dx, whose sum over the pieces stays in f32, and the piece's part of dw.  That
// is four products of 2 rows model vocab flops where keeping the logits takes
// three, and a workspace that does not grow with the vocabulary.  In f32 the
// pieces' logits are products of gemm.hpp in the workspace, and row kernels
// turn them into their cotangent in place.
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
constexpr int kPieceCols = 256;                 // a piece is a multiple of these

long long up(long long n, long long to) { return (n + to - 1) / to * to; }

// Tile and splits of a 16-bit product of M x N over K.
struct Shape {
    int tile, tiles_m, tiles_n, splits;
};
Shape shape_of(long long M, long long N, long long K, bool split) {
    Shape s{};
    const long long big = up(M, 256) / 256 * (up(N, 256) / 256);
    s.tile = big >= 192 ? 256 : 128;
    s.tiles_m = (int)(up(M, s.tile) / s.tile);
    s.tiles_n = (int)(up(N, s.tile) / s.tile);
    s.splits = 1;
    const long long t = (long long)s.tiles_m * s.tiles_n, nkb = up(K, 64) / 64;
    if (split && t < 256) s.splits = (int)std::max<long long>(1, std::min<long long>({512 / t, nkb / 4, 64}));
    return s;
}

struct Plan {
    bool head, value, grad;
    int st, esz, D, V, k, parts, slots, nblocks;
    long long rows, prows;
    float c;
    bool packx, packw;
    int Dp, piece, pieces, spiece;    // spiece: columns a pass of row sums takes at once
    long long ldz;
    size_t col, p, ent, start, count, most, lse, loss, coef, scale, pm, ps, pa, xp, wp, P, acc, part, total;
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
    q.parts = loss_parts(q.rows, (int)a.top);
    size_t at = 0;
    auto take = [&](long long bytes) {
        const size_t was = at;
        at += (size_t)up(std::max<long long>(bytes, 0), 256);
        return was;
    };
    const bool half = head && q.st != kF32;
    q.prows = up(q.rows, 64);
    q.nblocks = (int)(up(q.V, kCols) / kCols);
    q.col = take(4 * q.rows * q.k);
    q.p = take(4 * q.rows * q.k);
    q.ent = take(4 * q.rows);
    q.start = take(half && q.k > 4 ? 2 * q.rows * (q.nblocks + 1) : 0);
    q.count = take(4 * q.parts);
    q.most = take(4 * q.parts);
    q.lse = take(4 * q.rows);
    q.loss = take(4 * q.rows);
    q.coef = take(q.grad ? 4 * q.rows : 0);
    q.scale = take(4);
    q.slots = 0;
    if (!q.rows) {
        q.total = at;
        return q;
    }
    if (head) {
        // pieces of equal width, as wide as kPieceBytes allow
        const long long bytes = half ? 2 : 4;
        long long cols = kPieceBytes / (bytes * std::max<long long>(q.prows, 1)) / kPieceCols * kPieceCols;
        if (q.st == kF32) cols = std::min(cols, ((1ll << 31) - 1) / std::max<long long>(q.rows, 1) / kPieceCols * kPieceCols);
        cols = std::min(std::max<long long>(cols, kPieceCols), up(q.V, kPieceCols));
        q.pieces = (int)(up(q.V, cols) / cols);
        q.piece = (int)up((q.V + q.pieces - 1) / q.pieces, kPieceCols);
        q.pieces = (int)(up(q.V, q.piece) / q.piece);
    }
    if (half) {
        q.packx = q.D % 64 != 0;
        q.packw = (a.tied ? q.D : q.V) % 8 != 0;
        q.Dp = (int)up(q.D, 64);
        q.spiece = q.V;
        if (q.packw) q.spiece = q.piece;
        // (a launch stays below 2^32 threads)
        const long long rt = up(q.rows, 128) / 128;
        if (rt * (up(q.spiece, 128) / 128) > kMany)
            q.spiece = (int)std::max<long long>(kPieceCols, kMany / rt * 128 / kPieceCols * kPieceCols);
        q.slots = 0;
        for (long long v = 0; v < q.V && q.value; v += q.spiece)
            q.slots += shape_of(q.rows, std::min<long long>(q.spiece, q.V - v), q.D, false).tiles_n;
        q.xp = take(q.packx ? 2 * q.rows * q.Dp : 0);
        q.wp = take(!q.packw ? 0 : a.tied ? 2ll * q.piece * q.Dp : 2ll * q.D * up(q.piece, 64));
        if (q.grad) {
            const long long n = std::min<long long>(q.piece, q.V), pld = up(n, 64);
            q.P = take(2 * q.prows * pld);
            q.acc = take(a.dx && q.pieces > 1 ? 4 * q.rows * q.D : 0);
            long long part = 0;
            for (long long v = 0; v < q.V; v += q.piece) {
                const long long w = std::min<long long>(q.piece, q.V - v);
                const Shape x = shape_of(q.rows, q.D, up(w, 64), true);
                const Shape y = shape_of(a.tied ? w : q.D, a.tied ? q.D : w, q.prows, true);
                if (a.dx && x.splits > 1) part = std::max(part, 4 * x.splits * q.rows * q.D);
                if (a.dw && y.splits > 1) part = std::max(part, 4ll * y.splits * q.D * w);
            }
            q.part = take(part);
        }
    } else if (head) {
        q.ldz = up(std::min(q.piece, q.V), 4);
        const long long n = std::min<long long>(q.piece, q.V);
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
        q.part = take(part);
        (void)n;
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
    bool mean_done = false;

    template <typename T>
    T* at(size_t off) const { return (T*)(w + off); }

    hipError_t half_gemm(const LossGemm& g, LossEpi epi, bool akc, bool bkc, int tile) const {
        return q.st == kBF16 ? loss_gemm_bf16(g, epi, akc, bkc, tile, s) : loss_gemm_f16(g, epi, akc, bkc, tile, s);
    }

    // What the products of columns [v0, v0 + n) take of x and w.
    struct Side {
        const unsigned short* p;
        long long stride;
        int rows, k;    // of w: columns and k that exist, as the logits' product sees them
    };
    hipError_t weights(long long v0, int n, bool pack, Side* o) const {
        const unsigned short* const wt = (const unsigned short*)a.w + (a.tied ? v0 * q.D : v0);
        if (!q.packw) {
            *o = Side{wt, a.tied ? q.D : q.V, n, q.D};
            return hipSuccess;
        }
        unsigned short* const dst = at<unsigned short>(q.wp);
        if (a.tied) {
            *o = Side{dst, q.Dp, n, q.Dp};
            return pack ? loss_pack(wt, q.D, n, q.D, dst, q.Dp, s) : hipSuccess;
        }
        const int ld = (int)up(n, 64);
        *o = Side{dst, ld, ld, q.D};
        return pack ? loss_pack(wt, q.V, q.D, n, dst, ld, s) : hipSuccess;
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
        g.splits = 1;
        g.c = q.c;
        g.t = t;
        g.col0 = (int)v0;
        g.cols = n;
        g.rows = q.rows;
        return g;
    }
    hipError_t out(LossGemm g, const Shape& h, bool akc, bool bkc) const {
        g.tiles_m = h.tiles_m;
        g.tiles_n = h.tiles_n;
        g.splits = h.splits;
        g.part = at<float>(q.part);
        g.scale = q.st == kF16 ? at<float>(q.scale) : nullptr;
        g.flag = a.flag;
        LOSS_TRY(half_gemm(g, kEpiOut, akc, bkc, h.tile));
        return h.splits > 1 ? loss_join(g, q.st, s) : hipSuccess;
    }

    hipError_t half(const float* lse) {
        Side x{(const unsigned short*)a.x, q.D, (int)q.rows, q.D};
        if (q.packx) {
            LOSS_TRY(loss_pack(a.x, q.D, q.rows, q.D, at<void>(q.xp), q.Dp, s));
            x = Side{at<unsigned short>(q.xp), q.Dp, (int)q.rows, q.Dp};
        }
        Side w;
        if (q.value) {
            int slot = 0;
            for (long long v = 0; v < q.V; v += q.spiece) {
                const int n = (int)std::min<long long>(q.spiece, q.V - v);
                LOSS_TRY(weights(v, n, true, &w));
                const Shape h = shape_of(q.rows, n, q.D, false);
                LossGemm g = logits(x, w, v, n, h);
                g.pm = at<float>(q.pm) + slot * q.rows;
                g.ps = at<float>(q.ps) + slot * q.rows;
                g.pa = at<float>(q.pa) + slot * q.rows;
                LOSS_TRY(half_gemm(g, kEpiStats, true, a.tied, h.tile));
                slot += h.tiles_n;
            }
        }
        LOSS_TRY(rows_of());
        for (long long v = 0; v < q.V && q.grad; v += q.piece) {
            const int n = (int)std::min<long long>(q.piece, q.V - v);
            const long long pld = up(n, 64);
            // (a vocabulary of one piece is packed already)
            LOSS_TRY(weights(v, n, !(q.value && q.pieces == 1 && q.spiece >= q.V), &w));
            const Shape h = shape_of(q.rows, n, q.D, false);
            LossGemm g = logits(x, w, v, n, h);
            g.lse = lse;
            g.coef = at<float>(q.coef);
            g.P = at<unsigned short>(q.P);
            g.pld = pld;
            g.prows = (int)q.prows;
            LOSS_TRY(half_gemm(g, kEpiP, true, a.tied, h.tile));
            if (a.dx) {
                // dx[r][d] += sum over the piece of P[r][v] w(v, d); P is zero past the piece
                LossGemm d{};
                d.A = g.P;
                d.sa = pld;
                d.arows = (int)q.rows;
                d.ka = (int)pld;
                d.B = w.p;
                d.sb = w.stride;
                d.brows = a.tied ? w.k : q.D;       // d
                d.kb = a.tied ? n : w.rows;         // v
                d.M = (int)q.rows;
                d.N = q.D;
                d.K = (int)pld;
                d.acc = at<float>(q.acc);
                d.acc_in = v > 0;
                const bool last = v + n >= q.V;
                d.C = last ? a.dx : nullptr;
                d.ldc = q.D;
                LOSS_TRY(out(d, shape_of(q.rows, q.D, pld, true), true, !a.tied));
            }
            if (a.dw) {
                LossGemm d{};
                const Side px{g.P, pld, (int)pld, (int)q.prows}, sx{x.p, x.stride, x.k, (int)q.rows};
                const Side& A = a.tied ? px : sx;
                const Side& B = a.tied ? sx : px;
                d.A = A.p;
                d.sa = A.stride;
                d.arows = A.rows;
                d.ka = A.k;
                d.B = B.p;
                d.sb = B.stride;
                d.brows = B.rows;
                d.kb = B.k;
                d.M = a.tied ? n : q.D;
                d.N = a.tied ? q.D : n;
                d.K = (int)q.prows;
                d.C = (unsigned short*)a.dw + (a.tied ? v * q.D : v);
                d.ldc = a.tied ? q.D : q.V;
                LOSS_TRY(out(d, shape_of(d.M, d.N, q.prows, true), false, false));
            }
        }
        return hipSuccess;
    }

    hipError_t gemm(GemmArgs g, const float* A, const float* B, float* C, const float* bias) const {
        g.A = A;
        g.B = B;
        g.C = C;
        g.bias = bias;
        g.bias_kind = bias ? 2 : 0;
        g.work = at<float>(q.part);
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
        m.t = t;
        return m;
    }
    LossJoint joint_args(const LossMatrix& m, void* out, long long ldo) const {
        LossJoint j{};
        j.m = m;
        j.temperature = (float)a.temperature;
        j.lse = a.lse;
        j.loss = loss_out();
        j.ct = a.ct;
        j.count = at<int>(q.count);
        j.parts = q.parts;
        j.out = out;
        j.ldo = ldo;
        j.flag = a.flag;
        return j;
    }
    // the value of logits in memory, as far as the rows' sums: whole where one
    // chunk has each row
    hipError_t value_of(const LossMatrix& m, int slot) const {
        const LossDone d{(float)a.temperature, lse_out(), loss_out()};
        return loss_stats(m, at<float>(q.pm), at<float>(q.ps), at<float>(q.pa), slot, q.slots == 1 ? &d : nullptr, s);
    }
    hipError_t single(const float* lse) {
        const float* const x = (const float*)a.x;
        float* const z = at<float>(q.P);
        auto logits = [&](long long v, int n) {
            return gemm(product_z(q, a.tied, n), x, (const float*)a.w + (a.tied ? v * q.D : v), z, nullptr);
        };
        // a vocabulary of one piece: its logits, then their cotangent in place
        const LossMatrix whole = matrix(z, q.ldz, kF32, 0, q.V);
        const bool once = q.value && q.grad && q.pieces == 1 && loss_joint_fits(whole);
        if (once) {
            LOSS_TRY(logits(0, q.V));
            LOSS_TRY(loss_joint(joint_args(whole, z, q.ldz), s));
        } else {
            int slot = 0;
            for (long long v = 0; v < q.V && q.value; v += q.piece) {
                const int n = (int)std::min<long long>(q.piece, q.V - v);
                LOSS_TRY(logits(v, n));
                LOSS_TRY(value_of(matrix(z, q.ldz, kF32, v, n), slot));
                slot += loss_chunks(q.rows, n);
            }
            LOSS_TRY(rows_of());
        }
        for (long long v = 0; v < q.V && q.grad; v += q.piece) {
            const int n = (int)std::min<long long>(q.piece, q.V - v);
            if (!once) {
                LOSS_TRY(logits(v, n));
                LOSS_TRY(loss_grad(matrix(z, q.ldz, kF32, v, n), lse, at<float>(q.coef), z, q.ldz, nullptr, s));
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
        if (q.value && q.grad && loss_joint_fits(m)) return loss_joint(joint_args(m, a.dx, q.V), s);
        if (q.value) LOSS_TRY(value_of(m, 0));
        LOSS_TRY(rows_of());
        if (!q.grad) return hipSuccess;
        return loss_grad(m, lse, at<float>(q.coef), a.dx, q.V, a.flag, s);
    }

    float* lse_out() const { return a.lse ? a.lse : at<float>(q.lse); }
    float* loss_out() const { return a.loss ? a.loss : at<float>(q.loss); }
    LossRows row_args() const {
        LossRows r{};
        r.pm = at<float>(q.pm);
        r.ps = at<float>(q.ps);
        r.pa = at<float>(q.pa);
        // (one chunk of logits in memory: the rows are done)
        r.slots = q.slots == 1 && (!q.head || q.st == kF32) ? 0 : q.slots;
        r.t = t;
        r.rows = q.rows;
        r.temperature = (float)a.temperature;
        if (q.value) {
            r.lse = lse_out();
            r.loss = loss_out();
            if (loss_rows_mean(q.rows)) r.mean = a.mean;
        }
        if (q.grad) {
            r.coef = at<float>(q.coef);
            r.ct = a.ct;
            r.mean_in = !a.ct && !q.value ? a.mean : nullptr;
            r.scale = q.head && q.st == kF16 ? at<float>(q.scale) : nullptr;
        }
        r.count = at<int>(q.count);
        r.most = at<float>(q.most);
        r.parts = q.parts;
        return r;
    }
    // the rows' sums joined, their cotangents' factors, and of few rows the mean
    hipError_t rows_of() {
        const LossRows r = row_args();
        if (!r.slots && !r.coef && !r.mean) return hipSuccess;
        mean_done = r.mean;
        return loss_rows(r, s);
    }

    hipError_t run() {
        LossPrep p{};
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
        p.start = q.head && q.st != kF32 && q.k > 4 ? at<unsigned short>(q.start) : nullptr;
        p.nblocks = q.nblocks;
        p.count = at<int>(q.count);
        p.most = at<float>(q.most);
        t = LossTarget{p.col, p.p, p.ent, p.start, q.k, q.nblocks};
        if (q.rows) {
            LOSS_TRY(loss_prep(p, s));
            const float* const lse = lse_out();
            LOSS_TRY(!q.head ? given(lse) : q.st == kF32 ? single(lse) : half(lse));
        } else if (q.grad && q.head && a.dw) {
            LOSS_TRY(loss_zero(a.dw, (long long)q.D * q.V * q.esz, s));
        }
        if (q.value && a.mean && !mean_done) LOSS_TRY(loss_mean(loss_out(), q.rows, p.count, q.parts, a.mean, s));
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
    const bool value = what & PRESK_HIP_LOSS_VALUE, grad = what & PRESK_HIP_LOSS_GRAD;
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
    const long long esz = st == kF32 ? 4 : 2, k = std::max<int64_t>(a.top, 1);
    const long long nx = a.rows * (head ? a.model : a.vocab) * esz, nw = head ? a.model * a.vocab * esz : 0;
    struct Span { const char* name; const void* p; long long bytes; int align; bool out, need; };
    const Span spans[] = {
        {"x", a.x, nx, (int)esz, false, true},
        {"w", a.w, nw, (int)esz, false, head},
        {"index", a.index, 8 * a.rows * k, 8, false, true},
        {"teacher", a.teacher, esz * a.rows * a.top, (int)esz, false, a.top > 0},
        {"ct", a.ct, grad ? 4 * a.rows : 0, 4, false, false},
        {"loss", a.loss, value ? 4 * a.rows : 0, 4, value, false},
        {"lse", a.lse, 4 * a.rows, 4, value, !value},
        {"mean", a.mean, 8, 4, value, !value && !a.ct},
        {"dx", a.dx, grad ? nx : 0, (int)esz, true, grad && !head},
        {"dw", a.dw, grad ? nw : 0, (int)esz, true, false},
        {"flag", a.flag, 4, 4, true, false},
        {"work", a.work, (long long)a.work_bytes, 16, true, true},
    };
    if (!head && (a.w || a.dw)) return no("w or dw where the logits are given");
    for (const Span& s : spans) {
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
    for (const Span& s : spans)
        for (const Span& o : spans)
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
    Call c{a, q, s, (char*)a.work, {}};
    return c.run();
}

hipError_t loss_check_run(const presk_hip_loss& a, int what, bool head, hipStream_t s, std::string* why) {
    *why = loss_check(a, what, head);
    if (!why->empty()) return hipSuccess;
    const Plan q = plan_of(a, what, head);
    *why = check_buffers(a, what, head, bytes_of(q));
    if (!why->empty()) return hipSuccess;
    Call c{a, q, s, (char*)a.work, {}};
    return c.run();
}

}  // namespace presk
