// The losses of a large vocabulary (loss.hip, loss_rows.hip, loss_gemm.hpp):
// softmax cross entropy and the divergence from a teacher's top logits, of
// given logits or of a head's product x . w.
#pragma once

#include <hip/hip_runtime.h>

#include <string>

#include "gemm.hpp"
#include "loss_buffers.hpp"
#include "presk_hip.h"

namespace presk {

// What the ABI's arguments ask for, checked on the host: "" or why not, the
// message starting with its code.  loss_check looks at the type and the sizes,
// loss_check_all at the buffers and the workspace too.  `head`: of x . w, else
// of given logits.
std::string loss_check(const presk_hip_loss& a, int what, bool head);
std::string loss_check_all(const presk_hip_loss& a, int what, bool head);
// the bytes of workspace a checked call needs
size_t loss_workspace(const presk_hip_loss& a, int what, bool head);
// the launches of a checked call, and with the check in front (`why` it was refused)
hipError_t loss_run(const presk_hip_loss& a, int what, bool head, hipStream_t s);
hipError_t loss_check_run(const presk_hip_loss& a, int what, bool head, hipStream_t s, std::string* why);

// ---- what the kernels share -------------------------------------------------

constexpr int kUnused = 0x7fffffff;    // a row's slot that names nothing (sorted last)
constexpr int kOutside = 0x7ffffffe;   // one that names no column of the vocabulary
constexpr int kParts = 1024;           // at most so many partial counts of a call's rows
constexpr int kCols = 64;              // columns a `start` entry stands for
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A row's target: `k` slots (column, weight) sorted by column, the weights'
// sum of p log p (NaN where a slot names no column), and, where k > 4, each
// 64-column block's first slot.  One column a row: the call's own index.
struct LossTarget {
    const long long* index;      // [rows] or null
    int vocab;
    const int* col;              // [rows][k]
    const float* p;              // [rows][k]
    const float* ent;            // [rows]
    const unsigned short* start; // [rows][nblocks + 1] or null
    int k, nblocks;
};

// One 16-bit product of the head (loss_gemm.hpp).  Operands lie k-contiguous
// (element (r, k) at r * s + k) or not ((r, k) at k * s + r).
struct LossGemm {
    const unsigned short *A, *B;
    long long sa, sb;
    int arows, brows;           // rows that exist (those past them are read from the last ones)
    int ka, kb;                 // k that exist
    int M, N, K;                // the product's extent (rows stored, k summed)
    bool two;                   // dx, dw: one operand is in two parts, summed (a2 or b2 bytes apart)
    long long a2, b2;
    int tiles_m, tiles_n, splits;
    // values: u = z * c, in units of log 2
    float c;
    LossTarget t;
    int col0, cols;             // the product's first column of the vocabulary, and how many exist
    long long rows;             // rows that exist
    float *pm, *ps, *pa;        // a column tile's maximum, sum and target part: [tile][rows]
    const float *lse, *coef;    // [rows]
    unsigned short* P;          // the logits' cotangent, [prows][pld], zero past rows and cols
    long long pld, plow;        // elements from P to its second part (0: none)
    int prows;
    // outputs
    void* C;                    // 16-bit, row stride ldc (null: the f32 sums stay in acc)
    long long ldc;
    float* acc;                 // [M][lda] f32: added to (acc_in), written where C is null
    long long lda;              // (a multiple of 4)
    bool acc_in;
    float* part;                // [splits][M][lda] f32 (splits > 1, and logits)
    const float* scale;         // the sums' factor, one float of device memory
    unsigned* flag;
};

enum LossEpi { kEpiStats, kEpiP, kEpiZ, kEpiDx, kEpiDw };

// What a launch of products may do beside them, in workgroups of its own: the
// mean of the counted rows' losses, and the counts of rows of one column each.
struct LossMean {
    const float* loss;           // null: nothing
    long long rows;
    const int* count;            // the counts of `parts`, or, with none taken,
    int parts;
    const long long* index;      // which of one column a row count
    float* mean;
};
struct LossPrep {
    const long long* index;      // null: nothing
    const void* teacher;
    const float* ct;
    int storage;
    long long rows;
    int vocab, top;
    float c;                    // log2 e / T
    int* col;
    float *p, *ent;
    unsigned short* start;
    int nblocks;
    int* count;                 // [parts]: counted rows
    float* most;                // [parts]: their largest |ct|
    int parts;
};

// tile: 256 (256 x 256 by eight waves), 128 (128 x 128 by four) or kDeep128
// (128 x 128 by eight, more blocks in flight)
constexpr int kDeep128 = 130;
hipError_t loss_gemm_bf16(const LossGemm& g, LossEpi epi, bool bkc, int tile, hipStream_t s);
hipError_t loss_gemm_f16(const LossGemm& g, LossEpi epi, bool bkc, int tile, hipStream_t s);
// z = x . w in f32 (kEpiZ, A k-contiguous), the rows' targets counted beside it
hipError_t loss_logits_bf16(const LossGemm& g, bool bkc, int tile, const LossPrep& p, hipStream_t s);
hipError_t loss_logits_f16(const LossGemm& g, bool bkc, int tile, const LossPrep& p, hipStream_t s);
// dx and dw in one launch (either may have no tiles), and the mean
hipError_t loss_pair_bf16(const LossGemm& x, const LossGemm& w, bool xbkc, int tile, const LossMean& m, hipStream_t s);
hipError_t loss_pair_f16(const LossGemm& x, const LossGemm& w, bool xbkc, int tile, const LossMean& m, hipStream_t s);

// ---- row kernels (loss_rows.hip) -------------------------------------------

// workgroups of a call's preparation, each of which leaves one count
int loss_parts(long long rows, int top);
hipError_t loss_prep(const LossPrep& a, hipStream_t s);

// Logits in memory, [rows][ld] from column col0 on, `cols` of them.
struct LossMatrix {
    const void* z;
    long long ld;
    int storage;                // Storage
    long long rows;
    int col0, cols;
    float c, nat;               // log2 e / T and 1 / T
    LossTarget t;
    int planes;                 // loss_stats and loss_joint in f32: the sum of so many, in order, ...
    long long plane;            // ... so many elements apart
};

// partials -> a row's lse and loss, and the factor of its cotangent
struct LossRows {
    const float *pm, *ps, *pa;  // [slots][rows]
    int slots;
    float unit, nat;            // of pm and pa: in log 2, and in natural logarithms of u
    LossTarget t;
    LossMatrix z;               // given logits whose target's part is taken here (null: it is in pa)
    long long rows;
    float temperature;
    float *lse, *loss;          // outputs, may be null
    float *top, *sum;           // the two parts of lse: the largest logit and log s (null: not kept)
    float* coef;                // [rows] or null
    const float* ct;
    const float* mean_in;       // {mean, count}: the count where the rows are not counted here
    const int* count;
    const float* most;
    int parts;
    float* scale;               // out: the factor of all rows, which coef is without (null: it has it)
    bool shift;                 // f16: coef by a power of two that its range holds best
    float* mean;                // {mean, count} or null: in the same launch where loss_rows_mean(rows)
};
bool loss_rows_mean(long long rows);
hipError_t loss_rows(const LossRows& a, hipStream_t s);
hipError_t loss_mean(const LossMean& m, hipStream_t s);

// partials [chunk][rows] from slot0 on; or, of one chunk, the rows' lse and loss
// themselves (`done`, its outputs may be null)
struct LossDone {
    float temperature;
    float *lse, *loss, *top, *sum;
};
int loss_chunks(long long rows, int cols);
hipError_t loss_stats(const LossMatrix& m, float* pm, float* ps, float* pa, int slot0, const LossDone* done, hipStream_t s);
// the same partials of few rows, without the target's part, beside loss_prep
// of a teacher's slots in one launch
bool loss_beside(const LossMatrix& m, int top);
hipError_t loss_stats_beside(const LossMatrix& m, float* pm, float* ps, const LossPrep& p, hipStream_t s);
// Where a cotangent goes: in the logits' type (in place or not), or f32 logits'
// in 16 bits, zero then past their columns, and past their rows up to `rows`.
struct LossTo {
    void* p;
    int storage;
    long long ld, rows;
    long long low;              // 16 bits of f32: elements to what the rounding left, rounded itself (0: not kept)
};
// the logits' cotangent, coef * (softmax - target), from the rows' lse or, with
// `top`, from its two parts, which hold more of it
hipError_t loss_grad(const LossMatrix& m, const float* top, const float* lse, const float* coef, const LossTo& to, unsigned* flag, hipStream_t s);
// both of whole rows, each read once and held in registers: lse, loss (either
// may be null) and the cotangent for ct, or for the mean over `count` (null ct)
struct LossJoint {
    LossMatrix m;
    float temperature;
    float *lse, *loss;
    const float* ct;
    const int* count;
    const float* most;
    int parts;
    float* scale;               // as in LossRows (f16 outputs shifted), where products follow
    LossTo to;
    unsigned* flag;
};
bool loss_joint_fits(const LossMatrix& m);
hipError_t loss_joint(const LossJoint& a, hipStream_t s);

// [rows][cols] 16-bit from row stride lds to ldd (a multiple of 8), zero past
// cols: two of them, either may have no rows
struct LossPack {
    const void* src;
    long long lds, rows;
    int cols;
    void* dst;
    int ldd;
};
hipError_t loss_pack(const LossPack& a, const LossPack& b, hipStream_t s);
hipError_t loss_zero(void* dst, long long bytes, hipStream_t s);
// the partials' sums of two products (of those that are split), in split order,
// times scale (plus acc): into C (16-bit, ldc) or acc
hipError_t loss_join(const LossGemm& x, const LossGemm& w, int storage, hipStream_t s);

}  // namespace presk
