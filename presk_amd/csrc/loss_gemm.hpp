// The 16-bit products of a head's loss (loss.hip):
//   kEpiStats  z = x . w, of which a column tile leaves each row's maximum, its
//              sum of exponentials and its target's logits alone;
//   kEpiP      z, leaving the logits' cotangent coef * (exp(u - lse) - t)
//              rounded to 16 bits, a piece of the vocabulary's;
//   kEpiZ      z in f32;
//   kEpiDx     dx += P . w^T and
//   kEpiDw     dw = x^T . P over the cotangent P of all or of a piece.
// 32x32x16 MFMAs over tiles of 256 x 256 by eight waves (128 x 64 a wave, one
// workgroup a CU) or 128 x 128 by four (64 x 64, two workgroups a CU), two
// 64-deep k-blocks in LDS, loaded straight into it; or 128 x 128 by eight (32 x
// 64) with four blocks.  The MFMAs take the operands' roles exchanged (D = B^T
// A^T), so that a lane holds one row's columns, four consecutive ones at a
// time: a row's maximum and sum are lane sums and one exchange between
// half-waves.
// Bound by the matrix cores at the clock their power leaves, 7 % apart from card
// to card.  4096 x 32000 in bf16: kEpiStats of 2048 rows 430 to 480 us (1250 to
// 1120 TFLOP/s), the matrix cores busy 58 % of the cycles with no LDS conflict;
// of 8192 rows kEpiZ with its 1.05 GB 1.80 to 2.03 ms (1190 to 1060), busy 66 %
// with 2 % of the LDS cycles conflicts, dx and dw 3.42 to 3.89 (1255 to 1105),
// 69 % with 0.6 %; the library's plain product of that size 1233 to 1257
// TFLOP/s.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>
#include <utility>

#include "loss_dev.hpp"

namespace presk {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

constexpr int BK = 64;

// One operand's 64-deep block in LDS, 16-byte chunks placed by an XOR swizzle
// (lane i of a wave's load fills slot i of the wave's 1 KB, the swizzle picks
// the chunk that it fetches), so that the fragment reads meet no bank twice:
//   k-contiguous, [row][8 chunks of 8 k]: chunk c of row r at 8 r + (c ^ ((r ^ (r >> 3)) & 7))
//   else, [k][ROWS / 8 chunks of 8 rows]: chunk j of k-row r at
//     (ROWS / 8) r + (j ^ (2 (r & 3) ^ 8 (r & 1)))
// Loads past the operand are moved to where it ends: a row to the last row
// (or last whole vector of rows), a k to the last k (or last whole vector), whose
// products meet a zero of the other operand or are not stored.  The
// addresses are the tile's origin (uniform, 64 bits) and a lane's 32-bit
// offset in the block.  The loads are inline assembly without an output; the
// kernel waits for them (wait_vm) before the barrier ahead of every read.
template <bool KC, int ROWS, int NTH>
struct Block16 {
    static constexpr int CPR = KC ? 8 : ROWS / 8;
    static constexpr int SLOTS = ROWS * BK / 8, ROUNDS = SLOTS / NTH, BYTES = SLOTS * 16;
    static_assert(SLOTS % NTH == 0 && (KC || ROWS % 128 == 0), "whole rounds, the swizzle inside a k-row");
    unsigned voff[ROUNDS];
    const char* origin;
    long long block_bytes;
    unsigned lds0;
    long long stride;
    int nk;                     // k that exist

    __device__ static __forceinline__ int swz(int r) {
        return KC ? ((r ^ (r >> 3)) & 7) : ((2 * (r & 3)) ^ (8 * (r & 1)));
    }
    __device__ __forceinline__ void init(const unsigned short* p, int rows, long long s, int row0, int k_exist, unsigned tile) {
        const int t = threadIdx.x;
        stride = s;
        nk = k_exist;
        origin = (const char*)(p + (KC ? (long long)row0 * s : (long long)row0));
        block_bytes = KC ? 2LL * BK : 2LL * BK * s;
#pragma unroll
        for (int q = 0; q < ROUNDS; ++q) {
            const int slot = q * NTH + t, r = slot / CPR, c = (slot % CPR) ^ swz(r);
            if (KC) {
                const int row = row0 + r < rows ? r : rows - 1 - row0;
                voff[q] = (unsigned)(2 * (row * s + 8 * c));
            } else {
                const int row = row0 + 8 * c + 8 <= rows ? 8 * c : rows - 8 - row0;
                voff[q] = (unsigned)(2 * (r * s + row));
            }
        }
        lds0 = __builtin_amdgcn_readfirstlane(tile + (unsigned)(t & ~63) * 16u);
    }
    // block kb, `part` bytes further on
    __device__ __forceinline__ void issue(int kb, unsigned stage, long long part) const {
        const char* const src = origin + kb * block_bytes + part;
        const int left = nk - kb * BK;      // k of this block that exist
        if (left >= BK) {
#pragma unroll
            for (int q = 0; q < ROUNDS; ++q)
                asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1"
                             : : "v"(voff[q]), "s"(src), "s"(__builtin_amdgcn_readfirstlane(lds0 + stage + (unsigned)(q * NTH * 16))) : "memory", "m0");
        } else {
            // a block in which the operand ends, or one past its end (then
            // the whole block is read from the last k): offsets may be negative,
            // so the address is the lane's own
            const int t = threadIdx.x;
#pragma unroll
            for (int q = 0; q < ROUNDS; ++q) {
                const int slot = q * NTH + t, r = slot / CPR, c = (slot % CPR) ^ swz(r);
                long long move = 0;
                if (KC) {
                    if (8 * c + 8 > left) move = 2LL * (left - 8 - 8 * c);
                } else if (r >= left) {
                    move = 2LL * (left - 1 - r) * stride;
                }
                const char* const at = src + voff[q] + move;
                asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off"
                             : : "v"(at), "s"(__builtin_amdgcn_readfirstlane(lds0 + stage + (unsigned)(q * NTH * 16))) : "memory", "m0");
            }
        }
    }
    // the 32x32x16 fragment: a lane's k = kk + 8 (lane >> 5) .. + 8 of row
    // base + (lane & 31): one 16-byte read, or two transposing ones
    __device__ static __forceinline__ u16x8 frag(const unsigned char* xs, int base, int kk, int lane) {
        if constexpr (KC) {
            const int r = base + (lane & 31), c = (kk >> 3) + (lane >> 5);
            return *(const u16x8*)(xs + (r * 8 + (c ^ swz(r))) * 16);
        } else {
            const int L = lane & 15, g = lane >> 4;
            const int r = kk + 8 * (g >> 1) + (L >> 2), col = base + 16 * (g & 1) + 4 * (L & 3);
            const int off = r * ROWS * 2 + (((col >> 3) ^ swz(r)) << 4) + (col & 7) * 2;
            const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(xs + off));
            const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(xs + off + 4 * ROWS * 2));
            u16x8 f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[e] = (unsigned short)lo[e];
                f[4 + e] = (unsigned short)hi[e];
            }
            return f;
        }
    }
};

// at most N of this thread's vector-memory operations outstanding
template <int N>
__device__ __forceinline__ void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// Wait until the block about to be read has landed, `later` blocks issued
// after it (NL loads a thread each) still in flight.
template <int NL, int L>
__device__ __forceinline__ void wait_blocks(int later) {
    if constexpr (L == 0) {
        wait_vm<0>();
    } else {
        if (later >= L) wait_vm<L * NL>();
        else wait_blocks<NL, L - 1>(later);
    }
}

// Blocks kt .. kt + sizeof(I) - 1 in stages I; the tail takes those below n.
template <typename F, int... I>
__device__ __forceinline__ void stage_round(F& f, int kt, std::integer_sequence<int, I...>) {
    (f(kt + I, std::integral_constant<int, I>{}), ...);
}
template <typename F, int... I>
__device__ __forceinline__ void stage_tail(F& f, int kt, int n, std::integer_sequence<int, I...>) {
    ((kt + I < n ? f(kt + I, std::integral_constant<int, I>{}) : void()), ...);
}

template <int ST>
__device__ __forceinline__ f32x16 mfma32(u16x8 a, u16x8 b, f32x16 acc) {
    if constexpr (ST == kBF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0, 0);
}

// two values rounded into one word, the first in its low half
template <int ST>
__device__ __forceinline__ unsigned narrow2(float a, float b) {
    if constexpr (ST == kBF16) {
        unsigned r;
        asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
        return r;
    } else {
        return (unsigned)pk_f32_to_f16(a) | (unsigned)pk_f32_to_f16(b) << 16;
    }
}

// The column, of the wave's 64, of a lane's sum e of column fragment j
__device__ __forceinline__ int col_of(int j, int e, int lane) { return j * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3); }

// A tile: WAM x WAN waves of (WM x 32) x 64.
template <int WM_, int NW_, int WAN_, int STAGES_>
struct Tile {
    static constexpr int WM = WM_, NW = NW_, WAN = WAN_, NTH = 64 * NW, BM = NW / WAN * WM * 32, BN = WAN * 64;
    static constexpr int STAGES = STAGES_, STAGE = (BM + BN) * BK * 2, CLD = BN + 8;
    static constexpr int OPER = STAGES * STAGE, CTILE = BM * CLD * 2;
    static constexpr int BYTES = OPER > CTILE ? OPER : CTILE;   // of LDS
};
typedef Tile<4, 8, 4, 2> Tile256;      // one workgroup a CU
typedef Tile<2, 4, 2, 2> Tile128;      // two
typedef Tile<1, 8, 2, 4> Tile128x8;    // one, three blocks ahead

// Item `id` of `total` of a product, a tile and a range of k; `id` counts from a
// workgroup whose number is a multiple of 8.
template <int ST, bool AKC, bool BKC, typename TL, int EPI, bool TWO = false>
__device__ __forceinline__ void tile_of(const LossGemm& g, unsigned id, unsigned total, unsigned char* smem) {
    constexpr int WM = TL::WM, NW = TL::NW, WAN = TL::WAN, WN = 2, NTH = TL::NTH, BM = TL::BM, BN = TL::BN;
    typedef Block16<AKC, BM, NTH> QA;
    typedef Block16<BKC, BN, NTH> QB;
    constexpr int STAGE = TL::STAGE, CLD = TL::CLD;
    static_assert(QA::BYTES + QB::BYTES == STAGE && 3 * WAN * BM * 4 <= TL::BYTES, "the tile's LDS");

    // Work order: workgroups are dealt to the 8 XCDs round robin; each XCD
    // takes one run of items, tiles GROUP rows at a time across the columns,
    // so that those in flight share panels in its L2.
    const unsigned tiles = (unsigned)g.tiles_m * (unsigned)g.tiles_n;
    const unsigned xcd = id % 8, q8 = total / 8, r8 = total % 8;
    const unsigned item = xcd * q8 + (xcd < r8 ? xcd : r8) + id / 8;
    const int split = (int)(item / tiles);
    const unsigned bid = item - (unsigned)split * tiles;
    constexpr unsigned GROUP = BM == 256 ? 4 : 8;
    const unsigned group_size = GROUP * (unsigned)g.tiles_n, grp = bid / group_size, first_m = grp * GROUP;
    const unsigned gm = (unsigned)g.tiles_m - first_m < GROUP ? (unsigned)g.tiles_m - first_m : GROUP;
    const unsigned in_grp = bid - grp * group_size, tn = in_grp / gm, tm = first_m + (in_grp - tn * gm);
    const int m0 = (int)tm * BM, n0 = (int)tn * BN;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / WAN * (WM * 32), wn = wave % WAN * 64;
    f32x16 acc[WM][WN];
#pragma unroll
    for (int i = 0; i < WM; ++i)
#pragma unroll
        for (int j = 0; j < WN; ++j) acc[i][j] = f32x16{};

    // split s of S takes k-blocks [s * n / S, (s + 1) * n / S)
    // (TWO, an operand in two parts: a block of each in turn, against the other
    // operand's same block)
    constexpr int two = TWO;
    const unsigned nkb = (unsigned)((g.K + BK - 1) / BK) << two, ns = (unsigned)g.splits;
    const int kb0 = (int)((unsigned)split * nkb / ns), nd = (int)(((unsigned)split + 1) * nkb / ns) - kb0;

    // Blocks kt + 1 .. kt + STAGES - 1 stream into their stages while block kt
    // is multiplied; each 16-k step's fragments are read during the step
    // before.  Before a block's last step this thread's loads of the next
    // block have landed, and a barrier has seen every thread's; it also retires
    // every read of the stage that the loads after it overwrite.
    QA qa;
    QB qb;
    constexpr int NS = TL::STAGES, LA = NS - 1, NL = QA::ROUNDS + QB::ROUNDS;
    static_assert(LA * NL < 64, "vmcnt holds the loads in flight");
    const unsigned lds = (unsigned)(size_t)(lds_void_t*)smem;
    qa.init(g.A, g.arows, g.sa, m0, g.ka, lds);
    qb.init(g.B, g.brows, g.sb, n0, g.kb, lds + QA::BYTES);
    auto fetch_a = [&](int kb, int st) { qa.issue((kb0 + kb) >> two, (unsigned)(st * STAGE), (kb0 + kb) & two ? g.a2 : 0); };
    auto fetch_b = [&](int kb, int st) { qb.issue((kb0 + kb) >> two, (unsigned)(st * STAGE), (kb0 + kb) & two ? g.b2 : 0); };
    u16x8 a[WM], b[WN];
    auto read = [&](const unsigned char* st, int kk) {
#pragma unroll
        for (int i = 0; i < WM; ++i) a[i] = QA::frag(st, wm + i * 32, kk, lane);
#pragma unroll
        for (int j = 0; j < WN; ++j) b[j] = QB::frag(st + QA::BYTES, wn + j * 32, kk, lane);
    };
    if (nd > 0) {
        const int pre = nd < LA ? nd : LA;
        for (int kb = 0; kb < pre; ++kb) {
            fetch_a(kb, kb);
            fetch_b(kb, kb);
        }
        wait_blocks<NL, LA - 1>(pre - 1);
        __syncthreads();
        read(smem, 0);
    }
    auto block = [&](int kt, auto stage) {
        constexpr int CUR = decltype(stage)::value;
        const unsigned char* const st = smem + CUR * STAGE;
#pragma unroll
        for (int kk = 0; kk < BK; kk += 16) {
            // one operand's loads a step: both at once hold the next reads up
            // (8192 x 4096 x 32000, loss and gradients, 7.17 ms, 7.06 so, 7.00
            // with the MFMAs' priority)
            if (kt + LA < nd) {
                if (kk == 0) fetch_a(kt + LA, (CUR + LA) % NS);
                if (kk == 16) fetch_b(kt + LA, (CUR + LA) % NS);
            }
            u16x8 ca[WM], cb[WN];
#pragma unroll
            for (int i = 0; i < WM; ++i) ca[i] = a[i];
#pragma unroll
            for (int j = 0; j < WN; ++j) cb[j] = b[j];
            if (kk + 16 < BK) {
                read(st, kk + 16);
            } else if (kt + 1 < nd) {
                const int last = kt + LA < nd - 1 ? kt + LA : nd - 1;   // the last block issued
                wait_blocks<NL, LA - 1>(last - (kt + 1));
                __syncthreads();
                read(smem + (CUR + 1) % NS * STAGE, 0);
            }
            // the reads stay ahead of this step's MFMAs
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int j = 0; j < WN; ++j) acc[i][j] = mfma32<ST>(cb[j], ca[i], acc[i][j]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    int kt = 0;
    for (; kt + NS <= nd; kt += NS) stage_round(block, kt, std::make_integer_sequence<int, NS>{});
    stage_tail(block, kt, nd, std::make_integer_sequence<int, NS - 1>{});
    __syncthreads();    // the stages are the epilogue's from here

    // The slots of row m's target in the wave's 64 columns: f(column, weight)
    // for each, in order.
    auto targets = [&](int m, auto f) {
        const bool in = m < g.rows;
        const int k = g.t.k, first = g.col0 + n0 + wn;
        long long e = 0, end = 0;
        if (in) {
            e = (long long)m * k;
            end = e + k;
            if (g.t.start) {
                const unsigned short* const s = g.t.start + (long long)m * (g.t.nblocks + 1);
                const int blk = first / kCols < g.t.nblocks ? first / kCols : g.t.nblocks - 1;
                const bool past = first / kCols >= g.t.nblocks;
                end = e + (past ? 0 : s[blk + 1]);
                e = e + (past ? 0 : s[blk]);
            }
        }
        while (__any(e < end)) {
            const bool on = e < end;
            const int s = (int)(e - (long long)m * k);
            const int col = on ? slot_col(g.t, m, s) - first : -1;
            const float p = on ? slot_p(g.t, m, s) : 0.f;
            if (__any(col >= 0 && col < 64)) f(col, p);
            ++e;
        }
    };

    if constexpr (EPI == kEpiStats) {
        float* const red = (float*)smem;    // [3][WAN][BM]
        const int h = lane >> 5;
        const bool edge = n0 + BN > g.cols;
#pragma unroll
        for (int i = 0; i < WM; ++i) {
            const int row = wm + i * 32 + (lane & 31);
            if (edge) {
#pragma unroll
                for (int j = 0; j < WN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (n0 + wn + col_of(j, e, lane) >= g.cols) acc[i][j][e] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < WN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, acc[i][j][e]);
            mx = fmaxf(mx, partner<32>(mx));
            const float mc = mx * g.c, base = mx == -INFINITY ? 0.f : mc;
            float s = 0.f, ta = 0.f;
#pragma unroll
            for (int j = 0; j < WN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], g.c, -base));
            targets(m0 + row, [&](int col, float p) {
                float v = 0.f;
                bool hit = false;
#pragma unroll
                for (int j = 0; j < WN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (col == col_of(j, e, lane)) {
                            v = acc[i][j][e];
                            hit = true;
                        }
                if (hit) ta += p * (v * g.c);
            });
            s += partner<32>(s);
            ta += partner<32>(ta);
            if (h == 0) {
                const int at = wave % WAN * BM + row;
                red[at] = mc;
                red[WAN * BM + at] = s;
                red[2 * WAN * BM + at] = ta;
            }
        }
        __syncthreads();
        for (int r = threadIdx.x; r < BM; r += NTH) {
            if (m0 + r >= g.rows) continue;
            float m = red[r], s = 0.f, ta = 0.f;
#pragma unroll
            for (int w = 1; w < WAN; ++w) m = fmaxf(m, red[w * BM + r]);
            const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int w = 0; w < WAN; ++w) {
                s += red[(WAN + w) * BM + r] * __builtin_amdgcn_exp2f(red[w * BM + r] - base);
                ta += red[(2 * WAN + w) * BM + r];
            }
            const long long at = (long long)tn * g.rows + m0 + r;
            g.pm[at] = m;
            g.ps[at] = s;
            g.pa[at] = ta;
        }
    } else if constexpr (EPI == kEpiP) {
        // (f16 cotangents stay below 2^15: no overflow to look for)
        unsigned short* const ct = (unsigned short*)smem;   // [BM][CLD]
        const bool edge = n0 + BN > g.cols;
#pragma unroll
        for (int i = 0; i < WM; ++i) {
            const int row = wm + i * 32 + (lane & 31), m = m0 + row;
            const bool in = m < g.rows;
            const float lse = in ? g.lse[m] * kLog2e : 0.f, coef = in ? g.coef[m] : 0.f;
#pragma unroll
            for (int j = 0; j < WN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], g.c, -lse));
            targets(m, [&](int col, float p) {
#pragma unroll
                for (int j = 0; j < WN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (col == col_of(j, e, lane)) acc[i][j][e] -= p;
            });
            if (edge) {
#pragma unroll
                for (int j = 0; j < WN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (n0 + wn + col_of(j, e, lane) >= g.cols) acc[i][j][e] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < WN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = coef == 0.f ? 0.f : acc[i][j][e] * coef;
        }
        // the tile rounded, then, of a P in two parts, what that left
        for (long long part = 0;; part = g.plow) {
#pragma unroll
            for (int i = 0; i < WM; ++i) {
                const int row = wm + i * 32 + (lane & 31);
#pragma unroll
                for (int j = 0; j < WN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint2 v;
                        v.x = narrow2<ST>(acc[i][j][4 * q], acc[i][j][4 * q + 1]);
                        v.y = narrow2<ST>(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
                        *(uint2*)&ct[row * CLD + wn + col_of(j, 4 * q, lane)] = v;
                    }
            }
            __syncthreads();
            constexpr int VPR = BN / 8;
            for (int u = threadIdx.x; u < BM * VPR; u += NTH) {
                const int r = u / VPR, c = u % VPR * 8;
                if (m0 + r < g.prows && n0 + c < g.pld)
                    *(u16x8*)(g.P + part + (long long)(m0 + r) * g.pld + n0 + c) = *(const u16x8*)&ct[r * CLD + c];
            }
            if (part == g.plow) break;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int j = 0; j < WN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const unsigned short h = ST == kBF16 ? pk_f32_to_bf16(acc[i][j][e]) : pk_f32_to_f16(acc[i][j][e]);
                        acc[i][j][e] = left_of(acc[i][j][e], ST == kBF16 ? pk_bf16_to_f32(h) : pk_f16_to_f32(h));
                    }
        }
    } else {
        const float scale = g.scale ? *g.scale : 1.f;
        const bool sums = EPI == kEpiZ || g.splits > 1 || !g.C;   // f32 (rows hold whole fours)
        float* const out = EPI == kEpiZ || g.splits > 1 ? g.part + (long long)split * g.M * g.lda : g.acc;
        float f = EPI == kEpiZ || g.splits > 1 ? 1.f : scale;
        if (EPI == kEpiDx && g.splits <= 1 && g.acc_in) {
            // the pieces before
#pragma unroll
            for (int i = 0; i < WM; ++i) {
                const int m = m0 + wm + i * 32 + (lane & 31);
                const float* const row = out + (long long)m * g.lda;
#pragma unroll
                for (int j = 0; j < WN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int n = n0 + wn + col_of(j, 4 * q, lane);
                        f32x4 v = {0.f, 0.f, 0.f, 0.f};
                        if (m < g.M && n < g.N) v = *(const f32x4*)(row + n);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = acc[i][j][4 * q + e] * f + v[e];
                    }
            }
            f = 1.f;
        }
        if (sums) {
            // 32 rows of the wave's 64 columns at a time through its own LDS,
            // so that a store is four rows' 256 bytes and not 32 rows' 32
            constexpr int LD = 68;
            static_assert(NW * 32 * LD * 4 <= TL::BYTES, "the waves' rows");
            float* const rows = (float*)smem + wave * (32 * LD);
#pragma unroll
            for (int i = 0; i < WM; ++i) {
#pragma unroll
                for (int j = 0; j < WN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        f32x4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e] * f;
                        *(f32x4*)&rows[(lane & 31) * LD + col_of(j, 4 * q, lane)] = v;
                    }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    const int r = 4 * p + (lane >> 4), c = 4 * (lane & 15);
                    const f32x4 v = *(const f32x4*)&rows[r * LD + c];
                    const int m = m0 + wm + i * 32 + r, n = n0 + wn + c;
                    if (m < g.M && n < g.N) *(f32x4*)(out + (long long)m * g.lda + n) = v;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        } else {
            unsigned short* const ct = (unsigned short*)smem;
            // the largest finite value (past the operands' ends stand values
            // from inside them, or 0)
            unsigned worst = 0;
#pragma unroll
            for (int i = 0; i < WM; ++i) {
                const int row = wm + i * 32 + (lane & 31);
#pragma unroll
                for (int j = 0; j < WN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            x[e] = acc[i][j][4 * q + e] * f;
                            if constexpr (ST == kF16) {
                                const unsigned b = pk_bits(x[e]) & 0x7fffffffu;
                                worst = max(worst, b < 0x7f800000u ? b : 0u);
                            }
                        }
                        uint2 v;
                        v.x = narrow2<ST>(x[0], x[1]);
                        v.y = narrow2<ST>(x[2], x[3]);
                        *(uint2*)&ct[row * CLD + wn + col_of(j, 4 * q, lane)] = v;
                    }
            }
            if (ST == kF16 && g.flag && pk_overflows_f16(pk_float(worst))) atomicOr(g.flag, 1u);
            __syncthreads();
            // 16 bytes a thread, at whatever element a row starts
            unsigned short* const C = (unsigned short*)g.C;
            constexpr int VPR = BN / 8;
            for (int u = threadIdx.x; u < BM * VPR; u += NTH) {
                const int r = u / VPR, c = u % VPR * 8;
                if (m0 + r >= g.M) continue;
                unsigned short* const at = C + (long long)(m0 + r) * g.ldc + n0 + c;
                const u16x8 v = *(const u16x8*)&ct[r * CLD + c];
                if (n0 + c + 8 <= g.N)
                    __builtin_memcpy(at, &v, 16);
                else
                    for (int e = 0; e < 7; ++e)
                        if (n0 + c + e < g.N) at[e] = v[e];
            }
        }
    }
}

template <int ST, bool AKC, bool BKC, typename TL, int EPI>
__global__ void __launch_bounds__(TL::NTH, 2) loss_gemm_kernel(LossGemm g) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[TL::BYTES];
    tile_of<ST, AKC, BKC, TL, EPI>(g, blockIdx.x, gridDim.x, smem);
}

// the logits in f32, and in workgroups past their items the rows' counts
template <int ST, bool BKC, typename TL>
__global__ void __launch_bounds__(TL::NTH, 2) loss_logits_kernel(LossGemm g, unsigned items, LossPrep p) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[TL::BYTES];
    if (blockIdx.x < items) tile_of<ST, true, BKC, TL, kEpiZ>(g, blockIdx.x, items, smem);
    else prep_one<TL::NTH>(p, (int)(blockIdx.x - items));
}

// dx (A the cotangent, k-contiguous), dw (neither operand), the mean
template <int ST, bool XBKC, typename TL, bool TWO>
__global__ void __launch_bounds__(TL::NTH, 2) loss_pair_kernel(LossGemm x, LossGemm w, unsigned nx, unsigned nx8, unsigned nw, LossMean m) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[TL::BYTES];
    const unsigned id = blockIdx.x;
    if (id < nx8) {
        if (id < nx) tile_of<ST, true, XBKC, TL, kEpiDx, TWO>(x, id, nx, smem);
    } else if (id < nx8 + nw) {
        tile_of<ST, false, false, TL, kEpiDw, TWO>(w, id - nx8, nw, smem);
    } else {
        write_mean<TL::NTH>(m);
    }
}

unsigned items_of(const LossGemm& g) { return (unsigned)g.tiles_m * (unsigned)g.tiles_n * (unsigned)g.splits; }

template <int ST, bool AKC, bool BKC, int EPI>
hipError_t launch(const LossGemm& g, int tile, hipStream_t s) {
    const unsigned grid = items_of(g);
    if (!grid) return hipSuccess;
    if (tile == 256) loss_gemm_kernel<ST, AKC, BKC, Tile256, EPI><<<grid, 512, 0, s>>>(g);
    else if (tile == kDeep128) loss_gemm_kernel<ST, AKC, BKC, Tile128x8, EPI><<<grid, 512, 0, s>>>(g);
    else loss_gemm_kernel<ST, AKC, BKC, Tile128, EPI><<<grid, 256, 0, s>>>(g);
    return hipGetLastError();
}

template <int ST>
hipError_t gemm(const LossGemm& g, LossEpi epi, bool bkc, int tile, hipStream_t s) {
    if (epi == kEpiStats) return bkc ? launch<ST, true, true, kEpiStats>(g, tile, s) : launch<ST, true, false, kEpiStats>(g, tile, s);
    if (epi == kEpiP) return bkc ? launch<ST, true, true, kEpiP>(g, tile, s) : launch<ST, true, false, kEpiP>(g, tile, s);
    return hipErrorInvalidValue;
}

template <int ST, bool BKC>
hipError_t logits_of(const LossGemm& g, int tile, const LossPrep& p, hipStream_t s) {
    const unsigned n = items_of(g), grid = n + (p.index ? (unsigned)p.parts : 0);
    if (tile == 256) loss_logits_kernel<ST, BKC, Tile256><<<grid, 512, 0, s>>>(g, n, p);
    else if (tile == kDeep128) loss_logits_kernel<ST, BKC, Tile128x8><<<grid, 512, 0, s>>>(g, n, p);
    else loss_logits_kernel<ST, BKC, Tile128><<<grid, 256, 0, s>>>(g, n, p);
    return hipGetLastError();
}

template <int ST, bool XBKC, bool TWO>
hipError_t pair_of(const LossGemm& x, const LossGemm& w, int tile, const LossMean& m, hipStream_t s) {
    const unsigned nx = items_of(x), nx8 = (nx + 7) / 8 * 8, nw = items_of(w), grid = nx8 + nw + (m.loss ? 1 : 0);
    if (!grid) return hipSuccess;
    if (tile == 256) loss_pair_kernel<ST, XBKC, Tile256, TWO><<<grid, 512, 0, s>>>(x, w, nx, nx8, nw, m);
    else if (tile == kDeep128) loss_pair_kernel<ST, XBKC, Tile128x8, TWO><<<grid, 512, 0, s>>>(x, w, nx, nx8, nw, m);
    else loss_pair_kernel<ST, XBKC, Tile128, TWO><<<grid, 256, 0, s>>>(x, w, nx, nx8, nw, m);
    return hipGetLastError();
}

template <int ST>
hipError_t pair(const LossGemm& x, const LossGemm& w, bool xbkc, int tile, const LossMean& m, hipStream_t s) {
    if (x.two) return xbkc ? pair_of<ST, true, true>(x, w, tile, m, s) : pair_of<ST, false, true>(x, w, tile, m, s);
    return xbkc ? pair_of<ST, true, false>(x, w, tile, m, s) : pair_of<ST, false, false>(x, w, tile, m, s);
}

}  // namespace

}  // namespace presk
