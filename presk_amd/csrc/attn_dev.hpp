// Attention's kernels (attn.hpp).
//
// A wave keeps 32 rows of one operand (queries, or in the keys' gradients keys)
// in registers, one a lane of each half-wave, and the others pass by in tiles
// through LDS.  Scores are taken with the tile's rows as the matrix
// instruction's rows, so that a lane holds one kept row's scores against 16 of
// 32 tile rows: a softmax's maximum and sum are lane sums and one exchange
// between half-waves, and the weights, rounded to the storage type, are the
// next product's second operand as they lie, the sum over the tile's rows
// taken in the order in which the lanes hold them; its first operand, the
// tile transposed, comes from transposing LDS reads (16 bits) or from a row's
// consecutive elements (f32).
#pragma once

#include <hip/hip_runtime.h>

#include "attn.hpp"
#include "loss_gemm.hpp"

namespace presk {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// A tile's rows of ND * 32 elements in LDS, PITCH of them apart, 16-byte chunk c
// of row r at chunk c ^ swz(r): eight (and sixteen) consecutive rows' same chunk,
// and four consecutive rows' same four chunks, lie in different banks.
template <int ST, int ND>
struct Geo {
    static constexpr int ES = ST == kF32 ? 4 : 2, PITCH = ND <= 2 ? 64 : ND <= 4 ? 128 : 256;
    static constexpr int ROW = PITCH * ES, CPR = ROW / 16, EPC = 16 / ES;
    static constexpr int STEPS = ND * 32 / (2 * EPC);     // 16-byte reads of a row a lane (its half of each pair of chunks)
    static constexpr int KSTEPS = ST == kF32 ? STEPS / 2 : STEPS;     // matrix instructions' k of a row
    static constexpr int TILE = ROW <= 256 ? 64 : 32;     // rows of a tile
    __host__ __device__ static constexpr int swz(int r) {
        if constexpr (CPR == 8) return ((r & 2) << 1) | ((r & 4) >> 1) | ((r ^ (r >> 3)) & 1);
        else return ((r & 1) << 2) | (((r >> 1) ^ (r >> 3)) & 1) << 3 | (r & 2) | ((r >> 2) & 1);
    }
};

// 16 bytes of a row
template <int ST> struct FragOf { typedef u16x8 T; };
template <> struct FragOf<kF32> { typedef f32x4 T; };

// A matrix instruction's eight elements a lane.  f32 in three parts of 8 bits
// each, rounded to nearest, which are all of its 24 down to 2^-110 (where the last
// part's come to bf16's smallest step, 2^-133: scaling that away is an instruction an
// element more, and a second pass for the large ones, on what these kernels are
// bound by).  Of a product's nine six are taken (the three left are below 2^-24 of it
// together, f32's own rounding), by bf16 instructions, of which six take 3/8 of the
// time of f32's own (64 x 6 heads x 256 x 64, causal: the value 63 -> 52 us, the
// queries' gradient 87 -> 68, the keys' 121 -> 105; bound now by the eleven vector
// instructions that two elements' parts take, in every wave that reads them).  An
// infinite element, or one that rounds to it, has a second part that is no number:
// what reads it is NaN.
template <int ST> struct Part { u16x8 p[1]; };
template <> struct Part<kF32> { u16x8 p[3]; };

// Two values rounded into one word.  (The compiler's own conversion: it knows that
// an exponential's result needs a wait before it is read, which assembly would not get.)
template <int ST>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    if constexpr (ST == kBF16) return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{a, b}), bf16x2));
    else return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{a, b}), f16x2));
}

__device__ __forceinline__ Part<kF32> parts_of(const float (&x)[8]) {
    unsigned w[3][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float a = x[2 * e], b = x[2 * e + 1];
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            w[n][e] = pack2<kBF16>(a, b);
            a -= __builtin_bit_cast(float, w[n][e] << 16);
            b -= __builtin_bit_cast(float, w[n][e] & 0xffff0000u);
        }
    }
    Part<kF32> f;
#pragma unroll
    for (int n = 0; n < 3; ++n) f.p[n] = __builtin_bit_cast(u16x8, i32x4{(int)w[n][0], (int)w[n][1], (int)w[n][2], (int)w[n][3]});
    return f;
}
// The elements as they are read, and their parts.
struct Raw32 { f32x4 a, b; };
template <int ST> struct RawOf { typedef Part<ST> T; };
template <> struct RawOf<kF32> { typedef Raw32 T; };
__device__ __forceinline__ Part<kF32> parts_of(f32x4 a, f32x4 b) {
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return parts_of(x);
}

__device__ __forceinline__ Part<kF32> part_of(const Raw32& r) { return parts_of(r.a, r.b); }
template <int ST>
__device__ __forceinline__ const Part<ST>& part_of(const Part<ST>& p) { return p; }

template <int ST>
__device__ __forceinline__ f32x16 mma_row(const Part<ST>& a, const Part<ST>& b, f32x16 acc) {
    if constexpr (ST == kF32) {
        // the smallest first
#pragma unroll
        for (int n = 2; n >= 0; --n)
#pragma unroll
            for (int i = 0; i <= n; ++i) acc = mfma32<kBF16>(a.p[i], b.p[n - i], acc);
        return acc;
    } else {
        return mfma32<ST>(a.p[0], b.p[0], acc);
    }
}

// The weights of 32 tile rows as a product's operand.
template <int ST>
struct Weights {
    u16x8 w[2];
    __device__ __forceinline__ void set(const f32x16& p) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            unsigned u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = pack2<ST>(p[8 * s + 2 * e], p[8 * s + 2 * e + 1]);
            w[s] = __builtin_bit_cast(u16x8, i32x4{(int)u[0], (int)u[1], (int)u[2], (int)u[3]});
        }
    }
};
// What that rounding left of p, in its place.
template <int ST>
__device__ __forceinline__ void left_in(f32x16& p, const Weights<ST>& w) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const unsigned short u = w.w[e >> 3][e & 7];
        p[e] = left_of(p[e], ST == kBF16 ? pk_bf16_to_f32(u) : pk_f16_to_f32(u));
    }
}
template <>
struct Weights<kF32> {
    Part<kF32> w[2];
    __device__ __forceinline__ void set(const f32x16& p) {
#pragma unroll
        for (int s = 0; s < 2; ++s) w[s] = parts_of(f32x4{p[8 * s], p[8 * s + 1], p[8 * s + 2], p[8 * s + 3]},
                                                    f32x4{p[8 * s + 4], p[8 * s + 5], p[8 * s + 6], p[8 * s + 7]});
    }
};

// The tile row, of 32, of a lane's sum e.
__device__ __forceinline__ int row_of(int e, int h) { return 8 * (e >> 2) + 4 * h + (e & 3); }

// Where a lane reads a tile: LDS addresses, of a tile's 32 rows by adding whole
// tiles to them.  A step's and a piece's chunks are a base's with bits flipped, so
// that a lane holds one address and not one a step: `row` its part of row lane &
// 31, `col` its first element of the transposed 32 rows.
template <int ST, int ND>
struct Places {
    typedef Geo<ST, ND> G;
    unsigned row, col;
    __device__ __forceinline__ void init(int lane) {
        const int h = lane >> 5, r = lane & 31;
        row = (unsigned)(r * G::ROW + ((h ^ G::swz(r)) << 4));
        if constexpr (ST == kF32) {
            const int el = ND * r;
            col = (unsigned)(4 * h * G::ROW + (((el >> 2) ^ h) << 4 | (el & 3) << 2));
        } else {
            const int L = lane & 15, g = (lane >> 4) & 1, q = 4 * h + (L >> 2);
            col = (unsigned)(q * G::ROW + (((2 * g + ((L & 3) >> 1)) ^ G::swz(q)) << 4) + 8 * (L & 1));
        }
    }
    // at `at` bytes of LDS.  The compiler does not see that they stay the same
    // from tile to tile, or it would keep every step's.
    __device__ __forceinline__ Places from(unsigned at) const {
        Places p{row + at, col + at};
        asm volatile("" : "+v"(p.row), "+v"(p.col));
        return p;
    }
};

template <typename T>
__device__ __forceinline__ T lds_read(unsigned at) {
    return *(__attribute__((address_space(3))) T*)at;
}

// A lane's part of its row at step `st` (its half of chunks 2 st and 2 st + 1; in
// f32 of the four from 4 st on).
template <int ST>
__device__ __forceinline__ typename RawOf<ST>::T frag_row(unsigned row, int st, unsigned off = 0) {
    if constexpr (ST == kF32) return Raw32{lds_read<f32x4>((row ^ (unsigned)(st << 6)) + off), lds_read<f32x4>((row ^ (unsigned)(st << 6 | 32)) + off)};
    else return Part<ST>{{lds_read<u16x8>((row ^ (unsigned)(st << 5)) + off)}};
}

// acc[n][dt] += X^T . w[n] over 32 rows of a tile, for NB blocks of kept rows.  f32
// takes a lane's elements of the head as ND consecutive ones, and adds the 32 rows'
// products to acc once: the twelve instructions that they take would each round at the
// size of all rows' sum (16384 rows: 2.0e-6 of it, root mean square, so 0.5e-6; the
// value takes 3 % longer for it, the gradients 2 to 6).
template <int ST, int ND, int NB, bool TIGHT = false>
__device__ __forceinline__ void mma_col(unsigned col, unsigned off, const Weights<ST> (&w)[NB], f32x16 (&acc)[NB][ND]) {
    typedef Geo<ST, ND> G;
    if constexpr (ST == kF32) {
        float x[2][ND][8];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // (the row without the half-wave's 4, which `col` has)
                const int r = 16 * q + 8 * (e >> 2) + (e & 3);
                const unsigned at = (col ^ (unsigned)(G::swz(r) << 4)) + (unsigned)(r * G::ROW) + off;
                if constexpr (ND == 4) {
                    const f32x4 v = lds_read<f32x4>(at);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[q][i][e] = v[i];
                } else {
                    const f32x2 v = lds_read<f32x2>(at);
                    x[q][0][e] = v[0], x[q][1][e] = v[1];
                }
            }
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                f32x16 t = f32x16{};
#pragma unroll
                for (int q = 0; q < 2; ++q) t = mma_row<kF32>(parts_of(x[q][dt]), w[n].w[q], t);
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[n][dt][e] += t[e];
            }
            // (TIGHT: two waves a SIMD do not hold the next elements' parts too)
            if constexpr (TIGHT && ND == 2) __builtin_amdgcn_sched_barrier(0);
        }
    } else {
        constexpr unsigned FLIP = (unsigned)((G::swz(8) ^ G::swz(0)) << 4);      // of a row 8 further on
        // (TIGHT: a fragment's reads one ahead of its products, and no further)
        v4i16 a, b;
        auto read = [&](int n) {
            const int s = n / ND, dt = n % ND;
            a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)((col ^ (unsigned)(dt << 6)) + (unsigned)(16 * s * G::ROW) + off));
            b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)((col ^ (unsigned)(dt << 6) ^ FLIP) + (unsigned)((16 * s + 8) * G::ROW) + off));
        };
        read(0);
#pragma unroll
        for (int i = 0; i < 2 * ND; ++i) {
            u16x8 f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[e] = (unsigned short)a[e];
                f[4 + e] = (unsigned short)b[e];
            }
            if (i + 1 < 2 * ND) read(i + 1);
            if (TIGHT) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < NB; ++n) acc[n][i % ND] = mfma32<ST>(f, w[n].w[i / ND], acc[n][i % ND]);
            if (TIGHT) __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// ---- loads ------------------------------------------------------------------------

// Elements of a row one at a time (rows that are not whole vectors): those past
// the head's end, and of rows that do not exist, are zero.
template <int ST>
__device__ __forceinline__ typename FragOf<ST>::T chunk_of(const void* row, int c, int d, bool in) {
    typename FragOf<ST>::T f;
    constexpr int EPC = ST == kF32 ? 4 : 8;
#pragma unroll
    for (int e = 0; e < EPC; ++e) {
        const bool here = in && c * EPC + e < d;
        if constexpr (ST == kF32) f[e] = here ? ((const float*)row)[c * EPC + e] : 0.f;
        else f[e] = here ? ((const unsigned short*)row)[c * EPC + e] : (unsigned short)0;
    }
    return f;
}

template <int ST>
__device__ __forceinline__ const void* row_at(const AttnTensor& t, int b, long long i, int h) {
    const long long n = (long long)b * t.batch + i * t.seq + (long long)h * t.head;
    return (const char*)t.p + n * (ST == kF32 ? 4 : 2);
}

// A kept row: a lane's 16 bytes of every step.  Rows that are no whole vectors
// pass through the lane's own 16 bytes a step of `lds` (the wave's 1 KB a step),
// in a loop that is not unrolled.
template <int ST, int ND, typename P>
__device__ __forceinline__ void load_kept(const AttnTensor& t, int b, long long i, int head, int d, bool in, int lane, unsigned char* lds,
                                          P (&x)[Geo<ST, ND>::KSTEPS]) {
    typedef typename FragOf<ST>::T F;
    constexpr int EACH = ST == kF32 ? 2 : 1;
    const void* const row = row_at<ST>(t, b, in ? i : 0, head);
    const int h = lane >> 5;
    if (t.vec) {
        F f[Geo<ST, ND>::STEPS];
#pragma unroll
        for (int st = 0; st < Geo<ST, ND>::STEPS; ++st) {
            const int c = 2 * st + h;
            f[st] = in && c * Geo<ST, ND>::EPC < d ? *(const F*)((const char*)row + 16 * c) : F{};
        }
#pragma unroll
        for (int st = 0; st < Geo<ST, ND>::KSTEPS; ++st) {
            if constexpr (ST != kF32) x[st].p[0] = f[st];
            else if constexpr (sizeof(P) == sizeof(Raw32)) x[st] = Raw32{f[EACH * st], f[EACH * st + 1]};
            else x[st] = parts_of(f[EACH * st], f[EACH * st + 1]);
        }
    } else {
        F* const mine = (F*)lds + lane;
#pragma unroll 1
        for (int st = 0; st < Geo<ST, ND>::STEPS; ++st) mine[64 * st] = chunk_of<ST>(row, 2 * st + h, d, in);
#pragma unroll
        for (int st = 0; st < Geo<ST, ND>::KSTEPS; ++st) {
            if constexpr (ST != kF32) x[st].p[0] = mine[64 * st];
            else if constexpr (sizeof(P) == sizeof(Raw32)) x[st] = Raw32{mine[64 * EACH * st], mine[64 * (EACH * st + 1)]};
            else x[st] = parts_of(mine[64 * EACH * st], mine[64 * (EACH * st + 1)]);
        }
    }
}

__device__ __forceinline__ i32x4 buffer_of(const void* p, unsigned bytes) {
    const unsigned long long u = (unsigned long long)p;
    return i32x4{__builtin_amdgcn_readfirstlane((int)(u & 0xffffffffu)), __builtin_amdgcn_readfirstlane((int)((u >> 32) & 0xffffu)),
                 __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}

// A tile of ROWS rows, loaded straight into LDS by NTH threads (lane i of a
// wave's load fills chunk i of the wave's 1 KB, the swizzle picks the chunk that
// it fetches).  The loads go through a buffer that ends where the tile's rows
// do: what lies past it, or past a row's end, is zero.  They are inline
// assembly without an output; the kernel waits for them (wait_vm) before the
// barrier ahead of every read.
template <int ST, int ND, int ROWS, int NTH>
struct Rows {
    typedef Geo<ST, ND> G;
    static constexpr int SLOTS = ROWS * G::CPR, ROUNDS = SLOTS / NTH, BYTES = SLOTS * 16, STEP = NTH / G::CPR;
    static constexpr int ALT = STEP >= 16 ? 1 : 16 / STEP;      // rounds until the swizzle repeats
    static_assert(SLOTS % NTH == 0 && NTH % G::CPR == 0, "whole rounds of whole rows");
    static constexpr int KEPT = ALT < ROUNDS ? ALT : ROUNDS;
    unsigned voff[KEPT];
    const char* base;
    long long stride;       // bytes
    int d, vec;
    unsigned lds0;

    __device__ __forceinline__ void init(const AttnTensor& t, int b, int head, int d_, int tid, unsigned lds) {
        base = (const char*)row_at<ST>(t, b, 0, head);
        stride = t.seq * G::ES;
        d = d_;
        vec = t.vec;
#pragma unroll
        for (int q = 0; q < KEPT; ++q) {
            const int slot = q * NTH + tid, r = slot / G::CPR, c = (slot % G::CPR) ^ G::swz(r);
            voff[q] = c * G::EPC < d ? (unsigned)(r * stride) + 16u * c : 0x80000000u;
        }
        lds0 = __builtin_amdgcn_readfirstlane(lds + (unsigned)(tid & ~63) * 16u);
    }
    // the rows from row0 on, of which `left` (1 or more) exist, at `at` bytes of LDS
    __device__ __forceinline__ void issue(long long row0, int left, unsigned at, unsigned char* smem, int tid) const {
        const char* const src = base + row0 * stride;
        if (vec) {
            const int n = left < ROWS ? left : ROWS;
            const i32x4 buf = buffer_of(src, (unsigned)((n - 1) * stride + d * G::ES));
#pragma unroll
            for (int q = 0; q < ROUNDS; ++q) {
                const unsigned off = voff[q % KEPT] + (unsigned)(q / KEPT * KEPT * STEP * (int)stride);
                asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                             : : "v"(off), "s"(buf), "s"(__builtin_amdgcn_readfirstlane(lds0 + at + (unsigned)(q * NTH * 16))) : "memory", "m0");
            }
        } else {
            const int n = left < ROWS ? left : ROWS;
            const auto buf = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(src), (short)0, (int)((n - 1) * stride + d * G::ES), 0x00020000);
#pragma unroll 1
            for (int q = 0; q < ROUNDS; ++q) {
                const int slot = q * NTH + tid, r = slot / G::CPR, c = (slot % G::CPR) ^ G::swz(r);
                const unsigned off = (unsigned)(r * (int)stride + 16 * c);
                typename FragOf<ST>::T f;
#pragma unroll
                for (int e = 0; e < G::EPC; ++e) {
                    const int o = c * G::EPC + e < d ? (int)(off + e * G::ES) : (int)0x80000000u;
                    if constexpr (ST == kF32) f[e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(buf, o, 0, 0));
                    else f[e] = __builtin_amdgcn_raw_buffer_load_b16(buf, o, 0, 0);
                }
                *(typename FragOf<ST>::T*)(smem + at + slot * 16) = f;
            }
        }
    }
};

// ---- stores -----------------------------------------------------------------------

// A wave's 32 rows of sums, a lane's times its own f, in the storage type: through
// the wave's 32 rows of `lds` (which no other wave reads any more), so that a row
// leaves in 16-byte vectors beside each other.  `where(r)`: row r's address, null
// where there is none.  GRAD: an element that is not finite counts as one that
// overflows, since the cotangents of the weights may have.
template <int ST, int ND, bool GRAD, typename W>
__device__ __forceinline__ void store_kept(const f32x16 (&acc)[ND], float f, int d, bool vec, bool live, W where, unsigned char* lds, int lane,
                                           unsigned* flag) {
    typedef Geo<ST, ND> G;
    typedef typename FragOf<ST>::T F;
    const int h = lane >> 5, r = lane & 31;
    bool ovf = false;
    if constexpr (ST == kF32) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int at = ND * row_of(e, h);
            unsigned char* const to = lds + r * G::ROW + ((((at >> 2) ^ G::swz(r)) << 4) | ((at & 3) << 2));
            if constexpr (ND == 4) *(f32x4*)to = f32x4{acc[0][e] * f, acc[1][e] * f, acc[2][e] * f, acc[3][e] * f};
            else *(f32x2*)to = f32x2{acc[0][e] * f, acc[1][e] * f};
        }
    } else {
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at = dt * 32 + 8 * g + 4 * h;
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = acc[dt][4 * g + e] * f;
                    if (ST == kF16) ovf |= GRAD ? !(__builtin_fabsf(x[e]) < 65520.f) : pk_overflows_f16(x[e]);
                }
                *(unsigned long long*)(lds + r * G::ROW + ((((at >> 3) ^ G::swz(r)) << 4) | ((at & 4) << 1))) =
                    pack2<ST>(x[0], x[1]) | (unsigned long long)pack2<ST>(x[2], x[3]) << 32;
            }
    }
    if (ovf && live && flag) atomicOr(flag, 1u);
    constexpr int EPC = G::EPC;
#pragma unroll 1
    for (int u = lane; u < 32 * G::CPR; u += 64) {
        const int row = u / G::CPR, c = u % G::CPR;
        if (c * EPC >= d) continue;
        char* const to = (char*)where(row);
        if (!to) continue;
        const F v = *(const F*)(lds + row * G::ROW + ((c ^ G::swz(row)) << 4));
        if (vec) {
            *(F*)(to + 16 * c) = v;
        } else {
#pragma unroll
            for (int e = 0; e < EPC; ++e)
                if (c * EPC + e < d) {
                    if constexpr (ST == kF32) ((float*)to)[c * EPC + e] = v[e];
                    else ((unsigned short*)to)[c * EPC + e] = v[e];
                }
        }
    }
}

// ---- which keys a query reads -------------------------------------------------------

struct Keys {
    int len;            // keys of the sequence
    int first;          // the first query's position
    __device__ __forceinline__ void init(const AttnArgs& a, int b) {
        const long long n = a.lens ? a.lens[b] : a.tk, f = a.first ? a.first[b] : a.first0;
        len = __builtin_amdgcn_readfirstlane((int)(n < 0 ? 0 : n > a.tk ? a.tk : n));
        first = __builtin_amdgcn_readfirstlane((int)(f < -(1 << 30) ? -(1 << 30) : f > 1 << 30 ? 1 << 30 : f));
    }
    // of query i: keys [lo, hi) (and of a mask's columns those whose bit is set)
    __device__ __forceinline__ int lo(const AttnArgs& a, int i) const {
        const int w = a.window ? first + i - a.window + 1 : 0;
        return w > 0 ? w : 0;
    }
    __device__ __forceinline__ int hi(const AttnArgs& a, int i) const {
        const int e = a.causal ? first + i + 1 : a.cols ? first + a.cols : len;
        return e < len ? e : len;
    }
    // of all queries up to i: keys below this one, from lo(i) on, whatever the mask
    __device__ __forceinline__ int sure(const AttnArgs& a, int i) const {
        const int e = a.causal ? first + i + 1 : a.cols ? first : len;
        return e < len ? e : len;
    }
};

// Whether the cotangents of the weights of queries i0 .. i1 enter their products
// in two parts, the rounding to 16 bits and what it left: where one of them reads
// fewer than 64 keys (or a mask says which).  Such rows have the largest
// gradients, and theirs are the errors of the stored output too; together with
// the rounding of the weights' cotangents these pass what the gradients' own
// rounding adds (documents of 256 tokens in bf16: 1.53 times the error of a float32
// computation whose outputs are rounded, in two parts 1.35).
template <int ST>
__device__ __forceinline__ bool fine_of(const AttnArgs& a, const Keys& keys, int i0, int i1) {
    return ST != kF32 && (a.cols || keys.hi(a, i0) - keys.lo(a, i0) < 64 || keys.hi(a, i1) - keys.lo(a, i1) < 64);
}

// The first and past the last set of `n` flags of 0 or not, `stride` apart, in lines
// l0 .. l1 `line` apart; (n, 0) where none is.  By a wave.
__device__ __forceinline__ void flagged(const unsigned char* f, int n, long long stride, int l0, int l1, long long line, int* lo, int* hi) {
    const int lane = threadIdx.x & 63;
    *lo = n, *hi = 0;
    for (int w = 0; w < n; w += 64) {
        int any = 0;
        if (w + lane < n)
            for (int l = l0; l <= l1; ++l) any |= f[(w + lane) * stride + l * line];
        const unsigned long long set = __ballot(any);
        if (!set) continue;
        if (*hi == 0) *lo = w + __builtin_ctzll(set);
        *hi = w + 64 - __builtin_clzll(set);
    }
}
// A mask's part of the keys [lo, hi) that the queries i0 .. i1 read.
__device__ __forceinline__ void by_mask(const AttnArgs& a, const Keys& keys, int b, int i0, int i1, int* lo, int* hi) {
    if (!a.any) return;
    const int blocks = (a.tq + 31) / 32;
    int w0, w1;
    flagged(a.any + (a.bits_batch ? (long long)b * blocks * a.words : 0), a.words, 1, i0 / 32, i1 / 32, a.words, &w0, &w1);
    const int end = w1 ? keys.first + 32 * w1 : keys.first, from = keys.first + 32 * w0;
    if (end < *hi) *hi = end;
    if (keys.first <= 0 && from > *lo) *lo = from;
}

// 32 bits of a mask's line from `rel` on: ones before it, zeros past it.  The line
// begins `line` words (below 2^30) from `bits`.  The two words are loaded a tile
// ahead (`load`, then `landed` where the tile's own loads have), as a wait for them
// where they are used would be one for the next tile's loads as well.
struct MaskBits {
    unsigned lo, hi;
    __device__ __forceinline__ void load(const unsigned* bits, unsigned line, int words, int rel) {
        const int q = rel >> 5;
        auto word = [&](int w) { return *(const unsigned*)((const char*)bits + 4u * (line + (unsigned)(w < 0 ? 0 : w < words ? w : words - 1))); };
        lo = word(q);
        hi = word(q + 1);
    }
    __device__ __forceinline__ void landed() { asm volatile("" : "+v"(lo), "+v"(hi)); }
    __device__ __forceinline__ unsigned at(int words, int rel) const {
        const int q = rel >> 5;
        const unsigned a = q < 0 ? ~0u : q < words ? lo : 0u, b = q + 1 < 0 ? ~0u : q + 1 < words ? hi : 0u;
        return (unsigned)(((unsigned long long)b << 32 | a) >> (rel & 31));
    }
};

// Bits [lo, hi) of 32.
__device__ __forceinline__ unsigned range_of(int lo, int hi) {
    const unsigned from = lo <= 0 ? ~0u : lo < 32 ? ~0u << lo : 0u, to = hi >= 32 ? ~0u : hi > 0 ? ~0u >> (32 - hi) : 0u;
    return from & to;
}
// x where bit row_of(e, h) of a lane's 32 is set, else `no`; `bits` are shifted by 4 h.
__device__ __forceinline__ float where_bit(unsigned bits, int e, float x, float no) {
    const int m = (int)(bits << (31 - 8 * (e >> 2) - (e & 3))) >> 31;
    return __builtin_bit_cast(float, (m & __builtin_bit_cast(int, x)) | (~m & __builtin_bit_cast(int, no)));
}

// Work order: workgroups are dealt to the 8 XCDs round robin; each takes one
// run of items, so that those of a head share its keys in one L2.
__device__ __forceinline__ unsigned item_of(unsigned id, unsigned total) {
    const unsigned xcd = id % 8, q8 = total / 8, r8 = total % 8;
    return xcd * q8 + (xcd < r8 ? xcd : r8) + id / 8;
}

// Item `unit` of the heads, `n` of them a key head: a key head's of all sequences
// after each other, so that an XCD's run has sequences of different lengths (8 of
// 704 to 2048 keys, 32 heads in groups of four, all keys: 555 -> 481 us, the
// gradients 1740 -> 1510; 8 of 128 to 1024, 16 heads: 84 -> 67, 261 -> 216).
__device__ __forceinline__ void head_of(const AttnArgs& a, int unit, int n, int* b, int* hk, int* head) {
    const int at = unit / n;
    *b = at % a.batch;
    *hk = at / a.batch;
    *head = *hk * n + unit % n;
}

// A share of a sequence's keys and its key head, of workgroups that have the whole
// group's rows: a share's heads, whose rows lie beside each other, on one XCD; a
// sequence's shares on different ones, a longer sequence's last ones in the end (32
// sequences of 2048 to 8192 keys, 8 key heads x 128: 150 us where an XCD has a run
// of a head's shares, 140 a run of a sequence's, 132 so).
__device__ __forceinline__ void share_of(const AttnArgs& a, unsigned id, int* b, int* hk, int* split) {
    const unsigned kv = (unsigned)a.kv, batch = (unsigned)a.batch, rounds = batch * (unsigned)a.splits / 8, whole = 8 * rounds * kv;
    const unsigned at = id < whole ? id / 8 : id - whole;
    const unsigned share = id < whole ? at / kv * 8 + id % 8 : 8 * rounds + at / kv;
    *hk = (int)(at % kv);
    *split = (int)(share / batch);
    *b = (int)((share % batch + batch - (unsigned)*split % batch) % batch);
}

// The place of an item among its XCD's.
__device__ __forceinline__ unsigned turn_of(unsigned item, unsigned total) {
    const unsigned q8 = total / 8, r8 = total % 8, more = r8 * (q8 + 1);      // (the items of the XCDs that have one more)
    return item < more ? item % (q8 + 1) : (item - more) % q8;
}

// Split `split` of the keys [lo, hi): `chunk` of them, the same for sequences of
// any length, so that its workgroups take equally long or have nothing to do.
__device__ __forceinline__ void cut(const AttnArgs& a, int split, int* lo, int* hi) {
    const long long from = *lo + (long long)split * a.chunk, to = from + a.chunk;
    *hi = to < *hi ? (int)to : *hi;
    *lo = from < *hi ? (int)from : *hi;
}

// ---- the value ----------------------------------------------------------------------

// Sums to and from LDS as a wave's lanes hold them, 16 bytes a lane at a time.
template <int ND>
__device__ __forceinline__ void give(unsigned char* at, int lane, const f32x16 (&acc)[ND], bool now) {
    if (!now) return;
    f32x4* const to = (f32x4*)at + lane;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) to[64 * (4 * dt + g)] = f32x4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
}
// acc = f acc + g (those)
template <int ND>
__device__ __forceinline__ void take(const unsigned char* at, int lane, f32x16 (&acc)[ND], float f, float g) {
    const f32x4* const from = (const f32x4*)at + lane;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 x = from[64 * (4 * dt + q)];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[dt][4 * q + e] = acc[dt][4 * q + e] * f + x[e] * g;
        }
}

// One workgroup: 128 rows of a head (of a group's heads beside each other), 32 a
// wave, over the keys that any of them reads, or a share of those.  SW 2: eight
// waves, two of which share 32 rows and take half of each tile's keys each.
// Bound by the matrix instructions, 42 % of the cycles, and the softmax's vector
// instructions, nearly as many, of which two waves a SIMD hide a part: 4 x 32 heads x 4096 x 128 in
// bf16, causal, 670 to 700 us, 800 TFLOP/s of the two products (all keys 895; a
// large library product 1149); 32 heads x 2048 x 128 55 us.  Of a small call a
// third is a launch, the first loads and the last stores (2 x 12 heads x 1024 x 64
// with a mask 20 us, of which 8 with no tile at all).
template <int ST, int ND, int SW>
__global__ void __launch_bounds__(256 * SW, ST == kF32 && ND >= 4 ? 1 : 2) attn_fwd_kernel(AttnArgs a) {
    typedef Geo<ST, ND> G;
    constexpr int TILE = G::TILE;
    typedef Rows<ST, ND, TILE, 256 * SW> Tile;
    constexpr int NB = TILE / 32 / SW;
    static_assert(NB >= 1, "a tile has a block for each");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[4 * Tile::BYTES + (SW == 2 ? 2048 : 0)];
    constexpr int PAIR = SW == 2 ? 4096 * ND : 32 * G::ROW;     // of LDS for the waves of the same rows
    static_assert(4 * Tile::BYTES >= 4 * PAIR, "the waves' sums in LDS");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;

    const int rw = wave & 3, kw = wave >> 2;      // which rows, and which of a tile's keys
    const int rows = a.tq * a.pack, tiles = (rows + kAttnTile - 1) / kAttnTile;
    const unsigned item = item_of(blockIdx.x, gridDim.x);
    const int split = (int)(item % (unsigned)a.splits);
    const unsigned at = item / (unsigned)a.splits;
    // a head's tiles from the last on, the longest ones first where they are causal
    // (where all workgroups are on the chip at once, two a CU, the heads that begin
    // past an XCD's first 32 from the first on, so that a CU has a long one and a short
    // one: 32 heads x 2048 x 128, causal, 71 -> 62 us)
    const int unit = (int)(at / (unsigned)tiles);
    const int turn = (int)(at % (unsigned)tiles);
    const bool second = SW == 1 && gridDim.x <= 512 && turn_of((unsigned)unit * (unsigned)(tiles * a.splits), gridDim.x) >= 32;
    const int tile = second ? turn : tiles - 1 - turn;
    int b, hk, hx;
    head_of(a, unit, a.per / a.pack, &b, &hk, &hx);
    const int r0 = tile * kAttnTile, r1 = (rows < r0 + kAttnTile ? rows : r0 + kAttnTile) - 1;

    Keys keys;
    keys.init(a, b);
    const int ifirst = r0 / a.pack, ilast = r1 / a.pack;
    int klo = keys.lo(a, ifirst), khi = keys.hi(a, ilast);
    by_mask(a, keys, b, ifirst, ilast, &klo, &khi);
    const int surelo = keys.lo(a, ilast), surehi = keys.sure(a, ifirst);
    int nt = khi > klo ? (khi - klo + TILE - 1) / TILE : 0;
    if (a.splits > 1) {
        cut(a, split, &klo, &khi);
        nt = khi > klo ? (khi - klo + TILE - 1) / TILE : 0;
    }

    // this lane's row
    const int r = r0 + rw * 32 + (lane & 31);
    const bool live = r < rows;
    const int i = (live ? r : r1) / a.pack, head = hx * a.pack + (live ? r : r1) % a.pack;
    const int rlo = keys.lo(a, i), rhi = keys.hi(a, i);
    const unsigned line = (unsigned)((b * a.bits_batch + i) * a.words);

    Tile kt, vt;
    const unsigned lds = (unsigned)(size_t)(lds_void_t*)smem;
    kt.init(a.k, b, hk, a.d, tid, lds);
    vt.init(a.v, b, hk, a.d, tid, lds + Tile::BYTES);
    auto fetch = [&](int t) {
        const unsigned stage = (unsigned)(t & 1) * 2 * Tile::BYTES;
        const int k0 = klo + t * TILE;
        kt.issue(k0, khi - k0, stage, smem, tid);
        vt.issue(k0, khi - k0, stage, smem + Tile::BYTES, tid);
    };
    unsigned char* const own = smem + wave * 32 * G::ROW;   // the wave's part of LDS where no tile is
    Part<ST> q[G::KSTEPS];
    load_kept<ST, ND>(a.q, b, i, head, a.d, live, lane, own, q);
    if (!a.q.vec) __syncthreads();
    if (nt > 0) fetch(0);

    f32x16 o[1][ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[0][dt] = f32x16{};
    float m = -INFINITY, l = 0.f;       // in log 2; this lane's part of the sum
    // what any of the wave's rows reads
    const int w0 = r0 + rw * 32, w1 = w0 + 31 < r1 ? w0 + 31 : r1;
    const int wlo = keys.lo(a, (w0 < r1 ? w0 : r1) / a.pack), whi = w0 <= r1 ? keys.hi(a, w1 / a.pack) : 0;

    Places<ST, ND> places;
    places.init(lane);
    places = places.from(lds);
    MaskBits ahead[NB], now[NB];
    auto load_bits = [&](int t) {
        if (a.cols)
#pragma unroll
            for (int kb = 0; kb < NB; ++kb) ahead[kb].load(a.bits, line, a.words, klo + t * TILE + (kw * NB + kb) * 32 - keys.first);
    };
    auto body = [&](bool masked, int t) {
        const int k0 = klo + t * TILE;
        const Places<ST, ND> at = places.from((unsigned)((t & 1) * 2 * Tile::BYTES + kw * NB * 32 * G::ROW));
        f32x16 s[NB];
        bool any[NB];
        float mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
            const int base = k0 + (kw * NB + kb) * 32;
            unsigned bits = ~0u;
            any[kb] = true;
            if (masked) {
                // keys that no row of the wave reads are passed over
                any[kb] = base < whi && base + 32 > wlo;
                if (any[kb] && a.cols) {
                    bits = now[kb].at(a.words, base - keys.first);
                    any[kb] = __any(bits);
                }
                if (!any[kb]) continue;
            }
            s[kb] = f32x16{};
#pragma unroll
            for (int st = 0; st < G::KSTEPS; ++st) s[kb] = mma_row<ST>(part_of(frag_row<ST>(at.row, st, kb * 32 * G::ROW)), q[st], s[kb]);
            if (masked) {
                bits = (bits & range_of(rlo - base, rhi - base)) >> (4 * h);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[kb][e] = where_bit(bits, e, s[kb][e], -INFINITY);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][e]);
        }
        mx = fmaxf(mx, partner<32>(mx)) * a.c;
        // the sums stay at an older maximum until one passes it by 2^8
        if (__any(mx > m + 8.f)) {
            const float top = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - base_of(top));
            m = top;
            l *= f;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[0][dt][e] *= f;
        }
        const float base = base_of(m);
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
            if (!any[kb]) continue;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[kb][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e], a.c, -base));
                sum += s[kb][e];
            }
            l += sum;
            Weights<ST> w[1];
            w[0].set(s[kb]);
            mma_col<ST, ND, 1>(at.col, Tile::BYTES + kb * 32 * G::ROW, w, o);
        }
    };
    if (nt > 0) load_bits(0);
    for (int t = 0; t < nt; ++t) {
        wait_vm<0>();
        if (a.cols)
#pragma unroll
            for (int kb = 0; kb < NB; ++kb) {
                ahead[kb].landed();
                now[kb] = ahead[kb];
            }
        __syncthreads();
        if (t + 1 < nt) {
            fetch(t + 1);
            load_bits(t + 1);
        }
        const int k0 = klo + t * TILE;
        body(k0 < surelo || k0 + TILE > surehi, t);
    }

    l += partner<32>(l);
    unsigned char* const pair = smem + rw * PAIR;      // the LDS of the waves of the same rows
    if constexpr (SW == 2) {
        // their sums meet
        __syncthreads();
        give<ND>(pair, lane, o[0], kw == 1);
        float* const mls = (float*)(smem + 4 * PAIR) + 128 * rw + lane;
        if (kw == 1) mls[0] = m, mls[64] = l;
        __syncthreads();
        if (kw == 1) return;    // (no barrier follows)
        const float m1 = mls[0], l1 = mls[64], top = fmaxf(m, m1), base = base_of(top);
        const float f0 = __builtin_amdgcn_exp2f(m - base), f1 = __builtin_amdgcn_exp2f(m1 - base);
        take<ND>(pair, lane, o[0], f0, f1);
        m = top;
        l = l * f0 + l1 * f1;
    } else {
        __syncthreads();
    }
    const long long row = ((long long)b * a.heads + head) * a.tq + i;
    if (a.splits > 1) {
        const long long all = (long long)a.batch * a.heads * a.tq, n = (long long)split * all + row;
        if (live && h == 0) *(f32x2*)(a.part_ml + 2 * n) = f32x2{m, l};
        if (live && l != 0.f) {     // (the join reads no sums of a row without keys)
            float* const out = a.part + n * (ND * 32);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *(f32x4*)(out + dt * 32 + 8 * g + 4 * h) = f32x4{o[0][dt][4 * g], o[0][dt][4 * g + 1], o[0][dt][4 * g + 2], o[0][dt][4 * g + 3]};
        }
        return;
    }
    store_kept<ST, ND, false>(o[0], l == 0.f ? 0.f : 1.f / l, a.d, a.o.vec, live, [&](int n) -> const void* {
        const int x = r0 + rw * 32 + n;
        return x < rows ? row_at<ST>(a.o, b, x / a.pack, hx * a.pack + x % a.pack) : nullptr;
    }, pair, lane, a.flag);
    if (a.lse && live && h == 0) a.lse[row] = l == 0.f ? -INFINITY : (base_of(m) + __builtin_log2f(l)) * kLn2;
}

// The sum in place `at` of a row's (dt, row_of) as an element of the head.
template <int ST, int ND>
__device__ __forceinline__ bool put(void* row, int at, int d, float v) {
    const int e = ST == kF32 ? ND * (at & 31) + (at >> 5) : at;
    if (e >= d) return false;
    if constexpr (ST == kF32) ((float*)row)[e] = v;
    else if constexpr (ST == kBF16) ((unsigned short*)row)[e] = pk_f32_to_bf16(v);
    else ((unsigned short*)row)[e] = pk_f32_to_f16(v);
    return ST == kF16 && pk_overflows_f16(v);
}

// Few rows (a group's heads beside each other, 32 at most) over many keys: all
// of a workgroup's NW waves have the same rows, and blocks of 32 keys in turn,
// which each loads for itself two at a time, so that no wave waits for another
// until their sums meet in LDS at the end.  Bound by reading the keys and values:
// 32 sequences of 2048 to 8192, 8 key heads x 128 in bf16, 132 us, 5.2 TB/s (a large
// copy reads and writes 4.9).
template <int ST, int ND, int NW>
__global__ void __launch_bounds__(64 * NW, 1) attn_few_kernel(AttnArgs a) {
    typedef Geo<ST, ND> G;
    typedef Rows<ST, ND, 32, 64> Tile;
    constexpr int STAGE = 2 * Tile::BYTES, WAVE = 2 * STAGE, NL = 2 * Tile::ROUNDS;
    static_assert(ND * 4096 <= WAVE, "a wave's sums in its part of LDS");
    __shared__ __attribute__((aligned(1024))) unsigned char smem[NW * WAVE];
    __shared__ float ml[NW][32][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;

    const int rows = a.tq * a.pack;
    int b, hk, split;
    share_of(a, blockIdx.x, &b, &hk, &split);

    Keys keys;
    keys.init(a, b);
    int klo = keys.lo(a, 0), khi = keys.hi(a, a.tq - 1);
    const int surelo = keys.lo(a, a.tq - 1), surehi = keys.sure(a, 0);
    cut(a, split, &klo, &khi);
    const int nblk = khi > klo ? (khi - klo + 31) / 32 : 0, nt = (nblk - wave + NW - 1) / NW;

    Tile kt, vt;
    const unsigned lds = (unsigned)(size_t)(lds_void_t*)smem + (unsigned)(wave * WAVE);
    unsigned char* const own = smem + wave * WAVE;
    kt.init(a.k, b, hk, a.d, lane, lds);
    vt.init(a.v, b, hk, a.d, lane, lds + Tile::BYTES);
    auto fetch = [&](int t) {
        const unsigned stage = (unsigned)(t & 1) * STAGE;
        const int k0 = klo + (t * NW + wave) * 32;
        kt.issue(k0, khi - k0, stage, own, lane);
        vt.issue(k0, khi - k0, stage, own + Tile::BYTES, lane);
    };

    // this lane's row
    const int r = lane & 31;
    const bool live = r < rows;
    const int i = live ? r / a.pack : a.tq - 1, head = hk * a.pack + (live ? r % a.pack : 0);
    const int rlo = keys.lo(a, i), rhi = keys.hi(a, i);
    const unsigned line = (unsigned)((b * a.bits_batch + i) * a.words);
    Part<ST> q[G::KSTEPS];
    if (!a.q.vec) {
        load_kept<ST, ND>(a.q, b, i, head, a.d, live, lane, own, q);
        __builtin_amdgcn_s_waitcnt(0xc07f);     // LDS: the reads are done before a tile lands there
        if (nt > 0) fetch(0);
    } else {
        if (nt > 0) fetch(0);
        load_kept<ST, ND>(a.q, b, i, head, a.d, live, lane, own, q);
    }
    const bool whole = a.k.vec && a.v.vec;

    f32x16 o[1][ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[0][dt] = f32x16{};
    float m = -INFINITY, l = 0.f;
    Places<ST, ND> places;
    places.init(lane);
    places = places.from(lds);
    for (int t = 0; t < nt; ++t) {
        __builtin_amdgcn_s_waitcnt(0xc07f);     // LDS: the last block's reads are done before its stage is loaded again
        if (t + 1 < nt) fetch(t + 1);
        if (t + 1 < nt && whole) wait_vm<NL>();
        else wait_vm<0>();
        const int k0 = klo + (t * NW + wave) * 32;
        const Places<ST, ND> at = places.from((unsigned)(t & 1) * STAGE);
        f32x16 s = f32x16{};
#pragma unroll
        for (int st = 0; st < G::KSTEPS; ++st) s = mma_row<ST>(part_of(frag_row<ST>(at.row, st)), q[st], s);
        if (k0 < surelo || k0 + 32 > surehi) {
            unsigned bits = ~0u;
            if (a.cols && k0 + 32 > keys.first) {
                MaskBits m;
                m.load(a.bits, line, a.words, k0 - keys.first);
                bits = m.at(a.words, k0 - keys.first);
            }
            bits = (bits & range_of(rlo - k0, rhi - k0)) >> (4 * h);
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = where_bit(bits, e, s[e], -INFINITY);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[e]);
        mx = fmaxf(mx, partner<32>(mx)) * a.c;
        if (__any(mx > m + 8.f)) {
            const float top = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - base_of(top));
            m = top;
            l *= f;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[0][dt][e] *= f;
        }
        const float base = base_of(m);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], a.c, -base));
            sum += s[e];
        }
        l += sum;
        Weights<ST> w[1];
        w[0].set(s);
        mma_col<ST, ND, 1>(at.col, Tile::BYTES, w, o);
    }
    l += partner<32>(l);

    // the waves' sums, each in the wave's own part of LDS as its lanes hold them
    f32x4* const sums = (f32x4*)own + lane;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) sums[64 * (4 * dt + g)] = f32x4{o[0][dt][4 * g], o[0][dt][4 * g + 1], o[0][dt][4 * g + 2], o[0][dt][4 * g + 3]};
    if (h == 0) ml[wave][r][0] = m, ml[wave][r][1] = l;
    __syncthreads();
    float top = -INFINITY, f[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, ml[w][r][0]);
    const float base = base_of(top);
    l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        f[w] = __builtin_amdgcn_exp2f(ml[w][r][0] - base);
        l += ml[w][r][1] * f[w];
    }
    const long long all = (long long)a.batch * a.heads * a.tq, row = ((long long)b * a.heads + head) * a.tq + i, n = split * all + row;
    if (wave == 0 && h == 0 && live) {
        if (a.splits > 1) *(f32x2*)(a.part_ml + 2 * n) = f32x2{top, l};
        else if (a.lse) a.lse[row] = l == 0.f ? -INFINITY : (base + __builtin_log2f(l)) * kLn2;
    }
    if (a.splits > 1 && l == 0.f) return;       // (the join reads no sums of it; no barrier follows)
    const float whole_f = l == 0.f ? 0.f : 1.f / l;
    void* const out = live ? const_cast<void*>(row_at<ST>(a.o, b, i, head)) : nullptr;
    bool ovf = false;
    for (int x = wave; x < 4 * ND; x += NW) {
        f32x4 v = f32x4{};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const f32x4 y = ((const f32x4*)(smem + w * WAVE) + lane)[64 * x];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += y[e] * f[w];
        }
        const int at = (x >> 2) * 32 + 8 * (x & 3) + 4 * h;     // its place among a row's sums
        if (!live) continue;
        if (a.splits > 1) {
            *(f32x4*)(a.part + n * (ND * 32) + at) = v;
            continue;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) ovf |= put<ST, ND>(out, at + e, a.d, v[e] * whole_f);
    }
    if (ovf && a.flag) atomicOr(a.flag, 1u);
}

// The splits' sums of a row joined, in order: by a wave (64 lanes, ND / 2 elements a
// lane), or, of many splits, by a workgroup's four, every fourth of them each.  A
// lane takes a split's maximum and sum, then all lanes the sums of those splits
// that have any, four loads at a time on the way.
template <int ST, int ND, int WAVES>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a) {
    constexpr int E = ND / 2;
    typedef float V __attribute__((ext_vector_type(E)));
    __shared__ float sums[4][ND * 32], sl[4];
    const long long all = (long long)a.batch * a.heads * a.tq;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long long row = WAVES == 4 ? blockIdx.x : (long long)blockIdx.x * 4 + wave;
    if (row >= all) return;
    const f32x2* const mls = (const f32x2*)a.part_ml + row;
    const int first = WAVES == 4 ? wave : 0;
    f32x2 ml = f32x2{-INFINITY, 0.f};
    if (first + WAVES * lane < a.splits) ml = mls[(first + WAVES * lane) * all];
    float m = ml[0];
    for (int s = WAVES == 4 ? lane : lane + 64; s < a.splits; s += 64) m = fmaxf(m, mls[s * all][0]);
    m = all_of<64>(m, nullptr, max_f);
    const float base = base_of(m);
    float l = 0.f, x[E];
#pragma unroll
    for (int q = 0; q < E; ++q) x[q] = 0.f;
    for (int s0 = first; s0 < a.splits; s0 += 64 * WAVES) {
        if (s0 > first) ml = s0 + WAVES * lane < a.splits ? mls[(s0 + WAVES * lane) * all] : f32x2{-INFINITY, 0.f};
        const float f = __builtin_amdgcn_exp2f(ml[0] - base);
        l += ml[1] * f;
        // (a split without keys has no sums)
        for (unsigned long long have = __ballot(ml[1] != 0.f); have;) {
            const int n = __builtin_popcountll(have);
            V v[4];
            float g[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = __builtin_ctzll(have);
                g[j] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), k));
                v[j] = *((const V*)(a.part + ((s0 + WAVES * k) * all + row) * (ND * 32)) + lane);
                if (j < 3 && j + 1 < n) have &= have - 1;
            }
            have &= have - 1;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < n)
#pragma unroll
                    for (int q = 0; q < E; ++q) x[q] += v[j][q] * g[j];
        }
    }
    l = all_of<64>(l, nullptr, add_f);
    const int i = (int)(row % a.tq), head = (int)(row / a.tq % a.heads), b = (int)(row / a.tq / a.heads);
    void* const out = const_cast<void*>(row_at<ST>(a.o, b, i, head));
    bool ovf = false;
    if constexpr (WAVES == 4) {
#pragma unroll
        for (int q = 0; q < E; ++q) sums[wave][E * lane + q] = x[q];
        if (lane == 0) sl[wave] = l;
        __syncthreads();
        l = sl[0] + sl[1] + sl[2] + sl[3];
    }
    const float f = l == 0.f ? 0.f : 1.f / l;
    if constexpr (WAVES == 4) {
        for (int at = threadIdx.x; at < ND * 32; at += 256)
            ovf |= put<ST, ND>(out, at, a.d, (sums[0][at] + sums[1][at] + sums[2][at] + sums[3][at]) * f);
    } else {
#pragma unroll
        for (int q = 0; q < E; ++q) ovf |= put<ST, ND>(out, E * lane + q, a.d, x[q] * f);
    }
    if (ovf && a.flag) atomicOr(a.flag, 1u);
    if (a.lse && (WAVES == 4 ? threadIdx.x : lane) == 0) a.lse[row] = l == 0.f ? -INFINITY : (base + __builtin_log2f(l)) * kLn2;
}

// ---- the gradients --------------------------------------------------------------------

// A row's -lse log2 e, and behind all of them its -sum do o.  16 lanes a row.  One
// pass over o and do: 4 x 4096 x 32 x 128 in bf16 57 us, 4.7 TB/s.
template <int ST>
__global__ void __launch_bounds__(256) attn_rows_kernel(AttnArgs a) {
    const long long all = (long long)a.batch * a.heads * a.tq, row = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool live = row < all;
    const long long n = live ? row : all - 1;
    // heads innermost: the rows of a position lie together
    const int head = (int)(n % a.heads), i = (int)(n / a.heads % a.tq), b = (int)(n / a.heads / a.tq);
    const int lane = threadIdx.x & 15;
    const void* const x = row_at<ST>(a.dout, b, i, head);
    const void* const y = row_at<ST>(a.o, b, i, head);
    float s = 0.f;
    constexpr int EPC = ST == kF32 ? 4 : 8;
    for (int c = lane; c * EPC < a.d; c += 16) {
        typedef typename FragOf<ST>::T F;
        const F u = a.dout.vec ? *(const F*)((const char*)x + 16 * c) : chunk_of<ST>(x, c, a.d, true);
        const F v = a.o.vec ? *(const F*)((const char*)y + 16 * c) : chunk_of<ST>(y, c, a.d, true);
#pragma unroll
        for (int e = 0; e < EPC; ++e) {
            if constexpr (ST == kF32) s += u[e] * v[e];
            else if constexpr (ST == kBF16) s += pk_bf16_to_f32(u[e]) * pk_bf16_to_f32(v[e]);
            else s += pk_f16_to_f32(u[e]) * pk_f16_to_f32(v[e]);
        }
    }
    s = all_of<16>(s, nullptr, add_f);
    if (live && lane == 0) {
        const long long at = ((long long)b * a.heads + head) * a.tq + i;
        const float lse = a.lse[at];
        // (a row that reads nothing: its weights are zero by the keys it may read)
        a.rows[at] = -base_of(lse) * kLog2e;
        a.rows[all + at] = -s;
    }
}

// In f16 the weights, most of them far below one, enter their product times 2^8.
constexpr float kShift = 8.f;
// Their cotangents, of whatever size the gradient's are (a mean loss's 10^-4 left
// them f16's last bits, and the gradients 4 times the error), times a power of two of
// the wave's own, 2^up: as large a one as leaves the largest so far below 2^15 (those
// of 2^-22 of it and more are whole), and one at least, so that those past f16 still
// show.  As with a softmax's maximum, the sums go along with it where it has to fall,
// then by so much that the largest is past 2^8.  (Gradients of 4 x 32 heads in groups
// of four x 4096 x 128, causal: 2400 us without it, 2540 so, 2730 with a power for each
// kept row, which takes registers; shorter ones 2 to 8 % more than without.)
constexpr int kUp = 60;     // (2^60 times the largest of them, 2^41, stays in f32)
template <int ND>
__device__ __forceinline__ void fit_f16(f32x16& s, f32x16 (&acc)[ND], int& up, bool live) {
    float mx = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, __builtin_fabsf(s[e]));
    // (a lane without a row has scores of 0, and weights of any size)
    mx = live ? mx : 0.f;
    if (up == 0 || !__any(mx > 32768.f)) return;
    const unsigned top = __builtin_amdgcn_readfirstlane(__builtin_bit_cast(unsigned, all_of<64>(mx, nullptr, max_f)));
    const int by = max(135 - (int)(top >> 23), -up);
    const float f = __builtin_ldexpf(1.f, by);
    up += by;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] *= f;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] *= f;
}
// The sums as they are.
template <int ND>
__device__ __forceinline__ void unfit_f16(f32x16 (&acc)[ND], int up) {
    const float f = __builtin_ldexpf(1.f, -up);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[dt][e] *= f;
}

// The queries' gradient: as the value's kernel, with the cotangent's rows beside
// the queries' (4 x 32 heads x 4096 x 128, causal, 840 to 880 us, 960 TFLOP/s of the
// three products, where a large library product has 1149).  Rows of a group's heads
// stand beside each other where a head's do not fill a workgroup, as there.
template <int ST, int ND, int SW>
constexpr int dq_lds() { return 4 * Rows<ST, ND, Geo<ST, ND>::TILE, 256 * SW>::BYTES; }
template <int ST, int ND, int SW>
__device__ __forceinline__ void dq_of(const AttnArgs& a, unsigned id, unsigned total, unsigned char* smem) {
    typedef Geo<ST, ND> G;
    constexpr int TILE = G::TILE;
    typedef Rows<ST, ND, TILE, 256 * SW> Tile;
    constexpr int NB = 1;
    constexpr int WROWS = 32 * NB, ROWS = 4 * WROWS, PAIR = SW == 2 ? 4096 * ND : 32 * G::ROW;
    static_assert(4 * Tile::BYTES >= 4 * PAIR, "the waves' sums in LDS");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;

    const int rw = wave & 3, kw = wave >> 2;      // which rows, and which of a tile's keys
    const int rows = a.tq * a.pack, tiles = (rows + ROWS - 1) / ROWS;
    const unsigned at = item_of(id, total);
    const int tile = tiles - 1 - (int)(at % (unsigned)tiles), unit = (int)(at / (unsigned)tiles);
    int b, hk, hx;
    head_of(a, unit, a.per / a.pack, &b, &hk, &hx);
    const int r0 = tile * ROWS, r1 = (rows < r0 + ROWS ? rows : r0 + ROWS) - 1;

    Keys keys;
    keys.init(a, b);
    const int ifirst = r0 / a.pack, ilast = r1 / a.pack;
    int klo = keys.lo(a, ifirst), khi = keys.hi(a, ilast);
    by_mask(a, keys, b, ifirst, ilast, &klo, &khi);
    const int surelo = keys.lo(a, ilast), surehi = keys.sure(a, ifirst);
    const int nt = khi > klo ? (khi - klo + TILE - 1) / TILE : 0;

    Tile kt, vt;
    const unsigned lds = (unsigned)(size_t)(lds_void_t*)smem;
    kt.init(a.k, b, hk, a.d, tid, lds);
    vt.init(a.v, b, hk, a.d, tid, lds + Tile::BYTES);
    auto fetch = [&](int t) {
        const unsigned stage = (unsigned)(t & 1) * 2 * Tile::BYTES;
        const int k0 = klo + t * TILE;
        kt.issue(k0, khi - k0, stage, smem, tid);
        vt.issue(k0, khi - k0, stage, smem + Tile::BYTES, tid);
    };
    unsigned char* const own = smem + wave * 32 * G::ROW;   // the wave's part of LDS where no tile is

    const int w0 = r0 + rw * WROWS, w1 = w0 + WROWS - 1 < r1 ? w0 + WROWS - 1 : r1;
    const int wfirst = (w0 < r1 ? w0 : r1) / a.pack, wlast = w1 / a.pack;
    const int wlo = keys.lo(a, wfirst), whi = w0 <= r1 ? keys.hi(a, wlast) : 0;
    const bool fine = fine_of<ST>(a, keys, wfirst, wlast);
    // this lane's row
    const bool live = w0 + (lane & 31) <= r1;
    const int mine = live ? w0 + (lane & 31) : r1, i = mine / a.pack, head = hx * a.pack + mine % a.pack;
    Part<ST> q[NB][G::KSTEPS], dout[NB][G::KSTEPS];
    float lse[NB], delta[NB];
    f32x16 dq[NB][ND];
    int up = kUp;       // (f16)
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        load_kept<ST, ND>(a.q, b, i, head, a.d, live, lane, own, q[n]);
        load_kept<ST, ND>(a.dout, b, i, head, a.d, live, lane, own, dout[n]);
        const float* const x = a.rows + ((long long)b * a.heads + head) * a.tq + i;
        lse[n] = x[0], delta[n] = x[(long long)a.batch * a.heads * a.tq];
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) dq[n][dt] = f32x16{};
    }
    if (!a.q.vec || !a.dout.vec) __syncthreads();
    if (nt > 0) fetch(0);

    Places<ST, ND> places;
    places.init(lane);
    places = places.from(lds);
    constexpr int MINE = TILE / 32 / SW;     // blocks of a tile that are the wave's
    MaskBits ahead[MINE], now[MINE];
    const unsigned line = (unsigned)((b * a.bits_batch + i) * a.words);
    auto load_bits = [&](int t) {
        if (a.cols)
#pragma unroll
            for (int x = 0; x < MINE; ++x) ahead[x].load(a.bits, line, a.words, klo + t * TILE + (kw + SW * x) * 32 - keys.first);
    };
    auto body = [&](bool masked, int t, int kb) {
        const int base = klo + t * TILE + kb * 32;
        const Places<ST, ND> at = places.from((unsigned)((t & 1) * 2 * Tile::BYTES + kb * 32 * G::ROW));
        unsigned bits[NB];
        if (masked) {
            // keys that no row of the wave reads are passed over
            if (base >= whi || base + 32 <= wlo) return;
            bits[0] = ~0u;
            if (a.cols) bits[0] = (MINE == 1 || kb < SW ? now[0] : now[MINE - 1]).at(a.words, base - keys.first);
            if (!__any(bits[0])) return;
        }
        f32x16 s[NB], dp[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n] = dp[n] = f32x16{};
#pragma unroll
        for (int st = 0; st < G::KSTEPS; ++st) {
            const auto fk = frag_row<ST>(at.row, st), fv = frag_row<ST>(at.row, st, Tile::BYTES);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                s[n] = mma_row<ST>(part_of(fk), q[n][st], s[n]);
                dp[n] = mma_row<ST>(part_of(fv), dout[n][st], dp[n]);
            }
        }
        Weights<ST> w[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const float row = ST == kF16 ? lse[n] + (float)up : lse[n];
#pragma unroll
            for (int e = 0; e < 16; ++e) s[n][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][e], a.c, row)) * (dp[n][e] + delta[n]);
            if (masked) {
                const unsigned in = (bits[n] & range_of(keys.lo(a, i) - base, keys.hi(a, i) - base)) >> (4 * h);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[n][e] = where_bit(in, e, s[n][e], 0.f);
            }
            if (ST == kF16) fit_f16<ND>(s[n], dq[n], up, live);
            w[n].set(s[n]);
        }
        mma_col<ST, ND, NB, ST == kF32>(at.col, 0, w, dq);
        if constexpr (ST != kF32)
            if (fine) {
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    left_in<ST>(s[n], w[n]);
                    w[n].set(s[n]);
                }
                mma_col<ST, ND, NB>(at.col, 0, w, dq);
            }
    };
    if (nt > 0) load_bits(0);
    for (int t = 0; t < nt; ++t) {
        wait_vm<0>();
        if (a.cols)
#pragma unroll
            for (int x = 0; x < MINE; ++x) {
                ahead[x].landed();
                now[x] = ahead[x];
            }
        __syncthreads();
        if (t + 1 < nt) {
            fetch(t + 1);
            load_bits(t + 1);
        }
        const int k0 = klo + t * TILE;
#pragma unroll 1
        for (int kb = kw; kb < TILE / 32; kb += SW) body(k0 < surelo || k0 + TILE > surehi, t, kb);
    }
    __syncthreads();
    if (ST == kF16) unfit_f16<ND>(dq[0], up);
    unsigned char* const pair = smem + rw * PAIR;      // the LDS of the waves of the same rows
    if constexpr (SW == 2) {
        give<ND>(pair, lane, dq[0], kw == 1);
        __syncthreads();
        if (kw == 1) return;
        take<ND>(pair, lane, dq[0], 1.f, 1.f);
    }
    store_kept<ST, ND, true>(dq[0], a.scale, a.d, a.dq.vec, live, [&](int x) -> const void* {
        return w0 + x <= r1 ? row_at<ST>(a.dq, b, (w0 + x) / a.pack, hx * a.pack + (w0 + x) % a.pack) : nullptr;
    }, pair, lane, a.flag);
}

// The keys' and values' gradients (DK, DV): a workgroup keeps 128 keys of a key
// head, 32 a wave, and the rows of all heads of its group that read any of them
// pass by, QT at a time.  SW 2: eight waves, two of which share 32 keys and take
// half of each tile's rows each.  VL: the values are kept in LDS, as the registers
// that two waves a SIMD have do not hold them too, and with eight waves, whose one
// workgroup a CU has the room, the keys beside them.  DQ: the queries' workgroups
// follow the `nkv` of the keys in one launch, where either would leave CUs idle
// (3 x 10 heads, 5 of keys, 777 x 1021 x 80, 120 and 210 workgroups: 38 + 18 -> 41
// us, in f16 44 with its cotangents' powers; 2 x 12 heads x 1024 x 64, 192 each:
// 27 + 24 -> 39).  With eight waves, or heads past 128, a tile's rows may be in parts
// of theirs (AttnArgs::parts), whose sums in f32 attn_sum_kernel adds.  4 x 32 heads
// in groups of four x 4096 x 128 in
// bf16, causal, 1400 to 1440 us, 775 TFLOP/s of the four products: matrix
// instructions in 40 % of the cycles, vector ones in 25, LDS in 30, each waiting for
// the others' results in turn with two waves a SIMD, which is what the registers
// hold (64 keys a wave and one wave a SIMD: 2070; waves' priorities raised for the
// products: 1490).
template <int ST, int ND, int SW, int QT, bool DK, bool DV, bool VL, int OCC, bool DQ>
__global__ void __launch_bounds__(256 * SW, OCC) attn_dkv_kernel(AttnArgs a, unsigned nkv) {
    typedef Geo<ST, ND> G;
    typedef Rows<ST, ND, QT, 256 * SW> Tile;
    constexpr int NB = 1, WKEYS = 32 * NB, KEYS = 4 * WKEYS, STAGE = 2 * Tile::BYTES + 512, PAIR = SW == 2 ? 4096 * ND : 32 * G::ROW;
    typedef Rows<ST, ND, KEYS, 256 * SW> Kept;
    constexpr bool KL = VL && SW == 2;
    constexpr int MINE_LDS = 2 * STAGE + (VL ? SW * Kept::BYTES : 0);
    __shared__ __attribute__((aligned(1024))) unsigned char smem[DQ && dq_lds<ST, ND, SW>() > MINE_LDS ? dq_lds<ST, ND, SW>() : MINE_LDS];
    if constexpr (DQ)
        if (blockIdx.x >= nkv) return dq_of<ST, ND, SW>(a, blockIdx.x - nkv, gridDim.x - nkv, smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;

    const int rw = wave & 3, kw = wave >> 2;      // which keys, and which of a tile's rows
    const int tiles = (a.tk + KEYS - 1) / KEYS;
    unsigned at = item_of(blockIdx.x, DQ ? nkv : gridDim.x);
    constexpr bool PARTS = SW == 2 || ND == 8;      // (the kernels of small launches)
    const int part = PARTS ? (int)(at % (unsigned)a.parts) : 0;
    if (PARTS) at /= (unsigned)a.parts;
    const int tile = (int)(at % (unsigned)tiles), unit = (int)(at / (unsigned)tiles);
    const int b = unit % a.batch, hk = unit / a.batch;
    const int k0 = tile * KEYS, k1 = a.tk < k0 + KEYS ? a.tk : k0 + KEYS;

    Keys keys;
    keys.init(a, b);
    // queries [ilo, ihi) read any of the keys from jlo on, below jhi
    auto queries = [&](int jlo, int jhi, int* ilo, int* ihi) {
        const int last = (jhi < keys.len ? jhi : keys.len) - 1;
        *ilo = 0, *ihi = a.tq;
        if (a.causal) {
            *ilo = jlo - keys.first > 0 ? jlo - keys.first : 0;
            if (a.window) {
                const long long e = (long long)last - keys.first + a.window;
                *ihi = (int)(e < a.tq ? e : a.tq);
            }
        }
        if (last < jlo || (a.cols && jlo >= keys.first + a.cols)) *ihi = 0;
    };
    int ilo, ihi, wlo, whi;
    queries(k0, k1, &ilo, &ihi);
    if (a.any && k0 >= keys.first && ihi > 0) {
        const int blocks = (a.tq + 31) / 32, c0 = k0 - keys.first, c1 = (k1 < keys.first + a.cols ? k1 : keys.first + a.cols) - 1 - keys.first;
        flagged(a.any + (a.bits_batch ? (long long)b * blocks * a.words : 0), blocks, a.words, c0 / 32, c1 / 32, 1, &ilo, &ihi);
        ilo *= 32;
        ihi = 32 * ihi < a.tq ? 32 * ihi : a.tq;
    }
    // tiles of rows, head after head, and of those this part's [t0, nt)
    const int nt1 = ihi > ilo ? (ihi - ilo + QT - 1) / QT : 0;
    int nt = nt1 * a.per, t0 = 0;
    int fi = ilo, fg = 0;       // the next tile's first row, and its head in the group
    if (PARTS && a.parts > 1) {
        const int share = (nt + a.parts - 1) / a.parts;
        t0 = part * share < nt ? part * share : nt;
        nt = t0 + share < nt ? t0 + share : nt;
        if (t0 < nt) fi = ilo + t0 % nt1 * QT, fg = t0 / nt1;
    }
    const int i00 = fi;
    const int jw = k0 + rw * WKEYS;      // the wave's first key
    queries(jw, jw + WKEYS < k1 ? jw + WKEYS : k1, &wlo, &whi);

    Tile qt, dt_;
    const unsigned lds = (unsigned)(size_t)(lds_void_t*)smem;
    auto fetch = [&](int t) {
        const int i0 = fi, head = hk * a.per + fg;
        const unsigned stage = (unsigned)(t & 1) * STAGE;
        fi += QT;
        if (fi >= ihi) fi = ilo, ++fg;
        if (i0 == ilo || t == t0) {
            qt.init(a.q, b, head, a.d, tid, lds);
            dt_.init(a.dout, b, head, a.d, tid, lds + Tile::BYTES);
        }
        // (rows past ihi are zeros, the cotangent's and both sums' too, and so add nothing
        // where no mask leaves them out)
        const int left = ihi - i0;
        qt.issue(i0, left, stage, smem, tid);
        dt_.issue(i0, left, stage, smem + Tile::BYTES, tid);
        if (wave < 2) {
            // (the lanes past the rows write zeros into the rest of 256 bytes)
            const float* const src = a.rows + (wave ? (long long)a.batch * a.heads * a.tq : 0) + ((long long)b * a.heads + head) * a.tq + i0;
            const i32x4 buf = buffer_of(src, (unsigned)((left < QT ? left : QT) * 4));
            asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dword %0, %1, 0 offen lds"
                         : : "v"(lane * 4), "s"(buf), "s"(__builtin_amdgcn_readfirstlane(lds + stage + 2 * Tile::BYTES + wave * 256)) : "memory", "m0");
        }
    };

    unsigned char* const own = smem + wave * 32 * G::ROW;   // the wave's part of LDS where no tile is
    typename RawOf<ST>::T k[KL ? 1 : NB][G::KSTEPS], v[VL ? 1 : NB][G::KSTEPS];
    f32x16 dk[NB][ND], dv[NB][ND];
    int up = kUp;       // of dk's (f16)
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int j = jw + 32 * n + (lane & 31);
        const bool live = j < k1 && j < keys.len;
        if (!KL) load_kept<ST, ND>(a.k, b, j, hk, a.d, live, lane, own, k[n]);
        if (DK && !VL) load_kept<ST, ND>(a.v, b, j, hk, a.d, live, lane, own, v[n]);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) dk[n][dt] = dv[n][dt] = f32x16{};
    }
    if (!a.k.vec || !a.v.vec) __syncthreads();
    if (nt > t0) {
        if (VL) {
            Kept vt;
            vt.init(a.v, b, hk, a.d, tid, lds);
            vt.issue(k0, (k1 < keys.len ? k1 : keys.len) - k0, 2 * STAGE, smem, tid);
            if (KL) {
                vt.init(a.k, b, hk, a.d, tid, lds);
                vt.issue(k0, (k1 < keys.len ? k1 : keys.len) - k0, 2 * STAGE + Kept::BYTES, smem, tid);
            }
        }
        fetch(t0);
    }

    // a mask's words of this lane's key (its rows come 32 at a time from a multiple
    // of 32 on), loaded a tile ahead as the queries' are
    constexpr int MINE = QT / 32 / SW;      // blocks of a tile that are the wave's
    const int col = jw + (lane & 31) - keys.first;
    const unsigned line = (unsigned)((b * a.bits_t_batch + (col < 0 ? 0 : col < a.cols ? col : a.cols - 1)) * a.words_t);
    unsigned ahead[MINE], now[MINE];
    auto load_bits = [&](int i0) {
        if (a.cols)
#pragma unroll
            for (int x = 0; x < MINE; ++x) {
                const int w = i0 / 32 + kw + SW * x;
                ahead[x] = *(const unsigned*)((const char*)a.bits_t + 4u * (line + (unsigned)(w < a.words_t ? w : a.words_t - 1)));
            }
    };
    // the tile's rows sub * 32 on, which are the queries i0 on
    Places<ST, ND> places;
    places.init(lane);
    places = places.from(lds);
    auto body = [&](bool masked, int t, int sub, int i0) {
        const unsigned stage = (unsigned)(t & 1) * STAGE;
        const Places<ST, ND> at = places.from(stage + (unsigned)(sub * 32 * G::ROW));
        const f32x4* const stats = (const f32x4*)(smem + stage + 2 * Tile::BYTES + 128 * sub + 16 * h);
        unsigned bits[NB];
        if (masked) {
            // rows that read none of the wave's keys are passed over
            if (i0 + 31 < wlo || i0 >= whi) return;
            bits[0] = !a.cols || col < 0 ? ~0u : col < a.cols ? MINE == 1 || sub < SW ? now[0] : now[MINE - 1] : 0u;
            if (!__any(bits[0])) return;
        }
        const unsigned kept = VL ? places.from((unsigned)(2 * STAGE + rw * WKEYS * G::ROW)).row : 0u;
        f32x16 s[NB], dp[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n] = dp[n] = f32x16{};
        // a step's reads a step ahead of its products, and no further, or the
        // registers do not hold them
        typedef typename RawOf<ST>::T F;
        F fq, fd, fv[NB], fk;
        auto read = [&](int st) {
            fq = frag_row<ST>(at.row, st);
            if (KL) fk = frag_row<ST>(kept, st, Kept::BYTES);
            if (DK) {
                fd = frag_row<ST>(at.row, st, Tile::BYTES);
                if (VL)
#pragma unroll
                    for (int n = 0; n < NB; ++n) fv[n] = frag_row<ST>(kept, st, 32 * n * G::ROW);
            }
        };
        read(0);
#pragma unroll
        for (int st = 0; st < G::KSTEPS; ++st) {
            const F cq = fq, cd = fd;
            F ck = KL ? fk : k[0][KL ? 0 : st], cv[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) cv[n] = VL ? fv[n] : v[VL ? 0 : n][st];
            // (the compiler would keep their parts, which the registers do not hold)
            if constexpr (ST == kF32) asm volatile("" : "+v"(ck.a), "+v"(ck.b), "+v"(cv[0].a), "+v"(cv[0].b));
            if (st + 1 < G::KSTEPS) read(st + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                s[n] = mma_row<ST>(part_of(cq), part_of(ck), s[n]);
                if (DK) dp[n] = mma_row<ST>(part_of(cd), part_of(cv[n]), dp[n]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        Weights<ST> w[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 x = stats[2 * g];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[n][4 * g + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][4 * g + e], a.c, ST == kF16 ? x[e] + kShift : x[e]));
            }
            if (masked) {
                const int j = jw + 32 * n + (lane & 31);
                // queries [qlo, qhi) of these 32 read it (and of a mask's columns those whose bit is set)
                const int qlo = a.causal ? j - keys.first - i0 : 0;
                const long long end = a.window ? (long long)j - keys.first + a.window - i0 : 32;
                const unsigned in = (bits[n] & range_of(qlo, (int)(end < 32 ? end : 32))) >> (4 * h);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[n][e] = where_bit(in, e, s[n][e], 0.f);
            }
            if (DV) w[n].set(s[n]);
        }
        // (f16's cotangents first, whose largest is looked for: the registers hold no
        // more beside the values' products)
        if (DV && ST != kF16) mma_col<ST, ND, NB, true>(at.col, Tile::BYTES, w, dv);
        if (DK) {
            const float fit = __builtin_ldexpf(1.f, up - (int)kShift);
            Weights<ST> z[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 x = stats[16 + 2 * g];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y = s[n][4 * g + e];
                        s[n][4 * g + e] = (ST == kF16 ? y * fit : y) * (dp[n][4 * g + e] + x[e]);
                    }
                }
                if (ST == kF16) fit_f16<ND>(s[n], dk[n], up, jw + (lane & 31) < (k1 < keys.len ? k1 : keys.len));
                z[n].set(s[n]);
            }
            mma_col<ST, ND, NB, true>(at.col, 0, z, dk);
            if constexpr (ST != kF32)
                if (fine_of<ST>(a, keys, i0, i0 + 31 < a.tq ? i0 + 31 : a.tq - 1)) {
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        left_in<ST>(s[n], z[n]);
                        z[n].set(s[n]);
                    }
                    mma_col<ST, ND, NB, true>(at.col, 0, z, dk);
                }
        }
        if (DV && ST == kF16) mma_col<ST, ND, NB, true>(at.col, Tile::BYTES, w, dv);
    };
    if (nt > t0) load_bits(i00);
    for (int t = t0, ti = i00; t < nt; ++t, ti = ti + QT < ihi ? ti + QT : ilo) {
        wait_vm<0>();
        if (a.cols)
#pragma unroll
            for (int x = 0; x < MINE; ++x) {
                asm volatile("" : "+v"(ahead[x]));
                now[x] = ahead[x];
            }
        __syncthreads();
        if (t + 1 < nt) {
            fetch(t + 1);
            load_bits(ti + QT < ihi ? ti + QT : ilo);
        }
#pragma unroll 1
        for (int sub = kw; sub < QT / 32; sub += SW) {
            const int i0 = ti + 32 * sub;
            const bool sure = (!a.causal || (jw + WKEYS - 1 <= keys.first + i0 && (!a.window || jw > keys.first + i0 + 31 - a.window))) &&
                              (!a.cols || jw + WKEYS <= keys.first) && i0 < ihi;
            body(!sure, t, sub, i0);
        }
    }
    __syncthreads();
    if (DK && ST == kF16) unfit_f16<ND>(dk[0], up);
    unsigned char* const pair = smem + rw * PAIR;      // the LDS of the waves of the same keys
    if constexpr (SW == 2) {
        static_assert(sizeof(smem) >= 4 * PAIR, "the waves' sums in LDS");
        give<ND>(pair, lane, dk[0], kw == 1);
        __syncthreads();
        if (kw == 0) take<ND>(pair, lane, dk[0], 1.f, 1.f);
        __syncthreads();
        give<ND>(pair, lane, dv[0], kw == 1);
        __syncthreads();
        if (kw == 1) return;
        take<ND>(pair, lane, dv[0], 1.f, 1.f);
    }
    const int j = jw + (lane & 31);
    const bool exists = j < k1;
    // (what a key past the sequence's end was given is dropped)
    if (j >= keys.len)
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) dk[0][dt] = dv[0][dt] = f32x16{};
    if (PARTS && a.parts > 1) {
        // (of eight waves those that have both halves)
        const long long all = (long long)a.batch * a.kv * a.tk, row = part * all + ((long long)b * a.kv + hk) * a.tk + j;
        if (exists)
#pragma unroll
            for (int g = 0; g < 4 * ND; ++g) {
                float* const to = a.part + row * (ND * 32) + g / 4 * 32 + 8 * (g & 3) + 4 * h;
                const f32x16 &x = dk[0][g / 4], &y = dv[0][g / 4];
                if (DK) *(f32x4*)to = f32x4{x[g % 4 * 4], x[g % 4 * 4 + 1], x[g % 4 * 4 + 2], x[g % 4 * 4 + 3]};
                if (DV) *(f32x4*)(to + a.parts * all * (ND * 32)) = f32x4{y[g % 4 * 4], y[g % 4 * 4 + 1], y[g % 4 * 4 + 2], y[g % 4 * 4 + 3]};
            }
        return;
    }
    auto where = [&](const AttnTensor& t) {
        return [&, t](int x) -> const void* { return jw + x < k1 ? row_at<ST>(t, b, jw + x, hk) : nullptr; };
    };
    if (DK && a.dk.p) store_kept<ST, ND, true>(dk[0], a.scale, a.d, a.dk.vec, exists, where(a.dk), pair, lane, a.flag);
    if (DV && a.dv.p) store_kept<ST, ND, true>(dv[0], ST == kF16 ? 0.00390625f : 1.f, a.d, a.dv.vec, exists, where(a.dv), pair, lane, a.flag);
}

template <int ST, int ND, int SW>
__global__ void __launch_bounds__(256 * SW, ND >= 8 || (ST == kF32 && ND >= 4) ? 1 : 2) attn_dq_kernel(AttnArgs a) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[dq_lds<ST, ND, SW>()];
    dq_of<ST, ND, SW>(a, blockIdx.x, gridDim.x, smem);
}
// The parts of the keys' and values' gradients summed, in order: four elements a
// thread, all of the one tensor's before the other's.
template <int ST, int ND>
__global__ void __launch_bounds__(256) attn_sum_kernel(AttnArgs a) {
    const long long all = (long long)a.batch * a.kv * a.tk, n = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long row = n / (8 * ND), line = row % all;
    if (row >= 2 * all) return;
    const bool value = row >= all;
    const AttnTensor& t = value ? a.dv : a.dk;
    const int at = (int)(n % (8 * ND)) * 4;
    if (!t.p || (ST != kF32 && at >= a.d)) return;
    const float* const from = a.part + ((value ? a.parts : 0) * all + line) * (ND * 32) + at;
    f32x4 x = f32x4{};
#pragma unroll 4
    for (int p = 0; p < a.parts; ++p) {
        const f32x4 y = *(const f32x4*)(from + p * all * (ND * 32));
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += y[e];
    }
    const float f = value ? ST == kF16 ? 0.00390625f : 1.f : a.scale;
    const int j = (int)(line % a.tk), hk = (int)(line / a.tk % a.kv), b = (int)(line / a.tk / a.kv);
    void* const out = const_cast<void*>(row_at<ST>(t, b, j, hk));
    bool ovf = false;
    if (ST != kF32 && t.vec) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] *= f;
            ovf |= ST == kF16 && !(__builtin_fabsf(x[e]) < 65520.f);
        }
        if constexpr (ST != kF32)
            *(unsigned long long*)((unsigned short*)out + at) = pack2<ST>(x[0], x[1]) | (unsigned long long)pack2<ST>(x[2], x[3]) << 32;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            ovf |= put<ST, ND>(out, at + e, a.d, x[e] * f) || (ST == kF16 && at + e < a.d && !(__builtin_fabsf(x[e] * f) < 65520.f));
    }
    if (ovf && a.flag) atomicOr(a.flag, 1u);
}

// ---- launches -----------------------------------------------------------------------------

// Workgroups of eight waves where four would leave SIMDs with a wave or none, which
// then waits for its own results: where a round of the CUs holds them all (2 x 12
// heads x 1024 x 64 with a mask, 192 of them: the value 27 -> 20 us, the queries'
// gradient 35 -> 24, the keys' 38 -> 27; but 384 of 2 x 24 heads, causal, 23 ->
// 29).
template <int ST, int ND>
bool eight(long long grid) {
    return Geo<ST, ND>::TILE == 64 && grid <= 256;
}

template <int ST, int ND>
hipError_t fwd(const AttnArgs& a, hipStream_t s) {
    const long long rows = (long long)a.tq * a.pack, units = (long long)a.batch * (a.heads / a.pack), all = (long long)a.batch * a.heads * a.tq;
    if (!all) return hipSuccess;
    if (rows <= kAttnFew) {
        // as many waves as 128 KB of LDS have two blocks of keys and values each for
        constexpr int NW = Geo<ST, ND>::ROW > 256 ? 2 : 4;
        attn_few_kernel<ST, ND, NW><<<(unsigned)(units * a.splits), 64 * NW, 0, s>>>(a);
    } else {
        const long long grid = (rows + kAttnTile - 1) / kAttnTile * units * a.splits;
        if (eight<ST, ND>(grid)) {
            if constexpr (Geo<ST, ND>::TILE == 64) attn_fwd_kernel<ST, ND, 2><<<(unsigned)grid, 512, 0, s>>>(a);
        } else {
            attn_fwd_kernel<ST, ND, 1><<<(unsigned)grid, 256, 0, s>>>(a);
        }
    }
    if (a.splits > 16) attn_join_kernel<ST, ND, 4><<<(unsigned)all, 256, 0, s>>>(a);
    else if (a.splits > 1) attn_join_kernel<ST, ND, 1><<<(unsigned)((all + 3) / 4), 256, 0, s>>>(a);
    return hipGetLastError();
}

template <int ST, int ND>
hipError_t bwd(const AttnArgs& a, hipStream_t s) {
    constexpr bool WIDE = Geo<ST, ND>::ROW == 256;      // (two waves a SIMD have no registers for the values too)
    const long long all = (long long)a.batch * a.heads * a.tq;
    if (all) attn_rows_kernel<ST><<<(unsigned)((all + 15) / 16), 256, 0, s>>>(a);
    const long long nq = a.dq.p ? ((long long)a.tq * a.pack + 127) / 128 * a.batch * (a.heads / a.pack) : 0;
    long long nkv = a.dk.p || a.dv.p ? (long long)((a.tk + 127) / 128) * a.batch * a.kv * a.parts : 0;
    const auto add_parts = [&] {
        const long long n = 2LL * a.batch * a.kv * a.tk * 8 * ND;
        if (a.parts > 1) attn_sum_kernel<ST, ND><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a);
    };
    if constexpr (Geo<ST, ND>::TILE == 64)
        if (nkv && (a.parts > 1 || eight<ST, ND>(nkv))) {      // (parts are those kernels' alone)
            // the queries' beside them, unless there are many short ones, whose own
            // launch has two workgroups a CU (14 x 64 heads in groups of eight x 40 x
            // 128: 45 us in one launch, 40 in two; but 6 x 48 x 333 x 96, 864
            // workgroups, 98 and 103, 40 x 2048 x 128, 640 of them, 241 and 284)
            const bool one = nq <= 256 || (nq <= 1024 && a.tk > 256);
            if (nq && one) attn_dkv_kernel<ST, ND, 2, 64, true, true, WIDE, 2, true><<<(unsigned)(nkv + nq), 512, 0, s>>>(a, (unsigned)nkv);
            else attn_dkv_kernel<ST, ND, 2, 64, true, true, WIDE, 2, false><<<(unsigned)nkv, 512, 0, s>>>(a, (unsigned)nkv);
            add_parts();
            if (one) return hipGetLastError();
            nkv = 0;
        }
    if (nq) {
        if (eight<ST, ND>(nq)) {
            if constexpr (Geo<ST, ND>::TILE == 64) attn_dq_kernel<ST, ND, 2><<<(unsigned)nq, 512, 0, s>>>(a);
        } else {
            attn_dq_kernel<ST, ND, 1><<<(unsigned)nq, 256, 0, s>>>(a);
        }
    }
    if (nkv) {
        if constexpr (ND == 8) {
            // (both sums of 256 elements and both kept rows do not fit the registers)
            if (a.dk.p) attn_dkv_kernel<ST, ND, 1, 32, true, false, false, 1, false><<<(unsigned)nkv, 256, 0, s>>>(a, (unsigned)nkv);
            if (a.dv.p) attn_dkv_kernel<ST, ND, 1, 32, false, true, false, 1, false><<<(unsigned)nkv, 256, 0, s>>>(a, (unsigned)nkv);
            add_parts();
        } else if constexpr (ST == kF32 && ND == 4) {
            attn_dkv_kernel<ST, ND, 1, 32, true, true, false, 1, false><<<(unsigned)nkv, 256, 0, s>>>(a, (unsigned)nkv);
        } else {
            attn_dkv_kernel<ST, ND, 1, WIDE ? 32 : 64, true, true, WIDE, 2, false><<<(unsigned)nkv, 256, 0, s>>>(a, (unsigned)nkv);
        }
    }
    return hipGetLastError();
}

template <int ST>
hipError_t fwd_nd(const AttnArgs& a, int nd, hipStream_t s) {
    if constexpr (ST != kF32)
        if (nd == 8) return fwd<ST, 8>(a, s);
    return nd == 2 ? fwd<ST, 2>(a, s) : nd == 4 ? fwd<ST, 4>(a, s) : hipErrorInvalidValue;
}
template <int ST>
hipError_t bwd_nd(const AttnArgs& a, int nd, hipStream_t s) {
    if constexpr (ST != kF32)
        if (nd == 8) return bwd<ST, 8>(a, s);
    return nd == 2 ? bwd<ST, 2>(a, s) : nd == 4 ? bwd<ST, 4>(a, s) : hipErrorInvalidValue;
}

}  // namespace

}  // namespace presk
