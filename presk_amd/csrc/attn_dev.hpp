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

// A tile's rows of ND * 32 elements in LDS, PITCH of them apart, 16-byte chunk c
// of row r at chunk c ^ swz(r): eight (and sixteen) consecutive rows' same chunk,
// and four consecutive rows' same four chunks, lie in different banks.
template <int ST, int ND>
struct Geo {
    static constexpr int ES = ST == kF32 ? 4 : 2, PITCH = ND <= 2 ? 64 : ND <= 4 ? 128 : 256;
    static constexpr int ROW = PITCH * ES, CPR = ROW / 16, EPC = 16 / ES;
    static constexpr int STEPS = ND * 32 / (2 * EPC);     // 16-byte reads of a row a lane (its half of each pair of chunks)
    static constexpr int TILE = ROW <= 256 ? 64 : 32;     // rows of a tile
    __device__ static __forceinline__ int swz(int r) {
        if constexpr (CPR == 8) return ((r & 2) << 1) | ((r & 4) >> 1) | ((r ^ (r >> 3)) & 1);
        else return ((r & 1) << 2) | (((r >> 1) ^ (r >> 3)) & 1) << 3 | (r & 2) | ((r >> 2) & 1);
    }
};

// 16 bytes of a row: one matrix instruction's k in 16 bits, four's in f32
template <int ST> struct FragOf { typedef u16x8 T; };
template <> struct FragOf<kF32> { typedef f32x4 T; };

template <int ST>
__device__ __forceinline__ f32x16 mma_row(typename FragOf<ST>::T a, typename FragOf<ST>::T b, f32x16 acc) {
    if constexpr (ST == kF32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], acc, 0, 0, 0);
        return acc;
    } else {
        return mfma32<ST>(a, b, acc);
    }
}

template <int ST>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    unsigned r;
    if constexpr (ST == kBF16) asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    else asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
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
template <>
struct Weights<kF32> {
    f32x16 w;
    __device__ __forceinline__ void set(const f32x16& p) { w = p; }
};

// The tile row, of 32, of a lane's sum e.
__device__ __forceinline__ int row_of(int e, int h) { return 8 * (e >> 2) + 4 * h + (e & 3); }

// A lane's part of row `row` of a tile at step `st`.
template <int ST, int ND>
__device__ __forceinline__ typename FragOf<ST>::T frag_row(const unsigned char* xs, int row, int st, int h) {
    typedef Geo<ST, ND> G;
    return *(const typename FragOf<ST>::T*)(xs + row * G::ROW + (((2 * st + h) ^ G::swz(row)) << 4));
}

// acc[dt] += X^T . w over the tile's rows row0 .. row0 + 31.  Of acc[dt]'s sum e
// a lane's element of the head is dim_of(dt, e).
template <int ST, int ND>
__device__ __forceinline__ void mma_col(const unsigned char* xs, int row0, const Weights<ST>& w, f32x16 (&acc)[ND], int lane) {
    typedef Geo<ST, ND> G;
    const int h = lane >> 5;
    if constexpr (ST == kF32) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int r = row0 + row_of(e, h), m = lane & 31, el = ND * m;
            const unsigned char* const at = xs + r * G::ROW + ((((el >> 2) ^ G::swz(r)) << 4) | ((el & 3) << 2));
            float x[ND];
            if constexpr (ND == 4) {
                const f32x4 v = *(const f32x4*)at;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = v[i];
            } else {
                const f32x2 v = *(const f32x2*)at;
                x[0] = v[0], x[1] = v[1];
            }
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[dt], w.w[e], acc[dt], 0, 0, 0);
        }
    } else {
        const int L = lane & 15, g = (lane >> 4) & 1;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int r = row0 + 16 * s + 4 * h + (L >> 2);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
                const int col = dt * 32 + 16 * g + 4 * (L & 3);
                const int lo = r * G::ROW + (((col >> 3) ^ G::swz(r)) << 4) + (col & 7) * 2;
                const int hi = (r + 8) * G::ROW + (((col >> 3) ^ G::swz(r + 8)) << 4) + (col & 7) * 2;
                const v4i16 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(xs + lo));
                const v4i16 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(xs + hi));
                u16x8 f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f[e] = (unsigned short)a[e];
                    f[4 + e] = (unsigned short)b[e];
                }
                acc[dt] = mfma32<ST>(f, w.w[s], acc[dt]);
            }
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

// A kept row: a lane's 16 bytes of every step.
template <int ST, int ND>
__device__ __forceinline__ void load_kept(const AttnTensor& t, int b, long long i, int head, int d, bool in, int h,
                                          typename FragOf<ST>::T (&x)[Geo<ST, ND>::STEPS]) {
    typedef typename FragOf<ST>::T F;
    const void* const row = row_at<ST>(t, b, in ? i : 0, head);
    if (t.vec) {
#pragma unroll
        for (int st = 0; st < Geo<ST, ND>::STEPS; ++st) {
            const int c = 2 * st + h;
            x[st] = in && c * Geo<ST, ND>::EPC < d ? *(const F*)((const char*)row + 16 * c) : F{};
        }
    } else {
#pragma unroll
        for (int st = 0; st < Geo<ST, ND>::STEPS; ++st) x[st] = chunk_of<ST>(row, 2 * st + h, d, in);
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
            for (int q = 0; q < ROUNDS; ++q) {
                const int slot = q * NTH + tid, r = slot / G::CPR, c = (slot % G::CPR) ^ G::swz(r);
                *(typename FragOf<ST>::T*)(smem + at + slot * 16) = chunk_of<ST>(src + (r < left ? r : 0) * stride, c, d, r < left);
            }
        }
    }
};

// ---- stores -----------------------------------------------------------------------

// A lane's row of sums times f into the storage type.
template <int ST, int ND>
__device__ __forceinline__ void store_kept(const AttnTensor& t, int b, long long i, int head, int d, const f32x16 (&acc)[ND], float f, int h,
                                           bool in, unsigned* flag) {
    if (!in) return;
    void* const row = const_cast<void*>(row_at<ST>(t, b, i, head));
    bool ovf = false;
    if constexpr (ST == kF32) {
        float* const out = (float*)row;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int at = ND * row_of(e, h);
            if (t.vec) {
                if (at < d) {
                    if constexpr (ND == 4) *(f32x4*)(out + at) = f32x4{acc[0][e] * f, acc[1][e] * f, acc[2][e] * f, acc[3][e] * f};
                    else *(f32x2*)(out + at) = f32x2{acc[0][e] * f, acc[1][e] * f};
                }
            } else {
#pragma unroll
                for (int dt = 0; dt < ND; ++dt)
                    if (at + dt < d) out[at + dt] = acc[dt][e] * f;
            }
        }
    } else {
        unsigned short* const out = (unsigned short*)row;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at = dt * 32 + 8 * g + 4 * h;
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = acc[dt][4 * g + e] * f;
                if (at >= d) continue;
                if (ST == kF16)
#pragma unroll
                    for (int e = 0; e < 4; ++e) ovf |= pk_overflows_f16(x[e]);
                const unsigned lo = pack2<ST>(x[0], x[1]), hi = pack2<ST>(x[2], x[3]);
                if (t.vec) {
                    *(unsigned long long*)(out + at) = lo | (unsigned long long)hi << 32;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at + e < d) out[at + e] = (unsigned short)((e < 2 ? lo : hi) >> (16 * (e & 1)));
                }
            }
    }
    if (ovf && flag) atomicOr(flag, 1u);
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

// 32 bits of a mask's line from `rel` on: ones before it, zeros past it.
__device__ __forceinline__ unsigned bits_at(const unsigned* line, int words, int rel) {
    if (rel <= -32) return ~0u;
    const int q = rel >> 5;
    const unsigned lo = q < 0 ? ~0u : q < words ? line[q] : 0u, hi = q + 1 < words ? line[q + 1] : 0u;
    return (unsigned)(((unsigned long long)hi << 32 | lo) >> (rel & 31));
}

// Work order: workgroups are dealt to the 8 XCDs round robin; each takes one
// run of items, so that those of a head share its keys in one L2.
__device__ __forceinline__ unsigned item_of(unsigned id, unsigned total) {
    const unsigned xcd = id % 8, q8 = total / 8, r8 = total % 8;
    return xcd * q8 + (xcd < r8 ? xcd : r8) + id / 8;
}

// ---- the value ----------------------------------------------------------------------

// One workgroup: 128 rows of a head (of a group's heads beside each other), 32 a
// wave, over the keys that any of them reads, or a share of those.
template <int ST, int ND>
__global__ void __launch_bounds__(256, 2) attn_fwd_kernel(AttnArgs a) {
    typedef Geo<ST, ND> G;
    typedef Rows<ST, ND, G::TILE, 256> Tile;
    constexpr int NB = G::TILE / 32;
    __shared__ __attribute__((aligned(16))) unsigned char smem[4 * Tile::BYTES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;

    const int rows = a.tq * a.pack, tiles = (rows + kAttnTile - 1) / kAttnTile, groups = a.heads / a.pack;
    const unsigned item = item_of(blockIdx.x, gridDim.x);
    const int split = (int)(item % (unsigned)a.splits);
    const unsigned at = item / (unsigned)a.splits;
    // (a head's tiles from the last on: the longest ones first where they are causal)
    const int tile = tiles - 1 - (int)(at % (unsigned)tiles), unit = (int)(at / (unsigned)tiles);
    const int b = unit / groups, hx = unit % groups, hk = hx * a.pack / a.per;
    const int r0 = tile * kAttnTile, r1 = (rows < r0 + kAttnTile ? rows : r0 + kAttnTile) - 1;

    Keys keys;
    keys.init(a, b);
    const int ifirst = r0 / a.pack, ilast = r1 / a.pack;
    int klo = keys.lo(a, ifirst), khi = keys.hi(a, ilast);
    const int surelo = keys.lo(a, ilast), surehi = keys.sure(a, ifirst);
    int nt = khi > klo ? (khi - klo + G::TILE - 1) / G::TILE : 0;
    if (a.splits > 1) {
        const int t0 = (int)((long long)nt * split / a.splits), t1 = (int)((long long)nt * (split + 1) / a.splits);
        const int end = klo + t1 * G::TILE;
        klo += t0 * G::TILE;
        khi = end < khi ? end : khi;
        nt = t1 - t0;
    }

    // this lane's row
    const int r = r0 + wave * 32 + (lane & 31);
    const bool live = r < rows;
    const int i = (live ? r : r1) / a.pack, head = hx * a.pack + (live ? r : r1) % a.pack;
    const int rlo = keys.lo(a, i), rhi = keys.hi(a, i);
    const unsigned* const line = a.cols ? a.bits + ((long long)b * a.bits_batch + i) * a.words : nullptr;

    Tile kt, vt;
    const unsigned lds = (unsigned)(size_t)(lds_void_t*)smem;
    kt.init(a.k, b, hk, a.d, tid, lds);
    vt.init(a.v, b, hk, a.d, tid, lds + Tile::BYTES);
    auto fetch = [&](int t) {
        const unsigned stage = (unsigned)(t & 1) * 2 * Tile::BYTES;
        const int k0 = klo + t * G::TILE;
        kt.issue(k0, khi - k0, stage, smem, tid);
        vt.issue(k0, khi - k0, stage, smem + Tile::BYTES, tid);
    };
    if (nt > 0) fetch(0);
    typename FragOf<ST>::T q[G::STEPS];
    load_kept<ST, ND>(a.q, b, i, head, a.d, live, h, q);

    f32x16 o[ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[dt] = f32x16{};
    float m = -INFINITY, l = 0.f;       // in log 2; this lane's part of the sum

    for (int t = 0; t < nt; ++t) {
        wait_vm<0>();
        __syncthreads();
        if (t + 1 < nt) fetch(t + 1);
        const int k0 = klo + t * G::TILE;
        const unsigned char* const ks = smem + (t & 1) * 2 * Tile::BYTES;
        const unsigned char* const vs = ks + Tile::BYTES;
        f32x16 s[NB];
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
            s[kb] = f32x16{};
#pragma unroll
            for (int st = 0; st < G::STEPS; ++st) s[kb] = mma_row<ST>(frag_row<ST, ND>(ks, kb * 32 + (lane & 31), st, h), q[st], s[kb]);
        }
        if (k0 < surelo || k0 + G::TILE > surehi) {
#pragma unroll
            for (int kb = 0; kb < NB; ++kb) {
                const int base = k0 + kb * 32;
                const unsigned bits = a.cols ? bits_at(line, a.words, base - keys.first) : ~0u;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int c = row_of(e, h), j = base + c;
                    s[kb][e] = j >= rlo && j < rhi && (bits >> c & 1) ? s[kb][e] : -INFINITY;
                }
            }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][e]);
        mx = fmaxf(mx, partner<32>(mx)) * a.c;
        // the sums stay at an older maximum until one passes it by 2^8
        if (__any(mx > m + 8.f)) {
            const float top = fmaxf(m, mx), f = __builtin_amdgcn_exp2f(m - base_of(top));
            m = top;
            l *= f;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[dt][e] *= f;
        }
        const float base = base_of(m);
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[kb][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e], a.c, -base));
                sum += s[kb][e];
            }
            l += sum;
            Weights<ST> w;
            w.set(s[kb]);
            mma_col<ST, ND>(vs, kb * 32, w, o, lane);
        }
    }

    l += partner<32>(l);
    const long long row = ((long long)b * a.heads + head) * a.tq + i;
    if (a.splits > 1) {
        const long long all = (long long)a.batch * a.heads * a.tq, n = (long long)split * all + row;
        if (live) {
            float* const out = a.part + n * (ND * 32);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *(f32x4*)(out + dt * 32 + 8 * g + 4 * h) = f32x4{o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]};
            if (h == 0) *(f32x2*)(a.part_ml + 2 * n) = f32x2{m, l};
        }
        return;
    }
    store_kept<ST, ND>(a.o, b, i, head, a.d, o, l == 0.f ? 0.f : 1.f / l, h, live, a.flag);
    if (a.lse && live && h == 0) a.lse[row] = l == 0.f ? -INFINITY : (base_of(m) + __builtin_log2f(l)) * kLn2;
}

// The splits' sums of a row joined: 64 lanes a row, ND / 2 elements a lane.
template <int ST, int ND>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a) {
    const long long all = (long long)a.batch * a.heads * a.tq, row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= all) return;
    const int lane = threadIdx.x & 63;
    float m = -INFINITY;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[2 * (s * all + row)]);
    const float base = base_of(m);
    float l = 0.f, x[ND / 2];
#pragma unroll
    for (int q = 0; q < ND / 2; ++q) x[q] = 0.f;
    for (int s = 0; s < a.splits; ++s) {
        const long long n = s * all + row;
        const f32x2 ml = *(const f32x2*)(a.part_ml + 2 * n);
        const float f = __builtin_amdgcn_exp2f(ml[0] - base);
        l += ml[1] * f;
#pragma unroll
        for (int q = 0; q < ND / 2; ++q) x[q] += a.part[n * (ND * 32) + q * 64 + lane] * f;
    }
    const float f = l == 0.f ? 0.f : 1.f / l;
    const int i = (int)(row % a.tq), head = (int)(row / a.tq % a.heads), b = (int)(row / a.tq / a.heads);
    void* const out = const_cast<void*>(row_at<ST>(a.o, b, i, head));
    bool ovf = false;
#pragma unroll
    for (int q = 0; q < ND / 2; ++q) {
        // (an element's place among a split's sums: attn_fwd_kernel's lanes)
        const int at = q * 64 + lane;
        const int e = ST == kF32 ? ND * (at & 31) + (at >> 5) : at;
        if (e >= a.d) continue;
        const float v = x[q] * f;
        if constexpr (ST == kF32) ((float*)out)[e] = v;
        else if constexpr (ST == kBF16) ((unsigned short*)out)[e] = pk_f32_to_bf16(v);
        else {
            ovf |= pk_overflows_f16(v);
            ((unsigned short*)out)[e] = pk_f32_to_f16(v);
        }
    }
    if (ovf && a.flag) atomicOr(a.flag, 1u);
    if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : (base + __builtin_log2f(l)) * kLn2;
}

// ---- the gradients --------------------------------------------------------------------

// A row's {-lse / scale, -sum do o}: the scores' products start from the one, the
// weights' cotangents from the other.  16 lanes a row.
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
        *(f32x2*)(a.rows + 2 * at) = f32x2{lse == -INFINITY ? 0.f : -lse / a.scale, -s};
    }
}

// The weights and their cotangents, from the products that started from the
// rows' sums: p = exp2(c s), ds = p dp.  In f16 the weights, most of them far below
// one, enter their product times 2^8.
constexpr float kShift = 8.f;

// The queries' gradient: as the value's kernel, with the cotangent's rows beside
// the queries'.
template <int ST, int ND>
__global__ void __launch_bounds__(256, ND == 8 || (ST == kF32 && ND == 4) ? 1 : 2) attn_dq_kernel(AttnArgs a) {
    typedef Geo<ST, ND> G;
    typedef Rows<ST, ND, G::TILE, 256> Tile;
    constexpr int NB = G::TILE / 32;
    __shared__ __attribute__((aligned(16))) unsigned char smem[4 * Tile::BYTES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;

    const int tiles = (a.tq + kAttnTile - 1) / kAttnTile;
    const unsigned at = item_of(blockIdx.x, gridDim.x);
    const int tile = tiles - 1 - (int)(at % (unsigned)tiles), unit = (int)(at / (unsigned)tiles);
    const int b = unit / a.heads, head = unit % a.heads, hk = head / a.per;
    const int r0 = tile * kAttnTile, r1 = (a.tq < r0 + kAttnTile ? a.tq : r0 + kAttnTile) - 1;

    Keys keys;
    keys.init(a, b);
    const int klo = keys.lo(a, r0), khi = keys.hi(a, r1), surelo = keys.lo(a, r1), surehi = keys.sure(a, r0);
    const int nt = khi > klo ? (khi - klo + G::TILE - 1) / G::TILE : 0;

    const int r = r0 + wave * 32 + (lane & 31);
    const bool live = r < a.tq;
    const int i = live ? r : r1;
    const int rlo = keys.lo(a, i), rhi = keys.hi(a, i);
    const unsigned* const line = a.cols ? a.bits + ((long long)b * a.bits_batch + i) * a.words : nullptr;

    Tile kt, vt;
    const unsigned lds = (unsigned)(size_t)(lds_void_t*)smem;
    kt.init(a.k, b, hk, a.d, tid, lds);
    vt.init(a.v, b, hk, a.d, tid, lds + Tile::BYTES);
    auto fetch = [&](int t) {
        const unsigned stage = (unsigned)(t & 1) * 2 * Tile::BYTES;
        const int k0 = klo + t * G::TILE;
        kt.issue(k0, khi - k0, stage, smem, tid);
        vt.issue(k0, khi - k0, stage, smem + Tile::BYTES, tid);
    };
    if (nt > 0) fetch(0);
    typename FragOf<ST>::T q[G::STEPS], dout[G::STEPS];
    load_kept<ST, ND>(a.q, b, i, head, a.d, live, h, q);
    load_kept<ST, ND>(a.dout, b, i, head, a.d, live, h, dout);
    const f32x2 st2 = *(const f32x2*)(a.rows + 2 * (((long long)b * a.heads + head) * a.tq + i));

    f32x16 dq[ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) dq[dt] = f32x16{};

    for (int t = 0; t < nt; ++t) {
        wait_vm<0>();
        __syncthreads();
        if (t + 1 < nt) fetch(t + 1);
        const int k0 = klo + t * G::TILE;
        const unsigned char* const ks = smem + (t & 1) * 2 * Tile::BYTES;
        const unsigned char* const vs = ks + Tile::BYTES;
        const bool sure = k0 >= surelo && k0 + G::TILE <= surehi;
#pragma unroll
        for (int kb = 0; kb < NB; ++kb) {
            f32x16 s, dp;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = st2[0], dp[e] = st2[1];
#pragma unroll
            for (int st = 0; st < G::STEPS; ++st) {
                s = mma_row<ST>(frag_row<ST, ND>(ks, kb * 32 + (lane & 31), st, h), q[st], s);
                dp = mma_row<ST>(frag_row<ST, ND>(vs, kb * 32 + (lane & 31), st, h), dout[st], dp);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(s[e] * a.c) * dp[e];
            if (!sure) {
                const int base = k0 + kb * 32;
                const unsigned bits = a.cols ? bits_at(line, a.words, base - keys.first) : ~0u;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int c = row_of(e, h), j = base + c;
                    s[e] = j >= rlo && j < rhi && (bits >> c & 1) ? s[e] : 0.f;
                }
            }
            Weights<ST> w;
            w.set(s);
            mma_col<ST, ND>(ks, kb * 32, w, dq, lane);
        }
    }
    store_kept<ST, ND>(a.dq, b, i, head, a.d, dq, a.scale, h, live, a.flag);
}

// The keys' and values' gradients: a workgroup keeps 128 keys of a key head, 32 a
// wave, and the rows of all heads of its group that read any of them pass by.
template <int ST, int ND>
__global__ void __launch_bounds__(256, ND == 8 || (ST == kF32 && ND == 4) ? 1 : 2) attn_dkv_kernel(AttnArgs a) {
    typedef Geo<ST, ND> G;
    typedef Rows<ST, ND, 32, 256> Tile;
    constexpr int STAGE = 2 * Tile::BYTES + 256;
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;

    const int tiles = (a.tk + kAttnTile - 1) / kAttnTile;
    const unsigned at = item_of(blockIdx.x, gridDim.x);
    const int tile = (int)(at % (unsigned)tiles), unit = (int)(at / (unsigned)tiles);
    const int b = unit / a.kv, hk = unit % a.kv;
    const int k0 = tile * kAttnTile, k1 = a.tk < k0 + kAttnTile ? a.tk : k0 + kAttnTile;

    Keys keys;
    keys.init(a, b);
    // queries [ilo, ihi) read any of the keys
    int ilo = 0, ihi = a.tq;
    const int last = (k1 < keys.len ? k1 : keys.len) - 1;
    if (a.causal) {
        ilo = k0 - keys.first > 0 ? k0 - keys.first : 0;
        if (a.window) {
            const long long e = (long long)last - keys.first + a.window;
            ihi = (int)(e < ihi ? e : ihi);
        }
    }
    if (a.cols && k0 >= keys.first + a.cols) ihi = 0;
    if (last < k0) ihi = 0;
    const int nt1 = ihi > ilo ? (ihi - ilo + 31) / 32 : 0, nt = nt1 * a.per;

    // this lane's key
    const int j = k0 + wave * 32 + (lane & 31);
    const bool exists = j < a.tk, live = exists && j < keys.len;
    const int jw = k0 + wave * 32;      // the wave's first
    // queries [qlo, qhi) read it (and of a mask's columns those whose bit is set)
    const int qlo = a.causal ? j - keys.first : 0;
    const long long qend = a.window ? (long long)j - keys.first + a.window : a.tq;
    const int qhi = (int)(qend < a.tq ? qend : a.tq);
    const int col = j - keys.first;
    const unsigned* const line =
        a.cols && col >= 0 && col < a.cols ? a.bits_t + ((long long)b * a.bits_t_batch + col) * a.words_t : nullptr;

    Tile qt, dt_;
    const unsigned lds = (unsigned)(size_t)(lds_void_t*)smem;
    auto fetch = [&](int t) {
        const int g = t / nt1, i0 = ilo + (t - g * nt1) * 32, head = hk * a.per + g;
        const unsigned stage = (unsigned)(t & 1) * STAGE;
        if (i0 == ilo) {
            qt.init(a.q, b, head, a.d, tid, lds);
            dt_.init(a.dout, b, head, a.d, tid, lds + Tile::BYTES);
        }
        const int left = a.tq - i0;
        qt.issue(i0, left, stage, smem, tid);
        dt_.issue(i0, left, stage, smem + Tile::BYTES, tid);
        if (wave == 0) {
            const float* const src = a.rows + 2 * (((long long)b * a.heads + head) * a.tq + i0);
            const i32x4 buf = buffer_of(src, (unsigned)((left < 32 ? left : 32) * 8));
            asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dword %0, %1, 0 offen lds"
                         : : "v"(lane * 4), "s"(buf), "s"(__builtin_amdgcn_readfirstlane(lds + stage + 2 * Tile::BYTES)) : "memory", "m0");
        }
    };
    if (nt > 0) fetch(0);
    typename FragOf<ST>::T k[G::STEPS], v[G::STEPS];
    load_kept<ST, ND>(a.k, b, j, hk, a.d, live, h, k);
    load_kept<ST, ND>(a.v, b, j, hk, a.d, live, h, v);
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) dk[dt] = dv[dt] = f32x16{};

    for (int t = 0; t < nt; ++t) {
        wait_vm<0>();
        __syncthreads();
        if (t + 1 < nt) fetch(t + 1);
        const int i0 = ilo + t % nt1 * 32;
        const unsigned char* const qs = smem + (t & 1) * STAGE;
        const unsigned char* const ds_ = qs + Tile::BYTES;
        const float* const stats = (const float*)(qs + 2 * Tile::BYTES);
        f32x16 s, dp;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 x = *(const f32x4*)(stats + 2 * (8 * g + 4 * h)), y = *(const f32x4*)(stats + 2 * (8 * g + 4 * h) + 4);
            s[4 * g] = x[0], s[4 * g + 1] = x[2], s[4 * g + 2] = y[0], s[4 * g + 3] = y[2];
            dp[4 * g] = x[1], dp[4 * g + 1] = x[3], dp[4 * g + 2] = y[1], dp[4 * g + 3] = y[3];
        }
#pragma unroll
        for (int st = 0; st < G::STEPS; ++st) s = mma_row<ST>(frag_row<ST, ND>(qs, lane & 31, st, h), k[st], s);
#pragma unroll
        for (int st = 0; st < G::STEPS; ++st) dp = mma_row<ST>(frag_row<ST, ND>(ds_, lane & 31, st, h), v[st], dp);
#pragma unroll
        for (int e = 0; e < 16; ++e)
            s[e] = ST == kF16 ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], a.c, kShift)) : __builtin_amdgcn_exp2f(s[e] * a.c);
        const bool sure = (!a.causal || (jw + 31 <= keys.first + i0 && (!a.window || jw > keys.first + i0 + 31 - a.window))) &&
                          (!a.cols || jw + 32 <= keys.first);
        if (!sure) {
            const unsigned bits = !a.cols || col < 0 ? ~0u : line ? bits_at(line, a.words_t, i0) : 0u;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int c = row_of(e, h), i = i0 + c;
                s[e] = i >= qlo && i < qhi && (bits >> c & 1) ? s[e] : 0.f;
            }
        }
        Weights<ST> w;
        w.set(s);
        mma_col<ST, ND>(ds_, 0, w, dv, lane);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = ST == kF16 ? s[e] * 0.00390625f * dp[e] : s[e] * dp[e];
        w.set(s);
        mma_col<ST, ND>(qs, 0, w, dk, lane);
    }
    if (!live)
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) dk[dt] = dv[dt] = f32x16{};
    if (a.dk.p) store_kept<ST, ND>(a.dk, b, j, hk, a.d, dk, a.scale, h, exists, a.flag);
    if (a.dv.p) store_kept<ST, ND>(a.dv, b, j, hk, a.d, dv, ST == kF16 ? 0.00390625f : 1.f, h, exists, a.flag);
}

// ---- launches -----------------------------------------------------------------------------

template <int ST, int ND>
hipError_t fwd(const AttnArgs& a, hipStream_t s) {
    const long long rows = (long long)a.tq * a.pack;
    const long long grid = (rows + kAttnTile - 1) / kAttnTile * a.batch * (a.heads / a.pack) * a.splits;
    if (!grid) return hipSuccess;
    attn_fwd_kernel<ST, ND><<<(unsigned)grid, 256, 0, s>>>(a);
    if (a.splits > 1) {
        const long long all = (long long)a.batch * a.heads * a.tq;
        attn_join_kernel<ST, ND><<<(unsigned)((all + 3) / 4), 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

template <int ST, int ND>
hipError_t bwd(const AttnArgs& a, hipStream_t s) {
    const long long all = (long long)a.batch * a.heads * a.tq;
    if (all) attn_rows_kernel<ST><<<(unsigned)((all + 15) / 16), 256, 0, s>>>(a);
    if (a.dq.p && all) attn_dq_kernel<ST, ND><<<(unsigned)((a.tq + kAttnTile - 1) / kAttnTile * a.batch * a.heads), 256, 0, s>>>(a);
    if ((a.dk.p || a.dv.p) && a.batch && a.tk)
        attn_dkv_kernel<ST, ND><<<(unsigned)((a.tk + kAttnTile - 1) / kAttnTile * a.batch * a.kv), 256, 0, s>>>(a);
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
