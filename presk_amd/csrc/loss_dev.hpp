// What the losses' kernels share on the device (loss.hpp).
#pragma once

#include <hip/hip_runtime.h>

#include "devfmt.hpp"
#include "loss.hpp"

namespace presk {

namespace {

// 2^((z - base) c): the difference first, in the logits' own units, so that a
// type's lowest value (a mask) beside another stays finite, which z c need not
__device__ __forceinline__ float exp2_of(float z, float c, float base) { return __builtin_amdgcn_exp2f((z - base) * c); }
// what is subtracted from z where the largest is m: a row of -inf has sum 0
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// Lane i's partner at step D of a reduction over 2 D lanes whose steps below D
// are done (each half of them holds one value): register moves, no LDS.
template <int D>
__device__ __forceinline__ float partner(float v) {
    const int b = __builtin_bit_cast(int, v);
    if constexpr (D == 1) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, b, 0xB1, 0xF, 0xF, false));        // quad_perm [1,0,3,2]
    else if constexpr (D == 2) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, b, 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
    else if constexpr (D == 4) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, b, 0x141, 0xF, 0xF, false));  // row_half_mirror
    else if constexpr (D == 8) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, b, 0x140, 0xF, 0xF, false));  // row_mirror
    else if constexpr (D == 16) {
        const auto p = __builtin_amdgcn_permlane16_swap((unsigned)b, (unsigned)b, false, false);
        return __builtin_bit_cast(float, threadIdx.x & 16 ? p[0] : p[1]);
    } else {
        const auto p = __builtin_amdgcn_permlane32_swap((unsigned)b, (unsigned)b, false, false);
        return __builtin_bit_cast(float, threadIdx.x & 32 ? p[0] : p[1]);
    }
}

// what the rounding of v to 16 bits left of it (nothing beside an infinity)
__device__ __forceinline__ float left_of(float v, float rounded) { return __builtin_fabsf(rounded) < INFINITY ? v - rounded : 0.f; }

// Over G threads (16, 64: as many lanes of a wave; more: the workgroup,
// through `red`, G / 64 floats): the same value in every one, met in a fixed tree.
template <int G, typename F>
__device__ __forceinline__ float all_of(float v, float* red, F op) {
    v = op(v, partner<1>(v));
    v = op(v, partner<2>(v));
    v = op(v, partner<4>(v));
    v = op(v, partner<8>(v));
    if constexpr (G > 16) {
        v = op(v, partner<16>(v));
        v = op(v, partner<32>(v));
    }
    if constexpr (G > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int w = 1; w < G / 64; ++w) v = op(v, red[w]);
    }
    return v;
}
__device__ __forceinline__ float add_f(float a, float b) { return a + b; }
__device__ __forceinline__ float max_f(float a, float b) { return fmaxf(a, b); }

// ---- a row's target ----------------------------------------------------------------

__device__ __forceinline__ int slot_col(const LossTarget& t, long long r, int e) {
    if (!t.index) return t.col[r * t.k + e];
    const long long y = t.index[r];
    return y < 0 ? kUnused : y >= t.vocab ? kOutside : (int)y;
}
__device__ __forceinline__ float slot_p(const LossTarget& t, long long r, int e) {
    if (!t.index) return t.p[r * t.k + e];
    const long long y = t.index[r];
    return y >= 0 && y < t.vocab ? 1.f : 0.f;
}
__device__ __forceinline__ float row_ent(const LossTarget& t, long long r) {
    if (!t.index) return t.ent[r];
    return t.index[r] >= t.vocab ? NAN : 0.f;
}
__device__ __forceinline__ bool counts(const LossTarget& t, long long r) {
    return t.index ? t.index[r] >= 0 : t.col[r * t.k] != kUnused;
}

// One column a row: how many rows count, and their largest |ct|, by T threads
// of workgroup `part`.
template <int T>
__device__ __forceinline__ void prep_one(const LossPrep& a, int part) {
    __shared__ float red[T / 64];
    float n = 0.f, most = 0.f;
    for (long long r = (long long)part * T + threadIdx.x; r < a.rows; r += (long long)a.parts * T)
        if (a.index[r] >= 0) {
            n += 1.f;
            if (a.ct) most = fmaxf(most, fabsf(a.ct[r]));
        }
    n = all_of<T>(n, red, add_f);
    most = all_of<T>(most, red, max_f);
    if (threadIdx.x == 0) {
        a.count[part] = (int)n;
        a.most[part] = most;
    }
}

// The exponent of the power of two that brings a call's largest cotangent
// factor to 2^14 .. 2^15, where f16 keeps its bits down to 2^-38 of it.
__device__ __forceinline__ int scale_exponent(float top) {
    if (!(top > 0.f && top < INFINITY)) return 0;
    int x;
    (void)frexpf(top, &x);
    return 15 - x < -100 ? -100 : 15 - x > 100 ? 100 : 15 - x;
}

// the mean of m.rows losses over the counted ones by T threads, in f64 (their
// order is the strides', then a tree)
template <int T>
__device__ __forceinline__ void write_mean(const LossMean& m) {
    __shared__ double red[T / 64];
    __shared__ int nred[T / 64];
    double s = 0.0;
    int n = 0;
    // (eight loads in flight)
    for (long long r0 = threadIdx.x; r0 < m.rows; r0 += 8 * T) {
        float l[8];
        long long y[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const bool in = r0 + q * T < m.rows;
            l[q] = in ? m.loss[r0 + q * T] : 0.f;
            y[q] = in && !m.parts ? m.index[r0 + q * T] : -1;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            s += (double)l[q];
            n += y[q] >= 0;
        }
    }
    for (int i = threadIdx.x; i < m.parts; i += T) n += m.count[i];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        s += __shfl_xor(s, d);
        n += __shfl_xor(n, d);
    }
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = s;
        nred[threadIdx.x >> 6] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < T / 64; ++w) {
            s += red[w];
            n += nred[w];
        }
        m.mean[0] = n ? (float)(s / n) : 0.f;
        m.mean[1] = (float)n;
    }
}

}  // namespace

}  // namespace presk
