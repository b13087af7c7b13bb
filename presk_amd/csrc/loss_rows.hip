// The row kernels of the losses (loss.hpp): a call's targets, the row sums and
// cotangents of logits in memory, and what joins a row's partial sums.
//
// A row's logits are taken as u = z * c in units of log 2 (c = log2 e / T), its
// sum of exponentials as sum 2^(u - m) with m the largest u: one fma and one
// v_exp_f32 (1 ulp) an element.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "devfmt.hpp"
#include "loss.hpp"

namespace presk {

namespace {

typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <int ST> struct Elem {
    typedef unsigned short S;
    static constexpr int V = 8;
};
template <> struct Elem<kF32> {
    typedef float S;
    static constexpr int V = 4;
};

template <int ST>
__device__ __forceinline__ float widen(typename Elem<ST>::S x) {
    if constexpr (ST == kF32) return x;
    else if constexpr (ST == kBF16) return pk_bf16_to_f32(x);
    else return pk_f16_to_f32(x);
}
template <int ST>
__device__ __forceinline__ typename Elem<ST>::S narrow(float v, bool& ovf) {
    if constexpr (ST == kF32) return v;
    else if constexpr (ST == kBF16) return pk_f32_to_bf16(v);
    else {
        ovf |= pk_overflows_f16(v);
        return pk_f32_to_f16(v);
    }
}

// 16 bytes at any alignment of the element
template <int ST>
struct Vec {
    typename Elem<ST>::S e[Elem<ST>::V];
};
template <int ST>
__device__ __forceinline__ Vec<ST> load_vec(const typename Elem<ST>::S* p) {
    Vec<ST> v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
template <int ST>
__device__ __forceinline__ void store_vec(typename Elem<ST>::S* p, const Vec<ST>& v) {
    __builtin_memcpy(p, &v, 16);
}

__device__ __forceinline__ float exp2_of(float z, float c, float base) { return __builtin_amdgcn_exp2f(__builtin_fmaf(z, c, -base)); }
// what is subtracted from u where the largest is m: a row of -inf has sum 0
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// (m, s) with another (m2, s2)
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float n = fmaxf(m, m2), b = base_of(n);
    s = s * __builtin_amdgcn_exp2f(m - b) + s2 * __builtin_amdgcn_exp2f(m2 - b);
    m = n;
}

// Over G threads (64: a wave; more: the workgroup, through `red`, G / 64
// floats): the same value in every one, the lanes met in a fixed tree.
template <int G, typename F>
__device__ __forceinline__ float all_of(float v, float* red, F op) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = op(v, __shfl_xor(v, d));
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

// ---- targets ------------------------------------------------------------------

// one column a row
__global__ void __launch_bounds__(256) prep_one_kernel(LossPrep a) {
    __shared__ float red[4];
    float n = 0.f, most = 0.f;
    for (long long r = (long long)blockIdx.x * 256 + threadIdx.x; r < a.rows; r += (long long)gridDim.x * 256) {
        const long long y = a.index[r];
        const bool on = y >= 0, out = y >= a.vocab;
        a.col[r] = !on ? kUnused : out ? kOutside : (int)y;
        a.p[r] = on && !out ? 1.f : 0.f;
        a.ent[r] = out ? NAN : 0.f;
        if (on) {
            n += 1.f;
            if (a.ct) most = fmaxf(most, fabsf(a.ct[r]));
        }
    }
    n = all_of<256>(n, red, add_f);
    most = all_of<256>(most, red, max_f);
    if (threadIdx.x == 0) {
        a.count[blockIdx.x] = (int)n;
        a.most[blockIdx.x] = most;
    }
}

// A teacher's slots: the softmax of those in use, sorted by column (a slot's
// place is how many come before it: columns below its own, or its own at an
// earlier slot, so the order is one whatever runs first).
template <int ST, int G>
__global__ void __launch_bounds__(256) prep_top_kernel(LossPrep a) {
    constexpr int R = 256 / G, KM = G == 64 ? 64 : 1024;
    __shared__ int in[R][KM], sorted[R][KM];
    __shared__ float red[4];
    __shared__ float tally[R][2];
    const int g = threadIdx.x / G, t = threadIdx.x % G, k = a.top;
    float n = 0.f, most = 0.f;
    for (long long r0 = (long long)blockIdx.x * R; r0 < a.rows; r0 += (long long)gridDim.x * R) {
        const long long r = r0 + g;
        const bool live = r < a.rows;
        typedef typename Elem<ST>::S S;
        auto logit = [&](int j) { return widen<ST>(((const S*)a.teacher)[r * k + j]); };
        float top = -INFINITY, used = 0.f, bad = 0.f;
        for (int j = t; j < k; j += G) {
            int col = kUnused;
            if (live) {
                const long long i = a.index[r * k + j];
                const float x = logit(j);
                if (i >= 0 && x != -INFINITY) {
                    col = i >= a.vocab ? kOutside : (int)i;
                    if (i >= a.vocab) bad = 1.f;
                    used = 1.f;
                    top = x > top || x != x ? x : top;
                }
            }
            in[g][j] = col;
        }
        // (a NaN among them is lost to the maximum and comes back in its term)
        top = all_of<G>(top, red, max_f);
        used = all_of<G>(used, red, max_f);
        bad = all_of<G>(bad, red, max_f);
        __syncthreads();
        float total = 0.f;
        for (int j = t; j < k; j += G)
            if (in[g][j] != kUnused) total += exp2_of(logit(j), a.c, top * a.c);
        total = all_of<G>(total, red, add_f);
        const float l2 = __builtin_amdgcn_logf(total);
        float ent = 0.f;
        for (int j = t; j < k; j += G) {
            const int col = in[g][j];
            int at = 0;
            for (int q = 0; q < k; ++q) at += in[g][q] < col || (in[g][q] == col && q < j);
            float p = 0.f;
            if (col != kUnused) {
                const float u = __builtin_fmaf(logit(j), a.c, -(top * a.c));
                p = __builtin_amdgcn_exp2f(u) / total;
                if (p != 0.f) ent += p * ((u - l2) * kLn2);
            }
            sorted[g][at] = col;
            if (live) {
                a.col[r * k + at] = col;
                a.p[r * k + at] = p;
            }
        }
        ent = all_of<G>(ent, red, add_f);
        __syncthreads();
        if (live && a.start) {
            for (int b = t; b <= a.nblocks; b += G) {
                int lo = 0, hi = k;
                while (lo < hi) {
                    const int mid = (lo + hi) / 2;
                    if (sorted[g][mid] < b * kCols) lo = mid + 1;
                    else hi = mid;
                }
                a.start[r * (a.nblocks + 1) + b] = (unsigned short)lo;
            }
        }
        if (live && t == 0) {
            a.ent[r] = bad != 0.f ? NAN : ent;
            if (used != 0.f) {
                n += 1.f;
                if (a.ct) most = fmaxf(most, fabsf(a.ct[r]));
            }
        }
        __syncthreads();
    }
    if (t == 0) {
        tally[g][0] = n;
        tally[g][1] = most;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int q = 1; q < R; ++q) {
            n += tally[q][0];
            most = fmaxf(most, tally[q][1]);
        }
        a.count[blockIdx.x] = (int)n;
        a.most[blockIdx.x] = most;
    }
}

// ---- a row's partial sums joined ------------------------------------------------

// 32 rows a workgroup, eight threads a row, each over every eighth slot.
__global__ void __launch_bounds__(256) rows_kernel(LossRows a) {
    __shared__ float red[4];
    const int q = threadIdx.x & 7;
    const long long r = (long long)blockIdx.x * 32 + threadIdx.x / 8;
    const bool live = r < a.rows;
    float count = 0.f, most = 0.f;
    if (a.coef) {
        if (a.count) {
            for (int i = threadIdx.x; i < a.parts; i += 256) {
                count += (float)a.count[i];
                most = fmaxf(most, a.most[i]);
            }
            count = all_of<256>(count, red, add_f);
            most = all_of<256>(most, red, max_f);
        }
        if (a.mean_in) count = a.mean_in[1];
    }
    float m = -INFINITY, s = 0.f, ta = 0.f;
    if (live) {
        for (int p = q; p < a.slots; p += 8) {
            const long long at = (long long)p * a.rows + r;
            join(m, s, a.pm[at], a.ps[at]);
            ta += a.pa[at];
        }
    }
#pragma unroll
    for (int d = 1; d < 8; d *= 2) {
        const float m2 = __shfl_xor(m, d), s2 = __shfl_xor(s, d);
        join(m, s, m2, s2);
        ta += __shfl_xor(ta, d);
    }
    if (a.coef) {
        // f16: a power of two brings the largest cotangent to 2^14 .. 2^15
        int e = 0;
        if (a.scale) {
            const float top = (a.ct ? most : 1.f / fmaxf(count, 1.f)) * a.temperature;
            if (top > 0.f && top < INFINITY) {
                int x;
                (void)frexpf(top, &x);
                e = 15 - x < -100 ? -100 : 15 - x > 100 ? 100 : 15 - x;
            }
            if (blockIdx.x == 0 && threadIdx.x == 0) *a.scale = ldexpf(1.f, -e);
        }
        if (live && q == 0) {
            float f = 0.f;
            if (a.t.col[r * a.t.k] != kUnused) {
                f = (a.ct ? a.ct[r] : 1.f / fmaxf(count, 1.f)) * a.temperature;
                if (a.scale) f = ldexpf(f, e);
                f += a.t.ent[r] != a.t.ent[r] ? NAN : 0.f;
            }
            a.coef[r] = f;
        }
    }
    if (live && q == 0 && a.slots) {
        const float ls = pk_logf(s);
        if (a.lse) a.lse[r] = __builtin_fmaf(m, kLn2, ls);
        if (a.loss) {
            // the largest logit against the target's before anything is added to it
            const float l = a.t.ent[r] + (__builtin_fmaf(m - ta, kLn2, ls));
            a.loss[r] = a.t.col[r * a.t.k] == kUnused ? 0.f : a.temperature * a.temperature * l;
        }
    }
}

__global__ void __launch_bounds__(1024) mean_kernel(const float* loss, long long rows, const int* count, int parts, float* mean) {
    __shared__ double red[16];
    __shared__ int nred[16];
    double s = 0.0;
    int n = 0;
    for (long long r = threadIdx.x; r < rows; r += 1024) s += (double)loss[r];
    for (int i = threadIdx.x; i < parts; i += 1024) n += count[i];
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
        for (int w = 1; w < 16; ++w) {
            s += red[w];
            n += nred[w];
        }
        mean[0] = n ? (float)(s / n) : 0.f;
        mean[1] = (float)n;
    }
}

// ---- logits in memory -------------------------------------------------------------

// Columns [lo, hi) of row r by G threads: the largest, the sum, the target's part.
template <int ST, int G>
__device__ __forceinline__ void row_stats(const LossMatrix& a, long long r, int lo, int hi, int t, float* red, float& m, float& s,
                                          float& ta) {
    typedef typename Elem<ST>::S S;
    constexpr int V = Elem<ST>::V;
    const S* const z = (const S*)a.z + r * a.ld;
    m = -INFINITY;
    s = 0.f;
    ta = 0.f;
    const int whole = lo + (hi - lo) / V * V;
    // four vectors in flight, their largest first, then one rescale for all
    constexpr int U = 4;
    for (int i = lo + t * V; i < whole; i += U * G * V) {
        Vec<ST> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * G * V < whole) v[u] = load_vec<ST>(z + i + u * G * V);
        float x = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * G * V < whole)
#pragma unroll
                for (int e = 0; e < V; ++e) x = fmaxf(x, widen<ST>(v[u].e[e]));
        const float n = fmaxf(m, x * a.c), b = base_of(n);
        s *= __builtin_amdgcn_exp2f(m - b);
        m = n;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * G * V < whole)
#pragma unroll
                for (int e = 0; e < V; ++e) s += exp2_of(widen<ST>(v[u].e[e]), a.c, b);
    }
    if (whole + t < hi) {
        const float x = widen<ST>(z[whole + t]);
        const float n = fmaxf(m, x * a.c), b = base_of(n);
        s = s * __builtin_amdgcn_exp2f(m - b) + exp2_of(x, a.c, b);
        m = n;
    }
    for (int e = t; e < a.t.k; e += G) {
        const int col = a.t.col[r * a.t.k + e] - a.col0;
        const float p = a.t.p[r * a.t.k + e];
        if (col >= lo && col < hi && p != 0.f) ta += p * (widen<ST>(z[col]) * a.c);
    }
    const float top = all_of<G>(m, red, max_f);
    s *= __builtin_amdgcn_exp2f(m - base_of(top));
    m = top;
    s = all_of<G>(s, red, add_f);
    ta = all_of<G>(ta, red, add_f);
}

// G 64: four rows a workgroup, a wave each; 256: a row's chunk a workgroup
template <int ST, int G>
__global__ void __launch_bounds__(256) stats_kernel(LossMatrix a, float* pm, float* ps, float* pa, int slot0, int chunk) {
    __shared__ float red[4];
    const long long r = G == 64 ? (long long)blockIdx.x * 4 + threadIdx.x / 64 : (long long)blockIdx.x;
    if (r >= a.rows) return;    // (whole waves; with G 256 never)
    const int t = threadIdx.x % G;
    const int lo = (int)blockIdx.y * chunk, hi = min(a.cols, lo + chunk);
    float m, s, ta;
    row_stats<ST, G>(a, r, lo, hi, t, red, m, s, ta);
    if (t == 0) {
        const long long at = (long long)(slot0 + blockIdx.y) * a.rows + r;
        pm[at] = m;
        ps[at] = s;
        pa[at] = ta;
    }
}

// The cotangent of one target slot's column: `e` is the first slot that names
// it; the weights of those after it that name it too are added in order.
__device__ __forceinline__ bool first_of(const LossTarget& t, long long at, int e, float& p) {
    const int col = t.col[at + e];
    if (e > 0 && t.col[at + e - 1] == col) return false;
    p = t.p[at + e];
    for (int q = e + 1; q < t.k && t.col[at + q] == col; ++q) p += t.p[at + q];
    return true;
}

// out = coef * (2^(u - lse) - t).  One target a row is met as its column
// passes; several are written after the row's other columns, by a thread each,
// once the stores of this workgroup (or wave) have reached memory.
template <int SI, int SO, int G>
__global__ void __launch_bounds__(256) grad_kernel(LossMatrix a, const float* lse, const float* coef, void* out, long long ldo,
                                                   unsigned* flag, int chunk) {
    typedef typename Elem<SI>::S S;
    typedef typename Elem<SO>::S T;
    constexpr int V = SI == kF32 ? 4 : 8;
    const long long r = G == 64 ? (long long)blockIdx.x * 4 + threadIdx.x / 64 : (long long)blockIdx.x;
    if (r >= a.rows) return;
    const int t = threadIdx.x % G, lo = (int)blockIdx.y * chunk, hi = min(a.cols, lo + chunk);
    const S* const z = (const S*)a.z + r * a.ld;
    T* const o = (T*)out + r * ldo;
    const float c = coef[r], l = lse[r] * kLog2e;
    const int k = a.t.k, one = k == 1 ? a.t.col[r] - a.col0 : -1;
    const long long at = r * k;
    bool ovf = false;
    // at most four slots a thread (1024 by 256; a wave has 64 or 1024 by 16)
    constexpr int E = 1024 / G;
    float zt[E];
    if (k > 1)
        for (int q = 0; q < E; ++q) {
            const int e = t + q * G;
            zt[q] = 0.f;
            if (e < k) {
                const int col = a.t.col[at + e] - a.col0;
                if (col >= lo && col < hi) zt[q] = widen<SI>(z[col]);
            }
        }
    auto value = [&](float x, int col) {
        const float g = exp2_of(x, a.c, l) - (col == one ? a.t.p[at] : 0.f);
        return narrow<SO>(c == 0.f ? 0.f : g * c, ovf);
    };
    if (k > 1) {
        // every thread's logits of the targets are read before the row is written
        __builtin_amdgcn_s_waitcnt(0);
        if constexpr (G > 64) __syncthreads();
    }
    const int whole = lo + (hi - lo) / V * V;
    for (int i = lo + t * V; i < whole; i += G * V) {
        const Vec<SI> v = load_vec<SI>(z + i);
        struct { T e[V]; } w;
#pragma unroll
        for (int e = 0; e < V; ++e) w.e[e] = value(widen<SI>(v.e[e]), i + e);
        __builtin_memcpy(o + i, &w, sizeof w);
    }
    if (whole + t < hi) o[whole + t] = value(widen<SI>(z[whole + t]), whole + t);
    if (k > 1) {
        __builtin_amdgcn_s_waitcnt(0);
        if constexpr (G > 64) __syncthreads();
        for (int q = 0; q < E; ++q) {
            const int e = t + q * G;
            if (e >= k) break;
            const int col = a.t.col[at + e] - a.col0;
            float p;
            if (col >= lo && col < hi && first_of(a.t, at, e, p))
                o[col] = narrow<SO>(c == 0.f ? 0.f : (exp2_of(zt[q], a.c, l) - p) * c, ovf);
        }
    }
    if (SO == kF16 && ovf && flag) atomicOr(flag, 1u);
}

// Whole rows, read once: R vectors a thread of G.
template <int ST, int G, int R>
__global__ void __launch_bounds__(G) joint_kernel(LossMatrix a, float temperature, float* lse, float* loss, const float* coef,
                                                  void* out, long long ldo, unsigned* flag) {
    typedef typename Elem<ST>::S S;
    constexpr int V = Elem<ST>::V;
    __shared__ float red[G / 64];
    const long long r = blockIdx.x;
    const int t = threadIdx.x, k = a.t.k, nv = a.cols / V, rest = a.cols - nv * V;
    const S* const z = (const S*)a.z + r * a.ld;
    const long long at = r * k;
    Vec<ST> v[R];
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (t + i * G < nv) v[i] = load_vec<ST>(z + (long long)(t + i * G) * V);
    const bool tail = t < rest;
    const float last = tail ? widen<ST>(z[nv * V + t]) : -INFINITY;
    constexpr int E = (1024 + G - 1) / G;
    float zt[E], ta = 0.f;
#pragma unroll
    for (int q = 0; q < E; ++q) {
        const int e = t + q * G;
        zt[q] = 0.f;
        if (e < k) {
            const int col = a.t.col[at + e];
            const float p = a.t.p[at + e];
            if (col < a.cols) {
                zt[q] = widen<ST>(z[col]);
                if (p != 0.f) ta += p * (zt[q] * a.c);
            }
        }
    }
    float m = last;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (t + i * G < nv)
#pragma unroll
            for (int e = 0; e < V; ++e) m = fmaxf(m, widen<ST>(v[i].e[e]));
    m = all_of<G>(m, red, max_f) * a.c;
    const float b = base_of(m);
    float s = tail ? exp2_of(last, a.c, b) : 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (t + i * G < nv)
#pragma unroll
            for (int e = 0; e < V; ++e) s += exp2_of(widen<ST>(v[i].e[e]), a.c, b);
    s = all_of<G>(s, red, add_f);
    ta = all_of<G>(ta, red, add_f);
    const float ls = pk_logf(s), l = __builtin_fmaf(m, kLn2, ls);
    if (t == 0) {
        if (lse) lse[r] = l;
        if (loss)
            loss[r] = a.t.col[at] == kUnused ? 0.f : temperature * temperature * (a.t.ent[r] + __builtin_fmaf(m - ta, kLn2, ls));
    }
    const float c = coef[r], l2 = l * kLog2e;
    S* const o = (S*)out + r * ldo;
    bool ovf = false;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (t + i * G < nv) {
            Vec<ST> w;
#pragma unroll
            for (int e = 0; e < V; ++e)
                w.e[e] = narrow<ST>(c == 0.f ? 0.f : exp2_of(widen<ST>(v[i].e[e]), a.c, l2) * c, ovf);
            store_vec<ST>(o + (long long)(t + i * G) * V, w);
        }
    if (tail) o[nv * V + t] = narrow<ST>(c == 0.f ? 0.f : exp2_of(last, a.c, l2) * c, ovf);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < E; ++q) {
        const int e = t + q * G;
        if (e >= k) break;
        const int col = a.t.col[at + e];
        float p;
        if (col < a.cols && first_of(a.t, at, e, p))
            o[col] = narrow<ST>(c == 0.f ? 0.f : (exp2_of(zt[q], a.c, l2) - p) * c, ovf);
    }
    if (ST == kF16 && ovf && flag) atomicOr(flag, 1u);
}

// ---- copies ------------------------------------------------------------------------

// rows of `cols` elements into rows of `ldd`, eight elements a thread, zero
// past cols
__global__ void __launch_bounds__(256) pack_kernel(const unsigned short* src, long long lds, long long rows, int cols,
                                                   unsigned short* dst, int ldd) {
    const unsigned vpr = (unsigned)ldd / 8;
    const long long n = rows * vpr;
    for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < n; u += (long long)gridDim.x * 256) {
        const long long r = u / vpr;
        const int c = (int)(u - r * vpr) * 8;
        const unsigned short* const p = src + r * lds + c;
        u16x8 v;
        if (c + 8 <= cols) {
            __builtin_memcpy(&v, p, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? p[e] : (unsigned short)0;
        }
        *(u16x8*)(dst + r * ldd + c) = v;
    }
}

__global__ void __launch_bounds__(256) zero_kernel(unsigned char* dst, long long bytes) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < bytes; i += (long long)gridDim.x * 256) dst[i] = 0;
}

template <int ST>
__global__ void __launch_bounds__(256) join_kernel(LossGemm g) {
    const long long n = (long long)g.M * g.N, i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float s = g.part[i];
    int p = 1;
    for (; p + 8 <= g.splits; p += 8) {
        float w[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) w[q] = g.part[(long long)(p + q) * n + i];
#pragma unroll
        for (int q = 0; q < 8; ++q) s += w[q];
    }
    for (; p < g.splits; ++p) s += g.part[(long long)p * n + i];
    if (g.scale) s *= *g.scale;
    if (g.acc_in) s += g.acc[i];
    if (g.C) {
        bool ovf = false;
        const long long m = i / g.N;
        ((unsigned short*)g.C)[m * g.ldc + (i - m * g.N)] = narrow<ST>(s, ovf);
        if (ovf && g.flag) atomicOr(g.flag, 1u);
    } else {
        g.acc[i] = s;
    }
}

unsigned blocks_of(long long n) { return (unsigned)std::min<long long>((n + 255) / 256, 16384); }

template <int ST>
hipError_t stats(const LossMatrix& m, float* pm, float* ps, float* pa, int slot0, int chunks, int chunk, hipStream_t s) {
    if (m.cols <= 1024)
        stats_kernel<ST, 64><<<dim3((unsigned)((m.rows + 3) / 4)), 256, 0, s>>>(m, pm, ps, pa, slot0, m.cols);
    else
        stats_kernel<ST, 256><<<dim3((unsigned)m.rows, (unsigned)chunks), 256, 0, s>>>(m, pm, ps, pa, slot0, chunk);
    return hipGetLastError();
}

template <int SI, int SO>
hipError_t grad(const LossMatrix& m, const float* lse, const float* coef, void* out, long long ldo, unsigned* flag, int chunks,
                int chunk, hipStream_t s) {
    if (m.cols <= 1024)
        grad_kernel<SI, SO, 64><<<dim3((unsigned)((m.rows + 3) / 4)), 256, 0, s>>>(m, lse, coef, out, ldo, flag, m.cols);
    else
        grad_kernel<SI, SO, 256><<<dim3((unsigned)m.rows, (unsigned)chunks), 256, 0, s>>>(m, lse, coef, out, ldo, flag, chunk);
    return hipGetLastError();
}

// a chunk's columns: whole vectors of a workgroup
int chunk_cols(int cols, int chunks) { return ((cols + chunks - 1) / chunks + 2047) / 2048 * 2048; }

template <int ST>
hipError_t joint(const LossMatrix& m, float temperature, float* lse, float* loss, const float* coef, void* out, long long ldo,
                 unsigned* flag, hipStream_t s) {
    const int nv = m.cols / Elem<ST>::V;
    const unsigned n = (unsigned)m.rows;
    if (nv <= 256 * 4) joint_kernel<ST, 256, 4><<<n, 256, 0, s>>>(m, temperature, lse, loss, coef, out, ldo, flag);
    else if (nv <= 512 * 8) joint_kernel<ST, 512, 8><<<n, 512, 0, s>>>(m, temperature, lse, loss, coef, out, ldo, flag);
    else if (nv <= 1024 * 8) joint_kernel<ST, 1024, 8><<<n, 1024, 0, s>>>(m, temperature, lse, loss, coef, out, ldo, flag);
    else joint_kernel<ST, 1024, 16><<<n, 1024, 0, s>>>(m, temperature, lse, loss, coef, out, ldo, flag);
    return hipGetLastError();
}

template <int ST>
hipError_t prep(const LossPrep& a, unsigned grid, hipStream_t s) {
    if (a.top <= 64) prep_top_kernel<ST, 64><<<grid, 256, 0, s>>>(a);
    else prep_top_kernel<ST, 256><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

int loss_parts(long long rows, int top) {
    const long long per = top == 0 ? 256 : top <= 64 ? 4 : 1;
    return (int)std::min<long long>((rows + per - 1) / per, kParts);
}

hipError_t loss_prep(const LossPrep& a, hipStream_t s) {
    const unsigned grid = (unsigned)loss_parts(a.rows, a.top);
    if (!grid) return hipSuccess;
    if (a.top == 0) {
        prep_one_kernel<<<grid, 256, 0, s>>>(a);
        return hipGetLastError();
    }
    switch (a.storage) {
        case kF32: return prep<kF32>(a, grid, s);
        case kBF16: return prep<kBF16>(a, grid, s);
        case kF16: return prep<kF16>(a, grid, s);
    }
    return hipErrorInvalidValue;
}

hipError_t loss_rows(const LossRows& a, hipStream_t s) {
    if (a.rows <= 0) return hipSuccess;
    rows_kernel<<<(unsigned)((a.rows + 31) / 32), 256, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t loss_mean(const float* loss, long long rows, const int* count, int parts, float* mean, hipStream_t s) {
    mean_kernel<<<1, 1024, 0, s>>>(loss, rows, count, parts, mean);
    return hipGetLastError();
}

// Few rows are cut into chunks until a thousand workgroups share them.
int loss_chunks(long long rows, int cols) {
    if (cols <= 1024) return 1;
    const long long want = std::min<long long>((1024 + rows - 1) / std::max<long long>(rows, 1), (cols + 2047) / 2048);
    const int chunk = chunk_cols(cols, (int)std::max<long long>(want, 1));
    return (cols + chunk - 1) / chunk;
}

hipError_t loss_stats(const LossMatrix& m, float* pm, float* ps, float* pa, int slot0, hipStream_t s) {
    if (m.rows <= 0 || m.cols <= 0) return hipSuccess;
    const int n = loss_chunks(m.rows, m.cols), chunk = chunk_cols(m.cols, n);
    switch (m.storage) {
        case kF32: return stats<kF32>(m, pm, ps, pa, slot0, n, chunk, s);
        case kBF16: return stats<kBF16>(m, pm, ps, pa, slot0, n, chunk, s);
        case kF16: return stats<kF16>(m, pm, ps, pa, slot0, n, chunk, s);
    }
    return hipErrorInvalidValue;
}

hipError_t loss_grad(const LossMatrix& m, const float* lse, const float* coef, void* out, long long ldo, int to, unsigned* flag,
                     hipStream_t s) {
    if (m.rows <= 0 || m.cols <= 0) return hipSuccess;
    const int n = loss_chunks(m.rows, m.cols), chunk = chunk_cols(m.cols, n);
    if (m.storage == kF32 && to == kF32) return grad<kF32, kF32>(m, lse, coef, out, ldo, flag, n, chunk, s);
    if (m.storage == kBF16 && to == kBF16) return grad<kBF16, kBF16>(m, lse, coef, out, ldo, flag, n, chunk, s);
    if (m.storage == kF16 && to == kF16) return grad<kF16, kF16>(m, lse, coef, out, ldo, flag, n, chunk, s);
    return hipErrorInvalidValue;
}

bool loss_joint_fits(const LossMatrix& m) { return m.cols / (m.storage == kF32 ? 4 : 8) <= 1024 * 16; }

hipError_t loss_joint(const LossMatrix& m, float temperature, float* lse, float* loss, const float* coef, void* out, long long ldo,
                      unsigned* flag, hipStream_t s) {
    if (m.rows <= 0) return hipSuccess;
    switch (m.storage) {
        case kF32: return joint<kF32>(m, temperature, lse, loss, coef, out, ldo, flag, s);
        case kBF16: return joint<kBF16>(m, temperature, lse, loss, coef, out, ldo, flag, s);
        case kF16: return joint<kF16>(m, temperature, lse, loss, coef, out, ldo, flag, s);
    }
    return hipErrorInvalidValue;
}

hipError_t loss_pack(const void* src, long long lds, long long rows, int cols, void* dst, int ldd, hipStream_t s) {
    const long long n = rows * (ldd / 8);
    if (n <= 0) return hipSuccess;
    pack_kernel<<<blocks_of(n), 256, 0, s>>>((const unsigned short*)src, lds, rows, cols, (unsigned short*)dst, ldd);
    return hipGetLastError();
}

hipError_t loss_zero(void* dst, long long bytes, hipStream_t s) {
    if (bytes <= 0) return hipSuccess;
    zero_kernel<<<blocks_of(bytes), 256, 0, s>>>((unsigned char*)dst, bytes);
    return hipGetLastError();
}

hipError_t loss_join(const LossGemm& g, int storage, hipStream_t s) {
    const long long n = (long long)g.M * g.N;
    if (n <= 0) return hipSuccess;
    const unsigned grid = (unsigned)((n + 255) / 256);
    if (storage == kBF16) join_kernel<kBF16><<<grid, 256, 0, s>>>(g);
    else join_kernel<kF16><<<grid, 256, 0, s>>>(g);
    return hipGetLastError();
}

}  // namespace presk
