// The row kernels of the losses (loss.hpp): a call's targets, the row sums and
// cotangents of logits in memory, and what joins a row's partial sums.
//
// A row's sum of exponentials is taken as sum 2^((z - m) c), c = log2 e / T and m
// the largest logit: a difference, a product and one v_exp_f32 (1 ulp) an
// element.  Largest logits and targets stay in the logits' units: a row of the
// type's lowest value alone, which a mask may leave, has a finite loss.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "loss_dev.hpp"

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

// 16 bytes of a row, at any alignment of the element, as four words
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4 load_vec(const void* p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
__device__ __forceinline__ void store_vec(void* p, u32x4 v) { __builtin_memcpy(p, &v, 16); }
// the same past the caches, of what no cache will hold until it is used
typedef u32x4 u32x4u __attribute__((aligned(2)));
template <bool NT>
__device__ __forceinline__ u32x4 load_row(const void* p) {
    if constexpr (NT) return __builtin_nontemporal_load((const u32x4u*)p);
    else return load_vec(p);
}
template <bool NT>
__device__ __forceinline__ void store_row(void* p, u32x4 v) {
    if constexpr (NT) __builtin_nontemporal_store(v, (u32x4u*)p);
    else store_vec(p, v);
}
// element e of a vector
template <int ST>
__device__ __forceinline__ float elem(u32x4 v, int e) {
    if constexpr (ST == kF32) return pk_float(v[e]);
    else return widen<ST>((unsigned short)(e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xffffu));
}
template <int ST>
__device__ __forceinline__ void set_elem(u32x4& v, int e, typename Elem<ST>::S x) {
    if constexpr (ST == kF32) v[e] = pk_bits(x);
    else if (e & 1) v[e / 2] |= (unsigned)x << 16;
    else v[e / 2] = x;
}
// A row's vectors start where its address is a multiple of 16: `head`
// elements come before, `rest` after the `n` vectors.  Those at the ends go to
// threads 0 .. head + rest - 1, one each (at most 14).
template <int ST>
struct Split {
    int head, n, rest;
    __device__ __forceinline__ Split(const void* row, int cols) {
        constexpr int V = Elem<ST>::V, B = 16 / V;
        head = (int)(((16 - ((size_t)row & 15)) & 15) / B);
        if (head > cols) head = cols;
        n = (cols - head) / V;
        rest = cols - head - n * V;
    }
    __device__ __forceinline__ int edge(int t) const { return t < head ? t : head + n * Elem<ST>::V + t - head; }
    __device__ __forceinline__ int edges() const { return head + rest; }
};

// (m, s) with another (m2, s2), the largest in `unit`s of log 2
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float unit) {
    const float n = fmaxf(m, m2), b = base_of(n);
    s = s * exp2_of(m, unit, b) + s2 * exp2_of(m2, unit, b);
    m = n;
}

// ---- targets ------------------------------------------------------------------

// one column a row: bound by its launch (16384 rows 3.5 us)
__global__ void __launch_bounds__(256) prep_one_kernel(LossPrep a) { prep_one<256>(a, (int)blockIdx.x); }

// A teacher's slots: the softmax of those in use, sorted by column (a slot's
// place is how many come before it: columns below its own, or its own at an
// earlier slot, so the order is one whatever runs first).  k^2 comparisons a row
// out of LDS: G threads a row, E slots a thread, as many rows a workgroup as
// their slots fit.  4096 rows of 64 slots 12 us, 30 with the list of blocks
// that the products without kept logits look their slots up in.
template <int ST, int G, int E>
__device__ __forceinline__ void prep_top(const LossPrep& a, unsigned block, unsigned blocks) {
    constexpr int R = 256 / G, KM = G * E;
    __shared__ __attribute__((aligned(16))) int in[R][KM + 4], sorted[R][KM];  // (rows four banks apart)
    __shared__ float red[4], tally[R][2];
    const int g = threadIdx.x / G, t = threadIdx.x % G, k = a.top;
    typedef typename Elem<ST>::S S;
    float n = 0.f, most = 0.f;
    for (long long r0 = (long long)block * R; r0 < a.rows; r0 += (long long)blocks * R) {
        const long long r = r0 + g;
        const bool live = r < a.rows;
        float x[E];
        int col[E];
        float top = -INFINITY, seen = 0.f;      // seen: 1 a used slot, 2 one outside the vocabulary
#pragma unroll
        for (int q = 0; q < E; ++q) {
            const int j = t + q * G;
            col[q] = kUnused;
            x[q] = -INFINITY;
            if (live && j < k) {
                const long long i = a.index[r * k + j];
                x[q] = widen<ST>(((const S*)a.teacher)[r * k + j]);
                if (i >= 0 && x[q] != -INFINITY) {
                    col[q] = i >= a.vocab ? kOutside : (int)i;
                    seen = fmaxf(seen, i >= a.vocab ? 2.f : 1.f);
                    top = fmaxf(top, x[q]);     // (a NaN comes back in its term)
                }
            }
            in[g][j] = col[q];
        }
        top = all_of<G>(top, red, max_f);
        seen = all_of<G>(seen, red, max_f);
        const float base = base_of(top);
        float total = 0.f;
#pragma unroll
        for (int q = 0; q < E; ++q)
            if (col[q] != kUnused) total += exp2_of(x[q], a.c, base);
        total = all_of<G>(total, red, add_f);   // (and the barrier that `in` needs)
        if constexpr (G <= 64) __syncthreads();
        int at[E];
#pragma unroll
        for (int q = 0; q < E; ++q) at[q] = 0;
        for (int j = 0; j < k; j += 4) {
            const int4 c4 = *(const int4*)&in[g][j];    // (past k: unused, after every slot in use)
            const int c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int q = 0; q < E; ++q) at[q] += c[e] < col[q] || (c[e] == col[q] && j + e < t + q * G);
        }
        const float l2 = __builtin_amdgcn_logf(total);
        float ent = 0.f;
#pragma unroll
        for (int q = 0; q < E; ++q) {
            if (t + q * G >= k) continue;
            float p = 0.f;
            if (col[q] != kUnused) {
                const float u = (x[q] - base) * a.c;
                p = __builtin_amdgcn_exp2f(u) / total;
                if (p != 0.f) ent += p * ((u - l2) * kLn2);
            }
            sorted[g][at[q]] = col[q];
            if (live) {
                a.col[r * k + at[q]] = col[q];
                a.p[r * k + at[q]] = p;
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
            a.ent[r] = seen > 1.f ? NAN : ent;
            if (seen != 0.f) {
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
        a.count[block] = (int)n;
        a.most[block] = most;
    }
}
template <int ST, int G, int E>
__global__ void __launch_bounds__(256) prep_top_kernel(LossPrep a) { prep_top<ST, G, E>(a, blockIdx.x, gridDim.x); }

// ---- a row's partial sums joined ------------------------------------------------

// A row's loss from its sum and how far its target lies below its largest logit
// (`gap`, of which `nat` is 1 of u): the largest against the target's before
// anything is added to it.
__device__ __forceinline__ float row_loss(const LossTarget& t, long long r, float temperature, float gap, float nat, float log_s) {
    if (!counts(t, r)) return 0.f;
    return temperature * temperature * (row_ent(t, r) + __builtin_fmaf(gap, nat, log_s));
}

// T / G rows a workgroup, G threads a row, each over every G-th slot; with a
// mean one workgroup has all the rows.  Bound by the partials' bytes and its
// launch: 8192 rows of 125 slots, 12 MB, 12.5 us; few rows of many slots take a
// wave each (8 rows of 250 and their mean 6.5 us).
template <int T, int G>
__global__ void __launch_bounds__(T) rows_kernel(LossRows a) {
    __shared__ float red[T / 64];
    const int q = threadIdx.x % G;
    const long long r = (long long)blockIdx.x * (T / G) + threadIdx.x / G;
    const bool live = r < a.rows;
    float count = 0.f, most = 0.f;
    if (a.coef) {
        for (int i = threadIdx.x; i < a.parts; i += T) {
            count += (float)a.count[i];
            most = fmaxf(most, a.most[i]);
        }
        count = all_of<T>(count, red, add_f);
        most = all_of<T>(most, red, max_f);
        const float n = a.mean_in ? a.mean_in[1] : count;
        // what all rows share is kept out of 16-bit cotangents (*scale)
        const float shared = a.ct ? a.temperature : a.temperature / fmaxf(n, 1.f);
        const int e = a.scale && a.shift ? scale_exponent(a.ct ? most : 1.f) : 0;
        if (a.scale && blockIdx.x == 0 && threadIdx.x == 0) *a.scale = ldexpf(shared, -e);
        if (live && q == 0) {
            float f = 0.f;
            if (counts(a.t, r)) {
                f = ldexpf((a.ct ? a.ct[r] : 1.f) * (a.scale ? 1.f : shared), e);
                f += row_ent(a.t, r) != row_ent(a.t, r) ? NAN : 0.f;
            }
            a.coef[r] = f;
        }
    }
    if (a.slots) {
        float m = -INFINITY, s = 0.f, ta = 0.f;
        if (live)
            for (int p = q; p < a.slots; p += G) {
                const long long at = (long long)p * a.rows + r;
                join(m, s, a.pm[at], a.ps[at], a.unit);
                if (!a.z.z) ta += a.pa[at];
            }
#pragma unroll
        for (int d = 1; d < G; d *= 2) {
            const float m2 = __shfl_xor(m, d), s2 = __shfl_xor(s, d);
            join(m, s, m2, s2, a.unit);
        }
        // given logits' target, below the largest
        float gap = 0.f;
        if (live && a.z.z)
            for (int e = q; e < a.t.k; e += G) {
                const int col = slot_col(a.t, r, e);
                const float p = slot_p(a.t, r, e);
                if (col >= a.z.cols || p == 0.f) continue;
                const long long at = r * a.z.ld + col;
                const float z = a.z.storage == kF32 ? ((const float*)a.z.z)[at] : a.z.storage == kBF16 ? widen<kBF16>(((const unsigned short*)a.z.z)[at])
                                                                                                       : widen<kF16>(((const unsigned short*)a.z.z)[at]);
                gap += p * (m - z);
            }
#pragma unroll
        for (int d = 1; d < G; d *= 2) {
            ta += __shfl_xor(ta, d);
            gap += __shfl_xor(gap, d);
        }
        if (!a.z.z) gap = m - ta;
        if (live && q == 0) {
            const float ls = pk_logf(s);
            if (a.lse) a.lse[r] = __builtin_fmaf(m, a.nat, ls);
            if (a.loss) a.loss[r] = row_loss(a.t, r, a.temperature, gap, a.nat, ls);
            if (a.top) {
                a.top[r] = m;
                a.sum[r] = ls;
            }
        }
    }
    if (a.mean) {
        __threadfence_block();
        __syncthreads();
        write_mean<T>(LossMean{a.loss, a.rows, a.count, a.parts, a.t.index, a.mean});
    }
}

// the mean, in 64 bits, by one workgroup where no other launch has a place for
// it: 16384 rows 6.3 us, 256 rows 2.2
__global__ void __launch_bounds__(1024) mean_kernel(LossMean m) { write_mean<1024>(m); }

// ---- logits in memory -------------------------------------------------------------

// Columns [lo, hi) of row r by G threads: the largest logit, the sum and the
// target's part, or of a whole row how far that lies below the largest (`gap`).
template <int ST, int G>
__device__ __forceinline__ void row_stats(const LossMatrix& a, long long r, int lo, int hi, int t, float* red, bool gap, float& m,
                                          float& s, float& ta) {
    typedef typename Elem<ST>::S S;
    constexpr int V = Elem<ST>::V;
    const S* const z = (const S*)a.z + r * a.ld;
    const Split<ST> sp(z + lo, hi - lo);
    const S* const w = z + lo + sp.head;
    m = -INFINITY;
    s = 0.f;
    ta = 0.f;
    auto logit = [&](int col) {
        float x = widen<ST>(z[col]);
        if constexpr (ST == kF32)
            for (int p = 1; p < a.planes; ++p) x += z[p * a.plane + col];
        return x;
    };
    // four vectors in flight, their largest first, then one rescale for all
    constexpr int U = 4;
    for (int i = t; i < sp.n; i += U * G) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * G < sp.n) v[u] = load_vec(w + (long long)(i + u * G) * V);
        if constexpr (ST == kF32)
            for (int p = 1; p < a.planes; ++p)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i + u * G < sp.n) {
                        const u32x4 y = load_vec(w + p * a.plane + (long long)(i + u * G) * V);
#pragma unroll
                        for (int e = 0; e < V; ++e) v[u][e] = pk_bits(pk_float(v[u][e]) + pk_float(y[e]));
                    }
        float x = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * G < sp.n)
#pragma unroll
                for (int e = 0; e < V; ++e) x = fmaxf(x, elem<ST>(v[u], e));
        const float n = fmaxf(m, x), b = base_of(n);
        s *= exp2_of(m, a.c, b);
        m = n;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * G < sp.n)
#pragma unroll
                for (int e = 0; e < V; ++e) s += exp2_of(elem<ST>(v[u], e), a.c, b);
    }
    if (t < sp.edges()) {
        const float x = logit(lo + sp.edge(t));
        const float n = fmaxf(m, x), b = base_of(n);
        s = s * exp2_of(m, a.c, b) + exp2_of(x, a.c, b);
        m = n;
    }
    const float top = all_of<G>(m, red, max_f);
    s *= exp2_of(m, a.c, base_of(top));
    m = top;
    for (int e = t; e < a.t.k; e += G) {
        const int col = slot_col(a.t, r, e) - a.col0;
        const float p = slot_p(a.t, r, e);
        if (col >= lo && col < hi && p != 0.f) ta += p * (gap ? m - logit(col) : logit(col));
    }
    s = all_of<G>(s, red, add_f);
    ta = all_of<G>(ta, red, add_f);
}

// G 16, 64: 16 or four rows a workgroup; 256: a row's chunk a workgroup.  Bound
// by the logits' bytes, for few rows by its launch (64 x 50257 in f32, 12.9 MB
// out of the Infinity Cache, 5.2 us; 256 x 65 4.9).
template <int ST, int G>
__global__ void __launch_bounds__(256) stats_kernel(LossMatrix a, float* pm, float* ps, float* pa, int slot0, int chunk,
                                                    LossDone done, bool finish) {
    __shared__ float red[4];
    const long long r = G < 256 ? (long long)blockIdx.x * (256 / G) + threadIdx.x / G : (long long)blockIdx.x;
    if (r >= a.rows) return;    // (all threads of a row; with G 256 never)
    const int t = threadIdx.x % G;
    const int lo = (int)blockIdx.y * chunk, hi = min(a.cols, lo + chunk);
    float m, s, ta;
    row_stats<ST, G>(a, r, lo, hi, t, red, finish, m, s, ta);
    if (t != 0) return;
    if (finish) {
        const float ls = pk_logf(s);
        if (done.lse) done.lse[r] = __builtin_fmaf(m, a.nat, ls);
        if (done.loss) done.loss[r] = row_loss(a.t, r, done.temperature, ta, a.nat, ls);
        if (done.top) {
            done.top[r] = m;
            done.sum[r] = ls;
        }
    } else {
        const long long at = (long long)(slot0 + blockIdx.y) * a.rows + r;
        pm[at] = m;
        ps[at] = s;
        pa[at] = ta;
    }
}

// The same beside the targets of a teacher's slots, which the rows' launch then
// looks up: `parts` workgroups of prep_top, then a row's chunks after another's.
// For few rows, whose calls are their launches: 64 x 50257 in f32, 20 slots, and
// their mean 13.5 us of three kernels, 12.2 of two, 26.3 -> 23.5 a call.
template <int ST, int E>
__global__ void __launch_bounds__(256) stats_beside_kernel(LossMatrix a, float* pm, float* ps, int chunk, int chunks, LossPrep prep) {
    __shared__ float red[4];
    if (blockIdx.x < (unsigned)prep.parts) {
        prep_top<ST, 16, E>(prep, blockIdx.x, (unsigned)prep.parts);
        return;
    }
    const unsigned id = blockIdx.x - (unsigned)prep.parts, c = id % (unsigned)chunks;
    const long long r = id / (unsigned)chunks;
    const int lo = (int)c * chunk;
    float m, s, ta;
    row_stats<ST, 256>(a, r, lo, min(a.cols, lo + chunk), threadIdx.x, red, false, m, s, ta);
    if (threadIdx.x != 0) return;
    pm[c * a.rows + r] = m;
    ps[c * a.rows + r] = s;
}

// Whether slot e is the first that names its column; the weights of those
// after it that name it too are added in order.
__device__ __forceinline__ bool first_of(const LossTarget& t, long long r, int e, float& p) {
    const int col = slot_col(t, r, e);
    if (e > 0 && slot_col(t, r, e - 1) == col) return false;
    p = slot_p(t, r, e);
    for (int q = e + 1; q < t.k && slot_col(t, r, q) == col; ++q) p += slot_p(t, r, q);
    return true;
}

// c * (2^((z - b) cf - l) - p), 0 where c is 0 whatever the logit; `part` 1: what
// its rounding leaves
template <int ST>
__device__ __forceinline__ typename Elem<ST>::S cotangent(float z, float cf, float b, float l, float p, float c, int part, bool& ovf) {
    const float v = c == 0.f ? 0.f : (__builtin_amdgcn_exp2f(__builtin_fmaf(z - b, cf, -l)) - p) * c;
    const typename Elem<ST>::S h = narrow<ST>(v, ovf);
    return part ? narrow<ST>(left_of(v, widen<ST>(h)), ovf) : h;
}

// out = coef * (2^(u - lse) - t).  The target's columns are written after the
// row's others, by a thread each, once the stores of this workgroup (or wave)
// have reached memory.  SI the logits' type, SO the output's.  Bound by the
// bytes in and out; where value and gradient are one call and a row fits a
// workgroup's registers, joint_kernel reads the logits once instead of twice.
template <int SI, int SO, int G>
__global__ void __launch_bounds__(256) grad_kernel(LossMatrix a, const float* top, const float* lse, const float* coef, LossTo to,
                                                   unsigned* flag, int chunk) {
    typedef typename Elem<SI>::S S;
    typedef typename Elem<SO>::S O;
    constexpr int V = Elem<SI>::V;
    const long long r = G == 64 ? (long long)blockIdx.x * 4 + threadIdx.x / 64 : (long long)blockIdx.x;
    const int t = threadIdx.x % G, lo = (int)blockIdx.y * chunk, hi = min(a.cols, lo + chunk);
    O* o = (O*)to.p + r * to.ld + lo;
    const int end = (int)((hi == a.cols && SI != SO ? to.ld : hi) - lo);   // columns written
    const int parts = SI != SO && to.low ? 2 : 1;
    if (r >= a.rows) {
        for (int q = t; q < end && r < to.rows; q += G)
            for (int part = 0; part < parts; ++part) o[q + part * to.low] = (O)0;
        return;
    }
    const S* const z = (const S*)a.z + r * a.ld + lo;
    const float c = coef[r], b = top ? base_of(top[r]) : lse[r] / a.nat, l = top ? lse[r] * kLog2e : 0.f;
    const int k = a.t.k, first = a.col0 + lo, n = hi - lo;
    bool ovf = false;
    // the logits of the target's columns, before the row is written (in place)
    constexpr int E = 1024 / G;
    float zt[E];
    for (int q = 0; q < E && t + q * G < k; ++q) {
        const int col = slot_col(a.t, r, t + q * G) - first;
        zt[q] = col >= 0 && col < n ? widen<SI>(z[col]) : 0.f;
    }
    __builtin_amdgcn_s_waitcnt(0);
    if constexpr (G > 64) __syncthreads();
    const Split<SI> sp(z, n);
    constexpr int U = 2;
    for (int part = 0; part < parts; ++part, o += to.low) {
        for (int i = t; i < sp.n; i += U * G) {
            u32x4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * G < sp.n) v[u] = load_vec(z + sp.head + (long long)(i + u * G) * V);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * G < sp.n) {
                    O* const at = o + sp.head + (long long)(i + u * G) * V;
                    if constexpr (SI == SO) {
                        u32x4 w{};
#pragma unroll
                        for (int e = 0; e < V; ++e) set_elem<SO>(w, e, cotangent<SO>(elem<SI>(v[u], e), a.c, b, l, 0.f, c, 0, ovf));
                        store_vec(at, w);
                    } else {
                        O w[V];
#pragma unroll
                        for (int e = 0; e < V; ++e) w[e] = cotangent<SO>(elem<SI>(v[u], e), a.c, b, l, 0.f, c, part, ovf);
                        __builtin_memcpy(at, w, sizeof w);
                    }
                }
        }
        if (t < sp.edges()) o[sp.edge(t)] = cotangent<SO>(widen<SI>(z[sp.edge(t)]), a.c, b, l, 0.f, c, part, ovf);
        for (int q = n + t; q < end; q += G) o[q] = (O)0;
        __builtin_amdgcn_s_waitcnt(0);
        if constexpr (G > 64) __syncthreads();
        for (int q = 0; q < E && t + q * G < k; ++q) {
            const int e = t + q * G, col = slot_col(a.t, r, e) - first;
            float p;
            if (col >= 0 && col < n && first_of(a.t, r, e, p)) o[col] = cotangent<SO>(zt[q], a.c, b, l, p, c, part, ovf);
        }
    }
    if (SO == kF16 && ovf && flag) atomicOr(flag, 1u);
}

// Whole rows, read once: G threads a row (16, 64: 16 or four rows a workgroup), R
// vectors and E slots of the target each.  SI the logits' type, SO the output's.
// Bound by its row's bytes in and out: 8192 x 32000 in bf16, 1.05 GB, 215 us
// with the row past the caches (NT), 235 without; of 0.26 GB, which the
// Infinity Cache holds, 68 with and 63 without (8192 x 8000); f32 logits of
// 8192 x 32000 into bf16, 1.57 GB, 277 with and 300 without.
template <int SI, int SO, int G, int R, int E, bool NT, bool TWO>
__global__ void __launch_bounds__(G < 256 ? 256 : G, R <= 8 ? 8 : 4) joint_kernel(LossJoint a) {
    typedef typename Elem<SI>::S S;
    typedef typename Elem<SO>::S O;
    constexpr int V = Elem<SI>::V, T = G < 256 ? 256 : G;
    __shared__ float red[T / 64];
    const LossTarget& tg = a.m.t;
    // (a wave's row is one, and its addresses are a uniform base and 32 bits)
    const long long r = G == 16 ? (long long)blockIdx.x * 16 + threadIdx.x / 16
                        : G == 64 ? (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : (long long)blockIdx.x;
    const int t = threadIdx.x % G, k = tg.k, n = a.m.cols;
    O* o = (O*)a.to.p + r * a.to.ld;
    constexpr int parts = TWO ? 2 : 1;
    // (all threads of a row)
    if (r >= a.m.rows) {
        if (r < a.to.rows)
            for (long long c = t; c < a.to.ld; c += G)
                for (int part = 0; part < parts; ++part) o[c + part * a.to.low] = (O)0;
        return;
    }
    const S* const z = (const S*)a.m.z + r * a.m.ld;
    const float cf = a.m.c;
    const Split<SI> sp(z, n);
    const char* const zb = (const char*)(z + sp.head);
    const unsigned off = (unsigned)t * 16u;
    u32x4 v[R];
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (t + i * G < sp.n) v[i] = load_row<NT>(zb + i * G * 16 + off);
    const bool edge = t < sp.edges();
    auto logit = [&](int col) {
        float x = widen<SI>(z[col]);
        if constexpr (SI == kF32)
            for (int p = 1; p < a.m.planes; ++p) x += z[p * a.m.plane + col];
        return x;
    };
    const float last = edge ? logit(sp.edge(t)) : -INFINITY;
    if constexpr (SI == kF32)
        for (int p = 1; p < a.m.planes; ++p)
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (t + i * G < sp.n) {
                    const u32x4 w = load_vec(zb + p * a.m.plane * 4 + i * G * 16 + off);
#pragma unroll
                    for (int e = 0; e < V; ++e) v[i][e] = pk_bits(pk_float(v[i][e]) + pk_float(w[e]));
                }
    float zt[E], pt[E];
#pragma unroll
    for (int q = 0; q < E; ++q) {
        zt[q] = pt[q] = 0.f;
        if (t + q * G < k) {
            const int col = slot_col(tg, r, t + q * G);
            if (col < n) {
                zt[q] = logit(col);
                pt[q] = slot_p(tg, r, t + q * G);
            }
        }
    }
    // what all rows share is kept out of 16-bit cotangents (*scale)
    float c = a.ct ? a.ct[r] : 1.f, shared = a.temperature;
    if (!a.ct || a.scale) {
        float count = 0.f, most = 0.f;
        for (int i = t; i < a.parts; i += G) {
            count += (float)a.count[i];
            most = fmaxf(most, a.most[i]);
        }
        if (!a.ct) shared /= fmaxf(all_of<G>(count, red, add_f), 1.f);
        if (a.scale) {
            int e = 0;
            if constexpr (SO == kF16) e = scale_exponent(a.ct ? all_of<G>(most, red, max_f) : 1.f);
            c = ldexpf(c, e);
            if (r == 0 && t == 0) *a.scale = ldexpf(shared, -e);
        }
    }
    if (!a.scale) c *= shared;
    if (!counts(tg, r)) c = 0.f;
    else if (row_ent(tg, r) != row_ent(tg, r)) c = NAN;
    float m = last;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (t + i * G < sp.n)
#pragma unroll
            for (int e = 0; e < V; ++e) m = fmaxf(m, elem<SI>(v[i], e));
    // (every load of this thread has landed before the barriers below, and so
    // before any thread writes the row: the output may be the input)
    __builtin_amdgcn_s_waitcnt(0);
    m = all_of<G>(m, red, max_f);
    const float b = base_of(m);
    float gap = 0.f;
#pragma unroll
    for (int q = 0; q < E; ++q)
        if (pt[q] != 0.f) gap += pt[q] * (m - zt[q]);
    // (the vectors stay packed between the passes: their elements widened once
    // for all three would be twice the registers)
    auto packed = [&]() {
#pragma unroll
        for (int i = 0; i < R; ++i) asm volatile("" : "+v"(v[i]));
    };
    packed();
    float s = edge ? exp2_of(last, cf, b) : 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (t + i * G < sp.n)
#pragma unroll
            for (int e = 0; e < V; ++e) s += exp2_of(elem<SI>(v[i], e), cf, b);
    s = all_of<G>(s, red, add_f);
    gap = all_of<G>(gap, red, add_f);
    const float ls = pk_logf(s);
    if (t == 0) {
        if (a.lse) a.lse[r] = __builtin_fmaf(m, a.m.nat, ls);
        if (a.loss) a.loss[r] = row_loss(tg, r, a.temperature, gap, a.m.nat, ls);
    }
    const float l2 = ls * kLog2e;
    bool ovf = false;
    for (int part = 0; part < parts; ++part, o += a.to.low) {
        packed();
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (t + i * G < sp.n) {
                char* const at = (char*)(o + sp.head) + i * G * V * (int)sizeof(O) + (unsigned)t * (unsigned)(V * sizeof(O));
                if constexpr (SI == SO) {
                    u32x4 w{};
#pragma unroll
                    for (int e = 0; e < V; ++e) set_elem<SO>(w, e, cotangent<SO>(elem<SI>(v[i], e), cf, b, l2, 0.f, c, 0, ovf));
                    store_row<NT>(at, w);
                } else {
                    O w[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) w[e] = cotangent<SO>(elem<SI>(v[i], e), cf, b, l2, 0.f, c, part, ovf);
                    __builtin_memcpy(at, w, sizeof w);
                }
            }
        if (edge) o[sp.edge(t)] = cotangent<SO>(last, cf, b, l2, 0.f, c, part, ovf);
        if constexpr (SI != SO)
            for (long long q = n + t; q < a.to.ld; q += G) o[q] = (O)0;
        __builtin_amdgcn_s_waitcnt(0);
        if constexpr (G > 64) __syncthreads();
#pragma unroll
        for (int q = 0; q < E; ++q) {
            const int e = t + q * G;
            if (e >= k) break;
            const int col = slot_col(tg, r, e);
            float p;
            if (col < n && first_of(tg, r, e, p)) o[col] = cotangent<SO>(zt[q], cf, b, l2, p, c, part, ovf);
        }
    }
    if (SO == kF16 && ovf && a.flag) atomicOr(a.flag, 1u);
}

// ---- copies ------------------------------------------------------------------------

// rows of `cols` elements into rows of `ldd`, eight elements a thread, zero
// past cols; the first nb workgroups take a's.  Bound by its bytes, read at odd
// addresses: half of 1021 x 50257 in 16 bits and its states, 107 MB in and
// out, 20.8 us.
__global__ void __launch_bounds__(256) pack_kernel(LossPack a, LossPack b, unsigned nb) {
    const bool first = blockIdx.x < nb;
    const LossPack& k = first ? a : b;
    const long long at = first ? blockIdx.x : blockIdx.x - nb, stride = first ? nb : gridDim.x - nb;
    const unsigned vpr = (unsigned)k.ldd / 8;
    const long long n = k.rows * vpr;
    for (long long u = at * 256 + threadIdx.x; u < n; u += stride * 256) {
        const long long r = u / vpr;
        const int c = (int)(u - r * vpr) * 8;
        const unsigned short* const p = (const unsigned short*)k.src + r * k.lds + c;
        u16x8 v;
        if (c + 8 <= k.cols) {
            __builtin_memcpy(&v, p, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = c + e < k.cols ? p[e] : (unsigned short)0;
        }
        *(u16x8*)((unsigned short*)k.dst + r * k.ldd + c) = v;
    }
}

__global__ void __launch_bounds__(256) zero_kernel(unsigned char* dst, long long bytes) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < bytes; i += (long long)gridDim.x * 256) dst[i] = 0;
}

// Four columns of a row a thread, eight splits' loads in flight: bound by the
// partials' bytes (dx of 1999 x 1021 over 25 K columns 8.2 us, 12.2 with one
// column a thread).
template <int ST>
__device__ __forceinline__ void join_at(const LossGemm& g, unsigned i) {
    const unsigned quads = (unsigned)g.lda / 4, m = i / quads;
    const int c = (int)(i - m * quads) * 4;
    const long long n = (long long)g.M * g.lda, at = (long long)m * g.lda + c;
    f32x4 s = *(const f32x4*)(g.part + at);
    int p = 1;
    for (; p + 8 <= g.splits; p += 8) {
        f32x4 w[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) w[q] = *(const f32x4*)(g.part + (long long)(p + q) * n + at);
#pragma unroll
        for (int q = 0; q < 8; ++q) s += w[q];
    }
    for (; p < g.splits; ++p) s += *(const f32x4*)(g.part + (long long)p * n + at);
    if (g.scale) s *= *g.scale;
    if (g.acc_in) s += *(const f32x4*)(g.acc + at);
    if (!g.C) {
        *(f32x4*)(g.acc + at) = s;
        return;
    }
    unsigned short* const out = (unsigned short*)g.C + (long long)m * g.ldc + c;
    bool ovf = false;
    unsigned short h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bool o = false;
        h[e] = narrow<ST>(s[e], o);
        ovf |= o && c + e < g.N;
    }
    if (c + 4 <= g.N) __builtin_memcpy(out, h, 8);
    else
        for (int e = 0; e < 3; ++e)
            if (c + e < g.N) out[e] = h[e];
    if (ovf && g.flag) atomicOr(g.flag, 1u);
}
template <int ST>
__global__ void __launch_bounds__(256) join_kernel(LossGemm x, LossGemm w, unsigned nx) {
    const bool first = blockIdx.x < nx;
    const unsigned i = (first ? blockIdx.x : blockIdx.x - nx) * 256 + threadIdx.x;
    const LossGemm& g = first ? x : w;
    if (i < (unsigned)g.M * ((unsigned)g.lda / 4)) join_at<ST>(g, i);
}

unsigned blocks_of(long long n) { return (unsigned)std::min<long long>((n + 255) / 256, 16384); }

// a chunk's columns: whole vectors of a workgroup
int chunk_cols(int cols, int chunks) { return ((cols + chunks - 1) / chunks + 2047) / 2048 * 2048; }

template <int ST>
hipError_t stats(const LossMatrix& m, float* pm, float* ps, float* pa, int slot0, const LossDone* done, hipStream_t s) {
    const int chunks = loss_chunks(m.rows, m.cols), chunk = chunk_cols(m.cols, chunks);
    if (done && chunks > 1) return hipErrorInvalidValue;
    const LossDone d = done ? *done : LossDone{};
    if (m.cols <= 256)
        stats_kernel<ST, 16><<<dim3((unsigned)((m.rows + 15) / 16)), 256, 0, s>>>(m, pm, ps, pa, slot0, m.cols, d, done);
    else if (m.cols <= 1024)
        stats_kernel<ST, 64><<<dim3((unsigned)((m.rows + 3) / 4)), 256, 0, s>>>(m, pm, ps, pa, slot0, m.cols, d, done);
    else
        stats_kernel<ST, 256><<<dim3((unsigned)m.rows, (unsigned)chunks), 256, 0, s>>>(m, pm, ps, pa, slot0, chunk, d, done);
    return hipGetLastError();
}

template <int ST>
hipError_t stats_beside(LossMatrix m, float* pm, float* ps, const LossPrep& p, hipStream_t s) {
    const int chunks = loss_chunks(m.rows, m.cols), chunk = chunk_cols(m.cols, chunks);
    const unsigned grid = (unsigned)p.parts + (unsigned)(m.rows * chunks);
    m.t.k = 0;
    if (p.top <= 16) stats_beside_kernel<ST, 1><<<grid, 256, 0, s>>>(m, pm, ps, chunk, chunks, p);
    else if (p.top <= 32) stats_beside_kernel<ST, 2><<<grid, 256, 0, s>>>(m, pm, ps, chunk, chunks, p);
    else stats_beside_kernel<ST, 4><<<grid, 256, 0, s>>>(m, pm, ps, chunk, chunks, p);
    return hipGetLastError();
}

template <int SI, int SO>
hipError_t grad(const LossMatrix& m, const float* top, const float* lse, const float* coef, const LossTo& to, unsigned* flag, hipStream_t s) {
    const int chunks = loss_chunks(m.rows, m.cols), chunk = chunk_cols(m.cols, chunks);
    const unsigned rows = (unsigned)std::max(m.rows, to.rows);
    if (m.cols <= 1024) grad_kernel<SI, SO, 64><<<dim3((rows + 3) / 4), 256, 0, s>>>(m, top, lse, coef, to, flag, m.cols);
    else grad_kernel<SI, SO, 256><<<dim3(rows, (unsigned)chunks), 256, 0, s>>>(m, top, lse, coef, to, flag, chunk);
    return hipGetLastError();
}

template <int SI, int SO, int G, int R, bool NT, bool TWO>
void joint_of(const LossJoint& a, long long rows, hipStream_t s) {
    constexpr int T = G < 256 ? 256 : G;
    constexpr int per = T / G;
    const unsigned grid = (unsigned)((rows + per - 1) / per);
    if (a.m.t.k <= G) joint_kernel<SI, SO, G, R, 1, NT, TWO><<<grid, T, 0, s>>>(a);
    else joint_kernel<SI, SO, G, R, G == 16 ? 4 : 1024 / G, NT, TWO><<<grid, T, 0, s>>>(a);
}

template <int SI, int SO, bool NT, bool TWO = false>
hipError_t joint(const LossJoint& a, hipStream_t s) {
    const int nv = a.m.cols / Elem<SI>::V;
    const long long n = std::max(a.m.rows, a.to.rows);
    if (nv <= 16 * 4 && a.m.t.k <= 64) joint_of<SI, SO, 16, 4, NT, TWO>(a, n, s);
    else if (nv <= 64 * 4) joint_of<SI, SO, 64, 4, NT, TWO>(a, n, s);
    else if (nv <= 256 * 4) joint_of<SI, SO, 256, 4, NT, TWO>(a, n, s);
    else if (nv <= 512 * 8) joint_of<SI, SO, 512, 8, NT, TWO>(a, n, s);
    else if (nv <= 1024 * 8) joint_of<SI, SO, 1024, 8, NT, TWO>(a, n, s);
    else joint_of<SI, SO, 1024, 16, NT, TWO>(a, n, s);
    return hipGetLastError();
}
// of the caller's logits into the caller's buffer: past the caches where the two
// do not fit the last of them (256 MiB)
template <int ST>
hipError_t joint_rows(const LossJoint& a, hipStream_t s) {
    const bool nt = a.to.p != a.m.z && 2 * a.m.rows * a.m.cols * (ST == kF32 ? 4 : 2) > (256ll << 20);
    return nt ? joint<ST, ST, true>(a, s) : joint<ST, ST, false>(a, s);
}

template <int ST>
hipError_t prep(const LossPrep& a, unsigned grid, hipStream_t s) {
    if (a.top <= 16) prep_top_kernel<ST, 16, 1><<<grid, 256, 0, s>>>(a);
    else if (a.top <= 32) prep_top_kernel<ST, 16, 2><<<grid, 256, 0, s>>>(a);
    else if (a.top <= 64) prep_top_kernel<ST, 16, 4><<<grid, 256, 0, s>>>(a);
    else if (a.top <= 128) prep_top_kernel<ST, 64, 2><<<grid, 256, 0, s>>>(a);
    else if (a.top <= 256) prep_top_kernel<ST, 64, 4><<<grid, 256, 0, s>>>(a);
    else prep_top_kernel<ST, 256, 4><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

int loss_parts(long long rows, int top) {
    const long long per = top == 0 ? 256 : top <= 64 ? 16 : top <= 256 ? 4 : 1;
    return (int)std::min<long long>((rows + per - 1) / per, kParts);
}

hipError_t loss_prep(const LossPrep& a, hipStream_t s) {
    const unsigned grid = (unsigned)loss_parts(a.rows, a.top);
    if (!grid) return hipSuccess;
    if ((int)grid != a.parts) return hipErrorInvalidValue;
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

// few enough rows for one workgroup
bool loss_rows_mean(long long rows) { return rows <= 128; }

hipError_t loss_rows(const LossRows& a, hipStream_t s) {
    if (a.rows <= 0) return hipSuccess;
    if (a.mean) {
        if (!loss_rows_mean(a.rows) || !a.loss) return hipErrorInvalidValue;
        if (a.rows <= 16) rows_kernel<1024, 64><<<1, 1024, 0, s>>>(a);
        else rows_kernel<1024, 8><<<1, 1024, 0, s>>>(a);
    } else if (a.rows <= 1024 && a.slots > 64) {
        rows_kernel<256, 64><<<(unsigned)((a.rows + 3) / 4), 256, 0, s>>>(a);
    } else {
        rows_kernel<256, 8><<<(unsigned)((a.rows + 31) / 32), 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

hipError_t loss_mean(const LossMean& m, hipStream_t s) {
    mean_kernel<<<1, 1024, 0, s>>>(m);
    return hipGetLastError();
}

// Few rows are cut into chunks until a thousand workgroups share them.
int loss_chunks(long long rows, int cols) {
    if (cols <= 1024) return 1;
    const long long want = std::min<long long>((1024 + rows - 1) / std::max<long long>(rows, 1), (cols + 2047) / 2048);
    const int chunk = chunk_cols(cols, (int)std::max<long long>(want, 1));
    return (cols + chunk - 1) / chunk;
}

hipError_t loss_stats(const LossMatrix& m, float* pm, float* ps, float* pa, int slot0, const LossDone* done, hipStream_t s) {
    if (m.rows <= 0 || m.cols <= 0) return hipSuccess;
    switch (m.storage) {
        case kF32: return stats<kF32>(m, pm, ps, pa, slot0, done, s);
        case kBF16: return stats<kBF16>(m, pm, ps, pa, slot0, done, s);
        case kF16: return stats<kF16>(m, pm, ps, pa, slot0, done, s);
    }
    return hipErrorInvalidValue;
}

bool loss_beside(const LossMatrix& m, int top) { return loss_rows_mean(m.rows) && m.cols > 1024 && top >= 1 && top <= 64; }

hipError_t loss_stats_beside(const LossMatrix& m, float* pm, float* ps, const LossPrep& p, hipStream_t s) {
    if (!loss_beside(m, p.top) || p.parts != loss_parts(p.rows, p.top)) return hipErrorInvalidValue;
    switch (m.storage) {
        case kF32: return stats_beside<kF32>(m, pm, ps, p, s);
        case kBF16: return stats_beside<kBF16>(m, pm, ps, p, s);
        case kF16: return stats_beside<kF16>(m, pm, ps, p, s);
    }
    return hipErrorInvalidValue;
}

hipError_t loss_grad(const LossMatrix& m, const float* top, const float* lse, const float* coef, const LossTo& to, unsigned* flag, hipStream_t s) {
    if (m.rows <= 0 || m.cols <= 0) return hipSuccess;
    if (m.storage == kF32 && to.storage == kF32) return grad<kF32, kF32>(m, top, lse, coef, to, flag, s);
    if (m.storage == kBF16 && to.storage == kBF16) return grad<kBF16, kBF16>(m, top, lse, coef, to, flag, s);
    if (m.storage == kF16 && to.storage == kF16) return grad<kF16, kF16>(m, top, lse, coef, to, flag, s);
    if (m.storage == kF32 && to.storage == kBF16) return grad<kF32, kBF16>(m, top, lse, coef, to, flag, s);
    if (m.storage == kF32 && to.storage == kF16) return grad<kF32, kF16>(m, top, lse, coef, to, flag, s);
    return hipErrorInvalidValue;
}

bool loss_joint_fits(const LossMatrix& m) { return m.cols / (m.storage == kF32 ? 4 : 8) <= 1024 * 16; }

hipError_t loss_joint(const LossJoint& a, hipStream_t s) {
    if (a.m.rows <= 0) return hipSuccess;
    if (a.m.storage == kF32 && a.to.storage == kF32) return joint_rows<kF32>(a, s);
    if (a.m.storage == kBF16 && a.to.storage == kBF16) return joint_rows<kBF16>(a, s);
    if (a.m.storage == kF16 && a.to.storage == kF16) return joint_rows<kF16>(a, s);
    if (a.m.storage != kF32 || (a.to.storage != kBF16 && a.to.storage != kF16)) return hipErrorInvalidValue;
    // (two parts are few rows', which the caches hold)
    const bool bf = a.to.storage == kBF16;
    if (a.to.low) return bf ? joint<kF32, kBF16, false, true>(a, s) : joint<kF32, kF16, false, true>(a, s);
    if (4 * a.m.rows * a.m.ld > (256ll << 20)) return bf ? joint<kF32, kBF16, true>(a, s) : joint<kF32, kF16, true>(a, s);
    return bf ? joint<kF32, kBF16, false>(a, s) : joint<kF32, kF16, false>(a, s);
}

hipError_t loss_pack(const LossPack& a, const LossPack& b, hipStream_t s) {
    auto blocks = [](const LossPack& k) { return k.rows > 0 ? blocks_of(k.rows * (k.ldd / 8)) : 0u; };
    const unsigned na = blocks(a), n = na + blocks(b);
    if (!n) return hipSuccess;
    pack_kernel<<<n, 256, 0, s>>>(a, b, na);
    return hipGetLastError();
}

hipError_t loss_zero(void* dst, long long bytes, hipStream_t s) {
    if (bytes <= 0) return hipSuccess;
    zero_kernel<<<blocks_of(bytes), 256, 0, s>>>((unsigned char*)dst, bytes);
    return hipGetLastError();
}

hipError_t loss_join(const LossGemm& x, const LossGemm& w, int storage, hipStream_t s) {
    auto quads = [](const LossGemm& g) { return g.splits > 1 ? g.M * (g.lda / 4) : 0; };
    if (quads(x) >= 1ll << 30 || quads(w) >= 1ll << 30) return hipErrorInvalidValue;    // (few tiles are split)
    const unsigned nx = (unsigned)(quads(x) + 255) / 256, n = nx + (unsigned)(quads(w) + 255) / 256;
    if (!n) return hipSuccess;
    if (storage == kBF16) join_kernel<kBF16><<<n, 256, 0, s>>>(x, w, nx);
    else join_kernel<kF16><<<n, 256, 0, s>>>(x, w, nx);
    return hipGetLastError();
}

}  // namespace presk
