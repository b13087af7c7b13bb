// Each head of the queries and keys normed and rotated by its position (rotary.hpp):
//   n = x / sqrt(mean(x^2) + eps),  u = g n,
//   y = (u0 cos a - u1 sin a, u1 cos a + u0 sin a) of a pair (u0, u1), a = position * freq,
// and back: du the pair turned by -a, dg = sum du n, dx = (dn - n mean(dn n)) / sqrt(..)
// with dn = g du.
// A wave takes a token and some of its heads: a head is `lanes` lanes, each with two
// runs of EC elements that are each other's partners, so that no lane needs
// another's; the angles, the same for all of a token's heads, are worked out
// once.  They are turns in f64, of which whole quarters drop out before f32: a
// position of 10^6 keeps what an angle near zero has.
// Bound by its bytes, x read and y written once.
#include "rotary.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "gemm.hpp"
#include "heads.hpp"
#include "loss_dev.hpp"

namespace presk {

namespace {

int storage_code(const char* name) {
    const std::string t = name ? name : "";
    return t == "f32" ? kF32 : t == "bf16" ? kBF16 : t == "f16" ? kF16 : -1;
}

long long up(long long n, long long to) { return (n + to - 1) / to * to; }

struct RotTensor {
    void* p;
    long long batch, seq, head;
};

struct RotArgs {
    RotTensor x[2], y[2];        // q and k; of the gradient dy and dx, and the forward's x
    RotTensor in[2];
    const void* g[2];            // gains or null
    const double* freq;
    const long long* at;         // [batch][seq] or null
    int batch, seq, heads[2], d, rotary, norm, even;
    float eps;
    int lanes;                   // of a head, a power of two
    int per_wave, chunks;        // heads a wave takes of a token, and how many such there are
    float* part;                 // [workgroups][2][d]: the gains' gradients
    unsigned* flag;
};

template <int ST> struct Elem { typedef unsigned short T; };
template <> struct Elem<kF32> { typedef float T; };

template <int ST>
__device__ __forceinline__ float widen(typename Elem<ST>::T v) {
    if constexpr (ST == kF32) return v;
    else if constexpr (ST == kBF16) return pk_bf16_to_f32(v);
    else return pk_f16_to_f32(v);
}
template <int ST>
__device__ __forceinline__ typename Elem<ST>::T narrow(float v) {
    if constexpr (ST == kF32) return v;
    else if constexpr (ST == kBF16) return pk_f32_to_bf16(v);
    else return pk_f32_to_f16(v);
}

template <int ST, int EC>
struct alignas(EC * sizeof(typename Elem<ST>::T)) Run {
    typename Elem<ST>::T v[EC];
};

// cos and sin of `turns` quarter turns: the nearest whole one taken off in f64,
// the rest, at most pi / 4, by the series (to 2e-9).
__device__ __forceinline__ void turned(double quarters, float* c, float* s) {
    const double n = __builtin_rint(quarters);
    const float x = (float)((quarters - n) * 1.5707963267948966);
    const float z = x * x;
    float a = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
    a = __builtin_fmaf(z, a, 8.3333333e-3f);
    a = __builtin_fmaf(z, a, -1.6666667e-1f);
    const float sn = __builtin_fmaf(x * z, a, x);
    float b = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
    b = __builtin_fmaf(z, b, -1.3888889e-3f);
    b = __builtin_fmaf(z, b, 4.1666667e-2f);
    b = __builtin_fmaf(z, b, -0.5f);
    const float cs = __builtin_fmaf(z, b, 1.f);
    // (n mod 4 from the last bits: a position times a frequency stays far below 2^53)
    const int q = (int)((long long)n & 3);
    const float u = q & 1 ? sn : cs, v = q & 1 ? cs : sn;
    *c = q == 1 || q == 2 ? -u : u;
    *s = q >= 2 ? -v : v;
}

// The sum over a head's lanes, in every one of them.
__device__ __forceinline__ float over_lanes(float v, int lanes) {
    if (lanes > 1) v += partner<1>(v);
    if (lanes > 2) v += partner<2>(v);
    if (lanes > 4) v += partner<4>(v);
    if (lanes > 8) v += partner<8>(v);
    if (lanes > 16) v += partner<16>(v);
    if (lanes > 32) v += partner<32>(v);
    return v;
}

template <int ST, int EC, bool GRAD>
__global__ void __launch_bounds__(256) rotary_kernel(RotArgs a) {
    typedef typename Elem<ST>::T T;
    typedef Run<ST, EC> R;
    constexpr int K = EC == 1 ? 2 : 1;      // pairs of runs a lane (a head of 256 single elements)
    const int lane = threadIdx.x & 63, sub = lane / a.lanes, mine = lane % a.lanes, beside = 64 / a.lanes;
    const int pairs = a.rotary / (2 * EC), all = (a.d + 2 * EC - 1) / (2 * EC);

    // the first elements of this lane's two runs
    int e0[K], e1[K];
    bool in[K], in1[K], turns[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int p = mine + k * a.lanes;
        turns[k] = p < pairs;
        in[k] = p < all;
        if (turns[k]) {
            e0[k] = a.even ? 2 * EC * p : EC * p;
            e1[k] = a.even ? 2 * EC * p + EC : a.rotary / 2 + EC * p;
        } else {
            e0[k] = 2 * EC * p;
            e1[k] = e0[k] + EC;
        }
        in1[k] = in[k] && e1[k] < a.d;
    }
    // gains, and their gradients' sums
    float g0[2][K][EC], g1[2][K][EC], s0[2][K][EC], s1[2][K][EC];
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < EC; ++e) {
                const T* const g = (const T*)a.g[w];
                g0[w][k][e] = g && in[k] ? widen<ST>(g[e0[k] + e]) : 1.f;
                g1[w][k][e] = g && in1[k] ? widen<ST>(g[e1[k] + e]) : 1.f;
                s0[w][k][e] = s1[w][k][e] = 0.f;
            }
    bool ovf = false;

    const long long units = (long long)a.batch * a.seq * a.chunks;
    for (long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); unit < units; unit += (long long)gridDim.x * 4) {
        const long long token = unit / a.chunks;
        const int first = (int)(unit - token * a.chunks) * a.per_wave;
        const long long b = token / a.seq, i = token - b * a.seq;
        const double at = (double)(a.at ? a.at[token] : i);
        float cs[K][EC], sn[K][EC];
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int e = 0; e < EC; ++e) {
                cs[k][e] = 1.f, sn[k][e] = 0.f;
                // neighbours: the run's pairs are (e0 + 2 j, e0 + 2 j + 1), EC of them in the two runs
                if (turns[k]) turned(at * a.freq[EC * (mine + k * a.lanes) + e] * 0.6366197723675814, &cs[k][e], &sn[k][e]);
            }
        }
        const int total = a.heads[0] + a.heads[1], end = first + a.per_wave < total ? first + a.per_wave : total;
        for (int h0 = first; h0 < end; h0 += beside) {
            const int hh = h0 + sub;
            const bool live = hh < end;
            const int w = live && hh >= a.heads[0], head = live ? hh - (w ? a.heads[0] : 0) : 0;
            auto row = [&](const RotTensor& t0, const RotTensor& t1) {
                const RotTensor& t = w ? t1 : t0;
                return (T*)t.p + b * t.batch + i * t.seq + head * t.head;
            };
            const T* const xs = !GRAD ? row(a.x[0], a.x[1]) : a.norm ? row(a.in[0], a.in[1]) : nullptr;
            const T* const ds = GRAD ? row(a.x[0], a.x[1]) : nullptr;
            // the head's elements, normed; of the gradient its cotangent too
            float x0[K][EC], x1[K][EC], d0[K][EC], d1[K][EC];
            auto load = [&](const T* p, float (&u)[K][EC], float (&v)[K][EC]) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    R r0{}, r1{};
                    if (live && in[k]) r0 = *(const R*)(p + e0[k]);
                    if (live && in1[k]) r1 = *(const R*)(p + e1[k]);
#pragma unroll
                    for (int e = 0; e < EC; ++e) u[k][e] = widen<ST>(r0.v[e]), v[k][e] = widen<ST>(r1.v[e]);
                }
            };
            if (xs) load(xs, x0, x1);
            if (GRAD) load(ds, d0, d1);
            float rstd = 1.f;
            if (a.norm) {
                float ss = 0.f;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int e = 0; e < EC; ++e) ss += x0[k][e] * x0[k][e] + x1[k][e] * x1[k][e];
                ss = over_lanes(ss, a.lanes);
                rstd = 1.f / sqrtf(ss / (float)a.d + a.eps);
            }
            auto gain = [&](const float (&g)[2][K][EC], int k, int e) { return w ? g[1][k][e] : g[0][k][e]; };
            // a run's pairs: with neighbours paired, element j of the two runs read as one is turned with j ^ 1
            auto turn = [&](float (&u)[K][EC], float (&v)[K][EC], float sign) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if (EC > 1 && a.even) {
                        float z[2 * EC];
#pragma unroll
                        for (int e = 0; e < EC; ++e) z[e] = u[k][e], z[EC + e] = v[k][e];
#pragma unroll
                        for (int e = 0; e < EC; ++e) {
                            const float p = z[2 * e], q = z[2 * e + 1], s = sn[k][e] * sign;
                            z[2 * e] = p * cs[k][e] - q * s;
                            z[2 * e + 1] = q * cs[k][e] + p * s;
                        }
#pragma unroll
                        for (int e = 0; e < EC; ++e) u[k][e] = z[e], v[k][e] = z[EC + e];
                    } else {
#pragma unroll
                        for (int e = 0; e < EC; ++e) {
                            const float p = u[k][e], q = v[k][e], s = sn[k][e] * sign;
                            u[k][e] = p * cs[k][e] - q * s;
                            v[k][e] = q * cs[k][e] + p * s;
                        }
                    }
                }
            };
            if (!GRAD) {
                if (a.norm)
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int e = 0; e < EC; ++e) {
                            x0[k][e] = x0[k][e] * rstd * gain(g0, k, e);
                            x1[k][e] = x1[k][e] * rstd * gain(g1, k, e);
                        }
                turn(x0, x1, 1.f);
            } else {
                turn(d0, d1, -1.f);
                if (a.norm) {
                    float m = 0.f;
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int e = 0; e < EC; ++e) {
                            x0[k][e] *= rstd, x1[k][e] *= rstd;
                            const float t0 = d0[k][e] * x0[k][e], t1 = d1[k][e] * x1[k][e];
                            // (a lane without a head has zeros)
                            s0[0][k][e] += w ? 0.f : t0, s0[1][k][e] += w ? t0 : 0.f;
                            s1[0][k][e] += w ? 0.f : t1, s1[1][k][e] += w ? t1 : 0.f;
                            d0[k][e] *= gain(g0, k, e), d1[k][e] *= gain(g1, k, e);
                            m += d0[k][e] * x0[k][e] + d1[k][e] * x1[k][e];
                        }
                    m = over_lanes(m, a.lanes) / (float)a.d;
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int e = 0; e < EC; ++e) {
                            d0[k][e] = rstd * (d0[k][e] - x0[k][e] * m);
                            d1[k][e] = rstd * (d1[k][e] - x1[k][e] * m);
                        }
                }
            }
            T* const out = row(a.y[0], a.y[1]);
            auto store = [&](const float (&u)[K][EC], const float (&v)[K][EC]) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    R r0, r1;
#pragma unroll
                    for (int e = 0; e < EC; ++e) {
                        r0.v[e] = narrow<ST>(u[k][e]), r1.v[e] = narrow<ST>(v[k][e]);
                        if (ST == kF16) ovf |= live && in[k] && (pk_overflows_f16(u[k][e]) || (in1[k] && pk_overflows_f16(v[k][e])));
                    }
                    if (live && in[k]) *(R*)(out + e0[k]) = r0;
                    if (live && in1[k]) *(R*)(out + e1[k]) = r1;
                }
            };
            if (GRAD) store(d0, d1);
            else store(x0, x1);
        }
    }
    if (ovf && a.flag) atomicOr(a.flag, 1u);
    if (GRAD && a.part) {
        // the heads beside each other, then the four waves
        __shared__ float red[4][2][256];
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < EC; ++e) {
                    float u = s0[w][k][e], v = s1[w][k][e];
                    for (int step = a.lanes; step < 64; step *= 2) u += __shfl_xor(u, step), v += __shfl_xor(v, step);
                    if (sub == 0) {
                        if (in[k]) red[threadIdx.x >> 6][w][e0[k] + e] = u;
                        if (in1[k]) red[threadIdx.x >> 6][w][e1[k] + e] = v;
                    }
                }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * a.d; c += 256) {
            const int w = c / a.d, e = c - w * a.d;
            a.part[(long long)blockIdx.x * 2 * a.d + c] = red[0][w][e] + red[1][w][e] + red[2][w][e] + red[3][w][e];
        }
    }
}

// The gains' gradients: 64 of their elements a workgroup, the partial sums 16
// rows apart a wave, in order, then the waves'.
template <int ST>
__global__ void __launch_bounds__(1024) rotary_gains_kernel(const float* part, int parts, int d, void* dgq, void* dgk, unsigned* flag) {
    __shared__ float red[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
    float s = 0.f;
    if (c < 2 * d)
#pragma unroll 8
        for (int p = wave; p < parts; p += 16) s += part[(long long)p * 2 * d + c];
    red[wave][threadIdx.x & 63] = s;
    __syncthreads();
    if (wave || c >= 2 * d) return;
    s = 0.f;
    for (int w = 0; w < 16; ++w) s += red[w][threadIdx.x];
    void* const out = c < d ? dgq : dgk;
    if (!out) return;
    ((typename Elem<ST>::T*)out)[c < d ? c : c - d] = narrow<ST>(s);
    if (ST == kF16 && flag && pk_overflows_f16(s)) atomicOr(flag, 1u);
}

struct Plan {
    int st;
    bool gains;
    int parts = 0;
    size_t total = 0;
};

// Workgroups of a gradient with gains: each leaves one row of partial sums, so
// that they are no more than fill the chip twice.
constexpr int kParts = 1024;

Plan plan_of(const presk_hip_rot& a, int what) {
    Plan p;
    p.st = storage_code(a.dtype);
    p.gains = what == PRESK_HIP_ROT_GRAD && a.norm;
    if (p.gains) {
        const long long waves = a.batch * a.seq * (a.heads + a.kv_heads);
        p.parts = (int)std::max<long long>(1, std::min<long long>(kParts, (waves + 3) / 4));
        p.total = (size_t)up(8 * p.parts * a.head_dim, 256);
    }
    return p;
}

size_t bytes_of(const Plan& p) { return std::max<size_t>(p.total, 256); }

std::vector<HeadsBuffer> tensors(const presk_hip_rot& a, bool grad) {
    const auto t = [&](const char* n, const presk_hip_heads& t, bool k, bool out, bool need) {
        return HeadsBuffer{n, &t, a.batch, a.seq, k ? a.kv_heads : a.heads, a.head_dim, out, need};
    };
    if (!grad)
        return {t("q", a.q, false, false, true), t("k", a.k, true, false, true), t("yq", a.yq, false, true, true), t("yk", a.yk, true, true, true)};
    const bool x = a.norm != 0;
    return {t("dyq", a.dyq, false, false, true), t("dyk", a.dyk, true, false, true), t("dq", a.dq, false, true, true),
            t("dk", a.dk, true, true, true), t("q", a.q, false, false, x), t("k", a.k, true, false, x)};
}

std::vector<PlainBuffer> others(const presk_hip_rot& a, bool grad, int64_t work) {
    const int64_t esz = storage_code(a.dtype) == kF32 ? 4 : 2, g = a.norm ? esz * a.head_dim : 0;
    return {{"freq", a.freq, 4 * a.rotary, 8, false, true},
            {"at", a.at, 8 * a.batch * a.seq, 8, false, false},
            {"gq", a.gq, g, (int)esz, false, false},
            {"gk", a.gk, g, (int)esz, false, false},
            {"dgq", a.dgq, grad ? g : 0, (int)esz, true, false},
            {"dgk", a.dgk, grad ? g : 0, (int)esz, true, false},
            {"flag", a.flag, 4, 4, true, false},
            {"work", a.work, work, 16, true, grad && a.norm}};
}

template <int ST, bool GRAD>
hipError_t launch(RotArgs& g, int ec, unsigned grid, hipStream_t s) {
    if constexpr (ST != kF32)
        if (ec == 8) {
            rotary_kernel<ST, 8, GRAD><<<grid, 256, 0, s>>>(g);
            return hipGetLastError();
        }
    if (ec == 4) rotary_kernel<ST, 4, GRAD><<<grid, 256, 0, s>>>(g);
    else rotary_kernel<ST, 1, GRAD><<<grid, 256, 0, s>>>(g);
    return hipGetLastError();
}

}  // namespace

std::string rotary_check(const presk_hip_rot& a, int what) {
    auto no = [&](const std::string& why) { return std::string("E10001: head rotary: ") + why; };
    auto size = [&](const char* n, int64_t v) { return no(std::string(n) + " " + std::to_string(v)); };
    const int st = storage_code(a.dtype);
    if (st < 0) return std::string("E7005: head rotary in storage type `") + (a.dtype ? a.dtype : "") + "` (f32, bf16 or f16)";
    if (what != PRESK_HIP_ROT_VALUE && what != PRESK_HIP_ROT_GRAD) return no("what is neither VALUE nor GRAD");
    if (a.batch < 0 || a.batch >= 1 << 24) return size("batch", a.batch);
    if (a.seq < 0 || a.seq >= 1 << 28) return size("seq", a.seq);
    if (a.batch * a.seq >= 1ll << 31) return no("batch * seq past what a launch holds");
    if (a.heads < 1 || a.heads >= 1 << 16) return size("heads", a.heads);
    if (a.kv_heads < 0 || a.kv_heads >= 1 << 16) return size("kv_heads", a.kv_heads);
    if (a.head_dim < 1 || a.head_dim > 256) return size("head_dim", a.head_dim);
    if (a.rotary < 0 || a.rotary > a.head_dim || a.rotary % 2) return size("rotary", a.rotary);
    if (a.norm && !(a.eps >= 0.0 && a.eps <= 1e10)) return no("eps " + std::to_string(a.eps));
    if (!a.norm && (a.gq || a.gk || a.dgq || a.dgk)) return no("gains without a norm");
    return "";
}

std::string rotary_check_all(const presk_hip_rot& a, int what) {
    auto no = [&](const std::string& why) { return std::string("E10001: head rotary: ") + why; };
    if (std::string why = rotary_check(a, what); !why.empty()) return why;
    const bool grad = what == PRESK_HIP_ROT_GRAD;
    const int esz = storage_code(a.dtype) == kF32 ? 4 : 2;
    const std::vector<std::pair<int, int>> in_place{{2, 0}, {3, 1}};
    if (std::string why = buffers_check(tensors(a, grad), others(a, grad, (int64_t)a.work_bytes), esz, in_place); !why.empty()) return no(why);
    const Plan p = plan_of(a, what);
    if (p.total && a.work_bytes < bytes_of(p))
        return no("a workspace of " + std::to_string(a.work_bytes) + " bytes, " + std::to_string(bytes_of(p)) + " needed");
    return "";
}

size_t rotary_workspace(const presk_hip_rot& a, int what) { return bytes_of(plan_of(a, what)); }

void rotary_spans(const presk_hip_rot& a, int what, std::vector<Span>* rd, std::vector<Span>* wr) {
    const bool grad = what == PRESK_HIP_ROT_GRAD;
    buffers_spans(tensors(a, grad), others(a, grad, (int64_t)a.work_bytes), storage_code(a.dtype) == kF32 ? 4 : 2, rd, wr);
}

hipError_t rotary_run(const presk_hip_rot& a, int what, hipStream_t s) {
    const Plan p = plan_of(a, what);
    const bool grad = what == PRESK_HIP_ROT_GRAD;
    const int esz = p.st == kF32 ? 4 : 2;
    RotArgs g{};
    auto tensor = [](const presk_hip_heads& t) { return RotTensor{t.p, t.batch, t.seq, t.head}; };
    g.x[0] = tensor(grad ? a.dyq : a.q), g.x[1] = tensor(grad ? a.dyk : a.k);
    g.y[0] = tensor(grad ? a.dq : a.yq), g.y[1] = tensor(grad ? a.dk : a.yk);
    g.in[0] = tensor(a.q), g.in[1] = tensor(a.k);
    g.g[0] = a.gq, g.g[1] = a.gk;
    g.freq = a.freq;
    g.at = (const long long*)a.at;
    g.batch = (int)a.batch, g.seq = (int)a.seq, g.heads[0] = (int)a.heads, g.heads[1] = (int)a.kv_heads;
    g.d = (int)a.head_dim, g.rotary = (int)a.rotary, g.norm = a.norm != 0, g.even = a.even != 0;
    g.eps = (float)a.eps;
    g.flag = a.flag;
    const long long tokens = a.batch * a.seq;
    if (tokens) {
        // runs of 16 bytes where every tensor's rows, and the halves that are
        // paired, are whole ones
        auto fits = [&](int ec) {
            if (g.d % (2 * ec) || g.rotary % (2 * ec)) return false;
            for (const HeadsBuffer& b : tensors(a, grad)) {
                if (b.count() == 0 || (grad && !a.norm && !b.need)) continue;
                if ((uintptr_t)b.t->p % (uintptr_t)(ec * esz) || b.t->head % ec || b.t->seq % ec || b.t->batch % ec) return false;
            }
            return true;
        };
        const int ec = p.st != kF32 && fits(8) ? 8 : fits(4) ? 4 : 1;
        const int pairs = (g.d + 2 * ec - 1) / (2 * ec);
        g.lanes = 1;
        while (g.lanes < pairs && g.lanes < 64) g.lanes *= 2;
        // heads a wave: all of a token's, or as few as keep the chip full
        const int beside = 64 / g.lanes, total = g.heads[0] + g.heads[1];
        g.per_wave = (int)up(total, beside);
        while (g.per_wave > beside && tokens * ((total + g.per_wave - 1) / g.per_wave) < 4096) g.per_wave = (int)up(g.per_wave / 2, beside);
        g.chunks = (total + g.per_wave - 1) / g.per_wave;
        const long long waves = tokens * g.chunks;
        long long grid = (waves + 3) / 4;
        if (p.gains) {
            grid = std::min<long long>(grid, p.parts);
            g.part = (float*)a.work;
        } else {
            grid = std::min<long long>(grid, 1 << 20);
        }
        hipError_t e;
        if (p.st == kF32) e = grad ? launch<kF32, true>(g, ec, (unsigned)grid, s) : launch<kF32, false>(g, ec, (unsigned)grid, s);
        else if (p.st == kBF16) e = grad ? launch<kBF16, true>(g, ec, (unsigned)grid, s) : launch<kBF16, false>(g, ec, (unsigned)grid, s);
        else e = grad ? launch<kF16, true>(g, ec, (unsigned)grid, s) : launch<kF16, false>(g, ec, (unsigned)grid, s);
        if (e != hipSuccess) return e;
        if (!p.gains || (!a.dgq && !a.dgk)) return hipSuccess;
        const unsigned cols = (unsigned)((2 * g.d + 63) / 64);
        if (p.st == kF32) rotary_gains_kernel<kF32><<<cols, 1024, 0, s>>>(g.part, (int)grid, g.d, a.dgq, a.dgk, a.flag);
        else if (p.st == kBF16) rotary_gains_kernel<kBF16><<<cols, 1024, 0, s>>>(g.part, (int)grid, g.d, a.dgq, a.dgk, a.flag);
        else rotary_gains_kernel<kF16><<<cols, 1024, 0, s>>>(g.part, (int)grid, g.d, a.dgq, a.dgk, a.flag);
        return hipGetLastError();
    }
    if (p.gains && (a.dgq || a.dgk)) {
        // no tokens: the gains' gradients are zero
        const unsigned cols = (unsigned)((2 * g.d + 63) / 64);
        if (p.st == kF32) rotary_gains_kernel<kF32><<<cols, 1024, 0, s>>>(nullptr, 0, g.d, a.dgq, a.dgk, nullptr);
        else rotary_gains_kernel<kBF16><<<cols, 1024, 0, s>>>(nullptr, 0, g.d, a.dgq, a.dgk, nullptr);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace presk
