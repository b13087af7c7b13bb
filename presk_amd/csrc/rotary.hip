// Each head of the queries and keys normed and rotated by its position (rotary.hpp):
//   n = x / sqrt(mean(x^2) + eps),  u = g n,
//   y = (u0 cos a - u1 sin a, u1 cos a + u0 sin a) of a pair (u0, u1), a = position * freq,
// and back: du the pair turned by -a, dg = sum du n, dx = (dn - n mean(dn n)) / sqrt(..)
// with dn = g du.
// A wave takes a token and some of its heads of q, or of k: a head is `lanes` lanes,
// each with two runs of EC elements that are each other's partners, so that no lane
// needs another's; the angles, the same for all heads, are worked out once a wave.
// They are f64, of which whole quarter turns drop out before f32: a position of 10^6
// keeps what an angle near zero has.
// Bound by its bytes, x read and y written once, as long as the work on them stays
// at a few instructions an element: one kernel that told q from k and pairs from
// halves as it went took 47 an element, and 44 us for 2 x 4096 x (32 + 8) heads x 128
// in bf16, normed, and 114 for their gradients; these take 33.8 (a large copy's rate)
// and 59.8 (51 at that rate), and 4.9 for the gains' gradients.
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

// One of q and k.
struct RotSide {
    RotTensor in, x, y;          // what is turned (the forward's x, or dy), the forward's x, and the output
    const void* g;               // gains or null
    void* dg;
    int heads, chunks;           // heads of a token, and how many waves take them
    int blocks;                  // workgroups
};

struct RotArgs {
    RotSide side[2];
    const double* freq;
    const long long* at;         // [batch][seq] or null
    int batch, seq, d, rotary;
    float eps, per_d, sign;      // per_d 1 / d; sign -1 turns back
    int lanes;                   // of a head, a power of two
    int per_wave;                // heads a wave takes of a token
    float* part;                 // [workgroups][d]: the gains' gradients
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
    else if constexpr (ST == kBF16) return __builtin_bit_cast(unsigned short, (__bf16)v);
    else return __builtin_bit_cast(unsigned short, (_Float16)v);
}

template <int ST, int EC>
struct alignas(EC * sizeof(typename Elem<ST>::T)) Run {
    typename Elem<ST>::T v[EC];
};

// cos and sin of an angle: the nearest number of quarter turns taken off in f64, pi / 2
// in two parts by an fma each (Cody and Waite's reduction), the rest, at most pi / 4,
// by the series (to 2e-9).  An angle of 2^30 radians loses nothing that its f64 has:
// 4096 angles below it 6.6e-8 off, by one product with 2 / pi 1.8e-7.
__device__ __forceinline__ void turned(double angle, float* c, float* s) {
    const double n = __builtin_rint(angle * 0.63661977236758134);
    const float x = (float)__builtin_fma(-n, 6.1232339957367660e-17, __builtin_fma(-n, 1.5707963267948966, angle));
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

enum RotMode { kTurn, kNormed, kNormedGrad };

template <int ST, int EC, bool EVEN, RotMode MODE>
__global__ void __launch_bounds__(256) rotary_kernel(RotArgs a) {
    typedef typename Elem<ST>::T T;
    typedef Run<ST, EC> R;
    constexpr bool GRAD = MODE == kNormedGrad;
    constexpr int K = EC == 1 ? 2 : 1;      // pairs of runs a lane (a head of 256 single elements)
    constexpr int U = 2;                    // heads a lane whose loads are under way together (more of them cost waves)
    const bool second = blockIdx.x >= (unsigned)a.side[0].blocks;
    const RotSide& c = a.side[second];
    const int block = (int)blockIdx.x - (second ? a.side[0].blocks : 0);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int sub = lane / a.lanes, mine = lane % a.lanes, beside = 64 / a.lanes;
    const int pairs = a.rotary / (2 * EC), all = (a.d + 2 * EC - 1) / (2 * EC);

    // the first elements of this lane's two runs
    int e0[K], e1[K];
    bool in[K], in1[K], turns[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int p = mine + k * a.lanes;
        turns[k] = p < pairs;
        in[k] = p < all;
        const bool half = turns[k] && !EVEN;
        e0[k] = half ? EC * p : 2 * EC * p;
        e1[k] = half ? a.rotary / 2 + EC * p : 2 * EC * p + EC;
        in1[k] = in[k] && e1[k] < a.d;
    }
    // gains, and their gradients' sums
    float g0[K][EC], g1[K][EC], s0[K][EC], s1[K][EC];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < EC; ++e) {
            const T* const g = (const T*)c.g;
            g0[k][e] = g && in[k] ? widen<ST>(g[e0[k] + e]) : 1.f;
            g1[k][e] = g && in1[k] ? widen<ST>(g[e1[k] + e]) : 1.f;
            s0[k][e] = s1[k][e] = 0.f;
        }
    bool ovf = false;

    const long long units = (long long)a.batch * a.seq * c.chunks;
    for (long long unit = (long long)block * 4 + wave; unit < units; unit += (long long)c.blocks * 4) {
        const long long token = unit / c.chunks;
        const int first = (int)(unit - token * c.chunks) * a.per_wave;
        const int end = first + a.per_wave < c.heads ? first + a.per_wave : c.heads;
        const long long b = token / a.seq, i = token - b * a.seq;
        auto start = [&](const RotTensor& t) { return (T*)t.p + b * t.batch + i * t.seq; };
        T *const ip = start(c.in), *const xp = start(c.x), *const yp = start(c.y);
        R ri0[U][K], ri1[U][K], rx0[GRAD ? U : 1][K], rx1[GRAD ? U : 1][K];
        auto fetch = [&](int h0) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int head = h0 + u * beside + sub;
                auto load = [&](const T* p, R (&r0)[K], R (&r1)[K]) {
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        r0[k] = R{}, r1[k] = R{};
                        if (head < end && in[k]) r0[k] = *(const R*)(p + e0[k]);
                        if (head < end && in1[k]) r1[k] = *(const R*)(p + e1[k]);
                    }
                };
                load(ip + head * c.in.head, ri0[u], ri1[u]);
                if constexpr (GRAD) load(xp + head * c.x.head, rx0[u], rx1[u]);
            }
        };
        fetch(first);       // (under way while the angles are worked out)
        const double at = (double)(a.at ? a.at[token] : i);
        float cs[K][EC], sn[K][EC];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < EC; ++e) {
                cs[k][e] = 1.f, sn[k][e] = 0.f;
                // (neighbours paired: the two runs' EC pairs in order)
                if (turns[k]) turned(at * a.freq[EC * (mine + k * a.lanes) + e], &cs[k][e], &sn[k][e]);
                sn[k][e] *= a.sign;
            }
        for (int h0 = first; h0 < end; h0 += U * beside) {
            if (h0 > first) fetch(h0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int head = h0 + u * beside + sub;
                float v0[K][EC], v1[K][EC], x0[K][EC], x1[K][EC], rstd = 1.f;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int e = 0; e < EC; ++e) {
                        v0[k][e] = widen<ST>(ri0[u][k].v[e]), v1[k][e] = widen<ST>(ri1[u][k].v[e]);
                        if constexpr (GRAD) x0[k][e] = widen<ST>(rx0[u][k].v[e]), x1[k][e] = widen<ST>(rx1[u][k].v[e]);
                    }
                if constexpr (MODE != kTurn) {
                    float ss = 0.f;
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int e = 0; e < EC; ++e) {
                            const float p = GRAD ? x0[k][e] : v0[k][e], q = GRAD ? x1[k][e] : v1[k][e];
                            ss = __builtin_fmaf(p, p, __builtin_fmaf(q, q, ss));
                        }
                    // the hardware's root, refined once
                    const float m = __builtin_fmaf(over_lanes(ss, a.lanes), a.per_d, a.eps), r = __builtin_amdgcn_rsqf(m);
                    rstd = !(m >= 1e-30f && m <= 1e30f) ? 1.f / sqrtf(m) : __builtin_fmaf(__builtin_fmaf(-m * r, r, 1.f), 0.5f * r, r);
                    // (lanes without a head would have 1 / sqrt(eps), infinite for none, times
                    // their zeros in the gains' sums)
                    if (GRAD && head >= end) rstd = 0.f;
                }
                if constexpr (MODE == kNormed)
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int e = 0; e < EC; ++e) v0[k][e] *= rstd * g0[k][e], v1[k][e] *= rstd * g1[k][e];
                // turned: pair e of the two runs, or of the one that they make
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int e = 0; e < EC; ++e) {
                        float& p = EVEN && EC > 1 ? (2 * e < EC ? v0[k][2 * e % EC] : v1[k][2 * e % EC]) : v0[k][e];
                        float& q = EVEN && EC > 1 ? (2 * e < EC ? v0[k][(2 * e + 1) % EC] : v1[k][(2 * e + 1) % EC]) : v1[k][e];
                        const float p0 = p;
                        p = __builtin_fmaf(p0, cs[k][e], -(q * sn[k][e]));
                        q = __builtin_fmaf(q, cs[k][e], p0 * sn[k][e]);
                    }
                if constexpr (GRAD) {
                    float m = 0.f;
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int e = 0; e < EC; ++e) {
                            x0[k][e] *= rstd, x1[k][e] *= rstd;
                            // (a lane without a head has zeros)
                            s0[k][e] = __builtin_fmaf(v0[k][e], x0[k][e], s0[k][e]), s1[k][e] = __builtin_fmaf(v1[k][e], x1[k][e], s1[k][e]);
                            v0[k][e] *= g0[k][e], v1[k][e] *= g1[k][e];
                            m = __builtin_fmaf(v0[k][e], x0[k][e], __builtin_fmaf(v1[k][e], x1[k][e], m));
                        }
                    m = over_lanes(m, a.lanes) * a.per_d;
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int e = 0; e < EC; ++e) {
                            v0[k][e] = rstd * __builtin_fmaf(-x0[k][e], m, v0[k][e]);
                            v1[k][e] = rstd * __builtin_fmaf(-x1[k][e], m, v1[k][e]);
                        }
                }
                T* const out = yp + head * c.y.head;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    R r0, r1;
                    bool over = false;
#pragma unroll
                    for (int e = 0; e < EC; ++e) {
                        r0.v[e] = narrow<ST>(v0[k][e]), r1.v[e] = narrow<ST>(v1[k][e]);
                        if (ST == kF16) over |= pk_overflows_f16(v0[k][e]) || pk_overflows_f16(v1[k][e]);
                    }
                    if (head < end) {
                        if (in[k]) *(R*)(out + e0[k]) = r0;
                        if (in1[k]) *(R*)(out + e1[k]) = r1;
                        ovf |= over;
                    }
                }
            }
        }
    }
    if (ovf && a.flag) atomicOr(a.flag, 1u);
    if constexpr (GRAD) {
        // the heads beside each other, then the four waves
        __shared__ float red[4][256];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < EC; ++e) {
                float u = s0[k][e], v = s1[k][e];
                for (int step = a.lanes; step < 64; step *= 2) u += __shfl_xor(u, step), v += __shfl_xor(v, step);
                if (sub == 0) {
                    if (in[k]) red[wave][e0[k] + e] = u;
                    if (in1[k]) red[wave][e1[k] + e] = v;
                }
            }
        __syncthreads();
        for (int e = threadIdx.x; e < a.d; e += 256)
            a.part[(long long)blockIdx.x * a.d + e] = red[0][e] + red[1][e] + red[2][e] + red[3][e];
    }
}

// The gains' gradients: 64 of their elements a workgroup (of q's, then of k's), a
// sixteenth of the partial sums a wave, in order, then the waves'.
template <int ST>
__global__ void __launch_bounds__(1024) rotary_gains_kernel(const float* part, int parts_q, int parts_k, int d, void* dgq, void* dgk, unsigned* flag) {
    __shared__ float red[16][64];
    const int blocks = (d + 63) / 64, second = (int)blockIdx.x >= blocks;
    const int c = ((int)blockIdx.x - second * blocks) * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
    void* const out = second ? dgk : dgq;
    if (!out) return;
    const int first = second ? parts_q : 0, last = first + (second ? parts_k : parts_q);
    float s = 0.f;
    if (c < d)
#pragma unroll 8
        for (int p = first + wave; p < last; p += 16) s += part[(long long)p * d + c];
    red[wave][threadIdx.x & 63] = s;
    __syncthreads();
    if (wave || c >= d) return;
    s = 0.f;
    for (int w = 0; w < 16; ++w) s += red[w][threadIdx.x];
    ((typename Elem<ST>::T*)out)[c] = narrow<ST>(s);
    if (ST == kF16 && flag && pk_overflows_f16(s)) atomicOr(flag, 1u);
}

struct Plan {
    int st;
    bool gains;
    int parts = 0;
    size_t total = 0;
};

// Workgroups of a gradient with gains: each leaves one row of partial sums, so
// that they are no more than fill the chip.
constexpr int kParts = 1024;

Plan plan_of(const presk_hip_rot& a, int what) {
    Plan p;
    p.st = storage_code(a.dtype);
    p.gains = what == PRESK_HIP_ROT_GRAD && a.norm;
    if (p.gains) {
        const long long waves = a.batch * a.seq * (a.heads + a.kv_heads);
        p.parts = (int)std::max<long long>(2, std::min<long long>(kParts, (waves + 3) / 4 + 1));
        p.total = (size_t)up(4 * p.parts * a.head_dim, 256);
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

template <int ST, int EC, bool EVEN>
void launch_mode(const RotArgs& g, RotMode mode, unsigned grid, hipStream_t s) {
    if (mode == kTurn) rotary_kernel<ST, EC, EVEN, kTurn><<<grid, 256, 0, s>>>(g);
    else if (mode == kNormed) rotary_kernel<ST, EC, EVEN, kNormed><<<grid, 256, 0, s>>>(g);
    else rotary_kernel<ST, EC, EVEN, kNormedGrad><<<grid, 256, 0, s>>>(g);
}
template <int ST, int EC>
void launch_even(const RotArgs& g, bool even, RotMode mode, unsigned grid, hipStream_t s) {
    // (single elements are paired by their places alone)
    if (even) launch_mode<ST, EC, true>(g, mode, grid, s);
    else launch_mode<ST, EC, false>(g, mode, grid, s);
}
template <int ST>
hipError_t launch(const RotArgs& g, int ec, bool even, RotMode mode, unsigned grid, hipStream_t s) {
    if (ec == 4) launch_even<ST, 4>(g, even, mode, grid, s);
    else launch_even<ST, 1>(g, even, mode, grid, s);
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
    g.side[0] = RotSide{tensor(grad ? a.dyq : a.q), tensor(a.q), tensor(grad ? a.dq : a.yq), a.gq, a.dgq, (int)a.heads, 0, 0};
    g.side[1] = RotSide{tensor(grad ? a.dyk : a.k), tensor(a.k), tensor(grad ? a.dk : a.yk), a.gk, a.dgk, (int)a.kv_heads, 0, 0};
    g.freq = a.freq;
    g.at = (const long long*)a.at;
    g.batch = (int)a.batch, g.seq = (int)a.seq, g.d = (int)a.head_dim, g.rotary = (int)a.rotary;
    g.eps = (float)a.eps, g.per_d = 1.f / (float)a.head_dim, g.sign = grad ? -1.f : 1.f;
    g.flag = a.flag;
    g.part = (float*)a.work;
    const long long tokens = a.batch * a.seq;
    if (tokens) {
        // runs of 4 elements where every tensor's rows, and the halves that are
        // paired, are whole ones (of 8 in 16 bits the registers hold two waves a SIMD
        // of a gradient: 83 us, of 4 60; the value 44 and 33)
        auto fits = [&](int ec) {
            if (g.d % (2 * ec) || g.rotary % (2 * ec)) return false;
            for (const HeadsBuffer& b : tensors(a, grad)) {
                if (b.count() == 0 || (grad && !a.norm && !b.need)) continue;
                if ((uintptr_t)b.t->p % (uintptr_t)(ec * esz) || b.t->head % ec || b.t->seq % ec || b.t->batch % ec) return false;
            }
            return true;
        };
        const int ec = fits(4) ? 4 : 1;
        const int pairs = (g.d + 2 * ec - 1) / (2 * ec);
        g.lanes = 1;
        while (g.lanes < pairs && g.lanes < 64) g.lanes *= 2;
        // heads a wave: all of a token's, or as few as keep the chip full
        const int beside = 64 / g.lanes, most = std::max(g.side[0].heads, g.side[1].heads);
        g.per_wave = (int)up(most, beside);
        while (g.per_wave > beside && tokens * ((most + g.per_wave - 1) / g.per_wave) < 4096) g.per_wave = (int)up(g.per_wave / 2, beside);
        long long units[2], all = 0;
        for (int n = 0; n < 2; ++n) {
            g.side[n].chunks = (g.side[n].heads + g.per_wave - 1) / g.per_wave;
            units[n] = tokens * g.side[n].chunks;
            all += (units[n] + 3) / 4;
        }
        // workgroups: enough for every wave, or, of a gradient with gains, one for
        // each row of partial sums, shared out by the heads
        const long long limit = p.gains ? p.parts : 1 << 22;
        const double share = (double)a.heads / (double)(a.heads + a.kv_heads);
        for (int n = 0; n < 2; ++n) {
            const long long need = (units[n] + 3) / 4;
            const long long part = std::max<long long>(1, (long long)((double)(limit - 1) * (n ? 1.0 - share : share)));
            g.side[n].blocks = (int)(all <= limit ? need : std::min(need, part));
        }
        const unsigned grid = (unsigned)(g.side[0].blocks + g.side[1].blocks);
        const RotMode mode = !a.norm ? kTurn : grad ? kNormedGrad : kNormed;
        const bool even = a.even != 0;
        hipError_t e = p.st == kF32 ? launch<kF32>(g, ec, even, mode, grid, s)
                       : p.st == kBF16 ? launch<kBF16>(g, ec, even, mode, grid, s)
                                       : launch<kF16>(g, ec, even, mode, grid, s);
        if (e != hipSuccess) return e;
    }
    if (!p.gains || (!a.dgq && !a.dgk)) return hipSuccess;
    // (of no tokens: zeros)
    const unsigned cols = 2 * (unsigned)((g.d + 63) / 64);
    const int pq = g.side[0].blocks, pk = g.side[1].blocks;
    if (p.st == kF32) rotary_gains_kernel<kF32><<<cols, 1024, 0, s>>>(g.part, pq, pk, g.d, a.dgq, a.dgk, a.flag);
    else if (p.st == kBF16) rotary_gains_kernel<kBF16><<<cols, 1024, 0, s>>>(g.part, pq, pk, g.d, a.dgq, a.dgk, a.flag);
    else rotary_gains_kernel<kF16><<<cols, 1024, 0, s>>>(g.part, pq, pk, g.d, a.dgq, a.dgk, a.flag);
    return hipGetLastError();
}

}  // namespace presk
