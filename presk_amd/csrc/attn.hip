// Attention: what a call checks, its workspace and its launches (attn.hpp).
#include "attn.hpp"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "heads.hpp"

namespace presk {

namespace {

int storage_code(const char* name) {
    const std::string t = name ? name : "";
    return t == "f32" ? kF32 : t == "bf16" ? kBF16 : t == "f16" ? kF16 : -1;
}

long long up(long long n, long long to) { return (n + to - 1) / to * to; }

// 4 bytes' truth as 4 bits.
__device__ __forceinline__ unsigned truths(unsigned v) {
    return ((((v & 0x7f7f7f7fu) + 0x7f7f7f7fu) | v) >> 7 & 0x01010101u) * 0x01020408u >> 24;
}

// A byte mask's bits by rows and by columns, and which of its blocks of 32 x 32
// hold any: a wave takes 32 rows and 64 columns, a lane 32 columns of a row, from
// which a column's bits are a vote.  Reads each byte once (2 x 1024 x 1024 3.8 us,
// of which 3 are a launch's).
__global__ void __launch_bounds__(256) attn_mask_kernel(AttnMask m) {
    const int lane = threadIdx.x & 63, blocks = (m.tq + 31) / 32, pairs = (m.words + 1) / 2;
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (long long)m.nbatch * blocks * pairs) return;
    const int w = 2 * (int)(unit % pairs) + (lane >> 5);
    const long long line = unit / pairs, b = line / blocks;
    const int rb = (int)(line - b * blocks), i = 32 * rb + (lane & 31);
    unsigned bits = 0;
    if (i < m.tq && w < m.words) {
        const unsigned char* const src = m.mask + b * m.batch + i * m.row + 32LL * w;
        const int left = m.cols - 32 * w < 32 ? m.cols - 32 * w : 32;
        if (left == 32 && ((uintptr_t)src & 3) == 0) {
            unsigned v[8];
            if (((uintptr_t)src & 15) == 0) {
                *(uint4*)v = ((const uint4*)src)[0];
                *(uint4*)(v + 4) = ((const uint4*)src)[1];
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = ((const unsigned*)src)[q];
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) bits |= truths(v[q]) << (4 * q);
        } else {
            for (int e = 0; e < left; ++e) bits |= (src[e] ? 1u : 0u) << e;
        }
        m.bits[(b * m.tq + i) * m.words + w] = bits;
    }
    const unsigned long long any = __ballot(bits != 0);
    if ((lane & 31) == 0 && w < m.words) m.any[line * m.words + w] = (unsigned)(any >> lane) != 0;
    if (!m.bits_t) return;
    unsigned col = 0;
#pragma unroll
    for (int c = 0; c < 32; ++c) {
        const unsigned long long set = __ballot(bits >> c & 1);
        if ((lane & 31) == c) col = (unsigned)(set >> (lane & 32));
    }
    const int c = 32 * w + (lane & 31);
    if (c < m.cols) m.bits_t[(b * m.cols + c) * m.words_t + rb] = col;
}

// What a checked call launches.
struct Plan {
    int st, nd, pack = 1, splits = 1, chunk = 0, parts = 1;
    int words = 0, words_t = 0, nbits = 0;
    size_t bits = 0, bits_t = 0, any = 0, part = 0, ml = 0, rows = 0, total = 0;     // offsets in the workspace
};

// Keys a split of `items` workgroups' ranges: as many splits as come to `want`
// workgroups, of `least` keys at least.
int chunk_of(long long items, long long tk, long long want, long long least) {
    const long long splits = std::max<long long>(1, want / std::max<long long>(items, 1));
    return (int)std::min<long long>(up(std::max<long long>((tk + splits - 1) / splits, least), 128), 1 << 28);
}

Plan plan_of(const presk_hip_attn& a, int what) {
    Plan p;
    p.st = storage_code(a.dtype);
    p.nd = a.head_dim <= 64 ? 2 : a.head_dim <= 128 ? 4 : 8;
    const long long all = a.batch * a.heads * a.q_len;
    auto take = [&](long long bytes) {
        const size_t at = p.total;
        p.total += (size_t)up(bytes, 256);
        return at;
    };
    const bool grad = what == PRESK_HIP_ATTN_GRAD;
    if (a.mask_cols) {
        // (a mask that the sequences share is taken as theirs: the workspace is
        // one of the sizes alone)
        p.words = (int)up(a.mask_cols, 32) / 32;
        p.words_t = (int)up(a.q_len, 32) / 32;
        p.bits = take(4 * a.batch * a.q_len * p.words);
        if (grad) p.bits_t = take(4 * a.batch * a.mask_cols * p.words_t);
        p.any = take(a.batch * p.words_t * p.words);
    }
    const long long per = a.heads / a.kv_heads;
    if (a.q_len < kAttnTile) p.pack = (int)per;
    if (grad) {
        p.rows = take(8 * all);
        // the keys' and values' gradients in parts of their rows, where one
        // workgroup's tiles of 64 rows are more than a CU's share of all tiles, the
        // queries' among them (of a causal square's the longest has twice the mean):
        // to a workgroup a CU, and four tiles each at least (32 heads in groups of
        // four x 1024 x 128, causal, all gradients: 133 -> 82 us in four parts, 40
        // heads in groups of eight x 2048: 481 -> 250 in three; heads past 128, whose keys'
        // have launches of their own, whenever there is room)
        const long long units = a.batch * a.kv_heads * (up(a.k_len, kAttnTile) / kAttnTile);
        const long long span = a.window ? std::min<long long>(a.window + kAttnTile, 1 << 28) : 1 << 28;
        const long long own = per * (up(std::min<long long>(a.q_len, span), 64) / 64);
        const long long queries = a.batch * (a.heads / p.pack) * (up(a.q_len * p.pack, kAttnTile) / kAttnTile) * (up(std::min<long long>(a.k_len, span), 64) / 64);
        if ((p.st != kF32 || p.nd == 2) && units && own) {
            const long long mean = std::max<long long>(1, (units * own + queries) / (a.causal && !a.window ? 512 : 256));
            p.parts = (int)std::max<long long>(1, std::min({256 / units, own / 4, p.nd == 8 ? 256 : (own + mean / 2) / mean}));
        }
        if (p.parts > 1) p.part = take(8 * p.parts * a.batch * a.kv_heads * a.k_len * p.nd * 32);
        return p;
    }
    const long long rows = a.q_len * p.pack, units = a.batch * (a.heads / p.pack);
    // few rows in shares of the keys that come to four rounds of the CUs, a workgroup
    // each (32 sequences' single tokens over 8192 keys: 1024 132 us, 768 137, 2048 145)
    if (rows <= kAttnFew) {
        p.chunk = chunk_of(units, a.k_len, 1024, 256);
    } else {
        // others to one (8 x 24 drafted tokens over 4096: 34 us with the join, in two
        // rounds 35, in four 41), where the longest is so much shorter that it pays for
        // the join: 128 workgroups in two shares each of 4096 keys 77 -> 65 us, of 2048
        // 42 -> 40, but of 1024 26 -> 32; 64 in four of 1024 25 -> 23, in three of 600
        // 19 -> 23; in f32, whose keys take longer, 128 in two of 1024 53 -> 42
        p.chunk = chunk_of(up(rows, kAttnTile) / kAttnTile * units, a.k_len, 256, 256);
        if ((a.k_len - p.chunk) * (p.st == kF32 ? 2 : 1) < 768) p.chunk = 0;
    }
    p.splits = p.chunk ? (int)std::max<long long>(1, (a.k_len + p.chunk - 1) / p.chunk) : 1;
    if (p.splits > 1) {
        p.part = take(4 * all * p.splits * p.nd * 32);
        p.ml = take(8 * all * p.splits);
    }
    return p;
}

size_t bytes_of(const Plan& p) { return std::max<size_t>(p.total, 256); }

std::vector<HeadsBuffer> tensors(const presk_hip_attn& a, bool grad) {
    const auto q = [&](const char* n, const presk_hip_heads& t, bool out, bool need) {
        return HeadsBuffer{n, &t, a.batch, a.q_len, a.heads, a.head_dim, out, need};
    };
    const auto k = [&](const char* n, const presk_hip_heads& t, bool out, bool need) {
        return HeadsBuffer{n, &t, a.batch, a.k_len, a.kv_heads, a.head_dim, out, need};
    };
    std::vector<HeadsBuffer> v{q("q", a.q, false, true), k("k", a.k, false, true), k("v", a.v, false, true), q("o", a.o, !grad, true)};
    if (grad) {
        v.push_back(q("dout", a.dout, false, true));
        v.push_back(q("dq", a.dq, true, false));
        v.push_back(k("dk", a.dk, true, false));
        v.push_back(k("dv", a.dv, true, false));
    }
    return v;
}

std::vector<PlainBuffer> others(const presk_hip_attn& a, bool grad, int64_t work) {
    const int64_t mask = a.mask_cols && a.q_len && a.batch ? (a.batch - 1) * a.mask_batch + (a.q_len - 1) * a.mask_row + a.mask_cols : 0;
    return {{"lse", a.lse, 4 * a.batch * a.heads * a.q_len, 4, !grad, grad},
            {"lens", a.lens, 8 * a.batch, 8, false, false},
            {"first", a.first, 8 * a.batch, 8, false, false},
            {"mask", a.mask, mask, 1, false, true},
            {"flag", a.flag, 4, 4, true, false},
            {"work", a.work, work, 16, true, true}};
}

}  // namespace

std::string attn_check(const presk_hip_attn& a, int what) {
    auto no = [&](const std::string& why) { return std::string("E10001: attention: ") + why; };
    auto size = [&](const char* n, int64_t v) { return no(std::string(n) + " " + std::to_string(v)); };
    const int st = storage_code(a.dtype);
    if (st < 0) return std::string("E7005: attention in storage type `") + (a.dtype ? a.dtype : "") + "` (f32, bf16 or f16)";
    if (what != PRESK_HIP_ATTN_VALUE && what != PRESK_HIP_ATTN_GRAD) return no("what is neither VALUE nor GRAD");
    constexpr int64_t kMany = 1ll << 28;
    if (a.batch < 0 || a.batch >= 1 << 24) return size("batch", a.batch);
    if (a.heads < 1 || a.heads >= 1 << 16) return size("heads", a.heads);
    if (a.kv_heads < 1 || a.heads % a.kv_heads) return no("heads " + std::to_string(a.heads) + " are not whole groups of kv_heads " + std::to_string(a.kv_heads));
    if (a.q_len < 0 || a.q_len >= kMany) return size("q_len", a.q_len);
    if (a.k_len < 0 || a.k_len >= kMany) return size("k_len", a.k_len);
    if (a.head_dim < 1 || a.head_dim > 256) return size("head_dim", a.head_dim);
    if (st == kF32 && a.head_dim > 128) return "E7005: attention: head_dim " + std::to_string(a.head_dim) + " in f32 (to 128)";
    if (a.window < 0 || a.window >= kMany) return size("window", a.window);
    if (a.window && !a.causal) return no("a window without causal");
    if (a.mask_cols < 0 || a.mask_cols >= kMany) return size("mask_cols", a.mask_cols);
    if (a.mask_cols && a.causal) return no("a mask and causal");
    if (!(a.scale >= 1e-20 && a.scale <= 1e20)) return no("a scale of " + std::to_string(a.scale) + ", not in [1e-20, 1e20]");
    // workgroups of a launch
    const int64_t most = std::max(a.heads * (up(a.q_len, 16) / 16), a.kv_heads * (up(a.k_len, kAttnTile) / kAttnTile));
    if (a.batch * most >= 1ll << 31) return no("batch * heads * length past what a launch holds");
    if (a.mask_cols && a.batch * up(a.q_len, 32) * (up(a.mask_cols, 32) / 32) >= 1ll << 30)
        return no("a mask past what a launch holds");
    return "";
}

std::string attn_check_all(const presk_hip_attn& a, int what) {
    auto no = [&](const std::string& why) { return std::string("E10001: attention: ") + why; };
    if (std::string why = attn_check(a, what); !why.empty()) return why;
    const bool grad = what == PRESK_HIP_ATTN_GRAD;
    const int esz = storage_code(a.dtype) == kF32 ? 4 : 2;
    if (a.mask_cols) {
        if (a.mask_batch < 0 || a.mask_batch > 1ll << 40 || a.mask_row < 0 || a.mask_row > 1ll << 40) return no("a mask with a negative stride");
    }
    if (grad && !a.dq.p && !a.dk.p && !a.dv.p && a.batch * (a.q_len + a.k_len) > 0) return no("a gradient without an output");
    if (std::string why = buffers_check(tensors(a, grad), others(a, grad, (int64_t)a.work_bytes), esz); !why.empty()) return no(why);
    const size_t need = bytes_of(plan_of(a, what));
    if (a.work_bytes < need) return no("a workspace of " + std::to_string(a.work_bytes) + " bytes, " + std::to_string(need) + " needed");
    return "";
}

size_t attn_workspace(const presk_hip_attn& a, int what) { return bytes_of(plan_of(a, what)); }

void attn_spans(const presk_hip_attn& a, int what, std::vector<Span>* rd, std::vector<Span>* wr) {
    const bool grad = what == PRESK_HIP_ATTN_GRAD;
    buffers_spans(tensors(a, grad), others(a, grad, (int64_t)a.work_bytes), storage_code(a.dtype) == kF32 ? 4 : 2, rd, wr);
}

hipError_t attn_run(const presk_hip_attn& a, int what, hipStream_t s) {
    const Plan p = plan_of(a, what);
    const int esz = p.st == kF32 ? 4 : 2;
    char* const work = (char*)a.work;
    auto tensor = [&](const presk_hip_heads& t, int64_t seq, int64_t heads) {
        auto whole = [&](int64_t n, int64_t stride) { return n < 2 || stride * esz % 16 == 0; };
        const bool vec = (uintptr_t)t.p % 16 == 0 && a.head_dim * esz % 16 == 0 && whole(a.batch, t.batch) && whole(seq, t.seq) && whole(heads, t.head);
        // (a single row's stride may be anything, and the kernels multiply it by a tile's
        // row numbers: what they find past the row has to be zero)
        return AttnTensor{t.p, t.batch, seq < 2 ? a.head_dim : t.seq, t.head, vec};
    };
    auto queries = [&](const presk_hip_heads& t) { return tensor(t, a.q_len, a.heads); };
    auto keys = [&](const presk_hip_heads& t) { return tensor(t, a.k_len, a.kv_heads); };
    AttnArgs g{};
    g.q = queries(a.q);
    g.k = keys(a.k);
    g.v = keys(a.v);
    g.o = queries(a.o);
    g.dout = queries(a.dout);
    g.dq = queries(a.dq);
    g.dk = keys(a.dk);
    g.dv = keys(a.dv);
    g.lse = a.lse;
    g.lens = (const long long*)a.lens;
    g.first = (const long long*)a.first;
    g.first0 = a.k_len - (a.mask_cols ? a.mask_cols : a.q_len);
    g.batch = (int)a.batch;
    g.heads = (int)a.heads;
    g.kv = (int)a.kv_heads;
    g.per = (int)(a.heads / a.kv_heads);
    g.tq = (int)a.q_len;
    g.tk = (int)a.k_len;
    g.d = (int)a.head_dim;
    g.causal = a.causal != 0;
    g.window = (int)a.window;
    g.cols = (int)a.mask_cols;
    g.c = (float)(a.scale * 1.4426950408889634);
    g.scale = (float)a.scale;
    g.flag = a.flag;
    g.pack = p.pack;
    g.splits = p.splits;
    g.chunk = p.chunk;
    g.parts = p.parts;
    g.part = (float*)(work + p.part);
    g.part_ml = (float*)(work + p.ml);
    g.rows = (float*)(work + p.rows);
    if (a.mask_cols && a.batch && a.q_len) {
        const bool grad = what == PRESK_HIP_ATTN_GRAD;
        const int nb = a.mask_batch || a.batch == 1 ? (int)a.batch : 1;
        AttnMask m{a.mask, a.mask_batch, a.mask_row, nb, g.tq, g.cols, p.words, p.words_t, (unsigned*)(work + p.bits),
                   grad ? (unsigned*)(work + p.bits_t) : nullptr, (unsigned char*)(work + p.any)};
        const long long n = (long long)nb * p.words_t * ((p.words + 1) / 2);
        attn_mask_kernel<<<(unsigned)((n + 3) / 4), 256, 0, s>>>(m);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        g.bits = m.bits;
        g.bits_t = m.bits_t;
        g.any = a.mask_cols > 64 ? m.any : nullptr;     // (the few columns of a tree are one tile anyway)
        g.words = m.words;
        g.words_t = m.words_t;
        g.bits_batch = nb > 1 ? g.tq : 0;
        g.bits_t_batch = nb > 1 ? g.cols : 0;
    }
    if (what == PRESK_HIP_ATTN_GRAD)
        return p.st == kF32 ? attn_bwd_f32(g, p.nd, s) : p.st == kBF16 ? attn_bwd_bf16(g, p.nd, s) : attn_bwd_f16(g, p.nd, s);
    return p.st == kF32 ? attn_fwd_f32(g, p.nd, s) : p.st == kBF16 ? attn_fwd_bf16(g, p.nd, s) : attn_fwd_f16(g, p.nd, s);
}

}  // namespace presk
