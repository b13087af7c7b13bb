// Tensors of heads (presk_hip_heads) as the ABI's checks see them: host code alone.
#pragma once

#include <algorithm>
#include <array>
#include <cstdint>
#include <string>
#include <vector>

#include "branches.hpp"
#include "presk_hip.h"

namespace presk {

struct HeadsBuffer {
    const char* name;
    const presk_hip_heads* t;
    int64_t batch, seq, heads, d;
    bool out, need;

    int64_t count() const { return batch * seq * heads * d; }
    // elements from the first to past the last
    int64_t extent() const {
        return count() == 0 ? 0 : (batch - 1) * t->batch + (seq - 1) * t->seq + (heads - 1) * t->head + d;
    }
};

// a buffer of other bytes that a call reads or writes
struct PlainBuffer {
    const char* name;
    const void* p;
    int64_t bytes;
    int align;
    bool out, need;
};

// Why a tensor's strides are refused, or "".  The kernels reach a tile's rows by
// 32-bit offsets (of 128 rows below 2^31, which stands for an element that is
// not there); an output's elements are distinct.
inline std::string heads_check(const HeadsBuffer& b, int esz) {
    if (b.count() == 0) return "";
    if (!b.t->p) return b.need ? std::string(b.name) + " is null" : "";
    if ((uintptr_t)b.t->p % (uintptr_t)esz) return std::string(b.name) + " is not aligned to " + std::to_string(esz) + " bytes";
    constexpr int64_t kMost = 1ll << 40;
    for (int64_t s : {b.t->batch, b.t->seq, b.t->head})
        if (s < 0 || s > kMost) return std::string(b.name) + " has a stride of " + std::to_string(s);
    if (b.seq > 1 && b.t->seq < b.d) return std::string(b.name) + " has rows of " + std::to_string(b.d) + " elements " + std::to_string(b.t->seq) + " apart";
    if (b.seq > 1 && b.t->seq * esz >= 1ll << 24) return std::string(b.name) + " has rows 2^24 bytes apart or more";
    if (b.out) {
        std::vector<std::pair<int64_t, int64_t>> axes;   // stride, length
        if (b.batch > 1) axes.push_back({b.t->batch, b.batch});
        if (b.seq > 1) axes.push_back({b.t->seq, b.seq});
        if (b.heads > 1) axes.push_back({b.t->head, b.heads});
        std::sort(axes.begin(), axes.end());
        int64_t reach = b.d;
        for (const auto& [s, n] : axes) {
            if (s < reach) return std::string(b.name) + " has elements that meet";
            reach += s * (n - 1);
        }
    }
    return "";
}

// Whether two tensors' elements meet.  Where their bytes interleave (slices of a
// packed buffer's rows, of its batches, of its heads) they do not if some stride of
// theirs is a period in which both keep to places of their own: axes whose
// strides are multiples of it stay in place, the others spread a tensor out.
inline bool heads_meet(const HeadsBuffer& a, const HeadsBuffer& b, int esz) {
    if (a.count() == 0 || b.count() == 0 || !a.t->p || !b.t->p) return false;
    const uintptr_t x = (uintptr_t)a.t->p, y = (uintptr_t)b.t->p;
    if (!(x < y + (uintptr_t)(b.extent() * esz) && y < x + (uintptr_t)(a.extent() * esz))) return false;
    const int64_t gap = (int64_t)(y > x ? y - x : x - y);
    if (gap % esz) return true;
    typedef std::pair<int64_t, int64_t> Axis;      // stride, length
    typedef std::array<Axis, 3> Axes;
    auto axes = [](const HeadsBuffer& h) { return Axes{{{h.t->batch, h.batch}, {h.t->seq, h.seq}, {h.t->head, h.heads}}}; };
    const Axes as = axes(a), bs = axes(b);
    auto apart = [&](int64_t period) {
        auto width = [&](const Axes& v, int64_t d) {
            for (const Axis& e : v)
                if (e.second > 1 && e.first % period) d += (e.second - 1) * e.first;
            return d;
        };
        const int64_t wa = width(as, a.d), wb = width(bs, b.d);
        const int64_t at = y > x ? gap / esz % period : (period - gap / esz % period) % period;    // b's place in a's period
        return at >= wa && at + wb <= period;
    };
    for (const auto* v : {&as, &bs})
        for (const Axis& e : *v)
            if (e.second > 1 && e.first > 0 && apart(e.first)) return false;
    return true;
}

inline bool bytes_meet(const void* p, int64_t n, const void* q, int64_t m) {
    return p && q && n > 0 && m > 0 && (uintptr_t)p < (uintptr_t)q + (uintptr_t)m && (uintptr_t)q < (uintptr_t)p + (uintptr_t)n;
}

// The buffers of a call: presence, alignment, strides, and that no output meets
// another buffer (`same`: an output that may be the tensor it stands beside).
inline std::string buffers_check(const std::vector<HeadsBuffer>& ts, const std::vector<PlainBuffer>& ps, int esz,
                                 const std::vector<std::pair<int, int>>& same = {}) {
    for (const HeadsBuffer& b : ts)
        if (std::string why = heads_check(b, esz); !why.empty()) return why;
    for (const PlainBuffer& b : ps) {
        if (b.need && b.bytes > 0 && !b.p) return std::string(b.name) + " is null";
        if ((uintptr_t)b.p % (uintptr_t)b.align) return std::string(b.name) + " is not aligned to " + std::to_string(b.align) + " bytes";
    }
    for (size_t i = 0; i < ts.size(); ++i) {
        if (!ts[i].out || ts[i].count() == 0 || !ts[i].t->p) continue;
        for (size_t j = 0; j < ts.size(); ++j) {
            if (i == j || (ts[j].out && j < i)) continue;
            const presk_hip_heads &a = *ts[i].t, &b = *ts[j].t;
            const bool may = std::find(same.begin(), same.end(), std::make_pair((int)i, (int)j)) != same.end();
            if (may && a.p == b.p && a.batch == b.batch && a.seq == b.seq && a.head == b.head) continue;
            if (heads_meet(ts[i], ts[j], esz)) return std::string(ts[i].name) + " meets " + ts[j].name;
        }
    }
    for (size_t i = 0; i < ps.size(); ++i) {
        for (const HeadsBuffer& t : ts)
            if ((t.out || ps[i].out) && t.count() && bytes_meet(ps[i].p, ps[i].bytes, t.t->p, t.extent() * esz))
                return std::string(ps[i].name) + " meets " + t.name;
        for (size_t j = i + 1; j < ps.size(); ++j)
            if ((ps[i].out || ps[j].out) && bytes_meet(ps[i].p, ps[i].bytes, ps[j].p, ps[j].bytes))
                return std::string(ps[i].name) + " meets " + ps[j].name;
    }
    return "";
}

// The spans of a checked call for the planner of a sequence's branches (the
// flag, which any step only sets, orders none).
inline void buffers_spans(const std::vector<HeadsBuffer>& ts, const std::vector<PlainBuffer>& ps, int esz, std::vector<Span>* rd,
                          std::vector<Span>* wr) {
    for (const HeadsBuffer& t : ts)
        if (t.count() && t.t->p) (t.out ? wr : rd)->push_back({(uintptr_t)t.t->p, (uintptr_t)t.t->p + (size_t)(t.extent() * esz)});
    for (const PlainBuffer& b : ps)
        if (b.p && b.bytes > 0 && std::string(b.name) != "flag") (b.out ? wr : rd)->push_back({(uintptr_t)b.p, (uintptr_t)b.p + (size_t)b.bytes});
}

}  // namespace presk
