// The buffers of a loss (presk_hip_loss) and what a recorded step of one reads
// and writes: host code alone.
#pragma once

#include <algorithm>
#include <array>
#include <cstdint>
#include <cstring>
#include <vector>

#include "branches.hpp"
#include "presk_hip.h"

namespace presk {

// a checked call's buffers; what an argument's absence makes of no use has no bytes
struct LossBuffer {
    const char* name;
    const void* p;
    long long bytes;
    int align;
    bool out, need;
};

inline std::array<LossBuffer, 12> loss_buffers(const presk_hip_loss& a, int what, bool head) {
    const bool value = what & PRESK_HIP_LOSS_VALUE, grad = what & PRESK_HIP_LOSS_GRAD;
    const long long esz = std::strcmp(a.dtype, "f32") == 0 ? 4 : 2, k = std::max<int64_t>(a.top, 1);
    const long long nx = a.rows * (head ? a.model : a.vocab) * esz, nw = head ? a.model * a.vocab * esz : 0;
    return {{
        {"x", a.x, nx, (int)esz, false, true},
        {"w", a.w, nw, (int)esz, false, head},
        {"index", a.index, 8 * a.rows * k, 8, false, true},
        {"teacher", a.teacher, esz * a.rows * a.top, (int)esz, false, a.top > 0},
        {"ct", a.ct, grad ? 4 * a.rows : 0, 4, false, false},
        {"loss", a.loss, value ? 4 * a.rows : 0, 4, value, false},
        {"lse", a.lse, 4 * a.rows, 4, value, !value},
        {"mean", a.mean, 8, 4, value, !value && !a.ct},
        {"dx", a.dx, grad ? nx : 0, (int)esz, true, grad && !head},
        {"dw", a.dw, grad ? nw : 0, (int)esz, true, false},
        {"flag", a.flag, 4, 4, true, false},
        {"work", a.work, (long long)a.work_bytes, 16, true, true},
    }};
}

// The byte spans that a step of a sequence reads and writes, for the planner of
// its branches.  The flag is only ever set, by any step: it orders none.
inline void loss_spans(const presk_hip_loss& a, int what, bool head, std::vector<Span>* rd, std::vector<Span>* wr) {
    for (const LossBuffer& f : loss_buffers(a, what, head))
        if (f.p && f.bytes > 0 && f.p != a.flag)
            (f.out ? wr : rd)->push_back({(uintptr_t)f.p, (uintptr_t)f.p + (size_t)f.bytes});
}

}  // namespace presk
