// Attention in f32 (attn_dev.hpp).
#include "attn_dev.hpp"

namespace presk {

hipError_t attn_fwd_f32(const AttnArgs& a, int nd, hipStream_t s) { return fwd_nd<kF32>(a, nd, s); }
hipError_t attn_bwd_f32(const AttnArgs& a, int nd, hipStream_t s) { return bwd_nd<kF32>(a, nd, s); }

}  // namespace presk
