// Attention in bf16 (attn_dev.hpp).
#include "attn_dev.hpp"

namespace presk {

hipError_t attn_fwd_bf16(const AttnArgs& a, int nd, hipStream_t s) { return fwd_nd<kBF16>(a, nd, s); }
hipError_t attn_bwd_bf16(const AttnArgs& a, int nd, hipStream_t s) { return bwd_nd<kBF16>(a, nd, s); }

}  // namespace presk
