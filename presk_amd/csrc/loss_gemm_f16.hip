// The head's products in f16 storage (loss_gemm.hpp).
#include "loss_gemm.hpp"

namespace presk {

hipError_t loss_gemm_f16(const LossGemm& g, LossEpi epi, bool akc, bool bkc, int tile, hipStream_t s) {
    return dispatch<kF16>(g, epi, akc, bkc, tile, s);
}

}  // namespace presk
