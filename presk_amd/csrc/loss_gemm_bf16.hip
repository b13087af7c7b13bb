// The head's products in bf16 storage (loss_gemm.hpp).
#include "loss_gemm.hpp"

namespace presk {

hipError_t loss_gemm_bf16(const LossGemm& g, LossEpi epi, bool bkc, int tile, hipStream_t s) {
    return gemm<kBF16>(g, epi, bkc, tile, s);
}
hipError_t loss_logits_bf16(const LossGemm& g, bool bkc, int tile, const LossPrep& p, hipStream_t s) {
    return bkc ? logits_of<kBF16, true>(g, tile, p, s) : logits_of<kBF16, false>(g, tile, p, s);
}
hipError_t loss_pair_bf16(const LossGemm& x, const LossGemm& w, bool xbkc, int tile, const LossMean& m, hipStream_t s) {
    return pair<kBF16>(x, w, xbkc, tile, m, s);
}

}  // namespace presk
