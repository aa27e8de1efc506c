// gated_bf16.hip - the gated projection on bf16 operands (gated_tile.hpp).
#include "gated_tile.hpp"

namespace vcsr {

hipError_t launch_gated_bf16(const GatedGemm& g, const GemmPlan& p, hipStream_t st) {
    return tile::launch_gated_tiles<bf16>(g, p, st);
}

hipError_t launch_gated_grad_bf16(const TwinGemm& dw, const GemmPlan& p, const TwiceGemm& dx,
                                 const GemmPlan& q, const RowSum (&bias)[2], hipStream_t st) {
    return tile::launch_grad_of<bf16>(dw, p, dx, q, bias, st);
}

}  // namespace vcsr
