// gated_f32.hip - the gated projection on f32 operands (gated_tile.hpp).
#include "gated_tile.hpp"

namespace vcsr {

hipError_t launch_gated_f32(const GatedGemm& g, const GemmPlan& p, hipStream_t st) {
    return tile::launch_gated_tiles<float>(g, p, st);
}

hipError_t launch_gated_grad_f32(const TwinGemm& dw, const GemmPlan& p, const TwiceGemm& dx,
                                 const GemmPlan& q, const RowSum (&bias)[2], hipStream_t st) {
    return tile::launch_grad_of<float>(dw, p, dx, q, bias, st);
}

}  // namespace vcsr
