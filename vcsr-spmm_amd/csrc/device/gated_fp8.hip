// gated_fp8.hip - the gated projection on e4m3 operands (gated_tile.hpp).
#include "gated_tile.hpp"

namespace vcsr {

hipError_t launch_gated_fp8(const GatedGemm& g, const GemmPlan& p, hipStream_t st) {
    return tile::launch_gated_tiles<fp8>(g, p, st);
}

}  // namespace vcsr
