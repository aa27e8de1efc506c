// linear_fp8.hip - the dense product on e4m3 operands (linear_tile.hpp).
#include "linear_tile.hpp"

namespace vcsr {

hipError_t launch_gemm_fp8(const Gemm& g, const GemmPlan& p, hipStream_t st) {
    return tile::launch_layout<fp8, false, false>(g, p, st);
}

}  // namespace vcsr
