// linear_f32.hip - the dense product on f32 operands (linear_tile.hpp).
#include "linear_tile.hpp"

namespace vcsr {

hipError_t launch_gemm_f32(const Gemm& g, const GemmPlan& p, hipStream_t st) {
    if (g.p_cols) return tile::launch_layout<float, true, true>(g, p, st);   // dw
    if (g.q_cols) return tile::launch_layout<float, false, true>(g, p, st);  // dx
    return tile::launch_layout<float, false, false>(g, p, st);
}

hipError_t launch_pair_f32(const Gemm& dw, const GemmPlan& p, const Gemm& dx, const GemmPlan& q,
                           const RowSum& bias, hipStream_t st) {
    return tile::launch_pair<float>(dw, p, dx, q, bias, st);
}

}  // namespace vcsr
