// linear_bf16.hip - the dense product on bf16 operands (linear_tile.hpp).
#include "linear_tile.hpp"

namespace vcsr {

hipError_t launch_gemm_bf16(const Gemm& g, const GemmPlan& p, hipStream_t st) {
    if (g.p_cols) return tile::launch_layout<bf16, true, true>(g, p, st);   // dw
    if (g.q_cols) return tile::launch_layout<bf16, false, true>(g, p, st);  // dx
    return tile::launch_layout<bf16, false, false>(g, p, st);
}

hipError_t launch_pair_bf16(const Gemm& dw, const GemmPlan& p, const Gemm& dx, const GemmPlan& q,
                            const RowSum& bias, hipStream_t st) {
    return tile::launch_pair<bf16>(dw, p, dx, q, bias, st);
}

}  // namespace vcsr
