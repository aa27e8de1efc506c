// linear.hip - which kernel a dense product takes.
#include "dense.hpp"
#include "launch.hpp"
#include "linear_tile.hpp"

namespace vcsr {
namespace {

constexpr int64_t kCus = 256;

GemmPlan plan_of(const Gemm& g) {
    const int size = g.type == VCSR_F32 ? 4 : g.type == VCSR_BF16 ? 2 : 1;
    GemmPlan p{};
    auto tiles = [&](int64_t t) { return (g.I + t - 1) / t * (((int64_t)g.J + t - 1) / t); };
    p.tile_i = p.tile_j = g.type != VCSR_F32 && tiles(256) >= kCus * 3 / 4 ? 256 : tiles(128) >= kCus ? 128 : 64;
    const int64_t all = (g.R * size + tile::kStepBytes - 1) / tile::kStepBytes;
    // Few tiles: the sum is split until the chip has two blocks a compute unit,
    // at least 4 steps each.
    int64_t splits = 2 * kCus / tiles(p.tile_i);
    if (splits > all / 4) splits = all / 4;
    if (splits < 1) splits = 1;
    p.steps = (all + splits - 1) / splits;
    if (p.steps < 1) p.steps = 1;
    p.splits = (int32_t)((all + p.steps - 1) / p.steps);
    if (p.splits < 1) p.splits = 1;
    return p;
}

}  // namespace

size_t gemm_workspace(const Gemm& g) {
    if (g.I <= 0 || g.J <= 0) return 0;
    const GemmPlan p = plan_of(g);
    return p.splits > 1 ? (size_t)p.splits * (size_t)g.I * (size_t)tile::part_ld(g.J) * 4 : 0;
}

hipError_t launch_gemm(const Gemm& g, hipStream_t st) {
    if (g.I <= 0 || g.J <= 0) return hipSuccess;
    const GemmPlan p = plan_of(g);
    return g.type == VCSR_F32    ? launch_gemm_f32(g, p, st)
           : g.type == VCSR_BF16 ? launch_gemm_bf16(g, p, st)
                                 : launch_gemm_fp8(g, p, st);
}

}  // namespace vcsr
