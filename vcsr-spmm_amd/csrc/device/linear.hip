// linear.hip - which kernel a dense product takes.
#include "dense.hpp"
#include "launch.hpp"
#include "linear_tile.hpp"

namespace vcsr {
namespace {

constexpr int64_t kCus = 256;

GemmPlan plan_of(const Gemm& g, bool dma) {
    const int size = g.type == VCSR_F32 ? 4 : g.type == VCSR_BF16 ? 2 : 1;
    GemmPlan p{};
    p.dma = dma;
    auto tiles = [&](int64_t t) { return (g.I + t - 1) / t * (((int64_t)g.J + t - 1) / t); };
    p.tile_i = p.tile_j = p.dma && tiles(256) >= kCus * 3 / 4 ? 256 : tiles(128) >= kCus ? 128 : 64;
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

// Operands go straight to LDS where their rows lie on 16-byte boundaries in
// whole 16-byte pieces, and a tile's rows are within a buffer's range.
bool direct(const Gemm& g) {
    const int size = g.type == VCSR_F32 ? 4 : g.type == VCSR_BF16 ? 2 : 1;
    auto one = [&](const void* base, int64_t ld, int64_t row) {
        return ((uintptr_t)base | (uintptr_t)(ld * size) | (uintptr_t)(row * size)) % 16 == 0 &&
               ld * size * 256 < ((int64_t)1 << 31);
    };
    return one(g.p, g.ldp, g.p_cols ? g.I : g.R) && one(g.q, g.ldq, g.q_cols ? g.J : g.R);
}

}  // namespace

// Enough for either way of loading: alignment does not change what a caller
// has to provide.
size_t gemm_workspace(const Gemm& g) {
    if (g.I <= 0 || g.J <= 0) return 0;
    const int32_t a = plan_of(g, true).splits, b = plan_of(g, false).splits;
    const int32_t most = a > b ? a : b;
    return most > 1 ? (size_t)most * (size_t)g.I * (size_t)tile::part_ld(g.J) * 4 : 0;
}

hipError_t launch_gemm(const Gemm& g, hipStream_t st) {
    if (g.I <= 0 || g.J <= 0) return hipSuccess;
    const GemmPlan p = plan_of(g, direct(g));
    return g.type == VCSR_F32    ? launch_gemm_f32(g, p, st)
           : g.type == VCSR_BF16 ? launch_gemm_bf16(g, p, st)
                                 : launch_gemm_fp8(g, p, st);
}

}  // namespace vcsr
