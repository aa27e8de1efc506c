// linear.hip - which kernel a dense product takes.
#include "dense.hpp"
#include "launch.hpp"
#include "linear_tile.hpp"

namespace vcsr {
namespace {

constexpr int64_t kCus = tile::kCus;

// Measured on MI355X, tiles that fill the chip once: microseconds of one
// 128-byte step of the sum and of everything else of a tile, with 1 to `room`
// blocks on a compute unit.  A second and third block of 64 x 64 bf16 cost next to
// nothing (one alone waits for its loads), a fourth and fifth share the LDS
// pipe; FP32 tiles are bound by their matrix instructions throughout.
struct TileCost {
    int tile, room;
    float step[5], rest[5];
};
constexpr TileCost kF32[] = {
    {64, 5, {0.61f, 1.07f, 1.51f, 2.0f, 2.5f}, {4.2f, 4.8f, 5.7f, 6.2f, 6.6f}},
    {128, 2, {2.05f, 3.68f}, {8.7f, 10.4f}}};
constexpr TileCost kBf16[] = {
    {64, 5, {0.454f, 0.465f, 0.533f, 0.78f, 1.04f}, {3.4f, 3.8f, 4.0f, 4.8f, 5.6f}},
    {128, 2, {0.61f, 0.885f}, {5.7f, 7.6f}},
    {256, 1, {1.44f}, {10.5f}}};
constexpr TileCost kFp8[] = {
    {64, 5, {0.458f, 0.59f, 0.84f, 1.1f, 1.37f}, {4.0f, 4.3f, 4.7f, 5.0f, 5.3f}},
    {128, 2, {0.95f, 1.61f}, {7.0f, 7.3f}},
    {256, 1, {2.53f}, {11.4f}}};

// Of every tile and number of splits, the one with the least estimated time:
// whole rounds of blocks, what is left, and for a split sum the join (its launch,
// and the partial sums written and read at 4 TB/s).
GemmPlan plan_of(const Gemm& g) {
    const int size = g.type == VCSR_F32 ? 4 : g.type == VCSR_BF16 ? 2 : 1;
    const TileCost* costs = g.type == VCSR_F32 ? kF32 : g.type == VCSR_BF16 ? kBf16 : kFp8;
    const int n_costs = g.type == VCSR_F32 ? 2 : 3;
    const int64_t all = (g.R * size + tile::kStepBytes - 1) / tile::kStepBytes;
    // Up to 8 rows: W is read straight into the matrix layout, 6 to 9 us up to 32 MB of
    // it against 10 of the tiles (their join is a launch of its own).  Not where
    // few blocks would read long rows alone: 512 x 8000 bf16 16 us against 10.
    if (g.I <= 8 && !g.p_cols && !g.q_cols && (g.J >= 2048 || 16 * g.R * size <= 192 << 10))
        return GemmPlan{16, 16, 1, all};
    GemmPlan best{};
    float best_us = 0.f;
    for (int c = 0; c < n_costs; ++c) {
        const TileCost& t = costs[c];
        const int64_t tiles = (g.I + t.tile - 1) / t.tile * (((int64_t)g.J + t.tile - 1) / t.tile);
        // Transposing reads of both operands take a quarter longer in the big tile.
        const float slower = t.tile == 256 && g.p_cols ? 1.25f : 1.f;
        for (int64_t want = 1; want <= 128; want += want < 4 ? 1 : want / 2) {
            const int64_t steps = (all + want - 1) / want, splits = (all + steps - 1) / steps;
            if (want > 1 && (steps < 4 || tiles * splits > 8 * kCus)) break;
            const int64_t blocks = tiles * splits, round = kCus * t.room;
            const int64_t rounds = blocks / round, left = blocks - rounds * round;
            auto one = [&](int64_t b) {
                return (float)steps * t.step[b - 1] * slower + t.rest[b - 1];
            };
            float us = (float)rounds * one(t.room);
            if (left) us += one((left + kCus - 1) / kCus);
            if (splits > 1)
                us += 4.f + (float)((double)splits * (double)g.I * (double)g.J * 8e-6 / 4.0);
            if (best.splits == 0 || us < best_us) {
                best_us = us;
                best = GemmPlan{t.tile, t.tile, (int32_t)splits, steps};
            }
        }
    }
    return best;
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
