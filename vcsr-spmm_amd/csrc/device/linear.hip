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
// pipe; with loads three steps ahead instead of one, one or two blocks take two
// thirds of the time (1024^3 10.8 -> 8.0 us).  FP32 tiles are bound by their matrix
// instructions throughout, e4m3 ones by widening, and gain nothing from that, nor
// do the gradients' launches, which fill the chip with both products.
//
// The times are of operands by rows.  Gradients, whose operands lie by columns, are
// estimated with the same ones, which is too little for them (8192 x 2048 x 4096 bf16: dx
// 103 us by the table, 124 to 131 measured; dw in 128 tiles 121, 158 to 178).  So are gated
// projections, whose tile of 64 has other waves and another loader: of 9 to 512 rows the
// choice is up to a quarter slower than the best (359 x 4360 x 2078 bf16 42.9 us in tiles of
// 64, 33.8 in tiles of 128 and four parts).
struct TileCost {
    int tile, stages, room;
    float step[5], rest[5];
};
constexpr TileCost kF32[] = {
    {64, 2, 5, {0.61f, 1.07f, 1.51f, 2.0f, 2.5f}, {4.2f, 4.8f, 5.7f, 6.2f, 6.6f}},
    {128, 2, 2, {2.05f, 3.68f}, {8.7f, 10.4f}}};
constexpr TileCost kBf16[] = {
    {64, 2, 5, {0.454f, 0.465f, 0.533f, 0.78f, 1.04f}, {3.4f, 3.8f, 4.0f, 4.8f, 5.6f}},
    {128, 2, 2, {0.61f, 0.885f}, {5.7f, 7.6f}},
    {256, 2, 1, {1.44f}, {10.5f}},
    {64, 4, 2, {0.292f, 0.358f}, {3.3f, 4.1f}}};  // operands by rows only
constexpr TileCost kFp8[] = {
    {64, 2, 5, {0.458f, 0.59f, 0.84f, 1.1f, 1.37f}, {4.0f, 4.3f, 4.7f, 5.0f, 5.3f}},
    {128, 2, 2, {0.95f, 1.61f}, {7.0f, 7.3f}},
    {256, 2, 1, {2.53f}, {11.4f}}};

struct Costs {
    const TileCost* t;
    int n;
};
Costs costs_of(const Gemm& g) {
    if (g.type == VCSR_F32) return Costs{kF32, 2};
    if (g.type == VCSR_FP8) return Costs{kFp8, 3};
    return Costs{kBf16, g.p_cols || g.q_cols ? 3 : 4};
}
// Steps of the whole sum.
int64_t steps_of(const Gemm& g) {
    const int size = g.type == VCSR_F32 ? 4 : g.type == VCSR_BF16 ? 2 : 1;
    return (g.R * size + tile::kStepBytes - 1) / tile::kStepBytes;
}
int64_t tiles_of(const Gemm& g, int64_t t) {
    return (g.I + t - 1) / t * (((int64_t)g.J + t - 1) / t);
}
// Whether a launch of these blocks can be made: HIP has none of 2^32 threads or more.
bool launches(int64_t blocks, int tile) {
    return blocks * (tile == 256 ? 512 : 256) < (int64_t)1 << 32;
}
// A block's time with b blocks on its compute unit.  Transposing reads of both
// operands take a quarter longer in the big tile.
float block_us(const Gemm& g, const TileCost& t, int64_t steps, int64_t b) {
    const float slower = t.tile == 256 && g.p_cols ? 1.25f : 1.f;
    return (float)steps * t.step[b - 1] * slower + t.rest[b - 1];
}
// The join of a split sum: its launch, and the partial sums written and read at 4
// TB/s.
float join_us(const Gemm& g, int64_t splits) {
    return splits > 1 ? 4.f + (float)((double)splits * (double)g.I * (double)g.J * 2e-6) : 0.f;
}
// f(splits, steps) for every number of splits worth trying over `tiles` tiles.
template <class F>
void each_split(const Gemm& g, int64_t tiles, F&& f) {
    const int64_t all = steps_of(g);
    for (int64_t want = 1; want <= 128; want += want < 4 ? 1 : want / 2) {
        const int64_t steps = (all + want - 1) / want, splits = (all + steps - 1) / steps;
        if (want > 1 && (steps < 4 || tiles * splits > 8 * kCus)) break;
        f(splits, steps);
    }
}

// z and the residual on top of out: their time at 4 TB/s, half of it hidden where
// there is more than one round of blocks.  Both numbers stand on one size: 62451 x 128 x
// 128 FP32 with a residual, tiles of 64 in two rounds 30.3 us, of 128 in one 33.7.
float extra_us(const Gemm& g, bool rounds) {
    const double size = g.out_type == VCSR_F32 ? 4 : 2, count = (g.residual ? 1 : 0) + (g.z ? 1 : 0);
    return (float)((double)g.I * (double)g.J * size * count / 4e6) * (rounds ? 0.5f : 1.f);
}

// Of force_plan().
struct Forced {
    GemmPlan plan{};
    bool together = false;
};
thread_local Forced forced;
bool forced_takes(const Gemm& g) {
    if (forced.plan.tile == 16) return g.I <= 16 && !g.p_cols && !g.q_cols;
    const Costs c = costs_of(g);
    for (const TileCost* t = c.t; t < c.t + c.n; ++t)
        if (t->tile == forced.plan.tile && t->stages == forced.plan.stages) return true;
    return false;
}
GemmPlan forced_plan(const Gemm& g) {
    GemmPlan p = forced.plan;
    const int64_t all = steps_of(g), want = p.splits < all ? p.splits : all;
    p.steps = p.tile == 16 ? all : (all + want - 1) / want;
    p.splits = (int32_t)((all + p.steps - 1) / p.steps);
    if (p.rows <= 0 || p.rows >= g.I || p.splits > 1) p.rows = g.I;
    return p;
}

// Rows [from, g.I) of a product.
Gemm rows_from(Gemm g, int64_t from) {
    const int64_t size = g.type == VCSR_F32 ? 4 : g.type == VCSR_BF16 ? 2 : 1;
    const int64_t out = g.out_type == VCSR_F32 ? 4 : 2;
    g.I -= from;
    if (g.p) g.p = (const char*)g.p + from * size * (g.p_cols ? 1 : g.ldp);
    if (g.p_scale) g.p_scale += from;
    if (g.z) g.z = (char*)g.z + from * g.ldz * out;
    if (g.residual) g.residual = (const char*)g.residual + from * g.ldr * out;
    if (g.out) g.out = (char*)g.out + from * g.ldo * out;
    return g;
}
GatedGemm rows_from(GatedGemm g, int64_t from) {
    const int64_t out = g.out_type == VCSR_F32 ? 4 : 2;
    static_cast<Gemm&>(g) = rows_from(static_cast<const Gemm&>(g), from);
    if (g.z2) g.z2 = (char*)g.z2 + from * g.ldz * out;
    return g;
}

// Of every tile and number of splits, the one with the least estimated time:
// whole rounds of blocks, what is left, and the join.  Where a last round would
// leave most of the chip idle, the rows of the whole rounds go by themselves and the
// rest as a product of its own, in smaller tiles (5001 x 4096 x 4096 bf16: 320 tiles of
// 256 on 256 compute units).  splits = 0: no launch has that many blocks.
GemmPlan plan_of(const Gemm& g, float* us_out = nullptr, bool may_divide = true) {
    const int size = g.type == VCSR_F32 ? 4 : g.type == VCSR_BF16 ? 2 : 1;
    if (forced.plan.tile && forced_takes(g)) return forced_plan(g);
    // Up to 8 rows: W is read straight into the matrix layout, 6 to 9 us up to 32 MB of
    // it against 10 of the tiles (their join is a launch of its own).  Not where
    // few blocks would read long rows alone, past what a wave asks for at once: 512 x
    // 8000 bf16 16 us against 10.
    if (g.I <= 8 && !g.p_cols && !g.q_cols && (g.J >= 2048 || g.R * size <= 64 * 128) &&
        g.J <= (1 << 27) - 16) {  // blocks of 16 columns, fewer than 2^23 of 512 threads
        if (us_out) *us_out = 7.f;
        return GemmPlan{16, 1, 1, steps_of(g), g.I};
    }
    GemmPlan best{};
    float best_us = 0.f;
    const Costs c = costs_of(g);
    for (const TileCost* t = c.t; t < c.t + c.n; ++t) {
        const int64_t tiles = tiles_of(g, t->tile);
        each_split(g, tiles, [&](int64_t splits, int64_t steps) {
            const int64_t blocks = tiles * splits, round = kCus * t->room;
            const bool whole = launches(blocks, t->tile);
            const int64_t rounds = blocks / round, left = blocks - rounds * round;
            float us = (float)rounds * block_us(g, *t, steps, t->room) + join_us(g, splits) +
                       extra_us(g, rounds > 0);
            if (left) us += block_us(g, *t, steps, (left + kCus - 1) / kCus);
            if (whole && (best.splits == 0 || us < best_us)) {
                best_us = us;
                best = GemmPlan{t->tile, t->stages, (int32_t)splits, steps, g.I};
            }
            if (!may_divide || !whole || splits > 1 || rounds < 1 || !left) return;
            const int64_t per_row = ((int64_t)g.J + t->tile - 1) / t->tile;
            const int64_t first = rounds * round / per_row * t->tile;
            if (first < t->tile || first >= g.I) return;
            float rest_us = 0.f;
            if (plan_of(rows_from(g, first), &rest_us, false).splits == 0) return;
            us = (float)rounds * block_us(g, *t, steps, t->room) + extra_us(g, true) + rest_us + 2.f;
            if (us < best_us) {
                best_us = us;
                best = GemmPlan{t->tile, t->stages, 1, steps, first};
            }
        });
    }
    if (us_out) *us_out = best_us;
    return best;
}

// Both products in one launch, if that is estimated faster than one after the
// other: all blocks' time over the chip's room and part of a last block, or the
// longest block alone, and dw's join.  (8192 x 2048 x 4096 bf16: dw has 128 tiles of 256, dx 256.)
PairPlan plan_pair(const Gemm& dw, const Gemm& dx, bool may_divide = true) {
    float us_w = 0.f, us_x = 0.f;
    PairPlan best{false, plan_of(dw, &us_w, may_divide), plan_of(dx, &us_x, may_divide)};
    if (best.dw.splits == 0 || best.dx.splits == 0) return best;
    if (forced.plan.tile && forced_takes(dw)) {
        if (forced.together) {
            best.together = true;
            best.dx.splits = 1;
            best.dx.steps = steps_of(dx);
            best.dw.rows = dw.I;
            best.dx.rows = dx.I;
        }
        return best;
    }
    float best_us = us_w + us_x + 2.f;
    const Costs c = costs_of(dw);
    for (const TileCost* t = c.t; t < c.t + c.n; ++t) {
        const int64_t tiles_w = tiles_of(dw, t->tile), tiles_x = tiles_of(dx, t->tile);
        if (tiles_x > 64 * kCus) continue;  // long by itself: nothing to gain
        each_split(dw, tiles_w, [&](int64_t splits, int64_t steps) {
            const int64_t per_cu = (tiles_w * splits + tiles_x + kCus - 1) / kCus;
            const int64_t b = per_cu < t->room ? per_cu : t->room;
            const float one_w = block_us(dw, *t, steps, b), one_x = block_us(dx, *t, steps_of(dx), b);
            float us = ((float)(tiles_w * splits) * one_w + (float)tiles_x * one_x) /
                           (float)(kCus * b) + 0.25f * one_x;
            if (us < one_w) us = one_w;
            if (us < one_x) us = one_x;
            us += join_us(dw, splits);
            const int64_t blocks = (tiles_w * splits + 7) / 8 * 8 + tiles_x + (dw.I + 15) / 16;
            if (us < best_us && launches(blocks, t->tile)) {
                best_us = us;
                best = PairPlan{true, GemmPlan{t->tile, t->stages, (int32_t)splits, steps, dw.I},
                                GemmPlan{t->tile, t->stages, 1, steps_of(dx), dx.I}};
            }
        });
    }
    return best;
}

const GemmPlan& launchable(const GemmPlan& p) {
    if (p.splits == 0) throw Error(VCSR_ERANGE, "M, N: more tiles than a launch has blocks");
    return p;
}

size_t part_bytes(const Gemm& g, const GemmPlan& p) {
    if (p.rows < g.I) {
        const Gemm rest = rows_from(g, p.rows);
        return part_bytes(rest, plan_of(rest, nullptr, false));
    }
    return p.splits > 1 ? (size_t)p.splits * (size_t)g.I * (size_t)tile::part_ld(g.J) * 4 : 0;
}

hipError_t launch(const Gemm& g, const GemmPlan& p, hipStream_t st) {
    if (p.rows < g.I) {
        Gemm first = g;
        first.I = p.rows;
        const hipError_t e = launch(first, p, st);
        if (e != hipSuccess) return e;
        const Gemm rest = rows_from(g, p.rows);
        return launch(rest, plan_of(rest, nullptr, false), st);
    }
    return g.type == VCSR_F32    ? launch_gemm_f32(g, p, st)
           : g.type == VCSR_BF16 ? launch_gemm_bf16(g, p, st)
                                 : launch_gemm_fp8(g, p, st);
}

}  // namespace

// ----------------------------------------------------------- gated projection
namespace {

size_t part_bytes(const GatedGemm& g, const GemmPlan& p) {
    if (p.rows < g.I) {
        const GatedGemm rest = rows_from(g, p.rows);
        return part_bytes(rest, plan_of(rest, nullptr, false));
    }
    return p.splits > 1 ? (size_t)p.splits * (size_t)g.I * 8 * (size_t)tile::part_ld(g.J / 2) : 0;
}

hipError_t launch(const GatedGemm& g, const GemmPlan& p, hipStream_t st) {
    if (p.rows < g.I) {
        GatedGemm first = g;
        first.I = p.rows;
        const hipError_t e = launch(first, p, st);
        if (e != hipSuccess) return e;
        const GatedGemm rest = rows_from(g, p.rows);
        return launch(rest, plan_of(rest, nullptr, false), st);
    }
    return g.type == VCSR_F32    ? launch_gated_f32(g, p, st)
           : g.type == VCSR_BF16 ? launch_gated_bf16(g, p, st)
                                 : launch_gated_fp8(g, p, st);
}

// Planned as products of the same blocks: dw with the rows of both, dx with a sum as
// long as both.  Neither is divided into rows.
PairPlan plan_grad(const TwinGemm& dw, const TwiceGemm& dx) {
    Gemm w = dw, x = dx;
    w.I = 2 * dw.I;
    const int64_t step = tile::kStepBytes / (dx.type == VCSR_F32 ? 4 : 2);
    x.R = 2 * ((dx.R + step - 1) / step) * step;
    PairPlan p{};
    if (dw.out && dx.out)
        p = plan_pair(w, x, false);
    else if (dw.out)
        p.dw = plan_of(w, nullptr, false);
    else
        p.dx = plan_of(x, nullptr, false);
    // Room for the sums of dbias and for dw's halves rounded up, which come to fewer blocks.
    auto room = [](int64_t blocks, int tile) { return launches(blocks + (1 << 18), tile); };
    const int64_t blocks_w = p.dw.splits > 0 ? tiles_of(w, p.dw.tile) * p.dw.splits : 0;
    const int64_t blocks_x = p.dx.splits > 0 ? tiles_of(x, p.dx.tile) * p.dx.splits : 0;
    if (!p.together && !room(blocks_w, p.dw.tile)) p.dw.splits = 0;
    if (!p.together && !room(blocks_x, p.dx.tile)) p.dx.splits = 0;
    // Products in tiles of one size, of which one at most is split (the partial sums share
    // the workspace), are one launch: 8192 x 2048 x 4096 bf16 565 us, 574 in two; 9 x 384 x
    // 1551 FP32 with dx split 17, 21 in two; 500 x 1000 x 1500 bf16 42 and 46.
    const bool shared = (p.dw.splits == 1 && p.dx.splits > 0) ||
                        (p.dx.splits == 1 && p.dw.splits > 0);
    if (!forced.plan.tile && p.dw.tile == p.dx.tile && shared &&
        room(blocks_w + blocks_x, p.dw.tile))
        p.together = true;
    p.dw.rows = dw.I;
    p.dx.rows = dx.I;
    return p;
}
size_t dw_bytes(const TwinGemm& g, const GemmPlan& p) {
    return p.splits > 1 ? (size_t)p.splits * 2 * (size_t)g.I * (size_t)tile::part_ld(g.J) * 4 : 0;
}

}  // namespace

GemmPlan gated_plan(const GatedGemm& g) { return plan_of(g); }
size_t gated_workspace(const GatedGemm& g) {
    return g.I <= 0 ? 0 : part_bytes(g, launchable(plan_of(g)));
}
hipError_t launch_gated(const GatedGemm& g, hipStream_t st) {
    return g.I <= 0 ? hipSuccess : launch(g, plan_of(g), st);
}

PairPlan gated_grad_plan(const TwinGemm& dw, const TwiceGemm& dx) { return plan_grad(dw, dx); }
size_t gated_grad_workspace(const TwinGemm& dw, const TwiceGemm& dx) {
    const PairPlan p = plan_grad(dw, dx);
    const size_t a = dw.out ? dw_bytes(dw, launchable(p.dw)) : 0;
    const size_t b = dx.out ? part_bytes(dx, launchable(p.dx)) : 0;
    return a > b ? a : b;
}
hipError_t launch_gated_grad(const TwinGemm& dw, const TwiceGemm& dx, const RowSum (&bias)[2],
                             hipStream_t st) {
    const PairPlan p = plan_grad(dw, dx);
    const RowSum none[2] = {};
    auto go = [&](bool w, bool x, const RowSum(&sums)[2]) {
        GemmPlan a = p.dw, b = p.dx;
        if (!w) a.splits = 0;
        if (!x) b.splits = 0;
        return dw.type == VCSR_F32 ? launch_gated_grad_f32(dw, a, dx, b, sums, st)
                                   : launch_gated_grad_bf16(dw, a, dx, b, sums, st);
    };
    if (!dw.out || !dx.out || p.together) return go(dw.out, dx.out, bias);
    const hipError_t e = go(false, true, bias);
    return e != hipSuccess ? e : go(true, false, none);
}

GemmPlan gemm_plan(const Gemm& g) { return plan_of(g); }
PairPlan gemm_pair_plan(const Gemm& dw, const Gemm& dx) { return plan_pair(dw, dx); }
void force_plan(const GemmPlan& p, bool together) { forced = Forced{p, together}; }

size_t gemm_workspace(const Gemm& g) {
    return g.I <= 0 || g.J <= 0 ? 0 : part_bytes(g, launchable(plan_of(g)));
}

size_t gemm_pair_workspace(const Gemm& dw, const Gemm& dx) {
    const PairPlan p = plan_pair(dw, dx);
    const size_t a = part_bytes(dw, launchable(p.dw)), b = part_bytes(dx, launchable(p.dx));
    return a > b ? a : b;
}

hipError_t launch_gemm(const Gemm& g, hipStream_t st) {
    return g.I <= 0 || g.J <= 0 ? hipSuccess : launch(g, plan_of(g), st);
}

hipError_t launch_gemm_pair(const Gemm& dw, const Gemm& dx, const RowSum& bias, hipStream_t st) {
    const PairPlan p = plan_pair(dw, dx);
    if (p.together)
        return dw.type == VCSR_F32 ? launch_pair_f32(dw, p.dw, dx, p.dx, bias, st)
                                   : launch_pair_bf16(dw, p.dw, dx, p.dx, bias, st);
    hipError_t e = hipSuccess;
    if (bias.P > 0) e = launch_sum_rows(bias.part, bias.P, bias.C, bias.C, bias.out, st);
    if (e == hipSuccess) e = launch(dx, p.dx, st);
    return e != hipSuccess ? e : launch(dw, p.dw, st);
}

}  // namespace vcsr
