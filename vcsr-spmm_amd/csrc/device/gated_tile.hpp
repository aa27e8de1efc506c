// gated_tile.hpp - the gated projection and its gradients on linear_tile.hpp's tiles, for
// gated_f32.hip, gated_bf16.hip and gated_fp8.hip.
//
// Forward: out = act(x Wg^T) * (x Wu^T).  A tile's columns are half the one weight's and
// half the other's, 32 and 32 of each 64 that a wave has, so that the two sums of an
// output lie in one lane's registers and the epilogue multiplies them there: x is read
// once for both and neither sum goes through memory.
// Gradients: dx = dzg Wg + dzu Wu is one sum of both products' steps, dwg = dzg^T x and
// dwu = dzu^T x two halves of one launch.
//
// What bounds them, for rows x inputs x outputs: few rows the weights' read (1 x 4096 x
// 8192 bf16 25.3 us, 5.3 TB/s; FP32 53.6, 5.0 TB/s; e4m3 16.5, 4.1 TB/s), large FP32 ones
// the matrix units (4096^3 1981 us, 139 TFLOP/s), large bf16 ones the chip's power (8192 x
// 4096 x 8192 867 to 930 us, 1.18 to 1.27 PFLOP/s, the matrix units busy 57% at 2.0 GHz),
// e4m3 ones widening (5001 x 4096 x 4096 236 to 251 us, 1.34 to 1.42 PFLOP/s, 4096 rows of it
// in tiles of 256 and the rest in 128).  Gradients of 8192 x 2048 x 4096 bf16: the products some 500
// us of a pass' 558 (520 to 527 by themselves under a profiler), 1.1 PFLOP/s, busy 46% at 2.2
// GHz (transposing reads; keys without LDS conflicts change nothing); of 30011 x 130 x 257
// FP32 some 112 of 153 (128 under a profiler), busy 57%.  Farthest off are gradients with a
// narrow side, which write and read both dz for few products: 12102 x 66 x 3628 FP32 539 us,
// 7416 x 64 x 7913 bf16 222 to 239, where the bytes and products that cannot be done without
// are 150 and 68.
#pragma once

#include "linear_tile.hpp"

namespace vcsr {
namespace tile {

template <class T, int TILE, int STAGES>
__global__ __launch_bounds__(kThreads<TILE>) void gated_kernel(GatedGemm g, Part part) {
    __shared__ __attribute__((aligned(128))) uint8_t lds[kLds<TILE, STAGES>];
    gemm_block<T, TILE, STAGES, false, false>(g, part, blockIdx.x, lds);
}

// The partial sums of a split projection and the epilogue, as gemm_join_few_kernel and
// gemm_join_kernel: both weights' sums of 8 columns (or of one) a thread.
template <class O>
__global__ __launch_bounds__(256) void gated_join_few_kernel(GatedGemm g, int splits) {
    const int32_t J = g.J / 2;
    const int64_t ld = part_ld(J);
    const uint32_t per_row = (uint32_t)(ld / 8);
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t i = e / per_row;
    const int j = (int)(e - i * per_row) * 8;
    if (i >= g.I) return;
    float v[2][8] = {};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const float* const from = g.part + ((int64_t)s * g.I + i) * 2 * ld + j;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float p[8];
            load_vec(from + h * ld, 8, p);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[h][k] += p[k];
        }
    }
    if (J - j >= 8) {
        finish<O>(g, i, j, v[0], v[1]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float a[1] = {v[0][k]}, b[1] = {v[1][k]};
            if (j + k < J) finish<O>(g, i, j + k, a, b);
        }
    }
}
template <class O>
__global__ __launch_bounds__(256) void gated_join_kernel(GatedGemm g, int splits) {
    __shared__ float lds[2][8][32][9];
    const int32_t J = g.J / 2;
    const int64_t ld = part_ld(J);
    const uint32_t per_row = (uint32_t)(ld / 8);
    const int at = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int64_t e = (int64_t)blockIdx.x * 32 + at;
    const int64_t i = e / per_row;
    const int j = (int)(e - i * per_row) * 8;
    float v[2][8] = {};
    if (i < g.I) {
#pragma unroll 4
        for (int s = grp; s < splits; s += 8) {
            const float* const from = g.part + ((int64_t)s * g.I + i) * 2 * ld + j;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float p[8];
                load_vec(from + h * ld, 8, p);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[h][k] += p[k];
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < 8; ++k) lds[h][grp][at][k] = v[h][k];
    __syncthreads();
    // One column a thread from here.
    const int col = threadIdx.x & 7, own = threadIdx.x >> 3;
    const int64_t f = (int64_t)blockIdx.x * 32 + own;
    const int64_t row = f / per_row;
    const int c = (int)(f - row * per_row) * 8 + col;
    if (row >= g.I || c >= J) return;
    float a[1] = {lds[0][0][own][col]}, b[1] = {lds[1][0][own][col]};
#pragma unroll
    for (int q = 1; q < 8; ++q) {
        a[0] += lds[0][q][own][col];
        b[0] += lds[1][q][own][col];
    }
    finish<O>(g, row, c, a, b);
}

// Few rows of x (at most 16), as gemm_rows_kernel: a block takes 8 rows of each weight.
template <class T, class O, int UN>
__global__ __launch_bounds__(512) void gated_rows_kernel(GatedGemm g) {
    constexpr int WAVES = 8;
    __shared__ __attribute__((aligned(16))) float lds[WAVES][16][20];
    const int32_t J = g.J / 2;
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const int64_t j0 = (int64_t)blockIdx.x * 8;
    const int64_t jr = j0 + (lane & 7) < J ? j0 + (lane & 7) : J - 1;
    const T* const w = lane & 8 ? (const T*)g.q2 + jr * g.ldq2 : (const T*)g.q + jr * g.ldq;
    const f32x4 acc = rows_sum<T, UN>(g, w);
    *(f32x4*)&lds[wave][lane & 15][(lane >> 4) * 4] = acc;
    __syncthreads();
    const int row = threadIdx.x >> 3, col = threadIdx.x & 7;
    if (row >= 16 || row >= g.I || j0 + col >= J) return;
    float a[1] = {0.f}, b[1] = {0.f};
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
        a[0] += lds[k][row][col];
        b[0] += lds[k][row][8 + col];
    }
    finish<O>(g, row, (int)j0 + col, a, b);
}
template <class T, class O>
hipError_t launch_gated_rows(const GatedGemm& g, hipStream_t st) {
    const unsigned blocks = (unsigned)(((int64_t)g.J / 2 + 7) / 8);
    const int64_t lines = (g.R * (int64_t)sizeof(T) + 127) / 128;
    // Two blocks of four lines a unit rather than one of eight: 1 x 4096 x 8192 bf16 25.3
    // us (5.3 TB/s) against 30.7, FP32 53.6 and 62.9, 1 x 8192 x 8192 e4m3 24.5 and 29.2
    // (two sets of weights in turn, which the last cache helps); with fewer outputs (1 x 4096
    // x 1024) bf16 7.4 against 7.1, FP32 14.5 and 13.8.
    if (lines <= 16)
        gated_rows_kernel<T, O, 2><<<blocks, 512, 0, st>>>(g);
    else
        gated_rows_kernel<T, O, 4><<<blocks, 512, 0, st>>>(g);
    return hipGetLastError();
}

template <class T>
hipError_t launch_gated_tiles(const GatedGemm& g, const GemmPlan& p, hipStream_t st) {
    if (p.tile == 16)
        return g.out_type == VCSR_BF16 ? launch_gated_rows<T, bf16>(g, st)
                                       : launch_gated_rows<T, float>(g, st);
    const Part part = part_of(g, p);
    constexpr bool DEEP = sizeof(T) == 2;
    if (DEEP && p.tile == 64 && p.stages == 4) {
        if constexpr (DEEP) gated_kernel<T, 64, 4><<<part.blocks, kThreads<64>, 0, st>>>(g, part);
    } else if (p.tile == 64)
        gated_kernel<T, 64, 2><<<part.blocks, kThreads<64>, 0, st>>>(g, part);
    else if (p.tile == 128)
        gated_kernel<T, 128, 2><<<part.blocks, kThreads<128>, 0, st>>>(g, part);
    else if constexpr (sizeof(T) < 4)
        gated_kernel<T, 256, 2><<<part.blocks, kThreads<256>, 0, st>>>(g, part);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits <= 1) return e;
    const int64_t vectors = g.I * (part_ld(g.J / 2) / 8);
    const unsigned few = (unsigned)((vectors + 255) / 256), many = (unsigned)((vectors + 31) / 32);
    if (g.out_type == VCSR_BF16) {
        if (p.splits < 8)
            gated_join_few_kernel<bf16><<<few, 256, 0, st>>>(g, p.splits);
        else
            gated_join_kernel<bf16><<<many, 256, 0, st>>>(g, p.splits);
    } else {
        if (p.splits < 8)
            gated_join_few_kernel<float><<<few, 256, 0, st>>>(g, p.splits);
        else
            gated_join_kernel<float><<<many, 256, 0, st>>>(g, p.splits);
    }
    return hipGetLastError();
}

// ------------------------------------------------------------------ gradients
struct HalfGemm : Gemm {};  // one of dw's products

// dw's two products, from multiples of 8 on so that all keep their XCDs (dw_part's
// blocks are one's), then dx, then the sums of dbias' partial rows.  DW, DX: which of
// them there are.
template <class T, int TILE, int STAGES, bool DW, bool DX>
__global__ __launch_bounds__(kThreads<TILE>) void gated_grad_kernel(TwinGemm dw, Part dw_part,
                                                                    TwiceGemm dx, Part dx_part,
                                                                    RowSum bias0, RowSum bias1) {
    __shared__ __attribute__((aligned(128))) uint8_t lds[kLds<TILE, STAGES>];
    const uint32_t half = DW ? (dw_part.blocks + 7) & ~7u : 0;
    uint32_t b = blockIdx.x;
    if (b >= 2 * half) {
        b -= 2 * half;
        if (DX && b < dx_part.blocks) {
            gemm_block<T, TILE, STAGES, false, true>(dx, dx_part, b, lds);
            return;
        }
        b -= DX ? dx_part.blocks : 0;
        const uint32_t n = bias0.P > 0 ? (uint32_t)(((int64_t)bias0.C + 15) / 16) : 0;
        if (b < n)
            sum_columns<kThreads<TILE>>(bias0, b, lds);
        else
            sum_columns<kThreads<TILE>>(bias1, b - n, lds);
        return;
    }
    if constexpr (DW) {
        const bool second = b >= half;
        if (second) b -= half;
        if (b >= dw_part.blocks) return;
        HalfGemm g;
        static_cast<Gemm&>(g) = dw;
        g.p = second ? dw.p2 : dw.p;
        g.out = second ? dw.out2 : dw.out;
        g.ldo = second ? dw.ldo2 : dw.ldo;
        g.part = dw.part + (second ? (int64_t)dw_part.splits * dw.I * part_ld(dw.J) : 0);
        gemm_block<T, TILE, STAGES, true, true>(g, dw_part, b, lds);
    }
}

template <class T, bool DW, bool DX>
hipError_t launch_grad_parts(const TwinGemm& dw, const GemmPlan& p, const TwiceGemm& dx,
                             const GemmPlan& q, const RowSum (&bias)[2], hipStream_t st) {
    const Part a = DW ? part_of(dw, p) : Part{}, b = DX ? part_of(dx, q) : Part{};
    uint32_t blocks = (DW ? 2 * ((a.blocks + 7) & ~7u) : 0) + (DX ? b.blocks : 0);
    for (const RowSum& r : bias)
        if (r.P > 0) blocks += (uint32_t)(((int64_t)r.C + 15) / 16);
    const int tile = DW ? p.tile : q.tile;
    if (tile == 64)
        gated_grad_kernel<T, 64, 2, DW, DX>
            <<<blocks, kThreads<64>, 0, st>>>(dw, a, dx, b, bias[0], bias[1]);
    else if (tile == 128)
        gated_grad_kernel<T, 128, 2, DW, DX>
            <<<blocks, kThreads<128>, 0, st>>>(dw, a, dx, b, bias[0], bias[1]);
    else if constexpr (sizeof(T) < 4)
        gated_grad_kernel<T, 256, 2, DW, DX>
            <<<blocks, kThreads<256>, 0, st>>>(dw, a, dx, b, bias[0], bias[1]);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && DX) e = launch_join(dx, q.splits, st);
    if (e == hipSuccess && DW) e = launch_join(dw, p.splits, st, dw.out2, dw.ldo2);
    return e;
}
template <class T>
hipError_t launch_grad_of(const TwinGemm& dw, const GemmPlan& p, const TwiceGemm& dx,
                          const GemmPlan& q, const RowSum (&bias)[2], hipStream_t st) {
    if (p.splits > 0 && q.splits > 0)
        return launch_grad_parts<T, true, true>(dw, p, dx, q, bias, st);
    return p.splits > 0 ? launch_grad_parts<T, true, false>(dw, p, dx, q, bias, st)
                        : launch_grad_parts<T, false, true>(dw, p, dx, q, bias, st);
}

}  // namespace tile
}  // namespace vcsr
