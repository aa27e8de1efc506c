// rmsnorm.hip - RMS norm of x + residual and its gradient.
//
// Forward: t = x + residual, y = t * w / sqrt(mean(t^2) + eps).  One pass over
// memory: a row's t stays in registers between the sum of squares and the
// result, whatever y's type; for 8-bit y the row's scale needs max |t * w|,
// which is reduced together with the sum, since |y| = |t * w| * rstd.
// Gradient: with h = s * rstd, g = dy * w, dx = dsum + rstd * (g - h * mean(g
// h)); again one pass, the row's s and dy in registers.  dweight sums dy * h
// over the rows a block takes in registers, then over the blocks (colsum.hip),
// in a fixed order.  All of it is bound by memory: 32768 x 4096 bf16 with a residual
// to e4m3 163 us (5.8 TB/s), 62451 x 128 FP32 28 us (4.6 TB/s), the gradient of
// 16384 x 2050 bf16 67 us (4.0 TB/s), of 32768 x 4096 217 us (4.9 TB/s).
#include "dense.hpp"
#include "norm_rows.hpp"

namespace vcsr {
namespace {

using namespace norm;

// Whether max |t * w| stands for max |y| / rstd: it does not where that product is
// past FP32's range (or loses bits below it), which y = t * rstd * w need not be (1e-18
// * 1e-27, or 1e18 * 1e22).  y's own maximum is taken there.
__device__ __forceinline__ bool top_lost(float top) { return top < 0x1p-100f || top > 0x1p126f; }
template <int V>
__device__ __forceinline__ float y_top(const float (&t)[V], const float (&w)[V], float rstd,
                                       float top) {
#pragma unroll
    for (int i = 0; i < V; ++i) top = max_nan(top, __builtin_fabsf(t[i] * rstd * w[i]));
    return top;
}

// y's values of one vector.
template <class Y, int V>
__device__ __forceinline__ void write_y(Y* p, int n, const float (&t)[V], const float (&w)[V],
                                        float rstd, float scale) {
    float y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        y[i] = t[i] * rstd * w[i];
        if (sizeof(Y) == 1) y[i] = y[i] / scale;
    }
    store_vec(p, n, y);
}

// Rows of at most NV * 64 * WPR vectors, held in registers.  WPR = 1: groups of
// `lanes` (a power of two <= 64) lanes of a 256-thread block take a row each; WPR >
// 1: a block of WPR waves takes a row.
template <class X, class Y, int WPR, int NV>
__global__ __launch_bounds__(WPR > 1 ? 64 * WPR : 256) void rmsnorm_kernel(vcsr_rmsnorm_args a,
                                                                           int lanes) {
    constexpr int V = kVec<X>;
    __shared__ float lds[4 * WPR];
    const int tid = threadIdx.x;
    const int lane = WPR > 1 ? tid : tid & (lanes - 1);
    const int stride = WPR > 1 ? 64 * WPR : lanes;
    const int64_t row = WPR > 1 ? (int64_t)blockIdx.x
                                : (int64_t)blockIdx.x * (256 / lanes) + tid / lanes;
    const bool live = row < a.M;  // lanes past the last row still take part in the shuffles
    const int64_t at = live ? row : 0;
    float t[NV][V], w[NV][V];
    float sum = 0.f, top = 0.f;
    load_row((const X*)a.x + at * a.ldx, lane, stride, a.C, t);
    load_row(a.weight, lane, stride, a.C, w);
    if (a.residual) {
        float v[NV][V];
        load_row((const X*)a.residual + at * a.ldr, lane, stride, a.C, v);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) t[k][i] += v[k][i];
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            sum = __builtin_fmaf(t[k][i], t[k][i], sum);
            if (sizeof(Y) == 1) top = max_nan(top, __builtin_fabsf(t[k][i] * w[k][i]));
        }
    reduce_lanes(WPR > 1 ? 64 : lanes, sum, top);
    if (WPR > 1) reduce_waves<WPR>(lds, sum, top);
    if (!live) return;
    const float rstd = 1.f / __builtin_sqrtf(sum / (float)a.C + a.eps);
    if (a.rstd && lane == 0) a.rstd[row] = rstd;
    if (sizeof(Y) == 1 && top_lost(top)) {  // for all lanes of the row
        float unused = 0.f;
        top = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) top = y_top(t[k], w[k], rstd, top);
        reduce_lanes(WPR > 1 ? 64 : lanes, unused, top);
        if (WPR > 1) reduce_waves<WPR>(lds + 2 * WPR, unused, top);
    } else {
        top *= rstd;
    }
    const float scale = row_factor<Y>(top, a.y_scale, row, lane == 0);
    if (a.sum) store_row((X*)a.sum + row * a.ldsum, lane, stride, a.C, t);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            // 8 bits: the largest magnitude may come out a rounding over 448 and
            // still rounds to it.
            t[k][i] = t[k][i] * rstd * w[k][i];
            if (sizeof(Y) == 1) t[k][i] = t[k][i] / scale;
        }
    store_row((Y*)a.y + row * a.ldy, lane, stride, a.C, t);
}

// Longer rows: a block reads a row twice (the second time from the caches).  sum,
// which may be x or the residual, is written in the second pass, behind the reads
// of the same values by the same thread.
template <class X, class Y>
__global__ __launch_bounds__(1024) void rmsnorm_long_kernel(vcsr_rmsnorm_args a) {
    constexpr int V = kVec<X>, WAVES = 16;
    __shared__ float lds[4 * WAVES];
    const int64_t row = blockIdx.x;
    const X* x = (const X*)a.x + row * a.ldx;
    const X* r = a.residual ? (const X*)a.residual + row * a.ldr : nullptr;
    auto load_t = [&](int64_t c, float(&t)[V]) {
        const int n = a.C - c < V ? (int)(a.C - c) : V;
        load_vec(x + c, n, t);
        if (r) {
            float v[V];
            load_vec(r + c, n, v);
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] += v[i];
        }
        return n;
    };
    float sum = 0.f, top = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 1024 * V) {
        float t[V], w[V];
        const int n = load_t(c, t);
        load_vec(a.weight + c, n, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            sum = __builtin_fmaf(t[i], t[i], sum);
            if (sizeof(Y) == 1) top = max_nan(top, __builtin_fabsf(t[i] * w[i]));
        }
    }
    reduce_lanes(64, sum, top);
    reduce_waves<WAVES>(lds, sum, top);
    const float rstd = 1.f / __builtin_sqrtf(sum / (float)a.C + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
    if (sizeof(Y) == 1 && top_lost(top)) {
        float unused = 0.f;
        top = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 1024 * V) {
            float t[V], w[V];
            const int n = load_t(c, t);
            load_vec(a.weight + c, n, w);
            top = y_top(t, w, rstd, top);
        }
        reduce_lanes(64, unused, top);
        reduce_waves<WAVES>(lds + 2 * WAVES, unused, top);
    } else {
        top *= rstd;
    }
    const float scale = row_factor<Y>(top, a.y_scale, row, threadIdx.x == 0);
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 1024 * V) {
        float t[V], w[V];
        const int n = load_t(c, t);
        load_vec(a.weight + c, n, w);
        if (a.sum) store_vec((X*)a.sum + row * a.ldsum + c, n, t);
        write_y((Y*)a.y + row * a.ldy + c, n, t, w, rstd, scale);
    }
}

// Rows of fewer values than a vector: a thread takes a row.  Neighbouring threads'
// rows share lines, so memory bounds it: 4.2M x 3 FP32 with a residual 52 us (3.9
// TB/s), its gradient 50; with a block a row, as long ones have it, 19.5 and 32.7 ms.
template <class X, class Y>
__global__ __launch_bounds__(256) void rmsnorm_narrow_kernel(vcsr_rmsnorm_args a) {
    constexpr int V = kVec<X>;
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (row >= a.M) return;
    float t[V], w[V], sum = 0.f, top = 0.f;
    load_vec((const X*)a.x + row * a.ldx, a.C, t);
    load_vec(a.weight, a.C, w);
    if (a.residual) {
        float v[V];
        load_vec((const X*)a.residual + row * a.ldr, a.C, v);
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] += v[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sum = __builtin_fmaf(t[i], t[i], sum);
    const float rstd = 1.f / __builtin_sqrtf(sum / (float)a.C + a.eps);
    if (a.rstd) a.rstd[row] = rstd;
    if (sizeof(Y) == 1) {
        top = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < a.C) top = max_nan(top, __builtin_fabsf(t[i] * rstd * w[i]));
    }
    const float scale = row_factor<Y>(top, a.y_scale, row, true);
    if (a.sum) store_vec((X*)a.sum + row * a.ldsum, a.C, t);
    write_y((Y*)a.y + row * a.ldy, a.C, t, w, rstd, scale);
}

template <class X, class Y>
vcsr_rmsnorm_args rows_of(vcsr_rmsnorm_args a, int64_t first, int64_t count) {
    a.M = count;
    a.x = (const X*)a.x + first * a.ldx;
    if (a.residual) a.residual = (const X*)a.residual + first * a.ldr;
    if (a.sum) a.sum = (X*)a.sum + first * a.ldsum;
    a.y = (Y*)a.y + first * a.ldy;
    if (a.y_scale) a.y_scale += first;
    if (a.rstd) a.rstd += first;
    return a;
}

template <class X, class Y>
hipError_t launch_forward(const vcsr_rmsnorm_args& a, hipStream_t st) {
    constexpr int V = kVec<X>;
    const int64_t nv = ((int64_t)a.C + V - 1) / V;
    if (a.C < V) {
        rmsnorm_narrow_kernel<X, Y><<<(unsigned)((a.M + 255) / 256), 256, 0, st>>>(a);
        return hipGetLastError();
    }
    if (nv > 2048) {
        by_rows(a.M, 1024, [&](int64_t first, int64_t count) {
            rmsnorm_long_kernel<X, Y>
                <<<(unsigned)count, 1024, 0, st>>>(rows_of<X, Y>(a, first, count));
        });
        return hipGetLastError();
    }
    const int lanes = nv <= 64 ? next_pow2((int)nv) : 64;
    with_shape(row_shape(nv, 4), [&](auto wpr, auto k) {
        constexpr int W = decltype(wpr)::value, NV = decltype(k)::value;
        const int rows = W > 1 ? 1 : 256 / lanes;
        by_rows(a.M, W > 1 ? 64 * W : lanes, [&](int64_t first, int64_t count) {
            rmsnorm_kernel<X, Y, W, NV>
                <<<(unsigned)((count + rows - 1) / rows), W > 1 ? 64 * W : 256, 0, st>>>(
                    rows_of<X, Y>(a, first, count), lanes);
        });
    });
    return hipGetLastError();
}

// ------------------------------------------------------------------ gradient
// Rows of at most NV * 64 * WPR vectors (as above); each row group goes through
// rows blockIdx, blockIdx + gridDim, ... and keeps dweight of its columns in
// registers.  The weight stays in LDS: with it in registers too, 2050 bf16 columns
// leave room for three waves a SIMD instead of four.
template <class X, class D, int WPR, int NV>
__global__ __launch_bounds__(WPR > 1 ? 64 * WPR : 256) void rmsnorm_grad_kernel(
    vcsr_rmsnorm_grad_args a, float* part, int lanes) {
    constexpr int V = kVec<X>, COLS = (WPR > 1 ? 64 * WPR : 64) * NV * V;
    __shared__ float red[2][2 * WPR];
    __shared__ __attribute__((aligned(16))) float w_lds[COLS];
    const int tid = threadIdx.x;
    const int lane = WPR > 1 ? tid : tid & (lanes - 1);
    const int stride = WPR > 1 ? 64 * WPR : lanes;
    const int threads = WPR > 1 ? 64 * WPR : 256;
    const int rows = WPR > 1 ? 1 : 256 / lanes;
    const int sub = WPR > 1 ? 0 : tid / lanes;
    for (int c = tid; c < COLS; c += threads) w_lds[c] = c < a.C ? a.weight[c] : 0.f;
    __syncthreads();
    float dw[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = 0.f;
    const float inv_c = 1.f / (float)a.C;
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * rows; base < a.M;
         base += (int64_t)gridDim.x * rows, turn ^= 1) {
        const int64_t row = base + sub;
        const bool live = row < a.M;
        const int64_t at = live ? row : 0;
        float s[NV][V], d[NV][V], o[NV][V];
        const float rstd = a.rstd[at];
        float dot = 0.f, unused = 0.f;
        load_row((const X*)a.s + at * a.lds, lane, stride, a.C, s);
        load_row((const D*)a.dy + at * a.lddy, lane, stride, a.C, d);
        if (a.dsum) {
            load_row((const X*)a.dsum + at * a.lddsum, lane, stride, a.C, o);
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) o[k][i] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const float* const w = w_lds + (k * stride + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s[k][i] *= rstd;  // h
                if (WPR == 1 && !live) s[k][i] = d[k][i] = 0.f;
                dw[k][i] = __builtin_fmaf(d[k][i], s[k][i], dw[k][i]);
                d[k][i] *= w[i];  // g
                dot = __builtin_fmaf(d[k][i], s[k][i], dot);
            }
        }
        dot = sum_lanes(WPR > 1 ? 64 : lanes, dot);
        // Two sets of LDS slots in turn: the next row's sums do not meet this one's.
        if (WPR > 1) reduce_waves<WPR>(red[turn], dot, unused);
        if (!live) continue;
        const float mean = dot * inv_c;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) o[k][i] += rstd * (d[k][i] - s[k][i] * mean);
        store_row((X*)a.dx + row * a.lddx, lane, stride, a.C, o);
    }
    if (!part) return;
    float* out = part + (int64_t)blockIdx.x * a.C;
    if (WPR > 1) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * stride + lane) * V;
            if (c < a.C) store_vec(out + c, a.C - c, dw[k]);
        }
        return;
    }
    // A wave's row groups add up over its lanes, then the waves in LDS, one after
    // the other.
    for (int m = lanes; m < 64; m <<= 1)
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) dw[k][i] += __shfl_xor(dw[k][i], m);
    __syncthreads();
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        if (tid >> 6 == g && (tid & 63) < lanes)
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float* const p = w_lds + (k * stride + lane) * V + i;
                    *p = g ? *p + dw[k][i] : dw[k][i];
                }
        __syncthreads();
    }
    for (int c = tid; c < a.C; c += 256) out[c] = w_lds[c];
}

// Longer rows: a block per row, read twice; dweight apart (column by column).
template <class X, class D>
__global__ __launch_bounds__(1024) void rmsnorm_grad_long_kernel(vcsr_rmsnorm_grad_args a) {
    constexpr int V = kVec<X>, WAVES = 16;
    __shared__ float lds[2 * WAVES];
    const int64_t row = blockIdx.x;
    const X* s = (const X*)a.s + row * a.lds;
    const D* dy = (const D*)a.dy + row * a.lddy;
    const float rstd = a.rstd[row];
    float dot = 0.f, unused = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 1024 * V) {
        const int n = a.C - c < V ? (int)(a.C - c) : V;
        float h[V], g[V], w[V];
        load_vec(s + c, n, h);
        load_vec(dy + c, n, g);
        load_vec(a.weight + c, n, w);
#pragma unroll
        for (int i = 0; i < V; ++i) dot = __builtin_fmaf(g[i] * w[i], h[i] * rstd, dot);
    }
    dot = sum_lanes(64, dot);
    reduce_waves<WAVES>(lds, dot, unused);
    const float mean = dot / (float)a.C;
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 1024 * V) {
        const int n = a.C - c < V ? (int)(a.C - c) : V;
        float h[V], g[V], w[V], o[V];
        load_vec(s + c, n, h);
        load_vec(dy + c, n, g);
        load_vec(a.weight + c, n, w);
        if (a.dsum) {
            load_vec((const X*)a.dsum + row * a.lddsum + c, n, o);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] += rstd * (g[i] * w[i] - h[i] * rstd * mean);
        store_vec((X*)a.dx + row * a.lddx + c, n, o);
    }
}
// Its dweight: a thread per column over a block of rows.
template <class X, class D>
__global__ __launch_bounds__(256) void rmsnorm_dweight_kernel(vcsr_rmsnorm_grad_args a,
                                                              float* part) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.C) return;
    float t = 0.f;
    for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y)
        t = __builtin_fmaf(to_f32(((const D*)a.dy)[row * a.lddy + c]),
                           to_f32(((const X*)a.s)[row * a.lds + c]) * a.rstd[row], t);
    part[(int64_t)blockIdx.y * a.C + c] = t;
}

// Rows of fewer values than a vector: a thread takes rows blocks apart and keeps
// dweight in registers; lanes, then waves, add theirs up.
template <class X, class D>
__global__ __launch_bounds__(256) void rmsnorm_grad_narrow_kernel(vcsr_rmsnorm_grad_args a,
                                                                  float* part) {
    constexpr int V = kVec<X>;
    __shared__ float lds[4][V];
    float w[V], dw[V];
    load_vec(a.weight, a.C, w);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[i] = 0.f;
    const float inv_c = 1.f / (float)a.C;
    for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.M;
         row += (int64_t)gridDim.x * 256) {
        float h[V], g[V], o[V], dot = 0.f;
        const float rstd = a.rstd[row];
        load_vec((const X*)a.s + row * a.lds, a.C, h);
        load_vec((const D*)a.dy + row * a.lddy, a.C, g);
        if (a.dsum) {
            load_vec((const X*)a.dsum + row * a.lddsum, a.C, o);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            h[i] *= rstd;
            if (i < a.C) dw[i] = __builtin_fmaf(g[i], h[i], dw[i]);  // a factor may be infinite
            g[i] *= w[i];
            if (i < a.C) dot = __builtin_fmaf(g[i], h[i], dot);
        }
        const float mean = dot * inv_c;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] += rstd * (g[i] - h[i] * mean);
        store_vec((X*)a.dx + row * a.lddx, a.C, o);
    }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        dw[i] = sum_lanes(64, dw[i]);
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6][i] = dw[i];
    }
    __syncthreads();
    const int c = threadIdx.x;
    if (c < a.C)
        part[(int64_t)blockIdx.x * a.C + c] = ((lds[0][c] + lds[1][c]) + lds[2][c]) + lds[3][c];
}

// The gradient's row shape and blocks, each of which writes a row of partial
// dweight: two waves a SIMD.  With one a SIMD 16384 x 2050 bf16 takes 97 us, with
// two 68, with four 82 (twice the partial rows).
struct GradShape {
    int64_t nv;
    int lanes;
    RowShape row;
    bool narrow, in_registers;
    int32_t blocks;
};
GradShape grad_shape(const vcsr_rmsnorm_grad_args& a) {
    GradShape g;
    const int v = a.x_type == VCSR_F32 ? 4 : 8;
    g.nv = ((int64_t)a.C + v - 1) / v;
    g.lanes = g.nv <= 64 ? next_pow2((int)g.nv) : 64;
    g.row = row_shape(g.nv, 3);
    const int64_t rows = g.row.wpr > 1 ? 1 : 256 / g.lanes;
    const int64_t waves = g.row.wpr > 1 ? g.row.wpr : 4;
    const int64_t need = (a.M + rows - 1) / rows, most = 2048 / waves;
    g.blocks = (int32_t)(need < most ? need : most);
    if (need <= 4) g.blocks = 1;  // which then writes dweight itself
    g.narrow = a.C < v;
    g.in_registers = g.nv <= 2048 && !g.narrow;
    if (g.narrow) g.blocks = (int32_t)(a.M < 256 * 1024 ? (a.M + 255) / 256 : 1024);
    else if (!g.in_registers) g.blocks = (int32_t)(a.M < 64 ? a.M : 64);
    return g;
}

template <class X, class D>
hipError_t launch_grad(const vcsr_rmsnorm_grad_args& a, hipStream_t st) {
    const GradShape g = grad_shape(a);
    float* const part = !a.dweight ? nullptr : g.blocks == 1 ? a.dweight : (float*)a.workspace;
    if (g.narrow) {
        rmsnorm_grad_narrow_kernel<X, D><<<(unsigned)g.blocks, 256, 0, st>>>(a, part);
    } else if (!g.in_registers) {
        if (part)  // before dx, which may be s or dy itself
            rmsnorm_dweight_kernel<X, D>
                <<<dim3((unsigned)((a.C + 255) / 256), g.blocks), 256, 0, st>>>(a, part);
        by_rows(a.M, 1024, [&](int64_t first, int64_t count) {
            vcsr_rmsnorm_grad_args b = a;
            b.M = count;
            b.dy = (const D*)a.dy + first * a.lddy;
            b.s = (const X*)a.s + first * a.lds;
            b.rstd = a.rstd + first;
            if (a.dsum) b.dsum = (const X*)a.dsum + first * a.lddsum;
            b.dx = (X*)a.dx + first * a.lddx;
            rmsnorm_grad_long_kernel<X, D><<<(unsigned)count, 1024, 0, st>>>(b);
        });
    } else {
        with_shape(g.row, [&](auto wpr, auto k) {
            constexpr int W = decltype(wpr)::value, NV = decltype(k)::value;
            rmsnorm_grad_kernel<X, D, W, NV>
                <<<g.blocks, W > 1 ? 64 * W : 256, 0, st>>>(a, part, g.lanes);
        });
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !part || g.blocks == 1) return e;
    return launch_sum_rows(part, g.blocks, a.C, a.C, a.dweight, st);
}

}  // namespace

hipError_t launch_rmsnorm(const vcsr_rmsnorm_args& a, hipStream_t st) {
    if (a.M <= 0) return hipSuccess;
    if (a.x_type == VCSR_F32)
        return a.y_type == VCSR_F32    ? launch_forward<float, float>(a, st)
               : a.y_type == VCSR_BF16 ? launch_forward<float, bf16>(a, st)
                                       : launch_forward<float, fp8>(a, st);
    return a.y_type == VCSR_F32    ? launch_forward<bf16, float>(a, st)
           : a.y_type == VCSR_BF16 ? launch_forward<bf16, bf16>(a, st)
                                   : launch_forward<bf16, fp8>(a, st);
}

size_t rmsnorm_grad_workspace(const vcsr_rmsnorm_grad_args& a) {
    if (!a.dweight || a.M <= 0) return 0;
    const int32_t blocks = grad_shape(a).blocks;
    return blocks > 1 ? (size_t)blocks * (size_t)a.C * sizeof(float) : 0;
}

hipError_t launch_rmsnorm_grad(const vcsr_rmsnorm_grad_args& a, hipStream_t st) {
    if (a.M <= 0) {
        const int64_t bytes = (int64_t)a.C * 4;
        return a.dweight ? launch_zero(a.dweight, bytes, 1, bytes, st) : hipSuccess;
    }
    if (a.x_type == VCSR_F32)
        return a.y_type == VCSR_F32 ? launch_grad<float, float>(a, st)
                                    : launch_grad<float, bf16>(a, st);
    return a.y_type == VCSR_F32 ? launch_grad<bf16, float>(a, st) : launch_grad<bf16, bf16>(a, st);
}

}  // namespace vcsr
