// rmsnorm.hip - RMS norm of x + residual and its gradient.
//
// Forward: t = x + residual, y = t * w / sqrt(mean(t^2) + eps).  One pass over
// memory: a row's t stays in registers between the sum of squares and the
// result, whatever y's type; for 8-bit y the row's scale needs max |t * w|,
// which is reduced together with the sum, since |y| = |t * w| * rstd.
// Gradient: with h = s * rstd, g = dy * w, dx = dsum + rstd * (g - h * mean(g
// h)); again one pass, the row's s and dy in registers.  dweight sums dy * h
// over the rows a block takes in registers, then over the blocks (colsum.hip),
// in a fixed order.  All of it is bound by memory.
#include "dense.hpp"
#include "launch.hpp"

namespace vcsr {
namespace {

// Values of one lane's vector: 16 bytes of x.
template <class X>
constexpr int kVec = 16 / (int)sizeof(X);

// Sum and maximum over groups of `lanes` (a power of two <= 64) lanes.  The
// maximum keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) { return a > b || a != a ? a : b; }
__device__ __forceinline__ void reduce_lanes(int lanes, float& sum, float& top) {
    for (int m = 1; m < lanes; m <<= 1) {
        sum += __shfl_xor(sum, m);
        top = max_nan(top, __shfl_xor(top, m));
    }
}
__device__ __forceinline__ float sum_lanes(int lanes, float x) {
    for (int m = 1; m < lanes; m <<= 1) x += __shfl_xor(x, m);
    return x;
}
// The same over the block's waves; every wave calls it, in the same order of
// addition.
template <int WAVES>
__device__ __forceinline__ void reduce_waves(float* lds, float& sum, float& top) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        lds[w] = sum;
        lds[WAVES + w] = top;
    }
    __syncthreads();
    sum = lds[0];
    top = lds[WAVES];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        sum += lds[i];
        top = max_nan(top, lds[WAVES + i]);
    }
}

template <class Y>
__device__ __forceinline__ float row_factor(float rstd, float top, float* y_scale, int64_t row,
                                            bool writes) {
    if (sizeof(Y) != 1) return 1.f;
    float a = top * rstd;
    a = a < 1e-30f ? 1e-30f : a;  // a NaN stays one
    const float scale = a / 448.f;
    if (writes) y_scale[row] = scale;
    return scale;
}

// y's values of one vector.  8 bits: t * rstd * w / scale, where the largest
// magnitude may come out a rounding over 448 and still rounds to it.
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

// Rows of at most NV * LANES vectors, held in registers.  WAVES = 1: groups of
// `lanes` <= 64 lanes take a row each; WAVES > 1: a block takes a row.
template <class X, class Y, int WAVES, int NV>
__global__ __launch_bounds__(256) void rmsnorm_kernel(vcsr_rmsnorm_args a, int lanes) {
    constexpr int V = kVec<X>;
    __shared__ float lds[2 * WAVES];
    const int tid = threadIdx.x;
    const int lane = WAVES > 1 ? tid : tid & (lanes - 1);
    const int stride = WAVES > 1 ? 64 * WAVES : lanes;
    const int64_t row = WAVES > 1 ? (int64_t)blockIdx.x
                                  : (int64_t)blockIdx.x * (256 / lanes) + tid / lanes;
    const bool live = row < a.M;  // lanes past the last row still take part in the shuffles
    float t[NV][V];
    float sum = 0.f, top = 0.f;
    if (live) {
        const X* x = (const X*)a.x + row * a.ldx;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * stride + lane) * V;
            load_vec(x + c, c < a.C ? a.C - c : 0, t[k]);
        }
        if (a.residual) {
            const X* r = (const X*)a.residual + row * a.ldr;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = (k * stride + lane) * V;
                float v[V];
                load_vec(r + c, c < a.C ? a.C - c : 0, v);
#pragma unroll
                for (int i = 0; i < V; ++i) t[k][i] += v[i];
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) t[k][i] = 0.f;
    }
    float w[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * stride + lane) * V;
        load_vec(a.weight + c, c < a.C ? a.C - c : 0, w[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            sum = __builtin_fmaf(t[k][i], t[k][i], sum);
            if (sizeof(Y) == 1) top = max_nan(top, __builtin_fabsf(t[k][i] * w[k][i]));
        }
    }
    reduce_lanes(WAVES > 1 ? 64 : lanes, sum, top);
    if (WAVES > 1) reduce_waves<WAVES>(lds, sum, top);
    if (!live) return;
    const float rstd = 1.f / __builtin_sqrtf(sum / (float)a.C + a.eps);
    if (a.rstd && lane == 0) a.rstd[row] = rstd;
    const float scale = row_factor<Y>(rstd, top, a.y_scale, row, lane == 0);
    if (a.sum) {
        X* s = (X*)a.sum + row * a.ldsum;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * stride + lane) * V;
            if (c < a.C) store_vec(s + c, a.C - c, t[k]);
        }
    }
    Y* y = (Y*)a.y + row * a.ldy;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * stride + lane) * V;
        if (c < a.C) write_y(y + c, a.C - c, t[k], w[k], rstd, scale);
    }
}

// Longer rows: a block reads a row twice (the second time from the caches).
// sum, which may be x or the residual, is written in the second pass, behind
// the reads of the same values by the same thread.
template <class X, class Y>
__global__ __launch_bounds__(1024) void rmsnorm_long_kernel(vcsr_rmsnorm_args a) {
    constexpr int V = kVec<X>, WAVES = 16;
    __shared__ float lds[2 * WAVES];
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
    const float scale = row_factor<Y>(rstd, top, a.y_scale, row, threadIdx.x == 0);
    for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 1024 * V) {
        float t[V], w[V];
        const int n = load_t(c, t);
        load_vec(a.weight + c, n, w);
        if (a.sum) store_vec((X*)a.sum + row * a.ldsum + c, n, t);
        write_y((Y*)a.y + row * a.ldy + c, n, t, w, rstd, scale);
    }
}

int next_pow2(int n) {
    int p = 1;
    while (p < n) p <<= 1;
    return p;
}

template <class X, class Y>
hipError_t launch_forward(const vcsr_rmsnorm_args& a, hipStream_t st) {
    constexpr int V = kVec<X>;
    const int64_t nv = ((int64_t)a.C + V - 1) / V;
    if (nv <= 64) {
        const int lanes = next_pow2((int)nv), rows = 256 / lanes;
        rmsnorm_kernel<X, Y, 1, 1><<<(unsigned)((a.M + rows - 1) / rows), 256, 0, st>>>(a, lanes);
    } else if (nv <= 256) {
        rmsnorm_kernel<X, Y, 4, 1><<<(unsigned)a.M, 256, 0, st>>>(a, 64);
    } else if (nv <= 512) {
        rmsnorm_kernel<X, Y, 4, 2><<<(unsigned)a.M, 256, 0, st>>>(a, 64);
    } else if (nv <= 1024) {
        rmsnorm_kernel<X, Y, 4, 4><<<(unsigned)a.M, 256, 0, st>>>(a, 64);
    } else {
        rmsnorm_long_kernel<X, Y><<<(unsigned)a.M, 1024, 0, st>>>(a);
    }
    return hipGetLastError();
}

// ------------------------------------------------------------------ gradient
// Rows of at most NV * LANES vectors (as above); each row group goes through
// rows blockIdx, blockIdx + gridDim, ... and keeps dweight of its columns.
template <class X, class D, int WAVES, int NV>
__global__ __launch_bounds__(256) void rmsnorm_grad_kernel(vcsr_rmsnorm_grad_args a, float* part,
                                                           int lanes) {
    constexpr int V = kVec<X>;
    __shared__ float lds[2 * WAVES];
    __shared__ float dw_lds[WAVES > 1 ? 1 : 256 * V * NV];
    const int tid = threadIdx.x;
    const int lane = WAVES > 1 ? tid : tid & (lanes - 1);
    const int stride = WAVES > 1 ? 64 * WAVES : lanes;
    const int rows = WAVES > 1 ? 1 : 256 / lanes;
    const int sub = WAVES > 1 ? 0 : tid / lanes;
    float w[NV][V], dw[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * stride + lane) * V;
        load_vec(a.weight + c, c < a.C ? a.C - c : 0, w[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = 0.f;
    }
    const float inv_c = 1.f / (float)a.C;
    for (int64_t base = (int64_t)blockIdx.x * rows; base < a.M; base += (int64_t)gridDim.x * rows) {
        const int64_t row = base + sub;
        const bool live = row < a.M;
        float s[NV][V], d[NV][V];
        float rstd = 0.f, dot = 0.f, unused = 0.f;
        if (live) rstd = a.rstd[row];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * stride + lane) * V;
            const int n = live && c < a.C ? a.C - c : 0;
            load_vec((const X*)a.s + (live ? row * a.lds : 0) + c, n, s[k]);
            load_vec((const D*)a.dy + (live ? row * a.lddy : 0) + c, n, d[k]);
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                s[k][i] *= rstd;  // h
                dw[k][i] = __builtin_fmaf(d[k][i], s[k][i], dw[k][i]);
                d[k][i] *= w[k][i];  // g
                dot = __builtin_fmaf(d[k][i], s[k][i], dot);
            }
        dot = sum_lanes(WAVES > 1 ? 64 : lanes, dot);
        if (WAVES > 1) {
            reduce_waves<WAVES>(lds, dot, unused);
            __syncthreads();  // lds is written again for the next row
        }
        if (!live) continue;
        const float mean = dot * inv_c;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * stride + lane) * V;
            if (c >= a.C) continue;
            float o[V];
            if (a.dsum) {
                load_vec((const X*)a.dsum + row * a.lddsum + c, a.C - c, o);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] += rstd * (d[k][i] - s[k][i] * mean);
            store_vec((X*)a.dx + row * a.lddx + c, a.C - c, o);
        }
    }
    if (!part) return;
    float* out = part + (int64_t)blockIdx.x * a.C;
    if (WAVES > 1) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c = (k * stride + lane) * V;
            if (c < a.C) store_vec(out + c, a.C - c, dw[k]);
        }
        return;
    }
    // The block's row groups, summed in order.
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dw_lds[(sub * NV + k) * lanes * V + lane * V + i] = dw[k][i];
    __syncthreads();
    for (int c = tid; c < a.C; c += 256) {
        float t = 0.f;
        for (int g = 0; g < rows; ++g) t += dw_lds[g * NV * lanes * V + c];
        out[c] = t;
    }
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

// Vectors of a row, and the blocks the gradient's launch has (each writes a
// row of partial dweight): enough rows in flight for the chip, few partial
// rows beside the data.
struct GradShape {
    int64_t nv;
    int lanes;
    int32_t blocks;
};
GradShape grad_shape(const vcsr_rmsnorm_grad_args& a) {
    GradShape g;
    const int v = a.x_type == VCSR_F32 ? 4 : 8;
    g.nv = ((int64_t)a.C + v - 1) / v;
    g.lanes = g.nv <= 64 ? next_pow2((int)g.nv) : 64;
    const int64_t rows = g.nv <= 64 ? 256 / g.lanes : 1;
    const int64_t need = (a.M + rows - 1) / rows;
    g.blocks = (int32_t)(need < 1024 ? need : 1024);
    if (g.nv > 1024 && g.blocks > 64) g.blocks = 64;
    return g;
}

template <class X, class D>
hipError_t launch_grad(const vcsr_rmsnorm_grad_args& a, hipStream_t st) {
    const GradShape g = grad_shape(a);
    float* part = a.dweight ? (float*)a.workspace : nullptr;
    if (g.nv <= 64) {
        rmsnorm_grad_kernel<X, D, 1, 1><<<g.blocks, 256, 0, st>>>(a, part, g.lanes);
    } else if (g.nv <= 256) {
        rmsnorm_grad_kernel<X, D, 4, 1><<<g.blocks, 256, 0, st>>>(a, part, 64);
    } else if (g.nv <= 512) {
        rmsnorm_grad_kernel<X, D, 4, 2><<<g.blocks, 256, 0, st>>>(a, part, 64);
    } else if (g.nv <= 1024) {
        rmsnorm_grad_kernel<X, D, 4, 4><<<g.blocks, 256, 0, st>>>(a, part, 64);
    } else {
        rmsnorm_grad_long_kernel<X, D><<<(unsigned)a.M, 1024, 0, st>>>(a);
        if (part)
            rmsnorm_dweight_kernel<X, D>
                <<<dim3((unsigned)((a.C + 255) / 256), g.blocks), 256, 0, st>>>(a, part);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !part) return e;
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
    return (size_t)grad_shape(a).blocks * (size_t)a.C * sizeof(float);
}

hipError_t launch_rmsnorm_grad(const vcsr_rmsnorm_grad_args& a, hipStream_t st) {
    if (a.M <= 0)
        return a.dweight ? launch_zero(a.dweight, (int64_t)a.C * 4, st) : hipSuccess;
    if (a.x_type == VCSR_F32)
        return a.y_type == VCSR_F32 ? launch_grad<float, float>(a, st)
                                    : launch_grad<float, bf16>(a, st);
    return a.y_type == VCSR_F32 ? launch_grad<bf16, float>(a, st) : launch_grad<bf16, bf16>(a, st);
}

}  // namespace vcsr
