// layernorm.hip - layer norm of x + residual and its gradient.
//
// Forward: t = x + residual, d = t - mean(t), y = d * w / sqrt(mean(d^2) + eps) + b.
// One pass over memory: a row's t stays in registers while its sum, then the sum of
// the centred squares (a single sum of squares would lose the variance of rows whose
// mean is large), and for 8-bit y the largest |y| are reduced.
// Gradient: with h = (s - mean) * rstd, g = dy * w, dx = dsum + rstd * (g - mean(g) -
// h * mean(g h)); again one pass, the row's s and dy in registers, both sums reduced
// together.  dweight and dbias sum dy * h and dy over the rows a block takes in
// registers, then over the blocks (colsum.hip), in a fixed order.
// Memory bounds both: 62451 x 128 FP32 28 us (4.6 TB/s), 32768 x 4096 bf16 188 us, to
// e4m3 187; the gradient of 16384 x 2050 bf16 68 us (4.0 TB/s; 62 and, for the sums over
// the blocks, 6), of 32768 x 4096 208 us (5.2 TB/s), of 62451 x 128 FP32 27 to 30; of few
// long rows (822 x 4154 FP32) 21 to 22 us, 7 of them for both sums.  A single
// row of 4096 bf16 to e4m3 is a kernel of 4.2 us: two trips to memory and three sums.
#include "dense.hpp"
#include "norm_rows.hpp"

namespace vcsr {
namespace {

using namespace norm;

// t -> t - mean, zeros past the row's end.
template <int NV, int V>
__device__ __forceinline__ void centre(float (&t)[NV][V], float mean, int lane, int stride, int C) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i)
            t[k][i] = k + 1 < NV || (k * stride + lane) * V + i < C ? t[k][i] - mean : 0.f;
}

// Rows of at most NV * 64 * WPR vectors, held in registers.  WPR = 1: groups of
// `lanes` (a power of two <= 64) lanes of a 256-thread block take a row each; WPR >
// 1: a block of WPR waves takes a row.  Either goes on to rows gridDim further, with
// the weight and the bias in registers.
template <class X, class Y, int WPR, int NV>
__global__ __launch_bounds__(WPR > 1 ? 64 * WPR : 256) void layernorm_kernel(
    vcsr_layernorm_args a, int lanes) {
    constexpr int V = kVec<X>;
    __shared__ float red[3][WPR];
    const int tid = threadIdx.x;
    const int lane = WPR > 1 ? tid : tid & (lanes - 1);
    const int stride = WPR > 1 ? 64 * WPR : lanes;
    const int rows = WPR > 1 ? 1 : 256 / lanes;
    const int sub = WPR > 1 ? 0 : tid / lanes;
    const int wide = WPR > 1 ? 64 : lanes;
    float w[NV][V], b[NV][V];
    load_row(a.weight, lane, stride, a.C, w);
    if (a.bias) {
        load_row(a.bias, lane, stride, a.C, b);
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) b[k][i] = 0.f;
    }
    // The next row's loads are under way while a row is worked on.
    RawRow<X, NV, V> rx, rr;
    auto ask = [&](int64_t row) __attribute__((always_inline)) {
        const int64_t at = row < a.M ? row : 0;
        rx.load((const X*)a.x + at * a.ldx, lane, stride, a.C);
        if (a.residual) rr.load((const X*)a.residual + at * a.ldr, lane, stride, a.C);
    };
    const int64_t step = (int64_t)gridDim.x * rows;
    ask((int64_t)blockIdx.x * rows + sub);
    for (int64_t base = (int64_t)blockIdx.x * rows; base < a.M; base += step) {
        const int64_t row = base + sub;
        const bool live = row < a.M;  // lanes past the last row still take part in the shuffles
        float t[NV][V];
        rx.get(lane, stride, a.C, t);
        if (a.residual) {
            float v[NV][V];
            rr.get(lane, stride, a.C, v);
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) t[k][i] += v[k][i];
        }
        if (base + step < a.M) ask(row + step);
        float sum = 0.f, sq = 0.f, top = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) sum += t[k][i];
        sum = sum_lanes(wide, sum);
        if (WPR > 1) sum = sum_waves<WPR>(red[0], sum);
        // All of the row's loads are over: sum and y may lie over x or the residual.
        if (live && a.sum) store_row((X*)a.sum + row * a.ldsum, lane, stride, a.C, t);
        const float mean = sum / (float)a.C;
        centre(t, mean, lane, stride, a.C);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) sq = __builtin_fmaf(t[k][i], t[k][i], sq);
        sq = sum_lanes(wide, sq);
        if (WPR > 1) sq = sum_waves<WPR>(red[1], sq);
        const float rstd = 1.f / __builtin_sqrtf(sq / (float)a.C + a.eps);
        if (live && lane == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                t[k][i] = __builtin_fmaf(t[k][i] * rstd, w[k][i], b[k][i]);
                if (sizeof(Y) == 1) top = max_nan(top, __builtin_fabsf(t[k][i]));
            }
        if (sizeof(Y) == 1) {
            top = top_lanes(wide, top);
            if (WPR > 1) top = top_waves<WPR>(red[2], top);
            const float scale = row_factor<Y>(top, a.y_scale, row, live && lane == 0);
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) t[k][i] /= scale;
        }
        if (live) store_row((Y*)a.y + row * a.ldy, lane, stride, a.C, t);
    }
}

// Longer rows: a block reads a row three times (four for 8-bit y), from the caches
// after the first.  sum, which may be x or the residual, is written in the last pass,
// behind the reads of the same values by the same thread.
template <class X, class Y>
__global__ __launch_bounds__(1024) void layernorm_long_kernel(vcsr_layernorm_args a) {
    constexpr int V = kVec<X>, WAVES = 16;
    __shared__ float red[3][WAVES];
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
        const X* x = (const X*)a.x + row * a.ldx;
        const X* r = a.residual ? (const X*)a.residual + row * a.ldr : nullptr;
        auto each = [&](auto&& f) __attribute__((always_inline)) {
            for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 1024 * V) {
                const int n = a.C - c < V ? (int)(a.C - c) : V;
                float t[V];
                load_vec(x + c, n, t);
                if (r) {
                    float v[V];
                    load_vec(r + c, n, v);
#pragma unroll
                    for (int i = 0; i < V; ++i) t[i] += v[i];
                }
                f(c, n, t);
            }
        };
        float sum = 0.f, sq = 0.f, top = 0.f;
        each([&](int64_t, int, float(&t)[V]) {
#pragma unroll
            for (int i = 0; i < V; ++i) sum += t[i];
        });
        const float mean = sum_waves<WAVES>(red[0], sum_lanes(64, sum)) / (float)a.C;
        each([&](int64_t, int n, float(&t)[V]) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = i < n ? t[i] - mean : 0.f;
                sq = __builtin_fmaf(d, d, sq);
            }
        });
        sq = sum_waves<WAVES>(red[1], sum_lanes(64, sq));
        const float rstd = 1.f / __builtin_sqrtf(sq / (float)a.C + a.eps);
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        auto result = [&](int64_t c, int n, const float(&t)[V], float(&y)[V]) {
            float w[V], b[V];
            load_vec(a.weight + c, n, w);
#pragma unroll
            for (int i = 0; i < V; ++i) b[i] = 0.f;
            if (a.bias) load_vec(a.bias + c, n, b);
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] = __builtin_fmaf((t[i] - mean) * rstd, w[i], b[i]);
        };
        float scale = 1.f;
        if (sizeof(Y) == 1) {
            each([&](int64_t c, int n, float(&t)[V]) {
                float y[V];
                result(c, n, t, y);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i < n) top = max_nan(top, __builtin_fabsf(y[i]));
            });
            top = top_waves<WAVES>(red[2], top_lanes(64, top));
            scale = row_factor<Y>(top, a.y_scale, row, threadIdx.x == 0);
        }
        each([&](int64_t c, int n, float(&t)[V]) {
            float y[V];
            result(c, n, t, y);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (sizeof(Y) == 1) y[i] /= scale;
            if (a.sum) store_vec((X*)a.sum + row * a.ldsum + c, n, t);
            store_vec((Y*)a.y + row * a.ldy + c, n, y);
        });
    }
}

// Rows of fewer values than a vector: a thread takes a row.
template <class X, class Y>
__global__ __launch_bounds__(256) void layernorm_narrow_kernel(vcsr_layernorm_args a) {
    constexpr int V = kVec<X>;
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (row >= a.M) return;
    float t[V], w[V], b[V], sum = 0.f, sq = 0.f, top = 0.f;
    load_vec((const X*)a.x + row * a.ldx, a.C, t);
    load_vec(a.weight, a.C, w);
#pragma unroll
    for (int i = 0; i < V; ++i) b[i] = 0.f;
    if (a.bias) load_vec(a.bias, a.C, b);
    if (a.residual) {
        float v[V];
        load_vec((const X*)a.residual + row * a.ldr, a.C, v);
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] += v[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sum += t[i];
    if (a.sum) store_vec((X*)a.sum + row * a.ldsum, a.C, t);
    const float mean = sum / (float)a.C;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        t[i] = i < a.C ? t[i] - mean : 0.f;
        sq = __builtin_fmaf(t[i], t[i], sq);
    }
    const float rstd = 1.f / __builtin_sqrtf(sq / (float)a.C + a.eps);
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        t[i] = __builtin_fmaf(t[i] * rstd, w[i], b[i]);
        if (sizeof(Y) == 1 && i < a.C) top = max_nan(top, __builtin_fabsf(t[i]));
    }
    const float scale = row_factor<Y>(top, a.y_scale, row, true);
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (sizeof(Y) == 1) t[i] /= scale;
    store_vec((Y*)a.y + row * a.ldy, a.C, t);
}

template <class X, class Y>
hipError_t launch_forward(const vcsr_layernorm_args& a, hipStream_t st) {
    constexpr int V = kVec<X>;
    const int64_t nv = ((int64_t)a.C + V - 1) / V;
    if (a.C < V) {
        layernorm_narrow_kernel<X, Y><<<(unsigned)((a.M + 255) / 256), 256, 0, st>>>(a);
        return hipGetLastError();
    }
    if (nv > 2048) {
        const unsigned blocks = (unsigned)(a.M < 1 << 20 ? a.M : 1 << 20);
        layernorm_long_kernel<X, Y><<<blocks, 1024, 0, st>>>(a);
        return hipGetLastError();
    }
    const int lanes = nv <= 64 ? next_pow2((int)nv) : 64;
    with_shape(row_shape(nv, 4), [&](auto wpr, auto k) {
        constexpr int W = decltype(wpr)::value, NV = decltype(k)::value;
        const int64_t rows = W > 1 ? 1 : 256 / lanes, need = (a.M + rows - 1) / rows;
        // To 8 bits, with three sums a row, blocks that stay and have the next row under
        // way: 32768 x 4096 bf16 186 us, 195 with a block for each row; to bf16 that is
        // the faster one (8192 x 8192 FP32 189 against 204).
        const int64_t most = sizeof(Y) == 1 ? 32 * 256 / (W > 1 ? W : 4) : 1 << 20;
        layernorm_kernel<X, Y, W, NV>
            <<<(unsigned)(need < most ? need : most), W > 1 ? 64 * W : 256, 0, st>>>(a, lanes);
    });
    return hipGetLastError();
}

// ------------------------------------------------------------------ gradient
// Where a block's sums of dweight and dbias go: row blockIdx of partial rows `ld`
// apart, or (one block) the results themselves.
struct Sums {
    float *dweight, *dbias;
    int64_t ld;
};

// Rows of at most NV * 64 * WPR vectors (as above); each row group goes through rows
// blockIdx, blockIdx + gridDim, ... and keeps dweight and dbias of its columns in
// registers, the weight in LDS.
template <class X, class D, int WPR, int NV>
__global__ __launch_bounds__(WPR > 1 ? 64 * WPR : 256) void layernorm_grad_kernel(
    vcsr_layernorm_grad_args a, Sums out, int lanes) {
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
    float dw[NV][V], db[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
    const float inv_c = 1.f / (float)a.C;
    // The next row's loads are under way while a row is worked on (16384 x 2050 bf16 67.5 us,
    // 70.3 without; 822 x 4154 FP32 21.1 and 22.6), unless registers are short.
    constexpr bool AHEAD = NV < 4;
    RawRow<X, NV, V> rs, ro;
    RawRow<D, NV, V> rd;
    float next_rstd, next_mean;
    auto ask = [&](int64_t row) __attribute__((always_inline)) {
        const int64_t at = row < a.M ? row : 0;
        next_rstd = a.rstd[at];
        next_mean = a.mean[at];
        rs.load((const X*)a.s + at * a.lds, lane, stride, a.C);
        rd.load((const D*)a.dy + at * a.lddy, lane, stride, a.C);
        if (a.dsum) ro.load((const X*)a.dsum + at * a.lddsum, lane, stride, a.C);
    };
    const int64_t step = (int64_t)gridDim.x * rows;
    if (AHEAD) ask((int64_t)blockIdx.x * rows + sub);
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * rows; base < a.M; base += step, turn ^= 1) {
        const int64_t row = base + sub;
        const bool live = row < a.M;
        float s[NV][V], d[NV][V], o[NV][V];
        if (!AHEAD) ask(row);
        const float rstd = next_rstd, mean = next_mean;
        float all = 0.f, dot = 0.f;
        rs.get(lane, stride, a.C, s);
        rd.get(lane, stride, a.C, d);
        if (a.dsum) {
            ro.get(lane, stride, a.C, o);
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) o[k][i] = 0.f;
        }
        if (AHEAD && base + step < a.M) ask(row + step);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const float* const w = w_lds + (k * stride + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                // h, past the row's end zero: -mean * rstd may be infinite there.
                const bool in = k + 1 < NV || (k * stride + lane) * V + i < a.C;
                s[k][i] = in ? (s[k][i] - mean) * rstd : 0.f;
                if (WPR == 1 && !live) s[k][i] = d[k][i] = 0.f;
                dw[k][i] = __builtin_fmaf(d[k][i], s[k][i], dw[k][i]);
                db[k][i] += d[k][i];
                d[k][i] *= w[i];  // g
                all += d[k][i];
                dot = __builtin_fmaf(d[k][i], s[k][i], dot);
            }
        }
        all = sum_lanes(WPR > 1 ? 64 : lanes, all);
        dot = sum_lanes(WPR > 1 ? 64 : lanes, dot);
        // Two sets of LDS slots in turn: the next row's sums do not meet this one's.
        if (WPR > 1) sum_waves<WPR>(red[turn], all, dot);
        if (!live) continue;
        const float mean_g = all * inv_c, mean_gh = dot * inv_c;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i)
                o[k][i] += rstd * (d[k][i] - mean_g - s[k][i] * mean_gh);
        store_row((X*)a.dx + row * a.lddx, lane, stride, a.C, o);
    }
    auto write = [&](float* to, float(&v)[NV][V]) __attribute__((always_inline)) {
        if (!to) return;
        to += (int64_t)blockIdx.x * out.ld;
        if (WPR > 1) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int c = (k * stride + lane) * V;
                if (c < a.C) store_vec(to + c, a.C - c, v[k]);
            }
            return;
        }
        // A wave's row groups add up over its lanes, then the waves in LDS, one after
        // the other.
        for (int m = lanes; m < 64; m <<= 1)
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) v[k][i] += __shfl_xor(v[k][i], m);
        __syncthreads();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (tid >> 6 == g && (tid & 63) < lanes)
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float* const p = w_lds + (k * stride + lane) * V + i;
                        *p = g ? *p + v[k][i] : v[k][i];
                    }
            __syncthreads();
        }
        for (int c = tid; c < a.C; c += 256) to[c] = w_lds[c];
    };
    write(out.dweight, dw);
    write(out.dbias, db);
}

// Longer rows: a block per row, read twice; dweight and dbias apart (column by
// column).
template <class X, class D>
__global__ __launch_bounds__(1024) void layernorm_grad_long_kernel(vcsr_layernorm_grad_args a) {
    constexpr int V = kVec<X>, WAVES = 16;
    __shared__ float red[2][2 * WAVES];
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x, turn ^= 1) {
        const X* s = (const X*)a.s + row * a.lds;
        const D* dy = (const D*)a.dy + row * a.lddy;
        const float rstd = a.rstd[row], mean = a.mean[row];
        float all = 0.f, dot = 0.f;
        for (int64_t c = (int64_t)threadIdx.x * V; c < a.C; c += 1024 * V) {
            const int n = a.C - c < V ? (int)(a.C - c) : V;
            float h[V], g[V], w[V];
            load_vec(s + c, n, h);
            load_vec(dy + c, n, g);
            load_vec(a.weight + c, n, w);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                all = __builtin_fmaf(g[i], w[i], all);
                if (i < n) dot = __builtin_fmaf(g[i] * w[i], (h[i] - mean) * rstd, dot);
            }
        }
        all = sum_lanes(64, all);
        dot = sum_lanes(64, dot);
        sum_waves<WAVES>(red[turn], all, dot);
        const float mean_g = all / (float)a.C, mean_gh = dot / (float)a.C;
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
            for (int i = 0; i < V; ++i)
                o[i] += rstd * (g[i] * w[i] - mean_g - (h[i] - mean) * rstd * mean_gh);
            store_vec((X*)a.dx + row * a.lddx + c, n, o);
        }
    }
}
// Their dweight and dbias: a thread per column over a block of rows.
template <class X, class D>
__global__ __launch_bounds__(256) void layernorm_dweight_kernel(vcsr_layernorm_grad_args a,
                                                                Sums out) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.C) return;
    float t = 0.f, u = 0.f;
    for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
        const float d = to_f32(((const D*)a.dy)[row * a.lddy + c]);
        t = __builtin_fmaf(
            d, (to_f32(((const X*)a.s)[row * a.lds + c]) - a.mean[row]) * a.rstd[row], t);
        u += d;
    }
    if (out.dweight) out.dweight[(int64_t)blockIdx.y * out.ld + c] = t;
    if (out.dbias) out.dbias[(int64_t)blockIdx.y * out.ld + c] = u;
}

// Rows of fewer values than a vector: a thread takes rows blocks apart and keeps
// dweight and dbias in registers; lanes, then waves, add theirs up.
template <class X, class D>
__global__ __launch_bounds__(256) void layernorm_grad_narrow_kernel(vcsr_layernorm_grad_args a,
                                                                    Sums out) {
    constexpr int V = kVec<X>;
    __shared__ float lds[2][4][V];
    float w[V], dw[V], db[V];
    load_vec(a.weight, a.C, w);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[i] = db[i] = 0.f;
    const float inv_c = 1.f / (float)a.C;
    for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < a.M;
         row += (int64_t)gridDim.x * 256) {
        float h[V], g[V], o[V], all = 0.f, dot = 0.f;
        const float rstd = a.rstd[row], mean = a.mean[row];
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
            if (i >= a.C) continue;  // a factor may be infinite
            h[i] = (h[i] - mean) * rstd;
            dw[i] = __builtin_fmaf(g[i], h[i], dw[i]);
            db[i] += g[i];
            g[i] *= w[i];
            all += g[i];
            dot = __builtin_fmaf(g[i], h[i], dot);
        }
        const float mean_g = all * inv_c, mean_gh = dot * inv_c;
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] += rstd * (g[i] - mean_g - h[i] * mean_gh);
        store_vec((X*)a.dx + row * a.lddx, a.C, o);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        dw[i] = sum_lanes(64, dw[i]);
        db[i] = sum_lanes(64, db[i]);
        if ((threadIdx.x & 63) == 0) {
            lds[0][threadIdx.x >> 6][i] = dw[i];
            lds[1][threadIdx.x >> 6][i] = db[i];
        }
    }
    __syncthreads();
    const int c = threadIdx.x & 63, which = threadIdx.x >> 6;
    float* const to = which == 0 ? out.dweight : which == 1 ? out.dbias : nullptr;
    if (to && c < a.C) {
        const auto& v = lds[which];
        to[(int64_t)blockIdx.x * out.ld + c] = ((v[0][c] + v[1][c]) + v[2][c]) + v[3][c];
    }
}

// The gradient's row shape and blocks, each of which writes a row of partial dweight
// and dbias.
struct GradShape {
    int64_t nv;
    int lanes;
    RowShape row;
    bool narrow, in_registers;
    int32_t blocks;
};
GradShape grad_shape(const vcsr_layernorm_grad_args& a) {
    GradShape g;
    const int v = a.x_type == VCSR_F32 ? 4 : 8;
    g.nv = ((int64_t)a.C + v - 1) / v;
    g.lanes = g.nv <= 64 ? next_pow2((int)g.nv) : 64;
    g.row = row_shape(g.nv, 3);
    const int64_t rows = g.row.wpr > 1 ? 1 : 256 / g.lanes;
    const int64_t waves = g.row.wpr > 1 ? g.row.wpr : 4;
    const int64_t need = (a.M + rows - 1) / rows, most = 2048 / waves;
    g.blocks = (int32_t)(need < most ? need : most);
    if (need <= 4) g.blocks = 1;  // which then writes dweight and dbias itself
    g.narrow = a.C < v;
    g.in_registers = g.nv <= 2048 && !g.narrow;
    if (g.narrow) g.blocks = (int32_t)(a.M < 256 * 1024 ? (a.M + 255) / 256 : 1024);
    else if (!g.in_registers) g.blocks = (int32_t)(a.M < 64 ? a.M : 64);
    return g;
}

template <class X, class D>
hipError_t launch_grad(const vcsr_layernorm_grad_args& a, hipStream_t st) {
    const GradShape g = grad_shape(a);
    const bool sums = a.dweight || a.dbias;
    float* const part = (float*)a.workspace;  // partial rows of dweight, then of dbias
    Sums out{a.dweight, a.dbias, 0};
    if (g.blocks > 1)
        out = Sums{a.dweight ? part : nullptr,
                   a.dbias ? part + (a.dweight ? a.C : 0) : nullptr,
                   (a.dweight && a.dbias ? 2 : 1) * (int64_t)a.C};
    if (g.narrow) {
        layernorm_grad_narrow_kernel<X, D><<<(unsigned)g.blocks, 256, 0, st>>>(a, out);
    } else if (!g.in_registers) {
        if (sums)  // before dx, which may be s or dy itself
            layernorm_dweight_kernel<X, D>
                <<<dim3((unsigned)(((int64_t)a.C + 255) / 256), g.blocks), 256, 0, st>>>(a, out);
        const unsigned blocks = (unsigned)(a.M < 1 << 20 ? a.M : 1 << 20);
        layernorm_grad_long_kernel<X, D><<<blocks, 1024, 0, st>>>(a);
    } else {
        with_shape(g.row, [&](auto wpr, auto k) {
            constexpr int W = decltype(wpr)::value, NV = decltype(k)::value;
            layernorm_grad_kernel<X, D, W, NV>
                <<<g.blocks, W > 1 ? 64 * W : 256, 0, st>>>(a, out, g.lanes);
        });
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !sums || g.blocks == 1) return e;
    return launch_sum_row_pairs(part, g.blocks, a.C, out.ld, a.C, a.dweight ? a.dweight : a.dbias,
                                a.dweight ? a.dbias : nullptr, st);
}

}  // namespace

hipError_t launch_layernorm(const vcsr_layernorm_args& a, hipStream_t st) {
    if (a.M <= 0) return hipSuccess;
    if (a.x_type == VCSR_F32)
        return a.y_type == VCSR_F32    ? launch_forward<float, float>(a, st)
               : a.y_type == VCSR_BF16 ? launch_forward<float, bf16>(a, st)
                                       : launch_forward<float, fp8>(a, st);
    return a.y_type == VCSR_F32    ? launch_forward<bf16, float>(a, st)
           : a.y_type == VCSR_BF16 ? launch_forward<bf16, bf16>(a, st)
                                   : launch_forward<bf16, fp8>(a, st);
}

size_t layernorm_grad_workspace(const vcsr_layernorm_grad_args& a) {
    if ((!a.dweight && !a.dbias) || a.M <= 0) return 0;
    const int32_t blocks = grad_shape(a).blocks;
    const size_t rows = (a.dweight ? 1 : 0) + (a.dbias ? 1 : 0);
    return blocks > 1 ? rows * (size_t)blocks * (size_t)a.C * sizeof(float) : 0;
}

hipError_t launch_layernorm_grad(const vcsr_layernorm_grad_args& a, hipStream_t st) {
    if (a.M <= 0) {
        const int64_t bytes = (int64_t)a.C * 4;
        hipError_t e = hipSuccess;
        if (a.dweight) e = launch_zero(a.dweight, bytes, 1, bytes, st);
        if (e == hipSuccess && a.dbias) e = launch_zero(a.dbias, bytes, 1, bytes, st);
        return e;
    }
    if (a.x_type == VCSR_F32)
        return a.y_type == VCSR_F32 ? launch_grad<float, float>(a, st)
                                    : launch_grad<float, bf16>(a, st);
    return a.y_type == VCSR_F32 ? launch_grad<bf16, float>(a, st) : launch_grad<bf16, bf16>(a, st);
}

}  // namespace vcsr
