// colsum.hip - what the gradients sum over rows, in a fixed order: the partial
// rows of dweight and dbias, and dz = dy * act'(z) with the sums of its rows.
#include "common.hpp"
#include "dense.hpp"

namespace vcsr {
namespace {

// 16 columns a block, 64 threads a column: each adds every 64th partial row, then
// LDS adds the threads in order.
// blockIdx.y: of two sums, whose partial rows lie `next` apart, `out` or `out2`.
__global__ __launch_bounds__(1024) void sum_rows_kernel(const float* part, int32_t P, int32_t C,
                                                        int64_t ld, float* out, float* out2,
                                                        int64_t next) {
    __shared__ float lds[64][17];
    if (blockIdx.y) {
        part += next;
        out = out2;
    }
    const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
    // Neighbouring blocks, which share lines, on one XCD.
    const int64_t c = (int64_t)xcd_remap(blockIdx.x, gridDim.x) * 16 + col;
    float t = 0.f;
    if (c < C) {
#pragma unroll 8
        for (int32_t p = grp; p < P; p += 64) t += part[(int64_t)p * ld + c];
    }
    lds[grp][col] = t;
    __syncthreads();
    if (grp < 8) {
        t = lds[grp * 8][col];
#pragma unroll
        for (int g = 1; g < 8; ++g) t += lds[grp * 8 + g][col];
    }
    __syncthreads();
    if (grp < 8) lds[grp][col] = t;
    __syncthreads();
    if (grp == 0 && c < C) {
#pragma unroll
        for (int g = 1; g < 8; ++g) t += lds[g][col];
        out[c] = t;
    }
}

// A block takes `rows` rows of tx vectors of 16 bytes of dy: 256 / tx rows at a time,
// four of them under way together without a branch between their loads (rows past
// the block's end are its last one again and count for nothing).  Bound by memory:
// dy and z read once, dz written once (8192 x 4096 bf16 with gelu 37 to 40 us, 5.0 to
// 5.4 TB/s; 30011 x 257 FP32, whose rows begin anywhere in a line, 28 us, 3.3 TB/s).
// ENDS: how rows end: 0 in whole vectors, 1 inside one, 2 before the first is whole.
//
// For bf16 operands dz is rounded to bf16, also where dy and z are FP32: the products'
// matrix instruction takes no more.  Each dz moves by 2^-8 of itself at most, so a
// product's error stays small against its own terms; the gradients of 8192 x 2048 x 4096
// are 0.0023 from 64 bits, and 0.0017 with dz unrounded, which is their own last
// rounding.  Two bf16 parts of dz would keep its bits for twice the matrix work (some
// 280 of the call's 318 us again).
template <class D, class X, int ACT, int ENDS>
__global__ __launch_bounds__(256) void dz_kernel(vcsr_linear_grad_args a, X* dz, int64_t lddz,
                                                 float* part, int64_t rows, int tx) {
    constexpr int U = 4, V = 16 / (int)sizeof(D);
    __shared__ float lds[256 * V];
    const int ty_n = 256 / tx, ty = threadIdx.x / tx;
    const int64_t c = ((int64_t)blockIdx.x * tx + (threadIdx.x - ty * tx)) * V;
    const int n = c >= a.N ? 0 : a.N - c < V ? (int)(a.N - c) : V;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    const int64_t first = (int64_t)blockIdx.y * rows;
    const int64_t last = first + rows < a.M ? first + rows : a.M;
    if (n > 0 && ty < ty_n) {
        auto load = [&](const D* row, float(&v)[V]) __attribute__((always_inline)) {
            if (ENDS == 0)
                load_full(row + c, v);
            else if (ENDS == 1)
                load_tail(row, (int)c, a.N, v);
            else
                load_vec(row + c, n, v);
        };
        for (int64_t m = first + ty; m < last; m += U * ty_n) {
            float d[U][V], z[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = m + u * ty_n < last ? m + u * ty_n : last - 1;
                load((const D*)a.dy + r * a.lddy, d[u]);
                if (ACT != VCSR_ACT_NONE) load((const D*)a.z + r * a.ldz, z[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (m + u * ty_n >= last) continue;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (ACT != VCSR_ACT_NONE) d[u][i] *= act_grad_f32<ACT>(z[u][i]);
                    if (ENDS == 0 || i < n) sum[i] += d[u][i];
                }
                if (dz) store_vec(dz + (m + u * ty_n) * lddz + c, ENDS == 0 ? V : n, d[u]);
            }
        }
    }
    if (!part) return;
    if (ty < ty_n)
#pragma unroll
        for (int i = 0; i < V; ++i) lds[threadIdx.x * V + i] = sum[i];
    __syncthreads();
    for (int col = threadIdx.x; col < tx * V; col += 256) {
        const int64_t at = (int64_t)blockIdx.x * tx * V + col;
        if (at >= a.N) continue;
        float t = 0.f;
        for (int g = 0; g < ty_n; ++g) t += lds[g * tx * V + col];
        part[(int64_t)blockIdx.y * a.N + at] = t;
    }
}

// Vectors of a block's rows (even parts of a row's, at most 128, that leave few of
// its threads idle) and its rows: two
// passes of its threads at least, and few enough blocks of rows that their partial
// sums stay small.
struct DzShape {
    int tx;
    int64_t columns, rows, blocks;
};
DzShape dz_shape(int64_t M, int32_t N, int32_t dy_type) {
    DzShape s;
    const int64_t v = dy_type == VCSR_F32 ? 4 : 8, vectors = ((int64_t)N + v - 1) / v;
    double best = 0.0;
    for (int64_t k = (vectors + 127) / 128, end = k + 4; k < end; ++k) {
        const int64_t tx = (vectors + k - 1) / k, columns = (vectors + tx - 1) / tx;
        // Of the block's threads and of their vectors, those that are there.
        const double used = (double)(256 / tx * tx) * (double)vectors / (double)(tx * columns);
        if (used > best * 1.02) {
            best = used;
            s.tx = (int)tx;
            s.columns = columns;
        }
    }
    s.rows = 8 * (256 / s.tx);
    if (M <= 2 * s.rows) s.rows *= 2;  // one block of rows: no partial sums to add up
    while ((M + s.rows - 1) / s.rows > 1024) s.rows *= 2;
    s.blocks = (M + s.rows - 1) / s.rows;
    return s;
}

template <class D, class X, int ACT>
void launch_dz_act(const vcsr_linear_grad_args& a, X* dz, int64_t lddz, float* part,
                   hipStream_t st) {
    constexpr int V = 16 / (int)sizeof(D);
    const DzShape s = dz_shape(a.M, a.N, a.y_type);
    const dim3 grid((unsigned)s.columns, (unsigned)s.blocks);
    if (a.N % V == 0)
        dz_kernel<D, X, ACT, 0><<<grid, 256, 0, st>>>(a, dz, lddz, part, s.rows, s.tx);
    else if (a.N > V)
        dz_kernel<D, X, ACT, 1><<<grid, 256, 0, st>>>(a, dz, lddz, part, s.rows, s.tx);
    else
        dz_kernel<D, X, ACT, 2><<<grid, 256, 0, st>>>(a, dz, lddz, part, s.rows, s.tx);
}
template <class D, class X>
hipError_t launch_dz_typed(const vcsr_linear_grad_args& a, X* dz, int64_t lddz, float* part,
                           hipStream_t st) {
    switch (a.act) {
        case VCSR_ACT_RELU: launch_dz_act<D, X, VCSR_ACT_RELU>(a, dz, lddz, part, st); break;
        case VCSR_ACT_GELU: launch_dz_act<D, X, VCSR_ACT_GELU>(a, dz, lddz, part, st); break;
        case VCSR_ACT_SILU: launch_dz_act<D, X, VCSR_ACT_SILU>(a, dz, lddz, part, st); break;
        default: launch_dz_act<D, X, VCSR_ACT_NONE>(a, dz, lddz, part, st);
    }
    return hipGetLastError();
}

// The gated projection's, as dz_kernel: dy, z_gate and z_up read once, dz_gate and dz_up
// written once and rounded to the products' type, with zeros up to the end of their rows.
// That rounding is dz_kernel's choice, for its reason: the bf16 gradients of 8192 x 2048 x 4096
// are 0.0023 from 64 bits, and 0.0017, their own last rounding, with both dz unrounded.  The
// biases' sums take the unrounded values.
// Bound by memory: 8192 x 4096 bf16 59 us (5.7 TB/s); 30011 x 257 FP32, whose rows begin
// anywhere in a line, 35 us (4.6 TB/s), 48 with four rows' loads under way instead of two.
template <class D, class X, int ACT, int ENDS>
__global__ __launch_bounds__(256) void gated_dz_kernel(vcsr_gated_grad_args a, X* dz, int64_t lddz,
                                                       float* part_gate, float* part_up,
                                                       int64_t rows, int tx) {
    constexpr int U = 2, V = 16 / (int)sizeof(D);
    __shared__ float lds[2][256 * V];
    const int ty_n = 256 / tx, ty = threadIdx.x / tx;
    const int64_t c = ((int64_t)blockIdx.x * tx + (threadIdx.x - ty * tx)) * V;
    const int n = c >= a.N ? 0 : a.N - c < V ? (int)(a.N - c) : V;
    float sum[2][V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[0][i] = sum[1][i] = 0.f;
    const int64_t first = (int64_t)blockIdx.y * rows;
    const int64_t last = first + rows < a.M ? first + rows : a.M;
    if (n > 0 && ty < ty_n) {
        auto load = [&](const D* row, float(&v)[V]) __attribute__((always_inline)) {
            if (ENDS == 0)
                load_full(row + c, v);
            else if (ENDS == 1)
                load_tail(row, (int)c, a.N, v);
            else
                load_vec(row + c, n, v);
        };
        for (int64_t m = first + ty; m < last; m += U * ty_n) {
            float d[U][V], g[U][V], w[U][V];  // zeros behind the row's end
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = m + u * ty_n < last ? m + u * ty_n : last - 1;
                load((const D*)a.dy + r * a.lddy, d[u]);
                load((const D*)a.z_gate + r * a.ldz, g[u]);
                load((const D*)a.z_up + r * a.ldz, w[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (m + u * ty_n >= last) continue;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float z = g[u][i];
                    // Where dy * z_up passes FP32's range both are over 1, and what act' (1.13
                    // at most) brings back into it is formed by taking act' first.
                    const float slope = act_grad_f32<ACT>(z), both = d[u][i] * w[u][i];
                    g[u][i] = __builtin_isinf(both) ? d[u][i] * slope * w[u][i] : both * slope;
                    w[u][i] = d[u][i] * act_f32<ACT>(z);
                    if (ENDS == 0 || i < n) {
                        sum[0][i] += g[u][i];
                        sum[1][i] += w[u][i];
                    }
                }
                if (dz) {
                    X* const to = dz + (m + u * ty_n) * lddz + c;
                    store_vec(to, V, g[u]);
                    store_vec(to + a.M * lddz, V, w[u]);
                }
            }
        }
    } else if (dz && c < lddz && ty < ty_n) {
        for (int64_t m = first + ty; m < last; m += ty_n) {
            store_vec(dz + m * lddz + c, V, sum[0]);  // zeros
            store_vec(dz + (a.M + m) * lddz + c, V, sum[0]);
        }
    }
    if (!part_gate && !part_up) return;
    if (ty < ty_n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < V; ++i) lds[h][threadIdx.x * V + i] = sum[h][i];
    __syncthreads();
    for (int col = threadIdx.x; col < tx * V; col += 256) {
        const int64_t at = (int64_t)blockIdx.x * tx * V + col;
        if (at >= a.N) continue;
        float t[2] = {0.f, 0.f};
        for (int k = 0; k < ty_n; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) t[h] += lds[h][k * tx * V + col];
        if (part_gate) part_gate[(int64_t)blockIdx.y * a.N + at] = t[0];
        if (part_up) part_up[(int64_t)blockIdx.y * a.N + at] = t[1];
    }
}

template <class D, class X, int ACT>
void launch_gated_act(const vcsr_gated_grad_args& a, X* dz, int64_t lddz, float* part_gate,
                      float* part_up, hipStream_t st) {
    constexpr int V = 16 / (int)sizeof(D);
    const DzShape s = dz_shape(a.M, (int32_t)lddz, a.y_type);
    const dim3 grid((unsigned)s.columns, (unsigned)s.blocks);
    if (a.N % V == 0)
        gated_dz_kernel<D, X, ACT, 0>
            <<<grid, 256, 0, st>>>(a, dz, lddz, part_gate, part_up, s.rows, s.tx);
    else if (a.N > V)
        gated_dz_kernel<D, X, ACT, 1>
            <<<grid, 256, 0, st>>>(a, dz, lddz, part_gate, part_up, s.rows, s.tx);
    else
        gated_dz_kernel<D, X, ACT, 2>
            <<<grid, 256, 0, st>>>(a, dz, lddz, part_gate, part_up, s.rows, s.tx);
}
template <class D, class X>
hipError_t launch_gated_typed(const vcsr_gated_grad_args& a, X* dz, int64_t lddz, float* g,
                              float* u, hipStream_t st) {
    switch (a.act) {
        case VCSR_ACT_RELU: launch_gated_act<D, X, VCSR_ACT_RELU>(a, dz, lddz, g, u, st); break;
        case VCSR_ACT_GELU: launch_gated_act<D, X, VCSR_ACT_GELU>(a, dz, lddz, g, u, st); break;
        case VCSR_ACT_SILU: launch_gated_act<D, X, VCSR_ACT_SILU>(a, dz, lddz, g, u, st); break;
        default: launch_gated_act<D, X, VCSR_ACT_NONE>(a, dz, lddz, g, u, st);
    }
    return hipGetLastError();
}

// Rows of `n` 16-bit values, `ld` apart.
__global__ __launch_bounds__(256) void zero_kernel(uint16_t* p, int64_t ld, int64_t rows,
                                                   int64_t n) {
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256)
            p[r * ld + i] = 0;
}

}  // namespace

hipError_t launch_sum_row_pairs(const float* part, int32_t P, int32_t C, int64_t ld, int64_t next,
                                float* a, float* b, hipStream_t st) {
    // 64 threads a column, and fewer than 2^32 threads a launch.
    const int32_t most = b ? 1 << 24 : 1 << 25;
    for (int64_t c = 0; c < C; c += most) {
        const int32_t n = C - c < most ? (int32_t)(C - c) : most;
        sum_rows_kernel<<<dim3((unsigned)((n + 15) / 16), b ? 2 : 1), 1024, 0, st>>>(
            part + c, P, n, ld, a + c, b ? b + c : nullptr, next);
    }
    return hipGetLastError();
}
hipError_t launch_sum_rows(const float* part, int32_t P, int32_t C, int64_t ld, float* out,
                           hipStream_t st) {
    return launch_sum_row_pairs(part, P, C, ld, 0, out, nullptr, st);
}

int32_t dz_row_blocks(int64_t M, int32_t N, int32_t dy_type) {
    return (int32_t)dz_shape(M, N, dy_type).blocks;
}

hipError_t launch_dz(const vcsr_linear_grad_args& a, void* dz, int64_t lddz, float* part,
                     hipStream_t st) {
    if (a.y_type == VCSR_F32)
        return a.x_type == VCSR_F32
                   ? launch_dz_typed<float, float>(a, (float*)dz, lddz, part, st)
                   : launch_dz_typed<float, bf16>(a, (bf16*)dz, lddz, part, st);
    return a.x_type == VCSR_F32 ? launch_dz_typed<bf16, float>(a, (float*)dz, lddz, part, st)
                                : launch_dz_typed<bf16, bf16>(a, (bf16*)dz, lddz, part, st);
}

int32_t gated_row_blocks(int64_t M, int64_t lddz, int32_t dy_type) {
    return (int32_t)dz_shape(M, (int32_t)lddz, dy_type).blocks;
}

hipError_t launch_gated_dz(const vcsr_gated_grad_args& a, void* dz, int64_t lddz, float* g,
                           float* u, hipStream_t st) {
    if (a.y_type == VCSR_F32)
        return a.x_type == VCSR_F32
                   ? launch_gated_typed<float, float>(a, (float*)dz, lddz, g, u, st)
                   : launch_gated_typed<float, bf16>(a, (bf16*)dz, lddz, g, u, st);
    return a.x_type == VCSR_F32 ? launch_gated_typed<bf16, float>(a, (float*)dz, lddz, g, u, st)
                                : launch_gated_typed<bf16, bf16>(a, (bf16*)dz, lddz, g, u, st);
}

hipError_t launch_zero(void* p, int64_t ld, int64_t rows, int64_t bytes, hipStream_t st) {
    if (rows <= 0 || bytes <= 0) return hipSuccess;
    if (ld == bytes) {  // one row
        bytes *= rows;
        rows = 1;
    }
    const int64_t n = bytes / 2, columns = (n + 255) / 256, most = rows == 1 ? 4096 : 16;
    const dim3 grid((unsigned)(columns < most ? columns : most),
                    (unsigned)(rows < 4096 ? rows : 4096));
    zero_kernel<<<grid, 256, 0, st>>>((uint16_t*)p, ld / 2, rows, n);
    return hipGetLastError();
}

}  // namespace vcsr
