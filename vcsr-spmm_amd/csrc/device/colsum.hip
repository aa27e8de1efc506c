// colsum.hip - what the gradients sum over rows, in a fixed order: the partial
// rows of dweight and dbias, and dz = dy * act'(z) with the sums of its rows.
#include "dense.hpp"

namespace vcsr {
namespace {

// 16 columns a block, 64 threads a column: each adds every 64th partial row, then
// LDS adds the threads in order.
__global__ __launch_bounds__(1024) void sum_rows_kernel(const float* part, int32_t P, int32_t C,
                                                        int64_t ld, float* out) {
    __shared__ float lds[64][17];
    const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
    const int64_t c = (int64_t)blockIdx.x * 16 + col;
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

// A block takes `rows` rows of 8 * TX columns: TX threads of 8 columns a row, 256
// / TX rows at a time, two of them under way together.  Bound by memory: dy and z
// read once, dz written once.
template <class D, class X, int ACT>
__global__ __launch_bounds__(256) void dz_kernel(vcsr_linear_grad_args a, X* dz, int64_t lddz,
                                                 float* part, int64_t rows, int tx_log) {
    __shared__ float lds[256 * 8];
    const int TX = 1 << tx_log, TY = 256 >> tx_log;
    const int tx = threadIdx.x & (TX - 1), ty = threadIdx.x >> tx_log;
    const int64_t c = ((int64_t)blockIdx.x * TX + tx) * 8;
    const int n = c >= a.N ? 0 : a.N - c < 8 ? (int)(a.N - c) : 8;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const int64_t first = (int64_t)blockIdx.y * rows;
    const int64_t last = first + rows < a.M ? first + rows : a.M;
    if (n > 0) {
        for (int64_t m = first + ty; m < last; m += 2 * TY) {
            float d[2][8], z[2][8];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int64_t r = m + u * TY;
                if (r >= last) continue;
                load_vec((const D*)a.dy + r * a.lddy + c, n, d[u]);
                if (ACT != VCSR_ACT_NONE) load_vec((const D*)a.z + r * a.ldz + c, n, z[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int64_t r = m + u * TY;
                if (r >= last) continue;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (ACT != VCSR_ACT_NONE) d[u][i] *= act_grad_f32<ACT>(z[u][i]);
                    if (i >= n) d[u][i] = 0.f;  // act'(0) of what is not there
                    sum[i] += d[u][i];
                }
                if (dz) store_vec(dz + r * lddz + c, n, d[u]);
            }
        }
    }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) lds[(ty * TX + tx) * 8 + i] = sum[i];
    __syncthreads();
    for (int col = threadIdx.x; col < TX * 8; col += 256) {
        const int64_t at = (int64_t)blockIdx.x * TX * 8 + col;
        if (at >= a.N) continue;
        float t = 0.f;
        for (int g = 0; g < TY; ++g) t += lds[g * TX * 8 + col];
        part[(int64_t)blockIdx.y * a.N + at] = t;
    }
}

// Threads along a row (8, 16 or 32) and rows of a block: at least four passes of its
// threads, and few enough blocks of rows that their partial sums stay small.
struct DzShape {
    int tx_log;
    int64_t rows, blocks;
};
DzShape dz_shape(int64_t M, int32_t N) {
    DzShape s;
    // As wide as leaves few threads past the row's end.
    const int32_t vectors = (N + 7) / 8;
    s.tx_log = 5;
    while (s.tx_log > 3 && ((vectors + (1 << s.tx_log) - 1) >> s.tx_log << s.tx_log) >
                               vectors + vectors / 8)
        --s.tx_log;
    s.rows = 4 * (256 >> s.tx_log);
    while ((M + s.rows - 1) / s.rows > 1024) s.rows *= 2;
    s.blocks = (M + s.rows - 1) / s.rows;
    return s;
}

template <class D, class X>
hipError_t launch_dz_typed(const vcsr_linear_grad_args& a, X* dz, int64_t lddz, float* part,
                           hipStream_t st) {
    const DzShape s = dz_shape(a.M, a.N);
    const int cols = 8 << s.tx_log;
    const dim3 grid((unsigned)(((int64_t)a.N + cols - 1) / cols), (unsigned)s.blocks);
    switch (a.act) {
        case VCSR_ACT_RELU:
            dz_kernel<D, X, VCSR_ACT_RELU><<<grid, 256, 0, st>>>(a, dz, lddz, part, s.rows, s.tx_log);
            break;
        case VCSR_ACT_GELU:
            dz_kernel<D, X, VCSR_ACT_GELU><<<grid, 256, 0, st>>>(a, dz, lddz, part, s.rows, s.tx_log);
            break;
        case VCSR_ACT_SILU:
            dz_kernel<D, X, VCSR_ACT_SILU><<<grid, 256, 0, st>>>(a, dz, lddz, part, s.rows, s.tx_log);
            break;
        default:
            dz_kernel<D, X, VCSR_ACT_NONE><<<grid, 256, 0, st>>>(a, dz, lddz, part, s.rows, s.tx_log);
    }
    return hipGetLastError();
}

__global__ __launch_bounds__(256) void zero_kernel(uint8_t* p, int64_t bytes) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    for (int k = 0; k < 4; ++k)
        if (i + k < bytes) p[i + k] = 0;
}

}  // namespace

hipError_t launch_sum_rows(const float* part, int32_t P, int32_t C, int64_t ld, float* out,
                           hipStream_t st) {
    sum_rows_kernel<<<(unsigned)(((int64_t)C + 15) / 16), 1024, 0, st>>>(part, P, C, ld, out);
    return hipGetLastError();
}

int32_t dz_row_blocks(int64_t M, int32_t N) { return (int32_t)dz_shape(M, N).blocks; }

hipError_t launch_dz(const vcsr_linear_grad_args& a, void* dz, int64_t lddz, float* part,
                     hipStream_t st) {
    if (a.y_type == VCSR_F32)
        return a.x_type == VCSR_F32
                   ? launch_dz_typed<float, float>(a, (float*)dz, lddz, part, st)
                   : launch_dz_typed<float, bf16>(a, (bf16*)dz, lddz, part, st);
    return a.x_type == VCSR_F32 ? launch_dz_typed<bf16, float>(a, (float*)dz, lddz, part, st)
                                : launch_dz_typed<bf16, bf16>(a, (bf16*)dz, lddz, part, st);
}

hipError_t launch_zero(void* p, int64_t bytes, hipStream_t st) {
    if (bytes <= 0) return hipSuccess;
    zero_kernel<<<(unsigned)((bytes + 1023) / 1024), 256, 0, st>>>((uint8_t*)p, bytes);
    return hipGetLastError();
}

}  // namespace vcsr
