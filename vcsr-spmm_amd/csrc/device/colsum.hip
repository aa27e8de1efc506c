// colsum.hip - what the gradients sum over rows, in a fixed order: the partial
// rows of dweight and dbias, and dz = dy * act'(z) with the sums of its rows.
#include "dense.hpp"

namespace vcsr {
namespace {

// 32 columns a block, 32 threads a column: each adds every 32nd partial row,
// then LDS adds the threads in order.
__global__ __launch_bounds__(1024) void sum_rows_kernel(const float* part, int32_t P, int32_t C,
                                                        int64_t ld, float* out) {
    __shared__ float lds[32][33];
    const int col = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + col;
    float t = 0.f;
    if (c < C)
        for (int32_t p = grp; p < P; p += 32) t += part[(int64_t)p * ld + c];
    lds[grp][col] = t;
    __syncthreads();
    if (grp == 0 && c < C) {
        t = 0.f;
#pragma unroll
        for (int g = 0; g < 32; ++g) t += lds[g][col];
        out[c] = t;
    }
}

// A block takes kDzRows rows of 256 columns: 32 threads of 8 columns, 8 rows at
// a time.  Bound by memory: dy and z read once, dz written once.
constexpr int kDzRows = 64;

template <class D, class X>
__global__ __launch_bounds__(256) void dz_kernel(vcsr_linear_grad_args a, X* dz, int64_t lddz,
                                                 float* part, int64_t rows_per_block) {
    __shared__ float lds[8][256];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 256 + tx * 8;
    const int n = c >= a.N ? 0 : a.N - c < 8 ? (int)(a.N - c) : 8;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const int64_t first = (int64_t)blockIdx.y * rows_per_block;
    const int64_t last = first + rows_per_block < a.M ? first + rows_per_block : a.M;
    if (n > 0)
        for (int64_t m = first + ty; m < last; m += 8) {
            float d[8];
            load_vec((const D*)a.dy + m * a.lddy + c, n, d);
            if (a.act != VCSR_ACT_NONE) {
                float z[8];
                load_vec((const D*)a.z + m * a.ldz + c, n, z);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] *= act_grad_f32(a.act, z[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += i < n ? d[i] : 0.f;
            if (dz) store_vec(dz + m * lddz + c, n, d);
        }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) lds[ty][tx * 8 + i] = sum[i];
    __syncthreads();
    const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (col < a.N) {
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < 8; ++g) t += lds[g][threadIdx.x];
        part[(int64_t)blockIdx.y * a.N + col] = t;
    }
}

int64_t dz_rows_per_block(int64_t M) {
    // At most 4096 blocks of rows, whose partial rows stay small beside dz.
    int64_t rows = kDzRows;
    while ((M + rows - 1) / rows > 4096) rows *= 2;
    return rows;
}

__global__ __launch_bounds__(256) void zero_kernel(uint8_t* p, int64_t bytes) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    for (int k = 0; k < 4; ++k)
        if (i + k < bytes) p[i + k] = 0;
}

}  // namespace

hipError_t launch_sum_rows(const float* part, int32_t P, int32_t C, int64_t ld, float* out,
                           hipStream_t st) {
    sum_rows_kernel<<<(unsigned)((C + 31) / 32), 1024, 0, st>>>(part, P, C, ld, out);
    return hipGetLastError();
}

int32_t dz_row_blocks(int64_t M, int32_t N) {
    (void)N;
    const int64_t rows = dz_rows_per_block(M);
    return (int32_t)((M + rows - 1) / rows);
}

hipError_t launch_dz(const vcsr_linear_grad_args& a, void* dz, int64_t lddz, float* part,
                     hipStream_t st) {
    const int64_t rows = dz_rows_per_block(a.M);
    const dim3 grid((unsigned)(((int64_t)a.N + 255) / 256), (unsigned)((a.M + rows - 1) / rows));
    if (a.y_type == VCSR_F32) {
        if (a.x_type == VCSR_F32)
            dz_kernel<float, float><<<grid, 256, 0, st>>>(a, (float*)dz, lddz, part, rows);
        else
            dz_kernel<float, bf16><<<grid, 256, 0, st>>>(a, (bf16*)dz, lddz, part, rows);
    } else {
        if (a.x_type == VCSR_F32)
            dz_kernel<bf16, float><<<grid, 256, 0, st>>>(a, (float*)dz, lddz, part, rows);
        else
            dz_kernel<bf16, bf16><<<grid, 256, 0, st>>>(a, (bf16*)dz, lddz, part, rows);
    }
    return hipGetLastError();
}

hipError_t launch_zero(void* p, int64_t bytes, hipStream_t st) {
    if (bytes <= 0) return hipSuccess;
    zero_kernel<<<(unsigned)((bytes + 1023) / 1024), 256, 0, st>>>((uint8_t*)p, bytes);
    return hipGetLastError();
}

}  // namespace vcsr
