// dense.hpp - the dense operators' internal interface: 16-byte vectors of
// FP32, bf16 and e4m3 values at any alignment, and the launchers of
// rmsnorm.hip, linear*.hip, colsum.hip and adamw.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../../include/vcsr_spmm.h"

namespace vcsr {

typedef __bf16 bf16;
struct fp8 {  // one e4m3 code
    uint8_t bits;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// N values of T as they lie in memory, at the alignment of T alone: gfx950
// loads and stores up to 16 bytes at any byte address.
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T) < 4 ? sizeof(T) : 4))) Mem {
    T v[N];
};

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ float to_f32<bf16>(bf16 x) {
    return (float)x;
}

// The codes of four values, nearest even (a magnitude past 464 or a NaN gives
// e4m3's NaN).
__device__ __forceinline__ uint32_t fp8x4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
template <int B>
__device__ __forceinline__ float fp8_to_f32(uint32_t word) {
    return __builtin_amdgcn_cvt_f32_fp8((int)word, B);
}

// n <= N values of p into v, zeros behind them.
template <class T, int N>
__device__ __forceinline__ void load_vec(const T* p, int n, float (&v)[N]) {
    if (n >= N) {
        const Mem<T, N> m = *(const Mem<T, N>*)p;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_f32(m.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
    }
}
// The same for the values [c, c + N) of a row of C >= N values, without branches
// that would keep loads from being under way together: past the row's end, the
// row's last N values moved down (none for c >= C).
template <class T, int N>
__device__ __forceinline__ void load_tail(const T* row, int c, int C, float (&v)[N]) {
    const int back = c + N > C ? c + N - C : 0;
    const Mem<T, N> m = *(const Mem<T, N>*)(row + (back < N ? c - back : 0));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(m.v[i]);
#pragma unroll
    for (int s = 1; s < N; s <<= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float next = i + s < N ? v[i + s < N ? i + s : i] : 0.f;
            v[i] = back & s ? next : v[i];
        }
    if (back >= N)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.f;
}
template <class T, int N>
__device__ __forceinline__ void load_full(const T* p, float (&v)[N]) {
    const Mem<T, N> m = *(const Mem<T, N>*)p;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(m.v[i]);
}
// The first n <= N values of v to p, rounded to nearest even.
template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, int n, const float (&v)[N]) {
    if (n >= N) {
        Mem<T, N> m;
#pragma unroll
        for (int i = 0; i < N; ++i) m.v[i] = (T)v[i];
        *(Mem<T, N>*)p = m;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}
template <int N>
__device__ __forceinline__ void store_vec(fp8* p, int n, const float (&v)[N]) {
    static_assert(N % 4 == 0, "whole words");
    Mem<uint8_t, N> m;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const uint32_t w = fp8x4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        __builtin_memcpy(&m.v[i], &w, 4);
    }
    if (n >= N) {
        *(Mem<uint8_t, N>*)p = m;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i].bits = m.v[i];
    }
}

// act(z) and act'(z) in FP32.  gelu's 0.5 (1 + tanh u) is 1 / (1 + exp(-2u));
// the exponential is the hardware's base-2 one, whose relative error (some
// 2^-23 times the exponent) stays below FP32's own rounding of z + bias where
// the result is not negligible.
__device__ __forceinline__ float sigmoid_f32(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * x));
}
constexpr float kGelu2 = 1.5957691216f;  // 2 sqrt(2 / pi)
template <int ACT>
__device__ __forceinline__ float act_f32(float z) {
    if (ACT == VCSR_ACT_RELU) return z < 0.f ? 0.f : z;  // a NaN stays one
    if (ACT == VCSR_ACT_GELU)  // -log2(e) kGelu2 (z + 0.044715 z^3) in three operations
        return z * __builtin_amdgcn_rcpf(
                       1.f + __builtin_amdgcn_exp2f(
                                 z * __builtin_fmaf(z * z, -1.44269504f * kGelu2 * 0.044715f,
                                                    -1.44269504f * kGelu2)));
    if (ACT == VCSR_ACT_SILU) return z * sigmoid_f32(z);
    return z;
}
template <int ACT>
__device__ __forceinline__ float act_grad_f32(float z) {
    if (ACT == VCSR_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == VCSR_ACT_GELU) {
        const float p = sigmoid_f32(kGelu2 * (z + 0.044715f * z * z * z));
        // Where z^2 passes FP32's range, p (1 - p) is zero and stays the product: z^2 is
        // held at 2^80 there (fmin would take that for a NaN too, but p then is one).
        const float z2 = __builtin_fminf(z * z, 0x1p80f);
        return p + z * p * (1.f - p) * kGelu2 * (1.f + 0.134145f * z2);
    }
    if (ACT == VCSR_ACT_SILU) {
        const float p = sigmoid_f32(z);
        return p * (1.f + z * (1.f - p));
    }
    return 1.f;
}
// act by a runtime (wave-uniform) choice.
__device__ __forceinline__ float act_f32(int act, float z) {
    switch (act) {
        case VCSR_ACT_RELU: return act_f32<VCSR_ACT_RELU>(z);
        case VCSR_ACT_GELU: return act_f32<VCSR_ACT_GELU>(z);
        case VCSR_ACT_SILU: return act_f32<VCSR_ACT_SILU>(z);
        default: return z;
    }
}

// ------------------------------------------------------------- rmsnorm.hip
// The arguments are checked, and strides of 0 resolved, by the caller.
hipError_t launch_rmsnorm(const vcsr_rmsnorm_args& a, hipStream_t st);
hipError_t launch_rmsnorm_grad(const vcsr_rmsnorm_grad_args& a, hipStream_t st);
size_t rmsnorm_grad_workspace(const vcsr_rmsnorm_grad_args& a);

// -------------------------------------------------------------- colsum.hip
// out[c] = sum over p < P of part[p * ld + c] for c < C, in a fixed order.
hipError_t launch_sum_rows(const float* part, int32_t P, int32_t C, int64_t ld, float* out,
                           hipStream_t st);
// dz = dy * act'(z) in x_type (dz may be NULL) and, for each block of
// dz_row_blocks(M, N, type of dy), the sums of its rows of dz in `part` (ld N; may be NULL).
hipError_t launch_dz(const vcsr_linear_grad_args& a, void* dz, int64_t lddz, float* part,
                     hipStream_t st);
int32_t dz_row_blocks(int64_t M, int32_t N, int32_t dy_type);
// Zeros in `rows` rows of `bytes` bytes, `ld` bytes apart (all even, as FP32 and bf16
// matrices have them), by a kernel.
hipError_t launch_zero(void* p, int64_t ld, int64_t rows, int64_t bytes, hipStream_t st);

// ------------------------------------------------------------ linear*.hip
// out[i][j] = epilogue(sum_k P(i, k) Q(j, k)).  An operand lies by rows (k
// contiguous: P(i, k) = p[i * ldp + k]) or by columns (i contiguous: P(i, k) =
// p[k * ldp + i]).  The epilogue adds bias[j], writes z, applies act, adds the
// residual and writes out, all of `out_type`; scales belong to fp8 operands.
struct Gemm {
    int64_t I = 0, R = 0;  // rows of out, length of the sum
    int32_t J = 0;         // columns of out
    bool p_cols = false, q_cols = false;
    int32_t type = VCSR_F32, out_type = VCSR_F32, act = VCSR_ACT_NONE;
    const void *p = nullptr, *q = nullptr;
    int64_t ldp = 0, ldq = 0;
    const float *p_scale = nullptr, *q_scale = nullptr, *bias = nullptr;
    const void* residual = nullptr;
    int64_t ldr = 0;
    void* z = nullptr;
    int64_t ldz = 0;
    void* out = nullptr;
    int64_t ldo = 0;
    float* part = nullptr;  // partial sums of a split product (gemm_workspace bytes)
};
hipError_t launch_gemm(const Gemm& g, hipStream_t st);
// Throws VCSR_ERANGE for more tiles than a launch has blocks, as the pair's does.
size_t gemm_workspace(const Gemm& g);
// Partial rows of C columns still to be added up (none for P = 0).
struct RowSum {
    const float* part = nullptr;
    float* out = nullptr;
    int32_t P = 0, C = 0;
};
// dx and dw of one linear layer, in one launch where that is faster, and dbias.
hipError_t launch_gemm_pair(const Gemm& dw, const Gemm& dx, const RowSum& bias, hipStream_t st);
size_t gemm_pair_workspace(const Gemm& dw, const Gemm& dx);
// What a product's launch does: square tiles (16: the kernel for few rows), the
// splits of the sum, of `steps` steps of 128 bytes each (each writes partial sums),
// and how many of its rows (the rest are a product of their own).
struct GemmPlan {
    int tile;
    int stages;  // steps that have room in LDS
    int32_t splits;
    int64_t steps;
    int64_t rows;
};
// dw's and dx's; `together`: in one launch.
struct PairPlan {
    bool together;
    GemmPlan dw, dx;
};
GemmPlan gemm_plan(const Gemm& g);
PairPlan gemm_pair_plan(const Gemm& dw, const Gemm& dx);
// For tests: the calling thread's products take this tile, splits and (where `rows`
// is less than a product's) division of rows, as far as a product has them, and pairs
// go together or not; tile 0 ends it.
void force_plan(const GemmPlan& p, bool together);

hipError_t launch_gemm_f32(const Gemm& g, const GemmPlan& p, hipStream_t st);
hipError_t launch_gemm_bf16(const Gemm& g, const GemmPlan& p, hipStream_t st);
hipError_t launch_pair_f32(const Gemm& dw, const GemmPlan& p, const Gemm& dx, const GemmPlan& q,
                           const RowSum& bias, hipStream_t st);
hipError_t launch_pair_bf16(const Gemm& dw, const GemmPlan& p, const Gemm& dx, const GemmPlan& q,
                            const RowSum& bias, hipStream_t st);
hipError_t launch_gemm_fp8(const Gemm& g, const GemmPlan& p, hipStream_t st);

// --------------------------------------------------------------- adamw.hip
// One chunk of a tensor is kAdamwChunk values, a block's work.
constexpr int32_t kAdamwBlock = 256;
constexpr int32_t kAdamwChunk = 2048;
struct AdamwStep {  // a step's constants, rounded once from 64 bits
    float beta1, one_minus_beta1, beta2, one_minus_beta2, lr_over_bias1, inv_root_bias2, eps,
        grad_scale;
    double lr;
};
hipError_t launch_adamw(const vcsr_adamw_tensor* tensors, const int2* chunks, int32_t n_chunks,
                        const AdamwStep& s, hipStream_t st);

}  // namespace vcsr
