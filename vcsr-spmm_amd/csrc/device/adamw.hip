// adamw.hip - one AdamW step over all tensors of a plan in one launch.
//
// A block takes a chunk of 4096 values of one tensor, found through a table
// {tensor, first value / 4096} built with the plan.  A wave goes through the
// chunk's blocks of 256 values, four consecutive values a lane, so an 8-bit
// state's block maximum is one reduction over the wave and each state byte
// moves as part of a 4-byte word.  Everything is read and written once; bound
// by memory.  The arithmetic is FP32 with each operation rounded on its own
// (no fused multiply-adds), in the order of the header's formula, so a step
// does not depend on how the compiler contracts it.
#include "dense.hpp"

namespace vcsr {
namespace {

#pragma clang fp contract(off)

constexpr int kWaves = 4;

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const float y = __shfl_xor(x, m);
        x = x > y || x != x ? x : y;  // keeps a NaN
    }
    return x;
}
__device__ __forceinline__ float scale_of(float top) {
    top = wave_max(top);
    return (top < 1e-30f ? 1e-30f : top) / 448.f;
}
__device__ __forceinline__ float abs_max(float a, float b) {
    a = __builtin_fabsf(a);
    return a > b || a != a ? a : b;
}

// n values of a lane's four at p as a word of codes.
__device__ __forceinline__ uint32_t load_codes(const void* base, int64_t at, int n) {
    const uint8_t* p = (const uint8_t*)base + at;
    if (n >= 4) {
        const Mem<uint8_t, 4> m = *(const Mem<uint8_t, 4>*)p;
        uint32_t w;
        __builtin_memcpy(&w, &m, 4);
        return w;
    }
    uint32_t w = 0;
    for (int i = 0; i < 3; ++i)
        if (i < n) w |= (uint32_t)p[i] << (8 * i);
    return w;
}
__device__ __forceinline__ void store_codes(void* base, int64_t at, int n, uint32_t w) {
    uint8_t* p = (uint8_t*)base + at;
    if (n >= 4) {
        Mem<uint8_t, 4> m;
        __builtin_memcpy(&m, &w, 4);
        *(Mem<uint8_t, 4>*)p = m;
    } else {
        for (int i = 0; i < 3; ++i)
            if (i < n) p[i] = (uint8_t)(w >> (8 * i));
    }
}

template <bool F8>
__device__ __forceinline__ void step_block(const vcsr_adamw_tensor& t, const AdamwStep& s,
                                           int64_t at, int n) {
    const int lane = threadIdx.x & 63;
    float p[4], g[4], m[4], v[4];
    const int64_t block = at / kAdamwBlock;  // the same in every lane of the wave
    at += 4 * lane;
    n -= 4 * lane;
    if (n < 0) n = 0;
    load_vec(t.param + at, n, p);
    if (t.grad_type == VCSR_BF16)
        load_vec((const bf16*)t.grad + at, n, g);
    else
        load_vec((const float*)t.grad + at, n, g);
    if (F8) {
        const uint32_t mq = load_codes(t.m, at, n), vq = load_codes(t.v, at, n);
        const float ms = t.m_scale[block], vs = t.v_scale[block];
        m[0] = fp8_to_f32<0>(mq) * ms;
        m[1] = fp8_to_f32<1>(mq) * ms;
        m[2] = fp8_to_f32<2>(mq) * ms;
        m[3] = fp8_to_f32<3>(mq) * ms;
        v[0] = fp8_to_f32<0>(vq) * vs;
        v[1] = fp8_to_f32<1>(vq) * vs;
        v[2] = fp8_to_f32<2>(vq) * vs;
        v[3] = fp8_to_f32<3>(vq) * vs;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v[i] * v[i];
    } else {
        load_vec((const float*)t.m + at, n, m);
        load_vec((const float*)t.v + at, n, v);
    }
    const float keep = (float)(1.0 - s.lr * t.weight_decay);
    float root[4], m_top = 0.f, v_top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float gi = g[i] * s.grad_scale;
        m[i] = m[i] * s.beta1 + gi * s.one_minus_beta1;
        v[i] = v[i] * s.beta2 + (gi * gi) * s.one_minus_beta2;
        root[i] = __builtin_sqrtf(v[i]);
        p[i] = p[i] * keep - s.lr_over_bias1 * (m[i] / (root[i] * s.inv_root_bias2 + s.eps));
        m_top = abs_max(m[i], m_top);
        v_top = abs_max(root[i], v_top);
    }
    if (F8) {
        const float ms = scale_of(m_top), vs = scale_of(v_top);
        if (lane == 0) {
            t.m_scale[block] = ms;
            t.v_scale[block] = vs;
        }
        const uint32_t mq = fp8x4(m[0] / ms, m[1] / ms, m[2] / ms, m[3] / ms);
        uint32_t vq = fp8x4(root[0] / vs, root[1] / vs, root[2] / vs, root[3] / vs);
#pragma unroll
        for (int i = 0; i < 4; ++i)  // a nonzero root never gets the code of zero
            if (root[i] > 0.f && (vq >> (8 * i) & 0x7fu) == 0) vq |= 1u << (8 * i);
        store_codes(t.m, at, n, mq);
        store_codes(t.v, at, n, vq);
    } else {
        store_vec((float*)t.m + at, n, m);
        store_vec((float*)t.v + at, n, v);
    }
    store_vec(t.param + at, n, p);
    if (t.copy) store_vec((bf16*)t.copy + at, n, p);
}

__global__ __launch_bounds__(64 * kWaves) void adamw_kernel(const vcsr_adamw_tensor* tensors,
                                                            const int2* chunks, AdamwStep s) {
    const int2 c = chunks[blockIdx.x];
    const vcsr_adamw_tensor t = tensors[c.x];
    const int64_t first = (int64_t)c.y * kAdamwChunk;
    const int64_t end = first + kAdamwChunk < t.n ? first + kAdamwChunk : t.n;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    for (int64_t at = first + wave * kAdamwBlock; at < end; at += kWaves * kAdamwBlock) {
        const int n = end - at < kAdamwBlock ? (int)(end - at) : kAdamwBlock;
        if (t.state_type == VCSR_FP8)
            step_block<true>(t, s, at, n);
        else
            step_block<false>(t, s, at, n);
    }
}

}  // namespace

hipError_t launch_adamw(const vcsr_adamw_tensor* tensors, const int2* chunks, int32_t n_chunks,
                        const AdamwStep& s, hipStream_t st) {
    if (n_chunks <= 0) return hipSuccess;
    adamw_kernel<<<(unsigned)n_chunks, 64 * kWaves, 0, st>>>(tensors, chunks, s);
    return hipGetLastError();
}

}  // namespace vcsr
