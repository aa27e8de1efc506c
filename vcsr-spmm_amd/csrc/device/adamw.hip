// adamw.hip - one AdamW step over all tensors of a plan in one launch.
//
// A block takes a chunk of 2048 values of one tensor, found through a table
// {tensor, first value / 2048} built with the plan.  A wave takes two blocks of 256
// values of it, four consecutive values a lane, so an 8-bit state's block maximum is one
// reduction over the wave and each state byte moves as part of a 4-byte word; the
// loads of both blocks go out together, without branches between them where the
// blocks are whole.  Everything is read and written once; bound by memory: 201M
// values with 8-bit states, bf16 gradients and copies 611 to 637 us (5.1 to 5.3 TB/s),
// 1.05M with FP32 states 7.2 us.  The arithmetic is FP32 with each operation rounded on its own (no fused
// multiply-adds), in the order of the header's formula, so a step does not depend
// on how the compiler contracts it.
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

// A lane's n <= 4 values of a block as a word of codes.
template <bool WHOLE>
__device__ __forceinline__ uint32_t load_codes(const void* base, int64_t at, int n) {
    const uint8_t* p = (const uint8_t*)base + at;
    if (WHOLE) {
        const Mem<uint8_t, 4> m = *(const Mem<uint8_t, 4>*)p;
        uint32_t w;
        __builtin_memcpy(&w, &m, 4);
        return w;
    }
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) w |= (uint32_t)p[i] << (8 * i);
    return w;
}
template <bool WHOLE>
__device__ __forceinline__ void store_codes(void* base, int64_t at, int n, uint32_t w) {
    uint8_t* p = (uint8_t*)base + at;
    if (WHOLE) {
        Mem<uint8_t, 4> m;
        __builtin_memcpy(&m, &w, 4);
        *(Mem<uint8_t, 4>*)p = m;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) p[i] = (uint8_t)(w >> (8 * i));
}
template <bool WHOLE, class T>
__device__ __forceinline__ void load4(const T* p, int n, float (&v)[4]) {
    if (WHOLE)
        load_full(p, v);
    else
        load_vec(p, n, v);
}
template <bool WHOLE, class T>
__device__ __forceinline__ void store4(T* p, int n, const float (&v)[4]) {
    store_vec(p, WHOLE ? 4 : n, v);
}
__device__ __forceinline__ void decode(uint32_t q, float scale, float (&v)[4]) {
    v[0] = fp8_to_f32<0>(q) * scale;
    v[1] = fp8_to_f32<1>(q) * scale;
    v[2] = fp8_to_f32<2>(q) * scale;
    v[3] = fp8_to_f32<3>(q) * scale;
}

// U blocks of 256 values from `first`, `stride` values apart, of which the last
// ends at `end` at the latest.
template <class G, bool F8, bool WHOLE, int U>
__device__ __forceinline__ void step_blocks(const vcsr_adamw_tensor& t, const AdamwStep& s,
                                            int64_t first, int64_t stride, int64_t end) {
    const int lane = threadIdx.x & 63;
    float p[U][4], g[U][4], m[U][4], v[U][4], ms[U], vs[U];
    uint32_t mq[U], vq[U];
    int n[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = first + u * stride + 4 * lane;
        n[u] = WHOLE || end - at > 4 ? 4 : end < at ? 0 : (int)(end - at);
        load4<WHOLE>(t.param + at, n[u], p[u]);
        load4<WHOLE>((const G*)t.grad + at, n[u], g[u]);
        if (F8) {
            const int64_t block = (first + u * stride) / kAdamwBlock;
            mq[u] = load_codes<WHOLE>(t.m, at, n[u]);
            vq[u] = load_codes<WHOLE>(t.v, at, n[u]);
            ms[u] = t.m_scale[block];
            vs[u] = t.v_scale[block];
        } else {
            load4<WHOLE>((const float*)t.m + at, n[u], m[u]);
            load4<WHOLE>((const float*)t.v + at, n[u], v[u]);
        }
    }
    const float keep = (float)(1.0 - s.lr * t.weight_decay);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = first + u * stride + 4 * lane;
        if (F8) {
            decode(mq[u], ms[u], m[u]);
            decode(vq[u], vs[u], v[u]);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[u][i] = v[u][i] * v[u][i];
        }
        float root[4], m_top = 0.f, v_top = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float gi = g[u][i] * s.grad_scale;
            m[u][i] = m[u][i] * s.beta1 + gi * s.one_minus_beta1;
            v[u][i] = v[u][i] * s.beta2 + (gi * gi) * s.one_minus_beta2;
            root[i] = __builtin_sqrtf(v[u][i]);
            p[u][i] = p[u][i] * keep -
                      s.lr_over_bias1 * (m[u][i] / (root[i] * s.inv_root_bias2 + s.eps));
            m_top = abs_max(m[u][i], m_top);
            v_top = abs_max(root[i], v_top);
        }
        if (F8) {
            const int64_t block = (first + u * stride) / kAdamwBlock;
            const float mx = scale_of(m_top), vx = scale_of(v_top);
            if (lane == 0) {
                t.m_scale[block] = mx;
                t.v_scale[block] = vx;
            }
            const uint32_t a = fp8x4(m[u][0] / mx, m[u][1] / mx, m[u][2] / mx, m[u][3] / mx);
            uint32_t b = fp8x4(root[0] / vx, root[1] / vx, root[2] / vx, root[3] / vx);
#pragma unroll
            for (int i = 0; i < 4; ++i)  // a nonzero root never gets the code of zero
                if (root[i] > 0.f && (b >> (8 * i) & 0x7fu) == 0) b |= 1u << (8 * i);
            store_codes<WHOLE>(t.m, at, n[u], a);
            store_codes<WHOLE>(t.v, at, n[u], b);
        } else {
            store4<WHOLE>((float*)t.m + at, n[u], m[u]);
            store4<WHOLE>((float*)t.v + at, n[u], v[u]);
        }
        store4<WHOLE>(t.param + at, n[u], p[u]);
        if (t.copy) store4<WHOLE>((bf16*)t.copy + at, n[u], p[u]);
    }
}

template <class G, bool F8>
__device__ __forceinline__ void step_chunk(const vcsr_adamw_tensor& t, const AdamwStep& s,
                                           int64_t first, int wave) {
    constexpr int64_t stride = kWaves * kAdamwBlock;
    const int64_t at = first + wave * kAdamwBlock;
    if (first + kAdamwChunk <= t.n) {
        step_blocks<G, F8, true, kAdamwChunk / (int)stride>(t, s, at, stride, t.n);
    } else {
        for (int64_t b = at; b < t.n && b < first + kAdamwChunk; b += stride)
            step_blocks<G, F8, false, 1>(t, s, b, stride, t.n);
    }
}

__global__ __launch_bounds__(64 * kWaves) void adamw_kernel(const vcsr_adamw_tensor* tensors,
                                                            const int2* chunks, AdamwStep s) {
    const int2 c = chunks[blockIdx.x];
    const vcsr_adamw_tensor t = tensors[c.x];
    const int64_t first = (int64_t)c.y * kAdamwChunk;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (t.state_type == VCSR_FP8) {
        if (t.grad_type == VCSR_BF16)
            step_chunk<bf16, true>(t, s, first, wave);
        else
            step_chunk<float, true>(t, s, first, wave);
    } else {
        if (t.grad_type == VCSR_BF16)
            step_chunk<bf16, false>(t, s, first, wave);
        else
            step_chunk<float, false>(t, s, first, wave);
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
