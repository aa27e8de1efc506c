// norm_rows.hpp - what the norms (rmsnorm.hip, layernorm.hip) share: rows held in
// registers, sums over a row's lanes and waves, and the shapes that rows take.
#pragma once

#include <type_traits>

#include "dense.hpp"
#include "launch.hpp"

namespace vcsr {
namespace norm {

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

// One sum, two, or a maximum, with a barrier each; calls that follow one another
// take LDS of their own.
template <int WAVES>
__device__ __forceinline__ float sum_waves(float* lds, float x) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) x += lds[i];
    return x;
}
template <int WAVES>
__device__ __forceinline__ void sum_waves(float* lds, float& x, float& y) {
    if ((threadIdx.x & 63) == 0) {
        lds[threadIdx.x >> 6] = x;
        lds[WAVES + (threadIdx.x >> 6)] = y;
    }
    __syncthreads();
    x = lds[0];
    y = lds[WAVES];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
        x += lds[i];
        y += lds[WAVES + i];
    }
}
template <int WAVES>
__device__ __forceinline__ float top_waves(float* lds, float top) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
    __syncthreads();
    top = lds[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) top = max_nan(top, lds[i]);
    return top;
}
__device__ __forceinline__ float top_lanes(int lanes, float x) {
    for (int m = 1; m < lanes; m <<= 1) x = max_nan(x, __shfl_xor(x, m));
    return x;
}

// Scale of a row whose largest |y| is `top`.
template <class Y>
__device__ __forceinline__ float row_factor(float top, float* y_scale, int64_t row, bool writes) {
    if (sizeof(Y) != 1) return 1.f;
    const float a = top < 1e-30f ? 1e-30f : top;  // a NaN stays one
    const float scale = a / 448.f;
    if (writes) y_scale[row] = scale;
    return scale;
}

// A lane's NV vectors of a row of C >= V values: all but the last are whole.
template <class T, int NV, int V>
__device__ __forceinline__ void load_row(const T* row, int lane, int stride, int C,
                                         float (&v)[NV][V]) {
#pragma unroll
    for (int k = 0; k + 1 < NV; ++k) load_full(row + (k * stride + lane) * V, v[k]);
    load_tail(row, ((NV - 1) * stride + lane) * V, C, v[NV - 1]);
}
template <class T, int NV, int V>
__device__ __forceinline__ void store_row(T* row, int lane, int stride, int C,
                                          const float (&v)[NV][V]) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int c = (k * stride + lane) * V;
        if (k + 1 < NV)
            store_vec(row + c, V, v[k]);
        else if (c < C)
            store_vec(row + c, C - c, v[k]);
    }
}

// The same as it lies in memory, so that a row can be under way while the one before it is
// worked on.
template <class T, int NV, int V>
struct RawRow {
    Mem<T, V> m[NV];
    __device__ __forceinline__ static int back_of(int lane, int stride, int C) {
        const int c = ((NV - 1) * stride + lane) * V;
        return c + V > C ? c + V - C : 0;
    }
    __device__ __forceinline__ void load(const T* row, int lane, int stride, int C) {
#pragma unroll
        for (int k = 0; k + 1 < NV; ++k) m[k] = *(const Mem<T, V>*)(row + (k * stride + lane) * V);
        const int back = back_of(lane, stride, C);
        m[NV - 1] = *(const Mem<T, V>*)(row +
                                        (back < V ? ((NV - 1) * stride + lane) * V - back : 0));
    }
    // Its values, zeros past the row's end.
    __device__ __forceinline__ void get(int lane, int stride, int C, float (&v)[NV][V]) const {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) v[k][i] = to_f32(m[k].v[i]);
        const int back = back_of(lane, stride, C);
        if (C % V == 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[NV - 1][i] = back ? 0.f : v[NV - 1][i];
            return;
        }
#pragma unroll
        for (int s = 1; s < V; s <<= 1)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float next = i + s < V ? v[NV - 1][i + s < V ? i + s : i] : 0.f;
                v[NV - 1][i] = back & s ? next : v[NV - 1][i];
            }
#pragma unroll
        for (int i = 0; i < V; ++i) v[NV - 1][i] = back >= V ? 0.f : v[NV - 1][i];
    }
};

// A launch has fewer than 2^32 threads: more rows than that, at `threads` each, go
// in several.  launch(first, count) takes whole blocks of at most 256 rows.
template <class F>
void by_rows(int64_t M, int64_t threads, F&& launch) {
    const int64_t most = ((((int64_t)1 << 32) - 1) / threads) & ~(int64_t)255;
    for (int64_t first = 0; first < M; first += most)
        launch(first, M - first < most ? M - first : most);
}
inline int next_pow2(int n) {
    int p = 1;
    while (p < n) p <<= 1;
    return p;
}

// Waves of a row and vectors of a lane: the fewest idle vectors (2050 bf16 are 257
// vectors: 3 x 128 rather than 2 x 256), and where that leaves a choice two vectors
// a lane, whose loads are under way together (4096 bf16: 4 waves of 2 vectors 166
// us at 32768 rows, 8 waves of 1 206).  nv <= 2048.
struct RowShape {
    int wpr, nv;
};
inline RowShape row_shape(int64_t nv, int most_nv) {
    RowShape best{8, 4};
    int64_t slots = 1 << 30;
    for (int k : {2, 3, 1, 4})
        for (int wpr = 1; wpr <= 8; wpr <<= 1) {
            const int64_t s = (int64_t)wpr * 64 * k;
            if (s >= nv && s < slots && (k <= most_nv || s > 1536)) {
                slots = s;
                best = RowShape{wpr, k};
            }
        }
    return best;
}

// f.operator()<WPR, NV>() of a shape.
template <class F>
void with_shape(RowShape s, F&& f) {
    auto by_nv = [&](auto wpr) {
        constexpr int W = decltype(wpr)::value;
        switch (s.nv) {
            case 1: return f(std::integral_constant<int, W>{}, std::integral_constant<int, 1>{});
            case 2: return f(std::integral_constant<int, W>{}, std::integral_constant<int, 2>{});
            case 3: return f(std::integral_constant<int, W>{}, std::integral_constant<int, 3>{});
            default: return f(std::integral_constant<int, W>{}, std::integral_constant<int, 4>{});
        }
    };
    switch (s.wpr) {
        case 1: return by_nv(std::integral_constant<int, 1>{});
        case 2: return by_nv(std::integral_constant<int, 2>{});
        case 4: return by_nv(std::integral_constant<int, 4>{});
        default: return by_nv(std::integral_constant<int, 8>{});
    }
}

}  // namespace norm
}  // namespace vcsr
