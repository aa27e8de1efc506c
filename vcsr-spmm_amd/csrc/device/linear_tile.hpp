// linear_tile.hpp - the dense product on the matrix cores, for linear_f32.hip,
// linear_bf16.hip and linear_fp8.hip.
//
// out[i][j] = epilogue(sum_k P(i, k) Q(j, k)).  A block computes a TI x TJ tile
// of out; its WI x WJ waves take equal parts.  The sum goes in steps of 128
// bytes of k: both operands' tiles go straight from memory to LDS, one to three
// steps ahead of the one that is multiplied, and a wave multiplies 16 x 16 blocks
// with v_mfma_f32_16x16x4_f32 or _16x16x32_bf16.
//
// What bounds it: big bf16 products the chip's power (8192 x 4096 x 8192 with gelu
// 444 to 473 us, 1.16 to 1.24 PFLOP/s, the matrix units busy 57% at 1.8 to 2.15 GHz),
// FP32 ones the matrix units (4096^3 130 TFLOP/s, a large library product 127 to 155),
// e4m3 ones widening (4096 x 8192 x 4096 176 us, 1.56 PFLOP/s), few rows the weight's
// read.
//
// LDS tiles are TI (or TJ) x 128 bytes in 16-byte granules:
//   by rows     row r at r * 128, granule g of its k at slot g ^ key(r);
//   by columns  k-row k at k * TI * size, granule c of its i at slot c ^ key(k).
// The keys spread the granules that 16 lanes read together over all banks.
// A lane of the matrix instruction holds row (lane & 15) and, of each step, k in
// 16-byte granules (lane >> 4) + 4 s; any assignment of k to lanes is right as
// long as both operands use it.
//
// The matrix instruction's rows are out's columns: a lane then holds 4
// consecutive j of one i.  Within 32 columns, row a of block b stands for
// column (a >> 2) * 8 + b * 4 + (a & 3), so that two blocks give a lane 8
// consecutive j, a 16-byte store of bf16.
#pragma once

#include "common.hpp"
#include "dense.hpp"

namespace vcsr {
namespace tile {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t lds_byte;

constexpr int kStepBytes = 128;
constexpr int64_t kCus = 256;  // compute units
// Bytes a buffer descriptor covers, and an offset past them.
constexpr int kRange = 0x7fffffff;
constexpr uint32_t kPast = 0x80000000u;

// Granule keys of tiles by rows, for 16 consecutive rows (P) and for the rows
// that a block of Q stands for.
__device__ __forceinline__ int key_p(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ int key_q(int r) { return ((r >> 1) & 1) | ((r >> 2) & 6); }
template <bool Q>
__device__ __forceinline__ int key_rows(int r) {
    return Q ? key_q(r) : key_p(r);
}
// Key of k-row k of a tile by columns with GRAN granules a k-row.  bf16: 16 lanes
// read 4 k-rows, of each two granules (P) or halves of four (Q).  FP32: four groups
// of 16 lanes read k-rows 4 apart, of each four granules in a row (P) or every
// second (Q), which these keys put on different banks (35% of the LDS cycles were
// conflicts with one key for both).  For bf16's Q, keys that spread the granules
// further made 128 x 128 tiles slower (8192 x 2048 x 4096: 179 against 156 us).
template <class T, int GRAN, bool Q>
__device__ __forceinline__ int key_cols(int k) {
    if (sizeof(T) == 2) return (((k & 3) | ((k >> 1) & 4)) << 1) & (GRAN - 1);
    const int q = (k >> 2) & 3;
    return Q ? (q & 1) | (q >> 1) << 3 : q << 2;
}

struct Operand {
    const uint8_t* p;
    int64_t ld;     // bytes
    int64_t n;      // rows of the operand (i or j)
    int64_t first;  // of the tile
    int64_t bytes;  // from p to the end of its last row
};

// v moved down by `bytes` (0 to 15), zeros behind.
__device__ __forceinline__ u32x4 shift_down(u32x4 v, int bytes) {
    if (bytes & 8) v = u32x4{v.z, v.w, 0, 0};
    if (bytes & 4) v = u32x4{v.y, v.z, v.w, 0};
    const uint32_t b = bytes & 3;
    return u32x4{__builtin_amdgcn_alignbyte(v.y, v.x, b), __builtin_amdgcn_alignbyte(v.z, v.y, b),
                 __builtin_amdgcn_alignbyte(v.w, v.z, b), __builtin_amdgcn_alignbyte(0, v.w, b)};
}

// One operand's tile loader: NT threads bring ROWS x 128 bytes.  `GR` granules a
// thread; granule e = it * NT + tid of the tile lies at e * 16 in LDS.  SEG > 0:
// the tile's rows are runs of SEG rows, 2 * SEG apart.
template <class T, int ROWS, int NT, bool COLS, bool Q, int SEG = 0>
struct Loader {
    static constexpr int GR = ROWS * 8 / NT;
    static constexpr int EPG = 16 / (int)sizeof(T);
    static constexpr int BK = kStepBytes / (int)sizeof(T);
    static constexpr int KGRAN = ROWS * (int)sizeof(T) / 16;  // granules of a k-row (by columns)
    static_assert(ROWS * 8 % NT == 0, "whole granules");

    // k (relative to the step) and row of the first element of granule e.
    __device__ __forceinline__ static void place(int e, int& row, int& k) {
        if (COLS) {
            k = e / KGRAN;
            row = ((e % KGRAN) ^ key_cols<T, KGRAN, Q>(k)) * EPG;
        } else {
            row = e >> 3;
            k = ((e & 7) ^ key_rows<Q>(row)) * EPG;
        }
        if (SEG) row += row / (SEG ? SEG : 1) * SEG;
    }

    // Through registers, for a step that ends inside its 128 bytes or with the
    // operand: elements past the operand's rows or past k_end are zeros.  A
    // granule that ends outside is read ending at the last element, and shifted;
    // rows shorter than a granule go element by element.
    __device__ __forceinline__ static void fetch(const Operand& o, int64_t k0, int64_t k_end,
                                                 uint8_t* lds) {
        const int64_t total = COLS ? o.n : k_end;  // elements of a run
        u32x4 v[GR];
#pragma unroll
        for (int it = 0; it < GR; ++it) {
            int row, k;
            place(it * NT + (int)threadIdx.x, row, k);
            const int64_t kk = k0 + k, r = o.first + row;
            const int64_t run = COLS ? kk : r, pos = COLS ? r : kk;
            const bool in = (COLS ? kk < k_end : r < o.n) && pos < total;
            v[it] = u32x4{0, 0, 0, 0};
            if (in && total >= EPG) {
                const int back = total - pos < EPG ? (int)(EPG - (total - pos)) : 0;
                const Mem<T, EPG> m =
                    *(const Mem<T, EPG>*)((const T*)(o.p + run * o.ld) + (pos - back));
                __builtin_memcpy(&v[it], &m, 16);
                v[it] = shift_down(v[it], back * (int)sizeof(T));
            }
        }
#pragma unroll
        for (int it = 0; it < GR; ++it)
            *(u32x4*)(lds + (it * NT + (int)threadIdx.x) * 16) = v[it];
        if (total >= EPG) return;
#pragma unroll 1
        for (int it = 0; it < GR; ++it) {
            int row, k;
            place(it * NT + (int)threadIdx.x, row, k);
            const int64_t kk = k0 + k, r = o.first + row;
            const int64_t run = COLS ? kk : r, pos = COLS ? r : kk;
            if (COLS ? kk >= k_end : r >= o.n) continue;
#pragma unroll 1
            for (int i = 0; pos + i < total; ++i)
                ((T*)(lds + (it * NT + (int)threadIdx.x) * 16))[i] =
                    ((const T*)(o.p + run * o.ld))[pos + i];
        }
    }
    // Straight to LDS, whole steps only.  The hardware takes any byte address and
    // checks the range dword by dword.  off: byte offset of each of the thread's
    // granules from the tile's first k.  By columns, a granule that crosses the
    // last i goes on into the next k-row: its sums go nowhere.
    __device__ __forceinline__ static void offsets(const Operand& o, uint32_t (&off)[GR]) {
#pragma unroll
        for (int it = 0; it < GR; ++it) {
            int row, k;
            place(it * NT + (int)threadIdx.x, row, k);
            if (COLS) {
                off[it] = o.first + row < o.n ? (uint32_t)(k * o.ld) + row * (int)sizeof(T) : kPast;
            } else {  // rows past the last one read it again, or zeros where the tile has none
                const int64_t last = o.n - 1 - o.first;
                off[it] = last < 0 ? kPast
                                   : (uint32_t)((row < last ? row : last) * o.ld) +
                                         k * (int)sizeof(T);
            }
        }
    }
    __device__ __forceinline__ static void copy(const Operand& o, const uint32_t (&off)[GR],
                                                int64_t k0, lds_byte* lds) {
        const int64_t at = COLS ? k0 * o.ld + o.first * (int64_t)sizeof(T)
                                : o.first * o.ld + k0 * (int64_t)sizeof(T);
        const int64_t left = o.bytes - at;  // the descriptor's range is unsigned: none is 0
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(o.p + at), 0, left < 0 ? 0 : left < kRange ? (int)left : kRange, 0x00020000);
        const int wave = uniform((int)(threadIdx.x >> 6));
#pragma unroll
        for (int it = 0; it < GR; ++it)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rsrc, (__attribute__((address_space(3))) void*)(lds + (it * NT + wave * 64) * 16),
                16, off[it], 0, 0, 0);
    }
};

// The operand block of one matrix step: 16 rows (of wave-tile block `b`, first
// row `r0` of the wave's part) and granule step s.
template <class T, int ROWS, bool COLS, bool Q>
struct Reader;

// Row of the tile that lane row a of block b stands for.
template <bool Q>
__device__ __forceinline__ int tile_row(int r0, int b, int a) {
    return Q ? r0 + (b >> 1) * 32 + (a >> 2) * 8 + (b & 1) * 4 + (a & 3) : r0 + b * 16 + a;
}

template <class T, int ROWS, bool Q>
struct Reader<T, ROWS, false, Q> {
    __device__ __forceinline__ static u32x4 get(const uint8_t* lds, int r0, int b, int s) {
        const int lane = threadIdx.x & 63;
        const int r = tile_row<Q>(r0, b, lane & 15);
        const int g = (lane >> 4) + 4 * s;
        return *(const u32x4*)(lds + r * kStepBytes + ((g ^ key_rows<Q>(r)) << 4));
    }
};
// bf16 by columns: the transposing read gives lane t of 16 lanes element t of 4
// k-rows (lane t addresses 4 consecutive i of k-row t / 4).
template <int ROWS, bool Q>
struct Reader<bf16, ROWS, true, Q> {
    __device__ __forceinline__ static u32x4 get(const uint8_t* lds, int r0, int b, int s) {
        constexpr int GRAN = ROWS * 2 / 16;
        const int lane = threadIdx.x & 63, t = lane & 15;
        const int col = tile_row<Q>(r0, b, (t & 3) * 4);  // 4 consecutive ones from here
        u32x2 half[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = s * 32 + (lane >> 4) * 8 + h * 4 + (t >> 2);
            const int at = k * ROWS * 2 + (((col >> 3) ^ key_cols<bf16, GRAN, Q>(k)) << 4) +
                           (col & 7) * 2;
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(lds + at));
            __builtin_memcpy(&half[h], &v, 8);
        }
        return u32x4{half[0].x, half[0].y, half[1].x, half[1].y};
    }
};
template <int ROWS, bool Q>
struct Reader<float, ROWS, true, Q> {
    __device__ __forceinline__ static u32x4 get(const uint8_t* lds, int r0, int b, int s) {
        constexpr int GRAN = ROWS * 4 / 16;
        const int lane = threadIdx.x & 63;
        const int col = tile_row<Q>(r0, b, lane & 15);
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = s * 16 + (lane >> 4) * 4 + j;
            const int at = k * ROWS * 4 + (((col >> 2) ^ key_cols<float, GRAN, Q>(k)) << 4) +
                           (col & 3) * 4;
            v[j] = *(const uint32_t*)(lds + at);
        }
        return v;
    }
};

// acc (rows: Q's block, columns: P's block) += Q P^T over the k of one granule.
template <class T>
__device__ __forceinline__ f32x4 mma(const u32x4& q, const u32x4& p, f32x4 acc);
template <>
__device__ __forceinline__ f32x4 mma<bf16>(const u32x4& q, const u32x4& p, f32x4 acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q),
                                                   __builtin_bit_cast(bf16x8, p), acc, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mma<float>(const u32x4& q, const u32x4& p, f32x4 acc) {
    const f32x4 a = __builtin_bit_cast(f32x4, q), b = __builtin_bit_cast(f32x4, p);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc, 0, 0, 0);
    return acc;
}
// e4m3: the values become bf16 exactly and go through the bf16 instruction,
// whose sums are FP32.  The e4m3 instructions (16x16x32 and 16x16x128) align
// their products to the largest and drop bits: up to 2^-11.6 of the largest product
// was measured over 128 random terms.  That is far more than FP32's rounding, and of
// the largest product, not of each: a sum of many small ones beside it loses them.
__device__ __forceinline__ void widen(const u32x4& v, bf16x8 (&o)[2]) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], 1.f, false);
        const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[i], 1.f, true);
        o[i >> 1][(i & 1) * 4 + 0] = a[0];
        o[i >> 1][(i & 1) * 4 + 1] = a[1];
        o[i >> 1][(i & 1) * 4 + 2] = b[0];
        o[i >> 1][(i & 1) * 4 + 3] = b[1];
    }
}
// One granule of each operand, as the matrix instruction takes it.
template <class T>
struct Frag {
    u32x4 v;
    __device__ __forceinline__ void set(const u32x4& x) { v = x; }
};
template <>
struct Frag<fp8> {
    bf16x8 v[2];
    __device__ __forceinline__ void set(const u32x4& x) { widen(x, v); }
};
template <class T>
__device__ __forceinline__ f32x4 mma(const Frag<T>& q, const Frag<T>& p, f32x4 acc) {
    return mma<T>(q.v, p.v, acc);
}
template <>
__device__ __forceinline__ f32x4 mma<fp8>(const Frag<fp8>& q, const Frag<fp8>& p, f32x4 acc) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q.v[h], p.v[h], acc, 0, 0, 0);
    return acc;
}

// The epilogue of N consecutive columns from j of row i: scales, bias, z, act,
// residual, out.
template <class O, int N>
__device__ __forceinline__ void finish(const Gemm& g, int64_t i, int j, float (&v)[N]) {
    if (g.p_scale) {
        const float ps = g.p_scale[i];
        float qs[N];
        load_vec(g.q_scale + j, N, qs);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] *= ps * qs[k];
    }
    if (g.bias) {
        float b[N];
        load_vec(g.bias + j, N, b);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += b[k];
    }
    if (g.z) store_vec((O*)g.z + i * g.ldz + j, N, v);
    if (g.act != VCSR_ACT_NONE) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = act_f32(g.act, v[k]);
    }
    if (g.residual) {
        float r[N];
        load_vec((const O*)g.residual + i * g.ldr + j, N, r);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += r[k];
    }
    store_vec((O*)g.out + i * g.ldo + j, N, v);
}
// 8 columns of a row, or the first n of them (the others are its last one again),
// with all loads under way together.
template <class T>
__device__ __forceinline__ void load_cols(const T* p, int n, float (&v)[8]) {
    if (n == 8) {
        load_full(p, v);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = to_f32(p[k < n ? k : n - 1]);
    }
}

// Row length of the partial sums: whole vectors of 8.
__host__ __device__ inline int64_t part_ld(int32_t J) { return ((int64_t)J + 7) / 8 * 8; }

// Waits and barriers that nothing is moved across.
__device__ __forceinline__ void barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// All but the N newest of the wave's loads have arrived (and its LDS writes).
template <int N>
__device__ __forceinline__ void wait_loads() {
    if (N == 0)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
constexpr int kAhead = 8;  // loads a wave of gemm_turns has under way at a wait

// Where block b of a launch works: tile and part of the sum.  Blocks of one XCD
// take neighbouring tiles, `band` columns of tiles at a time, so that those that
// run together share Q's rows and a few of P's in its L2.
struct Place {
    int64_t i0, j0;
    uint32_t split;
};
template <int TI, int TJ>
__device__ __forceinline__ Place place_of(const Gemm& g, uint32_t block, uint32_t blocks,
                                          uint32_t splits) {
    constexpr uint32_t kBand = 4;
    const uint32_t ti = (uint32_t)((g.I + TI - 1) / TI);
    const uint32_t tj = (uint32_t)(((int64_t)g.J + TJ - 1) / TJ);
    const uint32_t b = xcd_remap(block, blocks);
    const uint32_t split = b % splits, t = b / splits;
    const uint32_t band = t / (kBand * ti), in_band = t - band * (kBand * ti);
    const uint32_t width = tj - band * kBand < kBand ? tj - band * kBand : kBand;
    return Place{(int64_t)(in_band / width) * TI, (int64_t)(band * kBand + in_band % width) * TJ,
                 split};
}

template <class T>
__device__ __forceinline__ int64_t extent(int64_t n, int64_t r, int64_t ld, bool cols) {
    return ((cols ? r - 1 : n - 1) * ld + (cols ? n : r)) * (int64_t)sizeof(T);
}

// acc of a wave -> out.  Each wave turns its part round in its own LDS room, a
// few blocks of rows at a time, so that its lanes go along rows of out: 8
// consecutive columns a lane, the same ones in every row.  (Stores straight from
// the matrix layout write half lines: 70 against 65 us for 8192 x 8192 at K = 128.)
// PLAIN: out alone, as the gradients need it.  WHOLE: all of the wave's columns
// are there (no branch then keeps loads and stores from being under way together).
template <class O, int ACT, bool PLAIN, bool PART, bool WHOLE, int FI, int FJ, int ROOM>
__device__ __forceinline__ void write_rows(const Gemm& g, const f32x4 (&acc)[FI][FJ], float* mine,
                                           int64_t i_first, int64_t j_first, uint32_t split) {
    constexpr int CW = FJ * 16, LD = CW + 4;  // 4 floats on: rows start in other banks
    constexpr int BLOCKS = ROOM / (16 * LD * 4);
    constexpr int XB = BLOCKS >= FI ? FI : BLOCKS >= FI / 2 ? FI / 2 : BLOCKS >= FI / 4 ? FI / 4 : 1;
    constexpr int LANES = CW / 8;  // of a row
    static_assert(BLOCKS >= 1 && FI % XB == 0 && 64 % LANES == 0, "rounds of whole blocks");
    const int lane = threadIdx.x & 63;
    const int col = lane % LANES * 8;
    const int64_t j = j_first + col;
    const int n = WHOLE || g.J - j > 8 ? 8 : (int)(g.J - j);
    float bias[8], scale[8];
    if (!PLAIN && !PART && n > 0) {
        if (g.bias) load_cols(g.bias + j, n, bias);
        if (g.q_scale) load_cols(g.q_scale + j, n, scale);
    }
#pragma unroll
    for (int r = 0; r < FI; r += XB) {
#pragma unroll
        for (int x = 0; x < XB; ++x)
#pragma unroll
            for (int y = 0; y < FJ; ++y)
                *(f32x4*)(mine + (x * 16 + (lane & 15)) * LD + (y >> 1) * 32 + (lane >> 4) * 8 +
                          (y & 1) * 4) = acc[r + x][y];
        __builtin_amdgcn_wave_barrier();
        if (n > 0) {
#pragma unroll
            for (int step = 0; step < XB * 16 * LANES / 64; ++step) {
                const int row = step * (64 / LANES) + lane / LANES;
                const int64_t i = i_first + r * 16 + row;
                if (i >= g.I) continue;
                const float* sums = mine + row * LD + col;
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = sums[k];
                if (PART) {
                    store_vec(g.part + ((int64_t)split * g.I + i) * part_ld(g.J) + j, 8, v);
                    continue;
                }
                if (!PLAIN) {
                    if (g.p_scale) {
                        const float ps = g.p_scale[i];
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] *= ps * scale[k];
                    }
                    if (g.bias) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] += bias[k];
                    }
                    if (g.z) store_vec((O*)g.z + i * g.ldz + j, n, v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = act_f32<ACT>(v[k]);
                    if (g.residual) {
                        float res[8];
                        load_cols((const O*)g.residual + i * g.ldr + j, n, res);
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] += res[k];
                    }
                }
                store_vec((O*)g.out + i * g.ldo + j, n, v);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}
template <class O, bool PLAIN, bool WHOLE, int ROOM, int FI, int FJ>
__device__ __forceinline__ void write_typed(const Gemm& g, const f32x4 (&acc)[FI][FJ], float* mine,
                                            int64_t i, int64_t j) {
    if (PLAIN || g.act == VCSR_ACT_NONE)
        write_rows<O, VCSR_ACT_NONE, PLAIN, false, WHOLE, FI, FJ, ROOM>(g, acc, mine, i, j, 0);
    else if (g.act == VCSR_ACT_RELU)
        write_rows<O, VCSR_ACT_RELU, PLAIN, false, WHOLE, FI, FJ, ROOM>(g, acc, mine, i, j, 0);
    else if (g.act == VCSR_ACT_GELU)
        write_rows<O, VCSR_ACT_GELU, PLAIN, false, WHOLE, FI, FJ, ROOM>(g, acc, mine, i, j, 0);
    else
        write_rows<O, VCSR_ACT_SILU, PLAIN, false, WHOLE, FI, FJ, ROOM>(g, acc, mine, i, j, 0);
}
template <bool PLAIN, int ROOM, int FI, int FJ>
__device__ __forceinline__ void write_out(const Gemm& g, const f32x4 (&acc)[FI][FJ], float* mine,
                                          int64_t i, int64_t j, int splits, uint32_t split) {
    if (splits > 1)
        write_rows<float, VCSR_ACT_NONE, true, true, false, FI, FJ, ROOM>(g, acc, mine, i, j, split);
    else if (j + FJ * 16 <= g.J && g.out_type == VCSR_BF16)
        write_typed<bf16, PLAIN, true, ROOM>(g, acc, mine, i, j);
    else if (j + FJ * 16 <= g.J)
        write_typed<float, PLAIN, true, ROOM>(g, acc, mine, i, j);
    else if (g.out_type == VCSR_BF16)
        write_typed<bf16, PLAIN, false, ROOM>(g, acc, mine, i, j);
    else
        write_typed<float, PLAIN, false, ROOM>(g, acc, mine, i, j);
}

// Whether the sum's last step goes through registers: its granules are not all
// whole.
template <class T>
__device__ __forceinline__ bool ragged_end(const Gemm& g, int64_t k_end, bool p_cols, bool q_cols) {
    constexpr int EPG = 16 / (int)sizeof(T), BK = kStepBytes / (int)sizeof(T);
    return k_end == g.R && ((g.R % BK) != 0 || (p_cols && g.I % EPG != 0) ||
                            (q_cols && g.J % EPG != 0));
}

// One of a launch's products: `blocks` blocks, each a tile and one of `splits`
// parts of the sum, of `steps` steps.
struct Part {
    int splits;
    int64_t steps;
    uint32_t blocks;
};

// Tiles whose blocks share a compute unit: a step's loads run under the other
// blocks' work as well as under the block's own.  STAGES steps have room in LDS, so
// loads go out STAGES - 1 steps ahead: two where five blocks share a unit, four
// where there are too few blocks to hide a trip to memory otherwise.
template <int TILE, int STAGES>
constexpr int kLds = STAGES * 2 * TILE * kStepBytes;
template <class T, int TI, int TJ, int WI, int WJ, int STAGES, bool PCOLS, bool QCOLS>
__device__ __forceinline__ void gemm_shared(const Gemm& g, const Part& part, uint32_t block,
                                            uint8_t* lds0) {
    constexpr int NT = 64 * WI * WJ;
    constexpr int FI = TI / WI / 16, FJ = TJ / WJ / 16;
    constexpr int BK = kStepBytes / (int)sizeof(T);
    static_assert(FJ % 2 == 0, "column blocks go in pairs");
    using LP = Loader<T, TI, NT, PCOLS, false>;
    using LQ = Loader<T, TJ, NT, QCOLS, true>;
    using RP = Reader<T, TI, PCOLS, false>;
    using RQ = Reader<T, TJ, QCOLS, true>;
    constexpr int kStage = (TI + TJ) * kStepBytes;
    const int splits = part.splits;
    const int64_t steps = part.steps;
    const Place at = place_of<TI, TJ>(g, block, part.blocks, (uint32_t)splits);
    const Operand P{(const uint8_t*)g.p, g.ldp * (int64_t)sizeof(T), g.I, at.i0,
                    extent<T>(g.I, g.R, g.ldp, PCOLS)};
    const Operand Q{(const uint8_t*)g.q, g.ldq * (int64_t)sizeof(T), g.J, at.j0,
                    extent<T>(g.J, g.R, g.ldq, QCOLS)};
    const int64_t k_first = (int64_t)at.split * steps * BK;
    const int64_t k_end = k_first + steps * BK < g.R ? k_first + steps * BK : g.R;

    const int wave = uniform((int)(threadIdx.x >> 6));
    const int ri = (wave / WJ) * (TI / WI), rj = (wave % WJ) * (TJ / WJ);
    f32x4 acc[FI][FJ];
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
        for (int y = 0; y < FJ; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto multiply = [&](const uint8_t* lp, const uint8_t* lq) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            Frag<T> p[FI];
#pragma unroll
            for (int x = 0; x < FI; ++x) p[x].set(RP::get(lp, ri, x, s));
#pragma unroll
            for (int y = 0; y < FJ; ++y) {
                Frag<T> q;
                q.set(RQ::get(lq, rj, y, s));
#pragma unroll
                for (int x = 0; x < FI; ++x) acc[x][y] = mma<T>(q, p[x], acc[x][y]);
            }
        }
    };
    const bool ragged = ragged_end<T>(g, k_end, PCOLS, QCOLS);
    const int64_t k_full = ragged ? k_first + (k_end - k_first - 1) / BK * BK : k_end;
    uint32_t op[LP::GR], oq[LQ::GR];
    LP::offsets(P, op);
    LQ::offsets(Q, oq);
    lds_byte* const to = (lds_byte*)lds0;
    constexpr int AHEAD = STAGES - 1;
    const int n = k_first < k_full ? (int)((k_full - k_first + BK - 1) / BK) : 0;
    auto ask = [&](int t) __attribute__((always_inline)) {
        lds_byte* const into = to + t % STAGES * kStage;
        LP::copy(P, op, k_first + (int64_t)t * BK, into);
        LQ::copy(Q, oq, k_first + (int64_t)t * BK, into + TI * kStepBytes);
    };
#pragma unroll
    for (int t = 0; t < AHEAD; ++t)
        if (t < n) ask(t);
    for (int t = 0; t < n; ++t) {
        // This step's tiles are in LDS (loads end in order; those of the steps behind
        // it may be under way), and all waves are done with the last step's.
        if (AHEAD > 1 && t + AHEAD - 1 < n)
            wait_loads<(AHEAD - 1) * (LP::GR + LQ::GR)>();
        else
            wait_loads<0>();
        barrier();
        if (t + AHEAD < n) ask(t + AHEAD);
        const uint8_t* const lp = lds0 + t % STAGES * kStage;
        multiply(lp, lp + TI * kStepBytes);
    }
    const int buf = n % STAGES;
    if (ragged) {
        LP::fetch(P, k_full, k_end, lds0 + buf * kStage);
        LQ::fetch(Q, k_full, k_end, lds0 + buf * kStage + TI * kStepBytes);
        __syncthreads();
        multiply(lds0 + buf * kStage, lds0 + buf * kStage + TI * kStepBytes);
    }
    __syncthreads();
    constexpr int ROOM = STAGES * kStage / (WI * WJ) / 16 * 16;
    write_out<PCOLS || QCOLS, ROOM>(g, acc, (float*)(lds0 + wave * ROOM), at.i0 + ri,
                                    at.j0 + rj, splits, at.split);
}

// 256 x 256 tiles, eight waves of 128 x 64, one block a compute unit.
//
// Two waves a SIMD take turns: while one multiplies, the other brings its next
// operands from LDS.  A step is four turns of 4 x 4 blocks: the upper 64 rows of
// the wave's part with both halves of k, then the lower 64.  The barrier before
// the loop puts waves 4 to 7 half a turn behind, and each half turn ends at a
// barrier of all waves.
//
// LDS holds two steps, each in three pieces: P's upper rows, P's lower rows and
// Q.  A step's Q and upper P have been read by all waves when those in front
// begin its third turn, and are asked for again there, two steps on; its lower P
// at the first turn of the next step.  So every load has six turns (some 3,000
// clocks of matrix work) to arrive, which covers a miss of L2: asking a step ahead for
// all of it left 58 of 468 us waiting at 8192 x 8192 x 4096.  Loads end in order:
// a wave waits until all but the 8 newest have, before its half turn that ends
// at the barrier behind which the first wave reads them.
template <class T, bool PCOLS, bool QCOLS>
__device__ __forceinline__ void gemm_turns(const Gemm& g, const Part& part, uint32_t block,
                                           uint8_t* lds) {
    constexpr int TI = 256, TJ = 256, NT = 512, WJ = 4, FI = 8, FJ = 4, H = 4;
    constexpr int BK = kStepBytes / (int)sizeof(T);
    constexpr int kP = TI / 2 * kStepBytes, kStage = (TI + TJ) * kStepBytes;
    using LP = Loader<T, TI / 2, NT, PCOLS, false, 64>;
    using LQ = Loader<T, TJ, NT, QCOLS, true>;
    using RP = Reader<T, TI / 2, PCOLS, false>;
    using RQ = Reader<T, TJ, QCOLS, true>;
    static_assert(LQ::GR + 2 * LP::GR == kAhead, "loads of a step");
    const int splits = part.splits;
    const int64_t steps = part.steps;
    const Place at = place_of<TI, TJ>(g, block, part.blocks, (uint32_t)splits);
    Operand P[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
        P[h] = Operand{(const uint8_t*)g.p, g.ldp * (int64_t)sizeof(T), g.I, at.i0 + h * 64,
                       extent<T>(g.I, g.R, g.ldp, PCOLS)};
    const Operand Q{(const uint8_t*)g.q, g.ldq * (int64_t)sizeof(T), g.J, at.j0,
                    extent<T>(g.J, g.R, g.ldq, QCOLS)};
    const int64_t k_first = (int64_t)at.split * steps * BK;
    const int64_t k_end = k_first + steps * BK < g.R ? k_first + steps * BK : g.R;
    const bool ragged = ragged_end<T>(g, k_end, PCOLS, QCOLS);
    const int n = (int)((k_end - k_first - (ragged ? 1 : 0)) / BK);  // whole steps

    const int wave = uniform((int)(threadIdx.x >> 6));
    const int wi = wave / WJ, wj = wave % WJ;
    f32x4 acc[FI][FJ];
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
        for (int y = 0; y < FJ; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};

    uint32_t op[2][LP::GR], oq[LQ::GR];
    LP::offsets(P[0], op[0]);
    LP::offsets(P[1], op[1]);
    LQ::offsets(Q, oq);
    lds_byte* const to = (lds_byte*)lds;
    auto ask_front = [&](int t) {  // Q and upper P of step t
        lds_byte* const into = to + (t & 1) * kStage;
        LQ::copy(Q, oq, k_first + (int64_t)t * BK, into + 2 * kP);
        LP::copy(P[0], op[0], k_first + (int64_t)t * BK, into);
    };
    auto ask_back = [&](int t) {  // lower P
        LP::copy(P[1], op[1], k_first + (int64_t)t * BK, to + (t & 1) * kStage + kP);
    };
    if (n > 0) ask_front(0), ask_back(0);
    if (n > 1) ask_front(1);
    wait_loads<0>();
    barrier();
    if (wi) barrier();
    for (int t = 0; t < n; ++t) {
        const uint8_t* const stage = lds + (t & 1) * kStage;
        Frag<T> p[H], q[2][FJ];
#pragma unroll
        for (int turn = 0; turn < 4; ++turn) {
            const int h = turn >> 1, s = turn & 1;
            if (h == 0)
#pragma unroll
                for (int y = 0; y < FJ; ++y) q[s][y].set(RQ::get(stage + 2 * kP, wj * 64, y, s));
#pragma unroll
            for (int x = 0; x < H; ++x) p[x].set(RP::get(stage + h * kP, wi * 64, x, s));
            if (turn == 0 && t + 1 < n) ask_back(t + 1);
            if (turn == 2 && t + 2 < n) ask_front(t + 2);
            if (turn == 1) {  // lower P of this step
                if (t + 1 < n) wait_loads<kAhead>();
                else wait_loads<0>();
            }
            if (turn == 3) {  // Q and upper P of the next
                if (t + 2 < n) wait_loads<kAhead>();
                else wait_loads<0>();
            }
            wait_lds();
            barrier();
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int x = 0; x < H; ++x)
#pragma unroll
                for (int y = 0; y < FJ; ++y)
                    acc[h * H + x][y] = mma<T>(q[s][y], p[x], acc[h * H + x][y]);
            __builtin_amdgcn_s_setprio(0);
            barrier();
        }
    }
    if (!wi) barrier();
    if (ragged) {
        uint8_t* const stage = lds + (n & 1) * kStage;
        const int64_t k = k_first + (int64_t)n * BK;
        LP::fetch(P[0], k, k_end, stage);
        LP::fetch(P[1], k, k_end, stage + kP);
        LQ::fetch(Q, k, k_end, stage + 2 * kP);
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            Frag<T> q[FJ];
#pragma unroll
            for (int y = 0; y < FJ; ++y) q[y].set(RQ::get(stage + 2 * kP, wj * 64, y, s));
#pragma unroll
            for (int x = 0; x < FI; ++x) {
                Frag<T> p;
                p.set(RP::get(stage + x / H * kP, wi * 64, x % H, s));
#pragma unroll
                for (int y = 0; y < FJ; ++y) acc[x][y] = mma<T>(q[y], p, acc[x][y]);
            }
        }
    }
    __syncthreads();
    constexpr int ROOM = 2 * kStage / 8;
    write_out<PCOLS || QCOLS, ROOM>(g, acc, (float*)(lds + wave * ROOM), at.i0 + wi * 128,
                                    at.j0 + wj * 64, splits, at.split);
}

// A tile of TILE x TILE by the code for its size.
template <class T, int TILE, int STAGES, bool PCOLS, bool QCOLS>
__device__ __forceinline__ void gemm_block(const Gemm& g, const Part& part, uint32_t block,
                                           uint8_t* lds) {
    if constexpr (TILE == 256)
        gemm_turns<T, PCOLS, QCOLS>(g, part, block, lds);
    else
        gemm_shared<T, TILE, TILE, 2, 2, STAGES, PCOLS, QCOLS>(g, part, block, lds);
}
template <int TILE>
constexpr int kThreads = TILE == 256 ? 512 : 256;

template <class T, int TILE, int STAGES, bool PCOLS, bool QCOLS>
__global__ __launch_bounds__(kThreads<TILE>) void gemm_kernel(Gemm g, Part part) {
    __shared__ __attribute__((aligned(128))) uint8_t lds[kLds<TILE, STAGES>];
    gemm_block<T, TILE, STAGES, PCOLS, QCOLS>(g, part, blockIdx.x, lds);
}

// Columns [16 * block, + 16) of the sum of partial rows, in a fixed order.
template <int THREADS>
__device__ __forceinline__ void sum_columns(const RowSum& r, uint32_t block, uint8_t* lds) {
    constexpr int G = THREADS / 16;
    float(*const t)[17] = (float(*)[17])lds;
    const int col = threadIdx.x & 15, grp = threadIdx.x >> 4;
    const int64_t c = (int64_t)block * 16 + col;
    float v = 0.f;
    if (c < r.C) {
#pragma unroll 8
        for (int32_t p = grp; p < r.P; p += G) v += r.part[(int64_t)p * r.C + c];
    }
    t[grp][col] = v;
    __syncthreads();
    if (grp == 0 && c < r.C) {
#pragma unroll
        for (int g = 1; g < G; ++g) v += t[g][col];
        r.out[c] = v;
    }
}

// Both products of a gradient in one launch: dw's blocks first, whose sums over the
// rows are long, then dx's (from a multiple of 8 on, so that both keep their XCDs),
// then those that add up dbias' partial rows.  Each product by itself leaves
// compute units idle at its end.
template <class T, int TILE, int STAGES>
__global__ __launch_bounds__(kThreads<TILE>) void gemm_pair_kernel(Gemm dw, Part dw_part, Gemm dx,
                                                                   Part dx_part, RowSum bias) {
    __shared__ __attribute__((aligned(128))) uint8_t lds[kLds<TILE, STAGES>];
    const uint32_t first = (dw_part.blocks + 7) & ~7u;
    if (blockIdx.x >= first + dx_part.blocks)
        sum_columns<kThreads<TILE>>(bias, blockIdx.x - first - dx_part.blocks, lds);
    else if (blockIdx.x >= first)
        gemm_block<T, TILE, STAGES, false, true>(dx, dx_part, blockIdx.x - first, lds);
    else if (blockIdx.x < dw_part.blocks)
        gemm_block<T, TILE, STAGES, true, true>(dw, dw_part, blockIdx.x, lds);
}

// The partial sums of a split product and the epilogue, for few parts: a thread
// adds those of 8 columns in order.
template <class O>
__global__ __launch_bounds__(256) void gemm_join_few_kernel(Gemm g, int splits) {
    const int64_t ld = part_ld(g.J);
    const uint32_t per_row = (uint32_t)(ld / 8);
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t i = e / per_row;
    const int j = (int)(e - i * per_row) * 8;
    if (i >= g.I) return;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        float p[8];
        load_vec(g.part + ((int64_t)s * g.I + i) * ld + j, 8, p);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += p[k];
    }
    if (g.J - j >= 8) {
        finish<O>(g, i, j, v);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float one[1] = {v[k]};
            if (j + k < g.J) finish<O>(g, i, j + k, one);
        }
    }
}

// For many parts (from 8): a block takes 32 vectors of 8 columns; 8 threads a vector add every eighth part, then LDS adds the
// eight in order: with few columns of out the parts' loads are what there is to
// run at once.
template <class O>
__global__ __launch_bounds__(256) void gemm_join_kernel(Gemm g, int splits) {
    __shared__ float lds[8][32][9];
    const int64_t ld = part_ld(g.J);
    const uint32_t per_row = (uint32_t)(ld / 8);
    const int at = threadIdx.x & 31, grp = threadIdx.x >> 5;
    const int64_t e = (int64_t)blockIdx.x * 32 + at;
    const int64_t i = e / per_row;
    const int j = (int)(e - i * per_row) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (i < g.I) {
#pragma unroll 4
        for (int s = grp; s < splits; s += 8) {
            float p[8];
            load_vec(g.part + ((int64_t)s * g.I + i) * ld + j, 8, p);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] += p[k];
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) lds[grp][at][k] = v[k];
    __syncthreads();
    // One column a thread from here.
    const int col = threadIdx.x & 7;
    const int64_t f = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    const int64_t row = f / per_row;
    const int c = (int)(f - row * per_row) * 8 + col;
    if (row >= g.I || c >= g.J) return;
    float sum[1] = {lds[0][threadIdx.x >> 3][col]};
#pragma unroll
    for (int q = 1; q < 8; ++q) sum[0] += lds[q][threadIdx.x >> 3][col];
    finish<O>(g, row, c, sum);
}

// One granule of a run of `total` elements from `pos`, zeros past its end; every
// element by itself where the run is shorter than a granule.
template <class T>
__device__ __forceinline__ u32x4 load_granule(const T* run, int64_t pos, int64_t total) {
    constexpr int EPG = 16 / (int)sizeof(T);
    u32x4 v{0, 0, 0, 0};
    if (pos >= total) return v;
    if (total >= EPG) {
        const int back = total - pos < EPG ? (int)(EPG - (total - pos)) : 0;
        const Mem<T, EPG> m = *(const Mem<T, EPG>*)(run + (pos - back));
        __builtin_memcpy(&v, &m, 16);
        return shift_down(v, back * (int)sizeof(T));
    }
    T t[EPG];
    __builtin_memset(t, 0, 16);
#pragma unroll
    for (int i = 0; i < EPG; ++i)
        if (pos + i < total) t[i] = run[pos + i];
    __builtin_memcpy(&v, t, 16);
    return v;
}

// Few rows of x (at most 16): what takes time is reading W once.  A block takes
// 16 rows of W; its 8 waves take its 128-byte lines in turn, UN lines of every
// row asked for at once and straight from memory into the matrix layout (all of a
// 4096-wide bf16 row, so that the chip has the whole W under way).  The waves'
// sums meet in LDS and are added in order: one launch, no partial sums in memory.
template <class T, class O, int UN>
__global__ __launch_bounds__(512) void gemm_rows_kernel(Gemm g) {
    constexpr int EPG = 16 / (int)sizeof(T), WAVES = 8;
    __shared__ __attribute__((aligned(16))) float lds[WAVES][16][20];
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const int64_t j0 = (int64_t)blockIdx.x * 16;
    const int64_t jr = j0 + (lane & 15) < g.J ? j0 + (lane & 15) : g.J - 1;
    const int64_t i = lane & 15;
    const T* const w = (const T*)g.q + jr * g.ldq;
    const T* const x = (const T*)g.p + (i < g.I ? i : 0) * g.ldp;
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
    const int64_t lines = (g.R + EPG * 8 - 1) / (EPG * 8);
    for (int64_t l0 = wave; l0 < lines; l0 += WAVES * UN) {
        u32x4 q[UN][2], p[UN][2];
        auto at = [&](int u, int h) { return ((l0 + WAVES * u) * 8 + h * 4 + (lane >> 4)) * EPG; };
        if ((l0 + WAVES * (UN - 1) + 1) * EPG * 8 <= g.R) {
#pragma unroll
            for (int u = 0; u < UN; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const Mem<T, EPG> m = *(const Mem<T, EPG>*)(w + at(u, h));
                    __builtin_memcpy(&q[u][h], &m, 16);
                }
#pragma unroll
            for (int u = 0; u < UN; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    p[u][h] = u32x4{0, 0, 0, 0};
                    if (i < g.I) {
                        const Mem<T, EPG> m = *(const Mem<T, EPG>*)(x + at(u, h));
                        __builtin_memcpy(&p[u][h], &m, 16);
                    }
                }
        } else {
#pragma unroll
            for (int u = 0; u < UN; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    q[u][h] = load_granule(w, at(u, h), g.R);
                    p[u][h] = u32x4{0, 0, 0, 0};
                    if (i < g.I) p[u][h] = load_granule(x, at(u, h), g.R);
                }
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                Frag<T> a, b;
                a.set(q[u][h]);
                b.set(p[u][h]);
                acc = mma<T>(a, b, acc);
            }
    }
    *(f32x4*)&lds[wave][lane & 15][(lane >> 4) * 4] = acc;
    __syncthreads();
    const int row = threadIdx.x >> 4, col = threadIdx.x & 15;
    if (row >= 16 || row >= g.I || j0 + col >= g.J) return;
    float sum[1] = {0.f};
#pragma unroll
    for (int k = 0; k < WAVES; ++k) sum[0] += lds[k][row][col];
    finish<O>(g, row, (int)j0 + col, sum);
}

template <class T, class O>
hipError_t launch_rows(const Gemm& g, hipStream_t st) {
    const unsigned blocks = (unsigned)(((int64_t)g.J + 15) / 16);
    const int64_t lines = (g.R * (int64_t)sizeof(T) + 127) / 128;
    if (lines <= 16)
        gemm_rows_kernel<T, O, 2><<<blocks, 512, 0, st>>>(g);
    else if (lines <= 32)
        gemm_rows_kernel<T, O, 4><<<blocks, 512, 0, st>>>(g);
    else
        gemm_rows_kernel<T, O, 8><<<blocks, 512, 0, st>>>(g);
    return hipGetLastError();
}

inline Part part_of(const Gemm& g, const GemmPlan& p) {
    const int64_t tiles = (g.I + p.tile - 1) / p.tile * (((int64_t)g.J + p.tile - 1) / p.tile);
    return Part{p.splits, p.steps, (uint32_t)(tiles * p.splits)};
}

inline hipError_t launch_join(const Gemm& g, int splits, hipStream_t st) {
    if (splits <= 1) return hipSuccess;
    const int64_t vectors = g.I * (part_ld(g.J) / 8);
    const unsigned few = (unsigned)((vectors + 255) / 256), many = (unsigned)((vectors + 31) / 32);
    if (g.out_type == VCSR_BF16) {
        if (splits < 8)
            gemm_join_few_kernel<bf16><<<few, 256, 0, st>>>(g, splits);
        else
            gemm_join_kernel<bf16><<<many, 256, 0, st>>>(g, splits);
    } else {
        if (splits < 8)
            gemm_join_few_kernel<float><<<few, 256, 0, st>>>(g, splits);
        else
            gemm_join_kernel<float><<<many, 256, 0, st>>>(g, splits);
    }
    return hipGetLastError();
}

template <class T, bool PCOLS, bool QCOLS>
hipError_t launch_layout(const Gemm& g, const GemmPlan& p, hipStream_t st) {
    if constexpr (!PCOLS && !QCOLS) {
        if (p.tile == 16)
            return g.out_type == VCSR_BF16 ? launch_rows<T, bf16>(g, st)
                                           : launch_rows<T, float>(g, st);
    }
    const Part part = part_of(g, p);
    constexpr bool DEEP = sizeof(T) == 2 && !PCOLS && !QCOLS;
    if (DEEP && p.tile == 64 && p.stages == 4) {
        if constexpr (DEEP)
            gemm_kernel<T, 64, 4, PCOLS, QCOLS><<<part.blocks, kThreads<64>, 0, st>>>(g, part);
    } else if (p.tile == 64)
        gemm_kernel<T, 64, 2, PCOLS, QCOLS><<<part.blocks, kThreads<64>, 0, st>>>(g, part);
    else if (p.tile == 128)
        gemm_kernel<T, 128, 2, PCOLS, QCOLS><<<part.blocks, kThreads<128>, 0, st>>>(g, part);
    else if constexpr (sizeof(T) < 4)
        gemm_kernel<T, 256, 2, PCOLS, QCOLS><<<part.blocks, kThreads<256>, 0, st>>>(g, part);
    hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_join(g, p.splits, st);
}

template <class T>
hipError_t launch_pair(const Gemm& dw, const GemmPlan& p, const Gemm& dx, const GemmPlan& q,
                       const RowSum& bias, hipStream_t st) {
    const Part a = part_of(dw, p), b = part_of(dx, q);
    const uint32_t blocks = ((a.blocks + 7) & ~7u) + b.blocks +
                            (bias.P > 0 ? (uint32_t)(((int64_t)bias.C + 15) / 16) : 0);
    if (p.tile == 64)
        gemm_pair_kernel<T, 64, 2><<<blocks, kThreads<64>, 0, st>>>(dw, a, dx, b, bias);
    else if (p.tile == 128)
        gemm_pair_kernel<T, 128, 2><<<blocks, kThreads<128>, 0, st>>>(dw, a, dx, b, bias);
    else if constexpr (sizeof(T) < 4)
        gemm_pair_kernel<T, 256, 2><<<blocks, kThreads<256>, 0, st>>>(dw, a, dx, b, bias);
    hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_join(dw, p.splits, st);
}

}  // namespace tile
}  // namespace vcsr
