// embed.hip - rows of a table by token (embedding) and the table's gradient.
//
// Forward: y[m] = scale * table[ids[m]], a copy that memory bounds.
// Gradient: dtable[v] = scale * sum of dy[m] over ids[m] = v.  Tokens are sorted by id,
// equal ones in the order they came, so that a row of the table is the sum of a run of
// sorted tokens and results repeat bit for bit (no atomics on values).  The sorted
// tokens are cut into chunks of E, a wave's work for 64 vectors of columns: it adds
// the rows of dy of each run in order and writes the run's row.  Runs of up to E tokens
// are the work of the chunk they start in, also past its end; longer ones (a few
// tokens make up much of a text) are added chunk by chunk, and their partial rows by
// another launch, in order.
// Memory bounds the lookup (65536 tokens of 2048 bf16 60 us: 5.6 TB/s with each row of the
// table that has a token read once) and most of the gradient (32768 tokens of 2048 bf16
// to 32768 x 2048 FP32 105 us: the sort 20 in four launches, the sums with the zeros 80,
// the join 5).  5001 tokens of 257 FP32, added, are three launches one after the other, 19.8 us:
// rank 7, sums 9, join 4.
#include "common.hpp"
#include "dense.hpp"
#include "launch.hpp"
#include "vecops.hpp"

namespace vcsr {
namespace {

// The FP32 values of 16 bytes.
__device__ __forceinline__ void widen(const u32x4& r, float (&v)[4], float) {
    const f32x4 f = __builtin_bit_cast(f32x4, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f[i];
}
__device__ __forceinline__ void widen(const u32x4& r, float (&v)[8], bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __builtin_bit_cast(float, r[i] << 16);
        v[2 * i + 1] = __builtin_bit_cast(float, r[i] & 0xffff0000u);
    }
}

// Of 4 and 8 bytes.
__device__ __forceinline__ void widen(uint32_t r, float (&v)[4], fp8) {
    v[0] = fp8_to_f32<0>(r);
    v[1] = fp8_to_f32<1>(r);
    v[2] = fp8_to_f32<2>(r);
    v[3] = fp8_to_f32<3>(r);
}
__device__ __forceinline__ void widen(uint64_t r, float (&v)[8], fp8) {
    float a[4], b[4];
    widen((uint32_t)r, a, fp8());
    widen((uint32_t)(r >> 32), b, fp8());
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
    }
}
__device__ __forceinline__ void widen(uint64_t r, float (&v)[4], bf16) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = __builtin_bit_cast(float, (uint32_t)(r >> (16 * i)) << 16);
}

// 16 bytes anywhere.
typedef u32x4 Any16 __attribute__((aligned(1)));

// What a call writes past the caches: as many bytes leave nothing there for whoever reads
// them next, half of the 256 MB that the last cache has.
constexpr int64_t kLarge = (int64_t)128 << 20;

// How rows end: in whole vectors of 16 bytes, inside one, or before the first is whole.
enum { kWhole = 0, kRagged = 1, kShort = 2 };
template <int V>
int ends_of(int32_t C) {
    return C % V == 0 ? kWhole : C > V ? kRagged : kShort;
}

// Values [c, c + V) of a row of C, for c a multiple of V: anything past the row's
// end.  No branch but for rows that are shorter than a vector.
// ONCE: of values that are read once.
template <class T, int ENDS, bool ONCE = false>
__device__ __forceinline__ u32x4 load16(const T* row, int64_t c, int64_t C) {
    constexpr int V = 16 / (int)sizeof(T);
    u32x4 r;
    if (ENDS == kShort) {
        T t[V];
        __builtin_memset(t, 0, 16);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c + i < C) t[i] = row[c + i];
        __builtin_memcpy(&r, t, 16);
        return r;
    }
    // A vector that reaches past the end is read ending with the row, and shifted.
    const int64_t back = c + V > C ? c + V - C : 0;
    const Any16* const from = (const Any16*)(row + (back < V ? c - back : 0));
    r = ONCE ? __builtin_nontemporal_load(from) : *from;
    return ENDS == kWhole ? r : shift_down(r, (int)(back & (V - 1)) * (int)sizeof(T));
}

// The same of V values of 4 or 8 bytes together.
template <class T, int V, int ENDS>
__device__ __forceinline__ auto load_bits(const T* row, int64_t c, int64_t C) {
    if constexpr (V * sizeof(T) == 16) {
        return load16<T, ENDS>(row, c, C);
    } else {
        using B = typename std::conditional<V * sizeof(T) == 8, uint64_t, uint32_t>::type;
        typedef B Any __attribute__((aligned(1)));
        if (ENDS == kShort) {
            T t[V];
            __builtin_memset(t, 0, sizeof(t));
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i < C) t[i] = row[c + i];
            return __builtin_bit_cast(B, t);
        }
        const int64_t back = c + V > C ? c + V - C : 0;
        const B r = *(const Any*)(row + (back < V ? c - back : 0));
        return ENDS == kWhole ? r : r >> ((int)(back & (V - 1)) * 8 * (int)sizeof(T));
    }
}

// ------------------------------------------------------------------- forward
// Values of a lane's vector: 16 bytes of the larger type, so that a wave's stores are
// whole lines (21082 tokens of 3824 e4m3 to bf16 41 us, 80 with 16 bytes of x a lane; 65536
// of 1024 bf16 to FP32 47 and 110).
template <class X, class Y>
constexpr int kForward = 16 / (int)(sizeof(X) > sizeof(Y) ? sizeof(X) : sizeof(Y));

// Stores past the caches, of whole 16 bytes; of bf16's 8 (rows of FP32) through them.
__device__ __forceinline__ void store_large(float* p, const float (&v)[4]) {
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}), (Any16*)p);
}
__device__ __forceinline__ void store_large(bf16* p, const float (&v)[8]) {
    Mem<bf16, 8> m;
#pragma unroll
    for (int k = 0; k < 8; ++k) m.v[k] = (bf16)v[k];
    u32x4 q;
    __builtin_memcpy(&q, &m, 16);
    __builtin_nontemporal_store(q, (Any16*)p);
}
__device__ __forceinline__ void store_large(bf16* p, const float (&v)[4]) { store_vec(p, 4, v); }

// Groups of `lanes` (a power of two <= 64) lanes take U rows each, of them NV vectors
// a lane from blockIdx.y's slab on; all loads go out together.  The table's rows stay
// in the caches, since tokens repeat; y, where it is large (whole rows alone), goes past
// them: 65536 tokens of 2048 bf16 60 us, 75 through them.
template <class X, class Y, int ENDS, int NV, int U, bool LARGE>
__global__ __launch_bounds__(256) void embed_kernel(vcsr_embed_args a, int lanes) {
    constexpr int V = kForward<X, Y>;
    const int lane = threadIdx.x & (lanes - 1);
    const int64_t first = ((int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes) * U;
    int32_t id[U];
    float f[U];
    decltype(load_bits<X, V, ENDS>((const X*)nullptr, 0, 0)) r[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        id[u] = first + u < a.M ? a.ids[first + u] : -1;
        if ((uint32_t)id[u] >= (uint32_t)a.V) id[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = id[u] < 0 ? 0 : id[u];
        const X* const row = (const X*)a.table + at * a.ldt;
        f[u] = sizeof(X) == 1 ? a.scale * a.table_scale[at] : a.scale;
#pragma unroll
        for (int k = 0; k < NV; ++k)
            r[u][k] = load_bits<X, V, ENDS>(
                row, (((int64_t)blockIdx.y * NV + k) * lanes + lane) * V, a.C);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (first + u >= a.M) continue;
        Y* const to = (Y*)a.y + (first + u) * a.ldy;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t c = (((int64_t)blockIdx.y * NV + k) * lanes + lane) * V;
            if (c >= a.C) continue;
            float v[V];
            widen(r[u][k], v, X());
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = id[u] < 0 ? 0.f : v[i] * f[u];
            if (LARGE)
                store_large(to + c, v);
            else
                store_vec(to + c, ENDS == kWhole || a.C - c > V ? V : (int)(a.C - c), v);
        }
    }
}

template <class X, class Y, int ENDS>
void launch_ends(const vcsr_embed_args& a, hipStream_t st) {
    constexpr int V = kForward<X, Y>;
    const int64_t nv = ((int64_t)a.C + V - 1) / V;
    int lanes = 1;
    while (lanes < 64 && lanes < nv) lanes *= 2;
    auto go = [&](auto nvec, auto rows) {
        constexpr int NV = decltype(nvec)::value, U = decltype(rows)::value;
        const int64_t per = 256 / lanes * U, slab = (int64_t)lanes * NV;
        const unsigned slabs = (unsigned)((nv + slab - 1) / slab);
        // A launch has fewer than 2^32 threads: more rows go in several.
        const int64_t most = per << 23;
        for (int64_t m = 0; m < a.M; m += most) {
            vcsr_embed_args b = a;
            b.M = a.M - m < most ? a.M - m : most;
            b.ids += m;
            b.y = (Y*)a.y + m * a.ldy;
            const dim3 grid((unsigned)((b.M + per - 1) / per), slabs);
            if (ENDS == kWhole && a.M * a.C * (int64_t)sizeof(Y) >= kLarge)
                embed_kernel<X, Y, ENDS, NV, U, ENDS == kWhole><<<grid, 256, 0, st>>>(b, lanes);
            else
                embed_kernel<X, Y, ENDS, NV, U, false><<<grid, 256, 0, st>>>(b, lanes);
        }
    };
    // Loads of a lane: of long rows (2048 bf16, 65536 tokens) four of one row 58 us, two of
    // two 70, one of four 65; of short ones (256) 12, 9.6 and 9.2.
    if (nv > 128)
        go(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
    else if (nv > 64)
        go(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
    else
        go(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
}
template <class X, class Y>
hipError_t launch_forward(const vcsr_embed_args& a, hipStream_t st) {
    switch (ends_of<kForward<X, Y>>(a.C)) {
        case kWhole: launch_ends<X, Y, kWhole>(a, st); break;
        case kRagged: launch_ends<X, Y, kRagged>(a, st); break;
        default: launch_ends<X, Y, kShort>(a, st);
    }
    return hipGetLastError();
}

// ---------------------------------------------------------------------- sort
// Key of a token: its id, or V (behind all others) for one outside the table.
__device__ __forceinline__ int32_t key_of(int32_t id, int32_t V) {
    return (uint32_t)id < (uint32_t)V ? id : V;
}

// A piece of 16 bytes of a span of zeros, the last one moved back to end with it.
template <bool LARGE>
__device__ __forceinline__ void zero_piece(uint8_t* p, int64_t bytes, int64_t i) {
    if (bytes >= 16) {
        Any16* const to = (Any16*)(p + (16 * i + 16 <= bytes ? 16 * i : bytes - 16));
        const u32x4 zero{0, 0, 0, 0};
        if (LARGE) __builtin_nontemporal_store(zero, to);
        else *to = zero;
    } else {
        for (int64_t b = 0; b < bytes; b += 2) *(uint16_t*)(p + b) = 0;
    }
}
// The rows of dtable, of which those without a token are to be cleared.  `owner` tells
// which: the first launch writes to owner[v] some token of id v, so that a row has one if
// its owner is a token of its id; what else lies there does not matter, and nothing has
// to be cleared first.  They are cleared beside the sums, past the caches where they are
// many (`large`): 32768 tokens and 32768 x 2048 FP32 take 105 us, 13 more with the zeros
// through the caches, 11 more with dy's loads through them, 24 more with every row cleared
// beside the sort and some written again.
struct Zeros {
    uint8_t* p;
    int64_t ld, bytes;  // of a row
    int64_t rows;
    const int32_t *owner, *ids;
    int32_t M;
    bool large;
};
// Rows of a group: 16 KB of them, 64 at most.
__host__ __device__ constexpr int64_t zero_group(int64_t bytes) {
    return bytes >= 16384 ? 1 : bytes > 256 ? 16384 / bytes : 64;
}
// Waves take groups of up to 64 rows, a lane a row to see which have a token (`met`).  Of
// rows that are shorter than 64 pieces the lanes take several at a time: 13307 tokens of 33
// FP32 to 32517 rows of bf16 are 30 us, 34 more one row after the other.
template <bool LARGE, class F>
__device__ __forceinline__ void zero_rows(const Zeros& z, int64_t wave, int64_t waves, F&& met) {
    const int lane = threadIdx.x & 63;
    const int64_t most = zero_group(z.bytes), pieces = (z.bytes + 15) / 16;
    for (int64_t r0 = wave * most; r0 < z.rows; r0 += waves * most) {
        const int rows = z.rows - r0 < most ? (int)(z.rows - r0) : (int)most;
        // With all lanes: met reads other lanes' tokens.
        const bool has = met(lane < rows ? r0 + lane : r0);
        const uint64_t kept = __ballot(lane < rows && has);
        if (!kept && z.ld == z.bytes) {
            for (int64_t i = lane; 16 * i < rows * z.bytes; i += 64)
                zero_piece<LARGE>(z.p + r0 * z.ld, rows * z.bytes, i);
            continue;
        }
        if (pieces < 64) {
            const int n = (int)pieces;
            for (int i = lane; i < rows * n; i += 64) {
                const int k = i / n;
                if (!(kept >> k & 1))
                    zero_piece<LARGE>(z.p + (r0 + k) * z.ld, z.bytes, i - k * n);
            }
            continue;
        }
        for (int k = 0; k < rows; ++k)
            if (!(kept >> k & 1))
                for (int64_t i = lane; 16 * i < z.bytes; i += 64)
                    zero_piece<LARGE>(z.p + (r0 + k) * z.ld, z.bytes, i);
    }
}
// Few tokens: each one's place is the number of tokens before it.  All keys go to LDS; a
// block takes 16 tokens, a lane one of them and a thirty-second of the keys, and LDS adds
// the parts.  Comparisons bound it, n * n of them: the whole gradient of 4000 tokens of 512
// bf16 is 16 us (by digits, below, 30), of 12000 33 (by digits 34 at 12500).
constexpr int kMostRanked = 12288;
__global__ __launch_bounds__(512) void rank_kernel(const int32_t* __restrict__ ids, int32_t n,
                                                   int32_t V, int32_t* __restrict__ keys,
                                                   int32_t* __restrict__ pos,
                                                   int32_t* __restrict__ owner) {
    __shared__ __attribute__((aligned(16))) int32_t all[kMostRanked];
    __shared__ int32_t count[32][17];
    const int t = threadIdx.x & 15, run = threadIdx.x >> 4;
    const int32_t i = (int32_t)blockIdx.x * 16 + t;
    const int32_t groups = (n + 3) / 4;
#pragma unroll 4
    for (int32_t g = threadIdx.x; g < groups; g += 512) {
        int32_t k[4];
        if (4 * g + 4 <= n) {
            const Mem<int32_t, 4> m = *(const Mem<int32_t, 4>*)(ids + 4 * g);
#pragma unroll
            for (int q = 0; q < 4; ++q) k[q] = key_of(m.v[q], V);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) k[q] = 4 * g + q < n ? key_of(ids[4 * g + q], V) : -1;
        }
        *(int4*)(all + 4 * g) = make_int4(k[0], k[1], k[2], k[3]);
    }
    __syncthreads();
    const int32_t key = i < n ? all[i] : V, own = i >> 2;
    const int32_t len = (groups + 31) / 32, g0 = run * len;
    const int32_t g1 = g0 + len < groups ? g0 + len : groups;
    // As unsigned numbers: what fills the last group (-1) is behind all keys, and a key
    // and one is at most 2^31.  Of equal keys those of lower tokens come first.
    int32_t before = 0;
#pragma unroll 4
    for (int32_t g = g0; g < g1; ++g) {
        const int4 k = *(const int4*)(all + 4 * g);
        const uint32_t limit = (uint32_t)key + (g < own ? 1 : 0);
        before += (uint32_t)k.x < limit ? 1 : 0;
        before += (uint32_t)k.y < limit ? 1 : 0;
        before += (uint32_t)k.z < limit ? 1 : 0;
        before += (uint32_t)k.w < limit ? 1 : 0;
    }
    count[run][t] = before;
    __syncthreads();
    if (run || i >= n) return;
#pragma unroll
    for (int w = 1; w < 32; ++w) before += count[w][t];
    for (int32_t j = 4 * own; j < i; ++j) before += all[j] == key ? 1 : 0;
    keys[before] = key;
    pos[before] = i;
    if (owner && key < V) owner[key] = i;
}

// More: by digits of up to 9 bits, the lowest first, two launches each.  A block takes a
// tile of `tile` keys in a row, each of its 4 waves a quarter; `pos` is null for the
// first digit, whose keys are the ids themselves.
// The blocks' counts are read kTogether at a time, all under way together: rows of zeros
// go up to a multiple of them (13 blocks: 39 us a gradient, 43 with a loop of its own for
// those).
constexpr int kDigits = 512, kTogether = 16;
struct Radix {
    const int32_t *keys, *pos;
    int32_t n, V, tile, shift, digits;
    int32_t* owner;  // of the first digit's counts, or null
};
__device__ __forceinline__ int32_t radix_key(const Radix& r, int64_t i) {
    const int32_t k = r.keys[i];
    return r.pos ? k : key_of(k, r.V);
}
__global__ __launch_bounds__(256) void digit_count_kernel(Radix r, int32_t* counts) {
    __shared__ int32_t lds[kDigits];
    for (int d = threadIdx.x; d < r.digits; d += 256) lds[d] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * r.tile;
    const int64_t last = first + r.tile < r.n ? first + r.tile : r.n;
#pragma unroll 4
    for (int64_t i = first + threadIdx.x; i < last; i += 256) {
        const int32_t k = radix_key(r, i);
        atomicAdd(&lds[(k >> r.shift) & (r.digits - 1)], 1);
        if (r.owner && k < r.V) r.owner[k] = (int32_t)i;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < r.digits; d += 256)
        counts[(int64_t)blockIdx.x * r.digits + d] = lds[d];
    if (blockIdx.x + 1 < gridDim.x) return;
    for (int32_t b = gridDim.x; b % kTogether; ++b)
        for (int d = threadIdx.x; d < r.digits; d += 256) counts[(int64_t)b * r.digits + d] = 0;
}
__global__ __launch_bounds__(256) void digit_place_kernel(Radix r, const int32_t* counts,
                                                          int32_t* keys, int32_t* pos) {
    __shared__ int32_t next[4][kDigits], base[kDigits], sums[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
    for (int d = tid; d < r.digits; d += 256)
#pragma unroll
        for (int w = 0; w < 4; ++w) next[w][d] = 0;
    // Digits [2 tid, 2 tid + 2): how many keys of them there are, and in blocks before.
    int32_t all[2] = {0, 0}, before[2] = {0, 0};
    if (2 * tid < r.digits) {
        for (int32_t b0 = 0; b0 < (int32_t)gridDim.x; b0 += kTogether)
#pragma unroll
            for (int32_t b = b0; b < b0 + kTogether; ++b) {
                const int2 c = *(const int2*)(counts + (int64_t)b * r.digits + 2 * tid);
                all[0] += c.x;
                all[1] += c.y;
                before[0] += b < (int32_t)blockIdx.x ? c.x : 0;
                before[1] += b < (int32_t)blockIdx.x ? c.y : 0;
            }
    }
    const int32_t two = all[0] + all[1], scan = wave_inclusive_scan(two, lane);
    if (lane == 63) sums[wave] = scan;
    __syncthreads();
    int32_t start = scan - two;
    for (int w = 0; w < wave; ++w) start += sums[w];
    if (2 * tid < r.digits) base[2 * tid] = start + before[0];
    if (2 * tid + 1 < r.digits) base[2 * tid + 1] = start + all[0] + before[1];
    // The wave's quarter: how many of each digit.
    const int64_t first = (int64_t)blockIdx.x * r.tile + (int64_t)wave * (r.tile / 4);
    int64_t last = first + r.tile / 4;
    if (last > r.n) last = r.n;
#pragma unroll 4
    for (int64_t i = first + lane; i < last; i += 64)
        atomicAdd(&next[wave][(radix_key(r, i) >> r.shift) & (r.digits - 1)], 1);
    __syncthreads();
    for (int d = tid; d < r.digits; d += 256) {
        int32_t at = base[d];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int32_t c = next[w][d];
            next[w][d] = at;
            at += c;
        }
    }
    __syncthreads();
    // 64 keys at a time, in order: lanes with one digit go behind one another.
    for (int64_t b = first; b < last; b += 64) {
        const bool in = b + lane < last;
        const int32_t key = in ? radix_key(r, b + lane) : 0;
        const int32_t from = in ? (r.pos ? r.pos[b + lane] : (int32_t)(b + lane)) : 0;
        const int d = (key >> r.shift) & (r.digits - 1);
        uint64_t same = __ballot(in);
        for (int bit = 1; bit < r.digits; bit <<= 1) {
            const uint64_t set = __ballot(d & bit);
            same &= d & bit ? set : ~set;
        }
        const int rank = __popcll(same & (((uint64_t)1 << lane) - 1));
        int32_t at = 0;
        if (in) at = next[wave][d] + rank;
        wave_sync();
        if (in && rank == 0) next[wave][d] = at + __popcll(same);
        wave_sync();
        if (in) {
            keys[at] = key;
            pos[at] = from;
        }
    }
}

// ------------------------------------------------------------------ gradient
// A chunk of E sorted tokens from `first` on, as a wave's lanes hold them: its keys and
// those of the chunks before and behind it (-1 and V where there is none).
struct Chunk {
    int32_t before, key, behind;
    // Which of the chunk's tokens, and how many behind it, the wave adds; tokens under
    // `lead` belong to a long run from before, those from `tail` on to one that goes on.
    int from, to, lead, tail;
};
__device__ __forceinline__ int count_equal(int32_t k, int32_t x, uint64_t mask) {
    return __popcll(__ballot(k == x) & mask);
}
__device__ __forceinline__ void find_runs(Chunk& c, bool first, int E, int32_t V) {
    const uint64_t mask = ~(uint64_t)0 >> (64 - E);
    const int32_t k0 = __builtin_amdgcn_readlane(c.key, 0);
    const int32_t kl = __builtin_amdgcn_readlane(c.key, E - 1);
    const bool joins = !first && __builtin_amdgcn_readlane(c.before, E - 1) == k0;
    const int valid = __popcll(__ballot(c.key < V) & mask);
    c.from = c.lead = 0;
    c.to = valid;
    c.tail = 2 * E;
    if (joins) {
        const int len = count_equal(c.key, k0, mask);
        if (count_equal(c.before, k0, mask) + len > E)
            c.lead = len;
        else
            c.from = len;
    }
    if (valid < E) return;
    const int more = count_equal(c.behind, kl, mask), own = count_equal(c.key, kl, mask);
    if (more == 0 || (own == E && joins)) return;
    if (own + more > E)
        c.tail = E - own;
    else
        c.to = E + more;
}
__device__ __forceinline__ Chunk load_chunk(const int32_t* keys, int64_t first, int64_t n, int E,
                                            int32_t V, int lane) {
    Chunk c;
    c.before = first > 0 && lane < E ? keys[first - E + lane] : -1;
    c.key = lane < E && first + lane < n ? keys[first + lane] : V;
    c.behind = lane < E && first + E + lane < n ? keys[first + E + lane] : V;
    return c;
}

struct Runs {
    const int32_t *keys, *pos;
    float* part;     // two partial rows a chunk: of a long run from before, and of one that goes on
    int64_t ldp;
    int64_t chunks;
    int E, slabs, width;  // tokens a chunk; slabs of `width` vectors of columns
    int64_t first;        // chunk (and slab) that the launch begins with
};
// Blocks of a launch, which has fewer than 2^32 threads.
constexpr int64_t kMostBlocks = (int64_t)1 << 23;

// SORTS: up to 64 tokens, which each wave sorts by itself; it adds the runs that begin
// among its E.  Blocks behind `sums` clear the rows of no token.
template <class D, class X, int ENDS, bool SORTS>
__global__ __launch_bounds__(256) void embed_sum_kernel(vcsr_embed_grad_args a, Runs r, Zeros z,
                                                        int32_t sums) {
    constexpr int V = 16 / (int)sizeof(D), U = 8;
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    if ((int32_t)blockIdx.x >= sums) {
        const int32_t key = SORTS && lane < a.M ? key_of(a.ids[lane], a.V) : a.V;
        auto met = [&](int64_t row) {
            if (!SORTS) {
                const uint32_t m = (uint32_t)z.owner[row];
                return m < (uint32_t)z.M && z.ids[m] == row;
            }
            bool any = false;
#pragma unroll
            for (int l = 0; l < 64; ++l) any |= __builtin_amdgcn_readlane(key, l) == row;
            return any;
        };
        const int64_t first = ((int64_t)blockIdx.x - sums) * 4 + wave;
        const int64_t waves = ((int64_t)gridDim.x - sums) * 4;
        if (z.large)
            zero_rows<true>(z, first, waves, met);
        else
            zero_rows<false>(z, first, waves, met);
        return;
    }
    const int64_t item = r.first + (int64_t)blockIdx.x * 4 + wave;
    const int64_t chunk = item / r.slabs;
    if (chunk >= r.chunks) return;
    const int E = SORTS ? 64 : r.E;
    Chunk k;
    int32_t pos, pos_behind = 0;
    if (SORTS) {
        const int32_t mine = lane < a.M ? key_of(a.ids[lane], a.V) : a.V;
        int rank = 0;
#pragma unroll
        for (int l = 0; l < 64; ++l) {
            const int32_t o = __builtin_amdgcn_readlane(mine, l);
            rank += o < mine || (o == mine && l < lane) ? 1 : 0;
        }
        k.key = __builtin_amdgcn_ds_permute(rank * 4, mine);
        pos = __builtin_amdgcn_ds_permute(rank * 4, lane);
        const int valid = __popcll(__ballot(k.key < a.V)), first = (int)chunk * r.E;
        const int32_t previous = __shfl_up(k.key, 1);  // with all lanes, lane 1 reads lane 0
        const uint64_t starts = __ballot(lane < valid && (lane == 0 || previous != k.key));
        // The first run that begins in a token from `at` on.
        auto start_from = [&](int at) {
            const uint64_t later = at < 64 ? starts >> at << at : 0;
            return later ? __builtin_ctzll(later) : valid;
        };
        k.from = start_from(first);
        k.to = start_from(first + r.E);
        k.lead = 0;
        k.tail = 64;
        k.behind = a.V;
    } else {
        k = load_chunk(r.keys, chunk * E, a.M, E, a.V, lane);
        pos = lane < E && chunk * E + lane < a.M ? r.pos[chunk * E + lane] : 0;
        pos_behind = lane < E && (chunk + 1) * E + lane < a.M ? r.pos[(chunk + 1) * E + lane] : 0;
        find_runs(k, chunk == 0, E, a.V);
    }
    const int64_t vec = (item - chunk * r.slabs) * r.width + lane;
    const bool live = lane < r.width && vec * V < a.C;
    const int64_t c = live ? vec * V : a.C;
    const int n = a.C - c < V ? (int)(a.C - c) : V;
    auto key_at = [&](int e) {
        return e < E ? __builtin_amdgcn_readlane(k.key, e)
                     : __builtin_amdgcn_readlane(k.behind, e - E);
    };
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    if (k.from >= k.to) return;
    int32_t key = key_at(k.from);
    // Two sets of U rows of dy: one is under way while the other is added.
    u32x4 v[2][U];
    auto load = [&](u32x4(&to)[U], int e) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = e + u < k.to ? e + u : k.to - 1;
            const int64_t m = at < E ? __builtin_amdgcn_readlane(pos, at)
                                     : __builtin_amdgcn_readlane(pos_behind, at - E);
            to[u] = load16<D, ENDS, true>((const D*)a.dy + m * a.lddy, c, a.C);
        }
    };
    auto add = [&](const u32x4(&from)[U], int e) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (e + u >= k.to) break;
            float d[V];
            widen(from[u], d, D());
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += d[i];
            const int32_t next = e + u + 1 < k.to ? key_at(e + u + 1) : -1;
            if (next == key) continue;
            if (live) {
                if (e + u < k.lead || e + u >= k.tail) {
                    float* const to =
                        r.part + (2 * chunk + (e + u < k.lead ? 0 : 1)) * r.ldp + c;
                    store_vec(to, V, acc);
                } else {
                    X* const to = (X*)a.dtable + (int64_t)key * a.lddt + c;
                    float o[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] = 0.f;
                    if (a.accumulate) load_vec(to, n, o);
#pragma unroll
                    for (int i = 0; i < V; ++i) o[i] = __builtin_fmaf(a.scale, acc[i], o[i]);
                    store_vec(to, n, o);
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.f;
            key = next;
        }
    };
    load(v[0], k.from);
    for (int e = k.from; e < k.to; e += 2 * U) {
        if (e + U < k.to) load(v[1], e + U);
        add(v[0], e);
        if (e + 2 * U < k.to) load(v[0], e + 2 * U);
        if (e + U < k.to) add(v[1], e + U);
    }
}

// The partial rows of the long run that begins in chunk blockIdx.x, 256 columns a
// block: each wave adds every fourth one, then LDS adds the waves, in order.  A run of very
// many tokens is a chain of loads in a few blocks: 65536 tokens of 512 bf16, all of one id, 98
// us (63 with ids as text has them), 2^20 of 128 608 (180).
template <class X>
__global__ __launch_bounds__(256) void embed_join_kernel(vcsr_embed_grad_args a, Runs r) {
    __shared__ float lds[4][64][5];
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const int64_t chunk = r.first + blockIdx.x, first = chunk * r.E;
    Chunk k = load_chunk(r.keys, first, a.M, r.E, a.V, lane);
    find_runs(k, chunk == 0, r.E, a.V);
    if (k.tail > r.E) return;
    const int32_t key = __builtin_amdgcn_readlane(k.key, r.E - 1);
    // The chunks behind it that begin with the run, one after the other.
    int64_t parts = 1;
    for (;;) {
        const int64_t at = (chunk + parts + lane) * r.E;
        const int more = __popcll(__ballot(at < a.M && r.keys[at < a.M ? at : 0] == key));
        parts += more;
        if (more < 64) break;
    }
    const int64_t c = ((int64_t)blockIdx.y * 64 + lane) * 4;
    float t[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.C) {
#pragma unroll 4
        for (int64_t p = wave; p < parts; p += 4) {
            float v[4];
            load_full(r.part + (2 * (chunk + p) + (p == 0 ? 1 : 0)) * r.ldp + c, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] += v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) lds[wave][lane][i] = t[i];
    __syncthreads();
    if (wave || c >= a.C) return;
#pragma unroll
    for (int w = 1; w < 4; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] += lds[w][lane][i];
    X* const to = (X*)a.dtable + (int64_t)key * a.lddt + c;
    const int n = a.C - c < 4 ? (int)(a.C - c) : 4;
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    if (a.accumulate) load_vec(to, n, o);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(a.scale, t[i], o[i]);
    store_vec(to, n, o);
}

// How the gradient's tokens are sorted and cut.
struct Shape {
    Runs runs{};
    int32_t passes = 0, tile = 0, bits = 0;  // of the sort by digits
    int64_t tiles = 0;
    size_t array = 0, counts = 0, owners = 0, parts = 0;  // bytes; an array of n numbers
    int arrays = 0;
    size_t bytes() const { return arrays * array + counts + owners + parts; }
};
size_t round_up(size_t n) { return (n + 255) / 256 * 256; }
Shape shape_of(const vcsr_embed_grad_args& a) {
    Shape s;
    const int64_t v = a.y_type == VCSR_F32 ? 4 : 8, nv = ((int64_t)a.C + v - 1) / v;
    const int64_t slabs = (nv + 63) / 64;
    s.runs.slabs = (int)slabs;
    s.runs.width = (int)((nv + slabs - 1) / slabs);
    s.runs.E = 64;
    s.runs.ldp = nv * v;
    // Enough waves to have the chip's loads under way: 4000 tokens of 512 bf16 with E = 8
    // 16 us, 16 20, 64 40; of 130000 E = 32 and 64 are alike.
    while (s.runs.E > 8 && a.M / s.runs.E * slabs < 2048) s.runs.E /= 2;
    s.runs.chunks = (a.M + s.runs.E - 1) / s.runs.E;
    if (a.M <= 64) return s;
    s.array = round_up((size_t)a.M * 4);
    s.arrays = 2;
    if (!a.accumulate) s.owners = round_up((size_t)a.V * 4);
    s.parts = round_up((size_t)s.runs.chunks * 2 * (size_t)s.runs.ldp * 4);
    if (a.M <= kMostRanked) return s;
    int bits = 1;
    while (bits < 31 && a.V >> bits) ++bits;
    s.passes = (bits + 8) / 9;
    s.bits = (bits + s.passes - 1) / s.passes;
    if (s.passes > 1) s.arrays = 4;
    // A short tile's 64 keys a turn against as many counts to read: 24000 tokens 41.8 us,
    // 45 with tiles from 1024; 130000 90, 94 with 256 blocks; 400000 171, 181 with 128.
    s.tile = 512;
    while ((a.M + s.tile - 1) / s.tile > (s.tile < 2048 ? 128 : 256)) s.tile *= 2;
    s.tiles = (a.M + s.tile - 1) / s.tile;
    const int64_t rows = (s.tiles + kTogether - 1) / kTogether * kTogether;
    s.counts = round_up((size_t)rows << s.bits << 2);
    return s;
}

// Blocks of 256 threads that clear these rows, a group a wave or more.
int32_t zero_blocks(const Zeros& z) {
    const int64_t rows = 4 * zero_group(z.bytes), need = (z.rows + rows - 1) / rows;
    return (int32_t)(need < 4096 ? need : 4096);
}

template <class D, class X, int ENDS>
hipError_t launch_sums(const vcsr_embed_grad_args& a, const Shape& s, const Zeros& z,
                       hipStream_t st) {
    Runs r = s.runs;
    const int64_t blocks = (r.chunks * r.slabs + 3) / 4;
    if (a.M <= 64) {
        embed_sum_kernel<D, X, ENDS, true>
            <<<(unsigned)blocks + (unsigned)zero_blocks(z), 256, 0, st>>>(a, r, z, (int32_t)blocks);
        return hipGetLastError();
    }
    for (int64_t b = 0; b < blocks; b += kMostBlocks) {
        const int64_t count = blocks - b < kMostBlocks ? blocks - b : kMostBlocks;
        r.first = 4 * b;
        const unsigned zeros = b == 0 ? (unsigned)zero_blocks(z) : 0;
        embed_sum_kernel<D, X, ENDS, false>
            <<<(unsigned)count + zeros, 256, 0, st>>>(a, r, z, (int32_t)count);
    }
    for (int64_t c = 0; c < r.chunks; c += kMostBlocks) {
        const int64_t count = r.chunks - c < kMostBlocks ? r.chunks - c : kMostBlocks;
        r.first = c;
        embed_join_kernel<X><<<dim3((unsigned)count, (unsigned)((a.C + 255) / 256)), 256, 0, st>>>(
            a, r);
    }
    return hipGetLastError();
}
template <class D, class X>
hipError_t launch_grad(const vcsr_embed_grad_args& a, const Shape& s, const Zeros& z,
                       hipStream_t st) {
    switch (ends_of<16 / (int)sizeof(D)>(a.C)) {
        case kWhole: return launch_sums<D, X, kWhole>(a, s, z, st);
        case kRagged: return launch_sums<D, X, kRagged>(a, s, z, st);
        default: return launch_sums<D, X, kShort>(a, s, z, st);
    }
}

}  // namespace

hipError_t launch_embed(const vcsr_embed_args& a, hipStream_t st) {
    if (a.M <= 0) return hipSuccess;
    if (a.table_type == VCSR_F32)
        return a.y_type == VCSR_F32 ? launch_forward<float, float>(a, st)
                                    : launch_forward<float, bf16>(a, st);
    if (a.table_type == VCSR_BF16)
        return a.y_type == VCSR_F32 ? launch_forward<bf16, float>(a, st)
                                    : launch_forward<bf16, bf16>(a, st);
    return a.y_type == VCSR_F32 ? launch_forward<fp8, float>(a, st)
                                : launch_forward<fp8, bf16>(a, st);
}

EmbedGradPlan embed_grad_plan(const vcsr_embed_grad_args& a) {
    if (a.M <= 0) return EmbedGradPlan{};
    const Shape s = shape_of(a);
    return EmbedGradPlan{a.M <= 64 ? 0 : a.M <= kMostRanked ? 1 : 2, s.passes, s.bits, s.tile,
                         s.runs.E};
}

size_t embed_grad_workspace(const vcsr_embed_grad_args& a) {
    return a.M > 0 ? shape_of(a).bytes() : 0;
}

hipError_t launch_embed_grad(const vcsr_embed_grad_args& a, hipStream_t st) {
    const int64_t size = a.table_type == VCSR_F32 ? 4 : 2;
    if (a.M <= 0)
        return a.accumulate ? hipSuccess
                            : launch_zero(a.dtable, a.lddt * size, a.V, a.C * size, st);
    Shape s = shape_of(a);
    char* const base = (char*)a.workspace;
    auto array = [&](int i) { return (int32_t*)(base + i * s.array); };
    int32_t* const counts = (int32_t*)(base + s.arrays * s.array);
    int32_t* const owner = s.owners ? (int32_t*)((char*)counts + s.counts) : nullptr;
    const Zeros zeros{(uint8_t*)a.dtable, a.lddt * size, a.C * size, a.accumulate ? 0 : a.V,
                      owner, a.ids, (int32_t)a.M, (int64_t)a.V * a.C * size >= kLarge};
    if (a.M > 64) {
        s.runs.keys = array(0);
        s.runs.pos = array(1);
        s.runs.part = (float*)((char*)counts + s.counts + s.owners);
    }
    if (a.M > 64 && a.M <= kMostRanked) {
        rank_kernel<<<(unsigned)((a.M + 15) / 16), 512, 0, st>>>(a.ids, (int32_t)a.M, a.V, array(0),
                                                                array(1), owner);
    } else if (a.M > 64) {
        for (int p = 0; p < s.passes; ++p) {
            const int to = (s.passes - 1 - p) % 2 * 2;  // the last digit's go to 0 and 1
            const Radix r{p ? array(2 - to) : a.ids, p ? array(3 - to) : nullptr, (int32_t)a.M, a.V,
                          s.tile, p * s.bits, 1 << s.bits, p ? nullptr : owner};
            digit_count_kernel<<<(unsigned)s.tiles, 256, 0, st>>>(r, counts);
            digit_place_kernel<<<(unsigned)s.tiles, 256, 0, st>>>(r, counts, array(to),
                                                                  array(to + 1));
        }
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.y_type == VCSR_F32)
        return a.table_type == VCSR_F32 ? launch_grad<float, float>(a, s, zeros, st)
                                        : launch_grad<float, bf16>(a, s, zeros, st);
    return a.table_type == VCSR_F32 ? launch_grad<bf16, float>(a, s, zeros, st)
                                    : launch_grad<bf16, bf16>(a, s, zeros, st);
}

}  // namespace vcsr
