// Attention over blocks of 64 keys that are chosen for each query: the choice, the lists as bits, and the operators row by row.
//
// Query i of batch entry b stands at position p = i + keys - queries.  For every head of keys and query there is a list of blocks; the query's
// `group` heads (heads / kv_heads) attend to the keys t of the listed blocks with t < length and, causal, t <= p.
//
// The kernels that multiply take a tile of queries through the union of its lists, so the lists are first turned into bits:
// bits[b, kv head][word w][block j], bit x set when query 32 w + x has block j on its list and it can hold a key for that query.
// A list is a set here: order and repetitions do not count, and entries that are no block are none.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <type_traits>

#include "common.cuh"

namespace vs {
namespace blocks {

constexpr int kBlock = 64;
constexpr int kMaxD = 128;
constexpr int kMaxBlocks = 16384;   // per sequence: scores of one query fit in shared memory
constexpr int kMaxQueries = 0x7fff0000;      // tiles and chunks of tiles that reach past the last query are counted in 32 bits
constexpr int kMaxCount = 0x7fffffff / 32;   // entries of a list: those of a word's 32 lists too

struct Shape {
    int batch, queries, keys, heads, kv_heads, d, count;
    int causal;
    int group;    // heads / kv_heads
    int blocks;   // of keys
    int words;    // of 32 queries
    const int32_t *lengths;   // tokens of each batch entry (queries == keys), or null: all

    __device__ __forceinline__ int length(int b) const { return lengths ? min(max(lengths[b], 0), keys) : keys; }
    __device__ __forceinline__ int rows(int b) const { return lengths ? min(max(lengths[b], 0), queries) : queries; }
    __device__ __forceinline__ int position(int i) const { return i + keys - queries; }
    // keys that query i may attend to end here
    __device__ __forceinline__ int end(int i, int len) const { return causal ? min(len, position(i) + 1) : len; }
};
struct Operand {   // [batch, tokens, heads, d], the last dimension contiguous; strides in elements
    const void *at;
    int64_t batch, token, head;
};

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T> __device__ __forceinline__ void load8(const T *p, float (&f)[8]) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    const T *h = reinterpret_cast<const T *>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32(h[i]);
}

// Two fused multiply-adds: one instruction on this part.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\nfma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// ---- lists as bits ------------------------------------------------------------------------------------------------
// One CTA takes a word of 32 queries: it collects their bits in shared memory and writes the word's row for all blocks, so that nothing has to
// be cleared beforehand.  Bound by the reading of the lists and the launch: 4 x 16384 lists of 16 blocks 5.8 us.
constexpr int kBitsThreads = 128, kBitsChunk = 4096;
__global__ void __launch_bounds__(kBitsThreads) bits_kernel(const Shape s, const int32_t *lists, uint32_t *bits, uint32_t *zero) {
    __shared__ uint32_t row[kBitsChunk];
    pdl_launch_dependents();
    const int64_t at = blockIdx.x;
    const int w = (int)(at % s.words);
    if (zero && w == 0)   // a word for each block of a head of keys
        for (int j = threadIdx.x; j < s.blocks; j += kBitsThreads) zero[at / s.words * s.blocks + j] = 0;
    const int b = (int)(at / s.words / s.kv_heads);
    const int len = s.length(b), rows = s.rows(b);
    const int32_t *list = lists + (at / s.words * s.queries + w * 32) * s.count;
    const int entries = min(32, s.queries - w * 32) * s.count;
    for (int base = 0; base < s.blocks; base += kBitsChunk) {
        const int n = min(kBitsChunk, s.blocks - base);
        for (int j = threadIdx.x; j < n; j += kBitsThreads) row[j] = 0;
        __syncthreads();
        for (int e = threadIdx.x; e < entries; e += kBitsThreads) {
            const int x = e / s.count, i = w * 32 + x, j = list[e] - base;
            if (j >= 0 && j < n && i < rows && (int64_t)(base + j) * kBlock < s.end(i, len)) atomicOr(row + j, 1u << x);
        }
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += kBitsThreads) bits[at * s.blocks + base + j] = row[j];
        __syncthreads();
    }
}

// ---- choosing -----------------------------------------------------------------------------------------------------
// Score of block j for query i: (sum of the group's query heads) . (mean of the block's keys), everything in 64 bits: its order decides whole
// numbers, and 32-bit sums in two orders disagree about blocks that are close.
// A bound on the norm of up to kMaxD elements from the fp32 sum of their squares, in any order: a square below 2^-126 is off by 2^-150 at most, and one below 2^-150
// counts as nothing, so the sum by d 2^-149 and its root by less than 2^-70.
__device__ __forceinline__ float norm_bound(float squares) { return fmaf(sqrtf(squares), 1.001f, 0x1p-70f); }
// Means: one CTA per (b, kv head, block), 8 dimensions to a thread, the tokens shared by groups of threads; in 64 bits, and in 32 with a bound on their norm.
// Bound by the latency of its few loads: 1024 blocks of 64 tokens, d = 128, 14 us (1.2 TB/s).
constexpr int kMeanThreads = 128;
template <typename T> __global__ void __launch_bounds__(kMeanThreads) means_kernel(const Shape s, const Operand k, double *means, float *means32, float *norms) {
    __shared__ double part[kMeanThreads * 8];
    __shared__ float squares;
    pdl_launch_dependents();
    if (threadIdx.x == 0) squares = 0.f;
    const int64_t at = blockIdx.x;
    const int j = (int)(at % s.blocks), h = (int)(at / s.blocks % s.kv_heads), b = (int)(at / s.blocks / s.kv_heads);
    const int first = j * kBlock, n = min(kBlock, s.length(b) - first);
    const int chunks = s.d / 8, groups = kMeanThreads / chunks, c = threadIdx.x % chunks, g = threadIdx.x / chunks;
    double sum[8] = {};
    if (g < groups) {
        const T *p = static_cast<const T *>(k.at) + b * k.batch + first * k.token + h * k.head + c * 8;
        for (int t = g; t < n; t += groups) {
            float f[8];
            load8(p + t * k.token, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += f[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) part[(g * chunks + c) * 8 + i] = sum[i];
    }
    __syncthreads();
    for (int x = threadIdx.x; x < s.d; x += kMeanThreads) {
        double total = 0;
        for (int y = 0; y < groups; ++y) total += part[y * s.d + x];
        total = n > 0 ? total / n : 0.0;
        means[at * s.d + x] = total;
        const float rounded = (float)total;
        means32[at * s.d + x] = rounded;
        atomicAdd(&squares, rounded * rounded);   // a bound, with room for the order of its sum
    }
    __syncthreads();
    if (threadIdx.x == 0) norms[at] = norm_bound(squares);
}

// Scores as whole numbers of the same order, above 0; what is no number counts as the lowest score.
__device__ __forceinline__ uint64_t sortable(double x) {
    x = x != x ? -DBL_MAX : fmin(fmax(x, -DBL_MAX), DBL_MAX);
    const uint64_t u = (uint64_t)__double_as_longlong(x == 0.0 ? 0.0 : x);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
// A warp takes the `want` highest of keys[0 .. n) (0: not to be had) into `taken` bits, ties to the lowest index.  keys lose what is taken.
__device__ __forceinline__ void take_best(uint64_t *keys, int n, int want, uint32_t *taken) {
    const int lane = threadIdx.x & 31;
    uint64_t best = 0;
    int at = 0x7fffffff;
    auto scan = [&]() {
        best = 0;
        at = 0x7fffffff;
        for (int j = lane; j < n; j += 32)
            if (keys[j] > best) { best = keys[j]; at = j; }
    };
    scan();
    for (int x = 0; x < want; ++x) {
        const uint32_t hi = (uint32_t)(best >> 32), top = __reduce_max_sync(~0u, hi);
        const uint32_t lo = hi == top ? (uint32_t)best : 0u, low = __reduce_max_sync(~0u, lo);
        if (!(top | low)) break;
        const int winner = __reduce_min_sync(~0u, hi == top && lo == low ? at : 0x7fffffff);
        if (at == winner) {
            keys[at] = 0;
            taken[at >> 5] |= 1u << (at & 31);   // words are shared by lanes of a warp, but one lane writes at a time
            scan();
        }
        __syncwarp();
    }
}
// The set bits in ascending order, -1 behind them.
__device__ __forceinline__ void write_list(const uint32_t *taken, int words, int count, int32_t *list) {
    const int lane = threadIdx.x & 31;
    int done = 0;
    for (int base = 0; base < words; base += 32) {
        uint32_t w = base + lane < words ? taken[base + lane] : 0u;
        int before = __popc(w);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(~0u, before, o);
            if (lane >= o) before += y;
        }
        const int total = __shfl_sync(~0u, before, 31);
        int at = done + before - __popc(w);
        for (; w; w &= w - 1) list[at++] = (base + lane) * 32 + __ffs(w) - 1;
        done += total;
    }
    for (int x = done + lane; x < count; x += 32) list[x] = -1;
}

// Most lists need no more than 32 bits: fp32 scores are off by E at most, and where the last block taken and the first left lie further apart than 2 E, the
// choice is that of 64 bits.  Where they do not, the scores from 2 E below the last one on are computed again in 64.
// Two kernels, over slabs of queries whose scores stay in L2: a product of the queries' sums with the means, and a ranking by a warp per query, which needs many warps
// to cover what it waits for and would not have them beside the product's tiles (in one kernel, with 16 warps an SM: 212 us at 16384 x 16384, 4 heads of keys,
// d = 128; fp64 throughout, as below: 525).  Now the product takes 76, bound by fp32 arithmetic and its shared memory, and the ranking 115, bound by instructions;
// with the means and the launches 245.  Queries with more than kMembers candidates that are all alike fall out of it: 4096 queries, 2 heads on one, 1024 blocks of zeros 120 ms against 0.53.
constexpr int kFastThreads = 256, kFastQueries = 64, kFastBlocks = 128, kFastPiece = 64, kFastPitch = kFastPiece + 4, kMembers = 256, kFastCount = 128;
constexpr int kFastMost = 1024;   // blocks of a sequence
__host__ __device__ constexpr int fast_pitch(int d) { return (d + 63) / 64 * 64 + 4; }
constexpr int fast_bytes(int d) { return (kFastQueries * fast_pitch(d) + kFastBlocks * kFastPitch) * 4; }
struct Slab {   // tiles of kFastQueries queries of a head of keys, from `first` on
    int64_t first, tiles;
    float *scores;   // [tiles][kFastQueries][blocks]
    float *errors;   // [tiles][kFastQueries]: steps of 2^-24 that a score is off by at most, for a mean of norm 1
};
struct FastTile {
    int b, h, i0, most;   // most: candidates of any query of the tile
    int64_t bh;
    __device__ __forceinline__ FastTile(const Shape &s, int64_t tile) {   // in 32 bits: every launch has fewer tiles
        const uint32_t tiles = (s.queries + kFastQueries - 1) / kFastQueries, pair = (uint32_t)tile / tiles;
        bh = pair;
        i0 = (int)((uint32_t)tile - pair * tiles) * kFastQueries;
        b = (int)(pair / (uint32_t)s.kv_heads);
        h = (int)(pair - (uint32_t)b * s.kv_heads);
        const int last = min(i0 + kFastQueries, s.rows(b)) - 1;
        most = last < i0 ? 0 : s.causal ? s.position(last) / kBlock : (s.length(b) + kBlock - 1) / kBlock;
    }
};
struct Members {   // of one warp: the query in 64 bits, the blocks to be ranked again, and which of all are taken
    double q[kMaxD];
    uint64_t keys[kMembers];
    int16_t index[kMembers];
    uint32_t taken[kMembers / 32];
    uint32_t all[kFastMost / 32];
};

__device__ __forceinline__ uint32_t sortable32(float x) {
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unsortable32(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// One query's `want` best of n candidates into `taken`, in 64 bits: those with fp32 scores from `from` on, or all.
template <typename T> __device__ __forceinline__ void take_exactly(const Shape &s, const T *q, int64_t q_head, const double *means, const float *scores, float from, bool all, int n,
                                                                   int want, uint32_t *taken, Members &m) {
    const int lane = threadIdx.x & 31;
    for (int x = lane; x < s.d; x += 32) {
        double sum = 0;
        for (int g = 0; g < s.group; ++g) sum += to_f32(q[g * q_head + x]);
        m.q[x] = sum;
    }
    __syncwarp();
    auto exact = [&](int j) {
        double dot = 0;
        const double *p = means + (int64_t)j * s.d;
        for (int x = 0; x < s.d; ++x) dot = fma(m.q[x], p[x], dot);
        return sortable(dot);
    };
    int count = 0;
    for (int base = 0; base < n; base += 32) {
        const bool mine = base + lane < n && (all || !(scores[base + lane] < from));
        const uint32_t some = __ballot_sync(~0u, mine);
        const int at = count + __popc(some & ((1u << lane) - 1));
        if (mine && at < kMembers) m.index[at] = (int16_t)(base + lane);
        count += __popc(some);
    }
    if (count <= kMembers) {
        for (int x = lane; x < kMembers / 32; x += 32) m.taken[x] = 0;
        __syncwarp();
        for (int x = lane; x < count; x += 32) m.keys[x] = exact(m.index[x]);
        __syncwarp();
        take_best(m.keys, count, want, m.taken);
        __syncwarp();
        for (int x = lane; x < count; x += 32)
            if (m.taken[x / 32] >> (x % 32) & 1u) atomicOr(taken + m.index[x] / 32, 1u << (m.index[x] % 32));
    } else {   // scores that are all alike: one block after another
        for (int x = 0; x < want; ++x) {
            uint64_t best = 0;
            int at = 0x7fffffff;
            for (int j = lane; j < n; j += 32) {
                if (taken[j / 32] >> (j % 32) & 1u) continue;
                const uint64_t key = exact(j);
                if (key > best) { best = key; at = j; }
            }
            const uint32_t hi = (uint32_t)(best >> 32), top = __reduce_max_sync(~0u, hi), lo = hi == top ? (uint32_t)best : 0u, low = __reduce_max_sync(~0u, lo);
            if (!(top | low)) break;
            const int winner = __reduce_min_sync(~0u, hi == top && lo == low ? at : 0x7fffffff);
            if (lane == 0) taken[winner / 32] |= 1u << (winner % 32);
            __syncwarp();
        }
    }
    __syncwarp();
}

// Scores of a tile: 64 queries against all candidates of any of them, 128 blocks and 64 dimensions at a time, 4 x 8 to a thread.
template <typename T> __global__ void __launch_bounds__(kFastThreads, 2) fast_score_kernel(const Shape s, const Operand q, const float *means32, const Slab slab) {
    extern __shared__ __align__(16) float fsm[];
    const int pitch = fast_pitch(s.d), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    float *sums = fsm, *piece = sums + kFastQueries * pitch;
    __shared__ float summands[kFastQueries];   // squares of the norms of the heads' magnitudes, summed
    pdl_launch_dependents();
    const int64_t index = slab.tiles - 1 - blockIdx.x;   // the last queries have most candidates: they go first
    const FastTile t(s, slab.first + index);
    if (t.most == 0) {
        pdl_wait();   // as every CTA: the kernels behind take the end of this one for the end of all before it
        return;
    }
    const int rows = s.rows(t.b), chunks = fast_pitch(s.d) / 8;   // of 8 dimensions, zeros behind the last
    const T *qp = static_cast<const T *>(q.at) + t.b * q.batch + t.h * s.group * q.head;
    for (int x = tid; x < kFastQueries * chunks; x += kFastThreads) {
        const int i = x / chunks, c = x % chunks * 8;
        float sum[8] = {}, size[8] = {};
        if (t.i0 + i < rows && c < s.d) {
#pragma unroll 8
            for (int g = 0; g < s.group; ++g) {
                float f[8];
                load8(qp + (t.i0 + i) * q.token + g * q.head + c, f);
#pragma unroll
                for (int y = 0; y < 8; ++y) {
                    sum[y] += f[y];
                    size[y] += fabsf(f[y]);
                }
            }
        }
        float square = 0.f;
#pragma unroll
        for (int y = 0; y < 8; ++y) square = fmaf(size[y], size[y], square);
        for (int o = chunks / 2; o; o >>= 1) square += __shfl_xor_sync(~0u, square, o);   // 8 or 16 neighbours have a query; all lanes are here
        if (c == 0) summands[i] = square;
#pragma unroll
        for (int y = 0; y < 8; y += 4) *reinterpret_cast<float4 *>(sums + i * pitch + c + y) = make_float4(sum[y], sum[y + 1], sum[y + 2], sum[y + 3]);
    }
    __syncthreads();
    static_assert(kFastThreads == 4 * kFastQueries, "four threads to a query's norm");
    {
        const float *p = sums + tid / 4 * pitch;
        float square = 0.f;   // of the norm of the sum
        for (int x = tid % 4; x < s.d; x += 4) square = fmaf(p[x], p[x], square);
#pragma unroll
        for (int o = 2; o; o >>= 1) square += __shfl_xor_sync(~0u, square, o);
        pdl_wait();   // the means are the kernel's before, and whoever reads the last slab is done
        // one rounding for each of the d terms of a product and those of its operands, relative to the sum; one for each of the group's additions, relative to what is added,
        // which the sum itself may be far below
        if (tid % 4 == 0) slab.errors[index * kFastQueries + tid / 4] = (s.d + 8) * norm_bound(square) + (s.group - 1) * norm_bound(summands[tid / 4]);
    }
    // queries 4 ty .. 4 ty + 3, blocks tx + 16 x
    const int tx = lane % 16, ty = warp * 2 + lane / 16;
    float *out = slab.scores + index * kFastQueries * s.blocks;
    auto product = [&](auto blocks_each, int base) {
        constexpr int kEach = decltype(blocks_each)::value;   // blocks of a thread
        const int width = min(16 * kEach, t.most - base);
        float2 acc[4][kEach];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int x = 0; x < kEach; ++x) acc[r][x] = make_float2(0.f, 0.f);
        for (int d0 = 0; d0 < s.d; d0 += kFastPiece) {
            __syncthreads();
            for (int x = tid; x < 16 * kEach * (kFastPiece / 4); x += kFastThreads) {
                const int j = x / (kFastPiece / 4), y = x % (kFastPiece / 4) * 4;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (j < width && d0 + y < s.d) v = __ldcg(reinterpret_cast<const float4 *>(means32 + (t.bh * s.blocks + base + j) * s.d + d0 + y));
                *reinterpret_cast<float4 *>(piece + j * kFastPitch + y) = v;
            }
            __syncthreads();
#pragma unroll 2
            for (int y = 0; y < kFastPiece; y += 4) {
                float4 v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = *reinterpret_cast<const float4 *>(sums + (ty * 4 + r) * pitch + d0 + y);
#pragma unroll
                for (int x = 0; x < kEach; ++x) {
                    const float4 a = *reinterpret_cast<const float4 *>(piece + (tx + 16 * x) * kFastPitch + y);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        acc[r][x] = fma2(make_float2(v[r].x, v[r].y), make_float2(a.x, a.y), acc[r][x]);
                        acc[r][x] = fma2(make_float2(v[r].z, v[r].w), make_float2(a.z, a.w), acc[r][x]);
                    }
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int x = 0; x < kEach; ++x)
                if (tx + 16 * x < width) out[(int64_t)(ty * 4 + r) * s.blocks + base + tx + 16 * x] = acc[r][x].x + acc[r][x].y;
    };
    for (int base = 0; base < t.most;) {
        const int left = t.most - base;
        if (left > 64) product(std::integral_constant<int, 8>(), base), base += 128;
        else if (left > 32) product(std::integral_constant<int, 4>(), base), base += 64;
        else product(std::integral_constant<int, 2>(), base), base += 32;
    }
}

// The list of one query from its n > want > 0 candidates' scores.  A lane holds kHeld of them in registers; more are read each time.
template <typename T, int kHeld> __device__ __forceinline__ void rank_row(const Shape &s, const FastTile &t, const Operand &q, int i, int own, int n, int want, const float *row,
                                                                          const float *error, const double *means, const float *mean_norms, int32_t *list, Members &m) {
    const int lane = threadIdx.x & 31;
    float v[kHeld], top = -FLT_MAX, low = FLT_MAX, norm = 0.f;
    bool number = true;
#pragma unroll
    for (int x = 0; x < kHeld; ++x) v[x] = lane + 32 * x < n ? __ldcg(row + lane + 32 * x) : -INFINITY;   // below every threshold
    for (int j = lane; j < n; j += 32) {
        const float m = __ldcg(mean_norms + t.bh * s.blocks + j);
        norm = m <= FLT_MAX ? fmaxf(norm, m) : INFINITY;
        number &= m <= FLT_MAX;
    }
#pragma unroll
    for (int x = 0; x < kHeld; ++x)
        if (lane + 32 * x < n) {
            number &= fabsf(v[x]) <= FLT_MAX;
            top = fmaxf(top, v[x]);
            low = fminf(low, v[x]);
        }
    for (int j = lane + 32 * kHeld; j < n; j += 32) {
        const float f = __ldcg(row + j);
        number &= fabsf(f) <= FLT_MAX;
        top = fmaxf(top, f);
        low = fminf(low, f);
    }
    float hi = unsortable32(__reduce_max_sync(~0u, sortable32(top))), lo = unsortable32(__reduce_min_sync(~0u, sortable32(low))), at = 0.5f * hi + 0.5f * lo;
    // besides, products and sums below 2^-126 are off by 2^-150 each
    const float off = 0x1p-24f * __ldcg(error) * __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(norm))) * 1.01f + 0x1p-120f;
    const bool usable = __all_sync(~0u, number) && off <= FLT_MAX;
    bool found = false;
    int reach_lo = n, reach_hi = 1;   // how many reach lo: more than `want`; and hi: fewer, or, at first, perhaps as many
    for (int step = 1; usable && step < 32; ++step) {
        if (!(at > lo && at < hi)) break;   // nothing between: scores that are alike
        int count = 0;
#pragma unroll
        for (int x = 0; x < kHeld; ++x) count += v[x] >= at;
        for (int j = lane + 32 * kHeld; j < n; j += 32) count += __ldcg(row + j) >= at;
        count = __reduce_add_sync(~0u, count);
        if (count == want) {
            found = true;
            break;
        }
        if (count > want) lo = at, reach_lo = count;
        else hi = at, reach_hi = count;
        // as if the scores between lay evenly; every third step halves, whatever they do
        const float part = step % 3 == 0 ? 0.5f : fminf(fmaxf(__fdividef(reach_lo - want - 0.5f, (float)max(1, reach_lo - reach_hi)), 0.05f), 0.95f);
        at = lo + (hi - lo) * part;
    }
    bool near = !found;
#pragma unroll
    for (int x = 0; x < kHeld; ++x) near |= fabsf(v[x] - at) <= off;
    for (int j = lane + 32 * kHeld; j < n; j += 32) near |= fabsf(__ldcg(row + j) - at) <= off;
    if (__any_sync(~0u, near)) {
        const int words = (s.blocks + 31) / 32;
        for (int x = lane; x < words; x += 32) m.all[x] = own >= 0 && own / 32 == x ? 1u << (own & 31) : 0u;
        __syncwarp();
        take_exactly(s, static_cast<const T *>(q.at) + t.b * q.batch + t.h * s.group * q.head + i * q.token, q.head, means + t.bh * s.blocks * s.d, row,
                     (found ? at : lo) - 2.f * off, !usable, n, want, m.all, m);
        write_list(m.all, words, s.count, list);
        return;
    }
    int before = 0;
#pragma unroll
    for (int x = 0; x < kHeld; ++x) {
        const bool mine = v[x] >= at;
        const uint32_t all = __ballot_sync(~0u, mine);
        if (mine) list[before + __popc(all & ((1u << lane) - 1))] = lane + 32 * x;
        before += __popc(all);
    }
    for (int base = 32 * kHeld; base < n; base += 32) {
        const bool mine = base + lane < n && __ldcg(row + base + lane) >= at;
        const uint32_t all = __ballot_sync(~0u, mine);
        if (mine) list[before + __popc(all & ((1u << lane) - 1))] = base + lane;
        before += __popc(all);
    }
    if (own >= 0 && lane == 0) list[s.count - 1] = own;
}
// The lists of a slab, a warp to a query: it narrows the interval between two scores until just as many reach a value as are wanted, a step being a comparison for each
// score of a lane and one sum over the warp (taking the best one after another costs several times that for each).
template <typename T> __global__ void __launch_bounds__(kFastThreads) fast_rank_kernel(const Shape s, const Operand q, const double *means, const float *mean_norms, const Slab slab,
                                                                                      int32_t *lists) {
    __shared__ Members members_all[kFastThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    const int64_t row_index = slab.tiles * kFastQueries - 1 - ((int64_t)blockIdx.x * (kFastThreads / 32) + warp);   // as the scores were made
    const FastTile t(s, slab.first + (row_index >> 6));
    const int i = t.i0 + (int)(row_index & 63);
    static_assert(kFastQueries == 64, "shifts");
    pdl_wait();
    if (i >= s.queries) return;
    const int rows = s.rows(t.b), own = s.causal ? s.position(i) / kBlock : -1, n = i >= rows ? 0 : s.causal ? own : t.most, want = s.count - (own >= 0);
    int32_t *list = lists + (t.bh * s.queries + i) * s.count;
    if (n <= want || want == 0) {   // all candidates, or none
        const int all = i >= rows ? 0 : want > 0 ? n + (own >= 0) : 0;   // the query's own block follows its candidates
        for (int x = lane; x < s.count; x += 32) list[x] = x < all ? x : want == 0 && i < rows && x == 0 ? own : -1;
        return;
    }
    const float *row = slab.scores + row_index * s.blocks, *error = slab.errors + row_index;
    if (n <= 64) rank_row<T, 2>(s, t, q, i, own, n, want, row, error, means, mean_norms, list, members_all[warp]);
    else if (n <= 128) rank_row<T, 4>(s, t, q, i, own, n, want, row, error, means, mean_norms, list, members_all[warp]);
    else rank_row<T, 8>(s, t, q, i, own, n, want, row, error, means, mean_norms, list, members_all[warp]);
}

// 64 bits throughout, for lists and sequences that the kernel above has no room for.
// One CTA scores QT queries of one head of keys against all their candidates, 64 blocks and 32 dimensions at a time, and each of its warps
// then takes the best of one query after another.  Shared memory: the queries' sums, a piece of the means, the scores.
constexpr int kScoreThreads = 256, kPiece = 32;
template <int QT> constexpr int64_t score_bytes(int blocks, int d) {
    return (int64_t)QT * (d + 1) * 8 + (int64_t)kBlock * (kPiece + 1) * 8 + (int64_t)QT * blocks * 8 + (int64_t)(kScoreThreads / 32) * ((blocks + 31) / 32) * 4;
}
template <typename T, int QT> __global__ void __launch_bounds__(kScoreThreads) score_kernel(const Shape s, const Operand q, const double *means, int32_t *lists) {
    extern __shared__ double sm[];
    double *sums = sm, *piece = sums + QT * (s.d + 1), *scores = piece + kBlock * (kPiece + 1);
    uint32_t *taken_all = reinterpret_cast<uint32_t *>(scores + (int64_t)QT * s.blocks);
    const int tiles = (s.queries + QT - 1) / QT;
    const int64_t bh = blockIdx.x / tiles;
    const int i0 = (int)(blockIdx.x % tiles) * QT, h = (int)(bh % s.kv_heads), b = (int)(bh / s.kv_heads);
    const int len = s.length(b), rows = s.rows(b), tid = threadIdx.x;
    const int last = min(i0 + QT, rows) - 1;   // last query of the tile that is there
    const int most = last < i0 ? 0 : s.causal ? s.position(last) / kBlock : (len + kBlock - 1) / kBlock;   // candidates of any of them

    const T *qp = static_cast<const T *>(q.at) + b * q.batch + h * s.group * q.head;
    for (int x = tid; x < QT * (s.d / 8); x += kScoreThreads) {
        const int i = x / (s.d / 8), c = x % (s.d / 8) * 8;
        double sum[8] = {};
        if (i0 + i < rows)
            for (int g = 0; g < s.group; ++g) {
                float f[8];
                load8(qp + (i0 + i) * q.token + g * q.head + c, f);
#pragma unroll
                for (int y = 0; y < 8; ++y) sum[y] += f[y];
            }
#pragma unroll
        for (int y = 0; y < 8; ++y) sums[i * (s.d + 1) + c + y] = sum[y];
    }
    constexpr int kRows = QT >= 16 ? QT / 16 : 1;   // queries of a thread; the 16 threads of a row of threads take 4 blocks each
    const int tx = tid % 16, ty = tid / 16;
    for (int base = 0; base < most; base += kBlock) {
        double acc[kRows][4] = {};
        for (int d0 = 0; d0 < s.d; d0 += kPiece) {
            const int width = min(kPiece, s.d - d0);
            __syncthreads();
            for (int x = tid; x < kBlock * kPiece; x += kScoreThreads) {
                const int j = x / kPiece, y = x % kPiece;
                piece[j * (kPiece + 1) + y] = base + j < most && y < width ? means[(bh * s.blocks + base + j) * s.d + d0 + y] : 0.0;
            }
            __syncthreads();
            if (ty * kRows < QT)
                for (int y = 0; y < width; ++y) {
                    double a[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) a[x] = piece[(tx + 16 * x) * (kPiece + 1) + y];
#pragma unroll
                    for (int r = 0; r < kRows; ++r) {
                        const double v = sums[(ty * kRows + r) * (s.d + 1) + d0 + y];
#pragma unroll
                        for (int x = 0; x < 4; ++x) acc[r][x] = fma(v, a[x], acc[r][x]);
                    }
                }
        }
        if (ty * kRows < QT)
#pragma unroll
            for (int r = 0; r < kRows; ++r)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (base + tx + 16 * x < most) scores[(int64_t)(ty * kRows + r) * s.blocks + base + tx + 16 * x] = acc[r][x];
    }
    __syncthreads();
    const int warp = tid >> 5, lane = tid & 31, words = (s.blocks + 31) / 32;
    uint32_t *taken = taken_all + warp * words;
    for (int r = warp; r < QT && i0 + r < s.queries; r += kScoreThreads / 32) {
        const int i = i0 + r, own = s.causal ? s.position(i) / kBlock : -1;
        int32_t *list = lists + (bh * s.queries + i) * s.count;
        const int n = i >= rows ? 0 : s.causal ? own : most;
        uint64_t *keys = reinterpret_cast<uint64_t *>(scores + (int64_t)r * s.blocks);
        for (int j = lane; j < n; j += 32) keys[j] = sortable(__longlong_as_double((long long)keys[j]));
        for (int x = lane; x < words; x += 32) taken[x] = i < rows && own >= 0 && own / 32 == x ? 1u << (own & 31) : 0u;
        __syncwarp();
        take_best(keys, n, s.count - (own >= 0), taken);
        __syncwarp();
        write_list(taken, words, s.count, list);
        __syncwarp();
    }
}

// ---- attention, row by row ------------------------------------------------------------------------------------------
// The operators straight from their formulas, on the CUDA cores, in fp32: a warp takes a row (query, head), its lanes the keys of a block two by two for
// the scores and then the dimensions for the sums.  Keys that a row does not attend to are not read, so what stands there cannot reach it, whatever it is.
// `redo`: one word per tile of `tile` queries (forward, dQ) or per block of keys (dK, dV); only those with a word that is not 0 are computed.
// Bound by reads of keys from L2, 64 d bytes twice for every row and block: all of 16384 x 16384, 32 heads on 4, d = 128, 16 blocks each, takes them 50 ms.
struct Args {
    Shape s;
    Operand q, k, v, out, grad_out;   // out and grad_out as q
    const uint32_t *bits;
    float *lse;           // [batch, heads, queries] base 2; +inf: the row attends to nothing
    float *delta;         // the same shape: rowsum(out o grad_out)
    uint32_t *most;       // as lse, fp16 alone: largest finite magnitude of a row of grad_out, as the bits of a float
    uint32_t *peak;       // [batch, kv_heads, blocks], fp16 alone: the largest of those of the rows that have listed a block
    const void *out_low;  // what rounding left of out, as out; or null
    void *result;         // out or grad_q, contiguous
    void *result_low;     // out_low or null
    void *grad_k, *grad_v;
    float *aside;         // sums that grad_kv_kernel has put aside, where a block can have more tiles than it sums at a stretch
    const uint32_t *redo;
    int tile;
    float scale;
};
constexpr int kRowThreads = 128, kRowWarps = kRowThreads / 32;
constexpr float kLog2e = 1.4426950408889634f;

template <typename T> __device__ __forceinline__ float dot_row(const float *a, const T *p, int d) {
    float sum = 0.f;
    for (int c = 0; c < d; c += 8) {
        float f[8];
        load8(p + c, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(a[c + i], f[i], sum);
    }
    return sum;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
    return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    return x;
}

template <typename T, bool kBackward> __global__ void __launch_bounds__(kRowThreads) rows_kernel(const Args a) {
    __shared__ float q_s[kRowWarps][kMaxD], g_s[kRowWarps][kMaxD];
    pdl_wait();
    const Shape &s = a.s;
    const int tiles = (s.queries + a.tile - 1) / a.tile, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t index = blockIdx.x; index < (int64_t)s.batch * s.kv_heads * tiles; index += gridDim.x) {
        if (a.redo && a.redo[index] == 0) continue;
        const int64_t bh = index / tiles;
        const int i0 = (int)(index % tiles) * a.tile, kvh = (int)(bh % s.kv_heads), b = (int)(bh / s.kv_heads), len = s.length(b);
        const T *kp = static_cast<const T *>(a.k.at) + b * a.k.batch + kvh * a.k.head;
        const T *vp = static_cast<const T *>(a.v.at) + b * a.v.batch + kvh * a.v.head;
        const float c = a.scale * kLog2e;
        for (int r = warp; r < a.tile * s.group; r += kRowWarps) {
            const int i = i0 + r / s.group, h = kvh * s.group + r % s.group;
            if (i >= s.queries) break;
            const int64_t row = ((int64_t)b * s.heads + h) * s.queries + i;
            const T *qp = static_cast<const T *>(a.q.at) + b * a.q.batch + (int64_t)i * a.q.token + h * a.q.head;
            const T *gp = kBackward ? static_cast<const T *>(a.grad_out.at) + b * a.grad_out.batch + (int64_t)i * a.grad_out.token + h * a.grad_out.head : nullptr;
            __syncwarp();
            for (int x = lane; x < s.d; x += 32) {
                q_s[warp][x] = to_f32(qp[x]);
                if (kBackward) g_s[warp][x] = to_f32(gp[x]);
            }
            __syncwarp();
            const int end = s.end(i, len);
            const uint32_t *bits = a.bits + (bh * s.words + (i >> 5)) * s.blocks;
            float top = -INFINITY, total = 0.f, acc[kMaxD / 32] = {};
            const float lse = kBackward ? a.lse[row] : 0.f, delta = kBackward ? a.delta[row] : 0.f;
            for (int j = 0; j < s.blocks; ++j) {
                if (!(bits[j] >> (i & 31) & 1u)) continue;
                const int n = min(kBlock, end - j * kBlock);
                float w[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int t = lane + 32 * x;
                    w[x] = -INFINITY;
                    if (t < n) w[x] = dot_row(q_s[warp], kp + (int64_t)(j * kBlock + t) * a.k.token, s.d) * c;
                }
                if (!kBackward) {
                    const float m = fmaxf(top, warp_max(fmaxf(w[0], w[1]))), base = m == -INFINITY ? 0.f : m;
                    const float shrink = exp2f(top - base);
                    w[0] = lane < n ? exp2f(w[0] - base) : 0.f;
                    w[1] = lane + 32 < n ? exp2f(w[1] - base) : 0.f;
                    total = total * shrink + warp_sum(w[0] + w[1]);
                    top = m;
#pragma unroll
                    for (int x = 0; x < kMaxD / 32; ++x) acc[x] *= shrink;
                } else {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int t = lane + 32 * x;
                        float ds = 0.f;
                        if (t < n) ds = exp2f(w[x] - lse) * (dot_row(g_s[warp], vp + (int64_t)(j * kBlock + t) * a.v.token, s.d) - delta) * a.scale;
                        w[x] = ds;
                    }
                }
                for (int t = 0; t < n; ++t) {
                    const float p = __shfl_sync(~0u, t < 32 ? w[0] : w[1], t & 31);
                    const T *row_t = (kBackward ? kp : vp) + (int64_t)(j * kBlock + t) * (kBackward ? a.k.token : a.v.token);
#pragma unroll
                    for (int x = 0; x < kMaxD / 32; ++x)
                        if (lane + 32 * x < s.d) acc[x] = fmaf(p, to_f32(row_t[lane + 32 * x]), acc[x]);
                }
            }
            const int64_t at = (((int64_t)b * s.queries + i) * s.heads + h) * s.d;
#pragma unroll
            for (int x = 0; x < kMaxD / 32; ++x)
                if (lane + 32 * x < s.d) {
                    const float y = kBackward ? acc[x] : total == 0.f ? 0.f : acc[x] / total;
                    const T high = from_f32<T>(y);
                    static_cast<T *>(a.result)[at + lane + 32 * x] = high;
                    if (!kBackward && a.result_low) static_cast<T *>(a.result_low)[at + lane + 32 * x] = from_f32<T>(y - to_f32(high));
                }
            if (!kBackward && lane == 0) a.lse[row] = total == 0.f ? INFINITY : top + log2f(total);
        }
    }
}

// dK and dV of the keys of one block: a warp takes a key, its lanes the queries of a word for the scores and then the dimensions for the sums.
template <typename T> __global__ void __launch_bounds__(kRowThreads) keys_kernel(const Args a) {
    __shared__ float k_s[kRowWarps][kMaxD], v_s[kRowWarps][kMaxD];
    pdl_wait();
    const Shape &s = a.s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float c = a.scale * kLog2e;
    for (int64_t index = blockIdx.x; index < (int64_t)s.batch * s.kv_heads * s.blocks; index += gridDim.x) {
        if (a.redo && a.redo[index] == 0) continue;
        const int64_t bh = index / s.blocks;
        const int j = (int)(index % s.blocks), kvh = (int)(bh % s.kv_heads), b = (int)(bh / s.kv_heads), len = s.length(b);
        for (int t = j * kBlock + warp; t < min(s.keys, (j + 1) * kBlock); t += kRowWarps) {
            float dk[kMaxD / 32] = {}, dv[kMaxD / 32] = {};
            if (t < len) {
                const T *kp = static_cast<const T *>(a.k.at) + b * a.k.batch + (int64_t)t * a.k.token + kvh * a.k.head;
                const T *vp = static_cast<const T *>(a.v.at) + b * a.v.batch + (int64_t)t * a.v.token + kvh * a.v.head;
                __syncwarp();
                for (int x = lane; x < s.d; x += 32) {
                    k_s[warp][x] = to_f32(kp[x]);
                    v_s[warp][x] = to_f32(vp[x]);
                }
                __syncwarp();
                for (int w = 0; w < s.words; ++w) {
                    const int i = w * 32 + lane;
                    const bool here = (a.bits[(bh * s.words + w) * s.blocks + j] >> lane & 1u) && t < s.end(i, len);
                    const uint32_t rows = __ballot_sync(~0u, here);
                    if (!rows) continue;
                    for (int g = 0; g < s.group; ++g) {
                        const int h = kvh * s.group + g;
                        const T *qp = static_cast<const T *>(a.q.at) + b * a.q.batch + h * a.q.head;
                        const T *gp = static_cast<const T *>(a.grad_out.at) + b * a.grad_out.batch + h * a.grad_out.head;
                        float p = 0.f, ds = 0.f;
                        if (here) {
                            const int64_t row = ((int64_t)b * s.heads + h) * s.queries + i;
                            p = exp2f(dot_row(k_s[warp], qp + (int64_t)i * a.q.token, s.d) * c - a.lse[row]);
                            ds = p * (dot_row(v_s[warp], gp + (int64_t)i * a.grad_out.token, s.d) - a.delta[row]) * a.scale;
                        }
                        for (uint32_t left = rows; left; left &= left - 1) {
                            const int x = __ffs(left) - 1;
                            const float px = __shfl_sync(~0u, p, x), dx = __shfl_sync(~0u, ds, x);
#pragma unroll
                            for (int y = 0; y < kMaxD / 32; ++y) {
                                const int e = lane + 32 * y;
                                if (e < s.d) {
                                    dv[y] = fmaf(px, to_f32(gp[(int64_t)(w * 32 + x) * a.grad_out.token + e]), dv[y]);
                                    dk[y] = fmaf(dx, to_f32(qp[(int64_t)(w * 32 + x) * a.q.token + e]), dk[y]);
                                }
                            }
                        }
                    }
                }
            }
            const int64_t at = (((int64_t)b * s.keys + t) * s.kv_heads + kvh) * s.d;
#pragma unroll
            for (int y = 0; y < kMaxD / 32; ++y)
                if (lane + 32 * y < s.d) {
                    static_cast<T *>(a.grad_k)[at + lane + 32 * y] = from_f32<T>(dk[y]);
                    static_cast<T *>(a.grad_v)[at + lane + 32 * y] = from_f32<T>(dv[y]);
                }
        }
    }
}

// rowsum(out o grad_out) of each row and, fp16, the largest magnitude of its grad_out that is a finite number; 0 of rows behind a sequence's end.  Eight dimensions to a lane, 16 lanes
// to a row.  Bound by the reading of its three operands: 262 144 rows, d = 128: 50 us (4.0 TB/s).
template <typename T> __global__ void __launch_bounds__(256) delta_kernel(const Args a) {
    const Shape &s = a.s;
    const int64_t at = (int64_t)blockIdx.x * 16 + threadIdx.x / 16, all = (int64_t)s.batch * s.queries * s.heads;
    const int c = threadIdx.x % 16 * 8;
    const int h = (int)(at % s.heads), i = (int)(at / s.heads % s.queries), b = (int)(at / s.heads / s.queries);
    pdl_wait();
    pdl_launch_dependents();
    float sum = 0.f, most = 0.f;
    if (at < all && c < s.d && i < s.rows(b)) {
        float o[8], g[8];
        load8(static_cast<const T *>(a.out.at) + b * a.out.batch + (int64_t)i * a.out.token + h * a.out.head + c, o);
        load8(static_cast<const T *>(a.grad_out.at) + b * a.grad_out.batch + (int64_t)i * a.grad_out.token + h * a.grad_out.head + c, g);
        if (a.out_low) {
            float low[8];
            load8(static_cast<const T *>(a.out_low) + at * s.d + c, low);
#pragma unroll
            for (int x = 0; x < 8; ++x) sum = fmaf(low[x], g[x], sum);
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            sum = fmaf(o[x], g[x], sum);
            if (std::is_same<T, __half>::value && fabsf(g[x]) <= FLT_MAX) most = fmaxf(most, fabsf(g[x]));
        }
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) {
        sum += __shfl_xor_sync(~0u, sum, o);
        if (std::is_same<T, __half>::value) most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
    }
    if (at < all && c == 0) {
        const int64_t row = ((int64_t)b * s.heads + h) * s.queries + i;
        a.delta[row] = sum;
        if (std::is_same<T, __half>::value) a.most[row] = __float_as_uint(most);
    }
}

// The largest of `most` among the rows that have listed a block: a CTA takes a word of 32 queries, all heads of the group.  Bound by its launch: a
// training step of 4 x 2048 queries and 16 heads takes 337 us with it and 331 with one maximum for the whole call.
__global__ void __launch_bounds__(kBitsThreads) peaks_kernel(const Args a) {
    __shared__ uint32_t query[32];
    const Shape &s = a.s;
    const int64_t at = blockIdx.x, bh = at / s.words;
    const int w = (int)(at % s.words), kvh = (int)(bh % s.kv_heads), b = (int)(bh / s.kv_heads), lane = threadIdx.x & 31, i = w * 32 + lane;
    if (threadIdx.x < 32) query[lane] = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    uint32_t most = 0;
    if (i < s.queries)
        for (int g = threadIdx.x >> 5; g < s.group; g += kBitsThreads / 32) most = max(most, __ldcg(a.most + ((int64_t)b * s.heads + kvh * s.group + g) * s.queries + i));
    atomicMax(query + lane, most);   // maxima: the order does not count
    __syncthreads();
    for (int j = threadIdx.x; j < s.blocks; j += kBitsThreads) {
        uint32_t rows = __ldcg(a.bits + at * s.blocks + j), top = 0;
        if (!rows) continue;
        for (; rows; rows &= rows - 1) top = max(top, query[__ffs(rows) - 1]);
        atomicMax(a.peak + bh * s.blocks + j, top);
    }
}

}  // namespace blocks
}  // namespace vs
