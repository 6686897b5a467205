// A cache of keys and values for single tokens: complete blocks of 64 tokens in 8 bits with a scale for each block and head, the newest ones in 16.
//
//   pages   codes[page][kv head][64][d] int8, scales[page][kv head] fp32, and of the keys sums[page][kv head][d] int16: the sum of a block's codes
//   rings   [tail][kv head][128][d] 16 bit: token t of the sequence whose ring it is stands at t % 128, for the tokens of the last two blocks
//   table   [sequence][max_blocks]: the page of each complete block
//
// A block is rounded once, when its last token arrives: scale = max |x| * fp32(1 / 127), code = rint(x / scale).
#pragma once
#include <type_traits>

#include "blocks.cuh"
#include "common.cuh"
#include "tc_ptx.cuh"

namespace vs {
namespace cache {

using blocks::from_f32;
using blocks::kBlock;
using blocks::load8;
using blocks::to_f32;

constexpr int kRing = 2 * kBlock;

struct Pages {
    int pages, tails, kv_heads, d;
    int8_t *codes[2];    // keys, values
    float *scales[2];
    int16_t *sums;
    void *rings[2];
};
struct Sequences {
    int count;
    const int32_t *table;     // [count][max_blocks]
    int max_blocks;
    const int32_t *tails;     // [count]
    const int32_t *lengths;   // [count]
    // page of block j of sequence r, or -1
    __device__ __forceinline__ int page(int r, int j, int pages) const {
        if (j < 0 || j >= max_blocks) return -1;
        const int p = table[(int64_t)r * max_blocks + j];
        return p >= 0 && p < pages ? p : -1;
    }
};

// Two 16-bit elements in a word.
template <typename T> struct Two;
template <> struct Two<__half> {
    static __device__ __forceinline__ uint32_t most(uint32_t x, uint32_t y) {   // magnitudes; what is no number stays
        const __half2 m = __hmax2_nan(__habs2(*reinterpret_cast<const __half2 *>(&x)), __habs2(*reinterpret_cast<const __half2 *>(&y)));
        return *reinterpret_cast<const uint32_t *>(&m);
    }
    static __device__ __forceinline__ float2 floats(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
    static __device__ __forceinline__ float larger(uint32_t x) {
        const float2 f = floats(x);
        return __uint_as_float(max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
    }
};
template <> struct Two<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t most(uint32_t x, uint32_t y) {
        const __nv_bfloat162 m = __hmax2_nan(__habs2(*reinterpret_cast<const __nv_bfloat162 *>(&x)), __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&y)));
        return *reinterpret_cast<const uint32_t *>(&m);
    }
    static __device__ __forceinline__ float2 floats(uint32_t x) { return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)); }
    static __device__ __forceinline__ float larger(uint32_t x) {
        const float2 f = floats(x);
        return __uint_as_float(max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
    }
};

// ---- appending ------------------------------------------------------------------------------------------------------
// One CTA takes one block of one sequence and head, keys or values: a block that becomes complete is gathered from ring and new tokens by asynchronous copies, reduced
// and rounded out of shared memory.  A CTA is a chain of waits, so what counts is how many of them an SM holds: 12 with 16 KB each (with the block in
// registers of 256 threads 5, and 40 us for 13 000 tokens of 8 heads, d = 128; now 33, 2.5 TB/s; one token for each of 64 sequences 8.6, bound by the launch and two
// dependent loads).  The CTA of a sequence's first block alone writes the ring, after it has read it.
constexpr int kAppendThreads = 128;
struct AppendArgs {
    Pages c;
    Sequences s;
    int tokens, touched;      // most new tokens of a sequence, most blocks they can touch
    const int32_t *counts;    // [count] or null: tokens each
    const void *at[2];        // new keys and values [count][tokens][kv heads][d]
    int64_t batch[2], token[2], head[2];
};
template <typename T> __global__ void __launch_bounds__(kAppendThreads, 12) append_kernel(const AppendArgs a) {
    __shared__ uint32_t most[kAppendThreads / 32];
    extern __shared__ __align__(16) uint4 tile[];   // [64][d / 8]
    int16_t *part = reinterpret_cast<int16_t *>(tile);   // [groups of tokens][d], once the block has been rounded
    const int kv = blockIdx.y, tid = threadIdx.x;
    // neighbouring CTAs take the heads of one block, whose tokens lie side by side
    const uint32_t block = blockIdx.x / (uint32_t)a.c.kv_heads;
    const int h = (int)(blockIdx.x - block * a.c.kv_heads), r = (int)(block / (uint32_t)a.touched), x = (int)(block - (uint32_t)r * a.touched);
    const int before = max(a.s.lengths[r], 0), fresh = a.counts ? min(max(a.counts[r], 0), a.tokens) : a.tokens, tail = a.s.tails[r];
    const int total = min(before, 0x7fffffff - fresh) + fresh, j = before / kBlock + x;
    const int d = a.c.d;
    if (tail < 0 || tail >= a.c.tails || fresh == 0) return;
    T *ring = static_cast<T *>(a.c.rings[kv]) + ((int64_t)tail * a.c.kv_heads + h) * kRing * d;
    const T *news = static_cast<const T *>(a.at[kv]) + r * a.batch[kv] + h * a.head[kv];
    const int chunks = d / 8, groups = kAppendThreads / chunks, c = tid % chunks, g = tid / chunks;   // 8 dimensions to a thread
    if (total / kBlock > j) {   // the same for all threads
        const uint32_t tile_at = tc::smem_u32(tile);
        for (int o = g; o < kBlock && g < groups; o += groups) {
            const int t = j * kBlock + o;
            tc::cp_async_16(tile_at + (o * chunks + c) * 16,
                            t < before ? ring + (int64_t)(t % kRing) * d + c * 8 : news + (int64_t)(t - before) * a.token[kv] + c * 8, 16);
        }
        tc::cp_async_commit();
        const int page = a.s.page(r, j, a.c.pages);
        auto block_max = [&](float mine) {   // of magnitudes; what is no number counts as the largest
            const uint32_t bits = __reduce_max_sync(~0u, __float_as_uint(mine) & 0x7fffffffu);
            if (tid % 32 == 0) most[tid / 32] = bits;
            __syncthreads();
            uint32_t all = 0;
#pragma unroll
            for (int w = 0; w < kAppendThreads / 32; ++w) all = max(all, most[w]);
            return all;
        };
        tc::cp_async_wait<0>();   // a thread reads what it has copied itself
        uint32_t high = 0;
        for (int o = g; o < kBlock && g < groups; o += groups) {
            const uint4 v = tile[o * chunks + c];
            high = Two<T>::most(high, Two<T>::most(Two<T>::most(v.x, v.y), Two<T>::most(v.z, v.w)));
        }
        uint32_t top = block_max(Two<T>::larger(high));
        const bool odd = top >= 0x7f800000u;   // something is not finite: it does not set the scale
        if (odd) {
            float mine = 0.f;
            for (int x4 = tid; x4 < kBlock * chunks * 4; x4 += kAppendThreads) {
                const float2 f = Two<T>::floats(reinterpret_cast<const uint32_t *>(tile)[x4]);
                if (fabsf(f.x) <= 3.402823466e38f) mine = fmaxf(mine, fabsf(f.x));
                if (fabsf(f.y) <= 3.402823466e38f) mine = fmaxf(mine, fabsf(f.y));
            }
            __syncthreads();   // (copies of all threads have been here since the barrier in the first maximum)
            top = block_max(mine);
        }
        if (page >= 0) {
            const float scale = __uint_as_float(top) * (1.f / 127.f);
            int8_t *codes = a.c.codes[kv] + ((int64_t)page * a.c.kv_heads + h) * kBlock * d;
            // x / scale correctly rounded decides the code, but only next to a half does it matter: elsewhere x times the reciprocal rounds the same way.  Adding
            // 1.5 * 2^23 rounds to a whole number whose low byte is the code.  Two elements to an instruction: this is what bounds a long prompt.
            constexpr float kWhole = 12582912.f;
            const bool exactly = odd || !(scale > 1e-30f);   // the reciprocal's own range
            const float inverse = exactly ? 0.f : 1.f / scale;
            uint32_t sum[8] = {};
            int count = 0;
#pragma unroll 2
            for (int o = g; o < kBlock && g < groups; o += groups) {
                const uint4 v = tile[o * chunks + c];
                const uint32_t in[4] = {v.x, v.y, v.z, v.w};
                uint32_t code[8];
                float off = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 q = blocks::fma2(Two<T>::floats(in[e]), make_float2(inverse, inverse), make_float2(0.f, 0.f));
                    const float2 whole = blocks::fma2(q, make_float2(1.f, 1.f), make_float2(kWhole, kWhole));
                    const float2 rest = blocks::fma2(blocks::fma2(whole, make_float2(1.f, 1.f), make_float2(-kWhole, -kWhole)), make_float2(-1.f, -1.f), q);
                    off = fmaxf(off, fmaxf(fabsf(rest.x), fabsf(rest.y)));
                    code[2 * e] = __float_as_uint(whole.x);
                    code[2 * e + 1] = __float_as_uint(whole.y);
                }
                if (exactly || off >= 0.4999f)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = Two<T>::floats(in[e]);
                        const float q[2] = {scale > 0.f ? rintf(__fdiv_rn(f.x, scale)) : 0.f, scale > 0.f ? rintf(__fdiv_rn(f.y, scale)) : 0.f};
#pragma unroll
                        for (int z = 0; z < 2; ++z) code[2 * e + z] = __float_as_uint((q[z] == q[z] ? fminf(fmaxf(q[z], -127.f), 127.f) : 0.f) + kWhole);
                    }
                ++count;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += code[e];
                uint32_t word[2];
#pragma unroll
                for (int e = 0; e < 8; e += 4)
                    word[e / 4] = __byte_perm(__byte_perm(code[e], code[e + 1], 0x0040), __byte_perm(code[e + 2], code[e + 3], 0x0040), 0x5410);
                *reinterpret_cast<uint2 *>(codes + (int64_t)o * d + c * 8) = make_uint2(word[0], word[1]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] -= count * __float_as_uint(kWhole);
            if (tid == 0) a.c.scales[kv][(int64_t)page * a.c.kv_heads + h] = scale;
            if (kv == 0) {
                __syncthreads();
                if (g < groups) {
                    // sums of a thread's codes, 16 bits each
                    *reinterpret_cast<uint4 *>(part + g * d + c * 8) = make_uint4(__byte_perm(sum[0], sum[1], 0x5410), __byte_perm(sum[2], sum[3], 0x5410),
                                                                                  __byte_perm(sum[4], sum[5], 0x5410), __byte_perm(sum[6], sum[7], 0x5410));
                }
                __syncthreads();
                for (int e = tid; e < d; e += kAppendThreads) {
                    int all = 0;
                    for (int y = 0; y < groups; ++y) all += part[y * d + e];
                    a.c.sums[((int64_t)page * a.c.kv_heads + h) * d + e] = (int16_t)all;
                }
            }
        }
    }
    if (x == 0) {
        __syncthreads();
        const int first = max(before, (total / kBlock - 1) * kBlock);
        if (g < groups)
            for (int t = first + g; t < total; t += groups)
                *reinterpret_cast<uint4 *>(ring + (int64_t)(t % kRing) * d + c * 8) =
                    *reinterpret_cast<const uint4 *>(news + (int64_t)(t - before) * a.token[kv] + c * 8);
    }
}

// ---- choosing blocks for single tokens --------------------------------------------------------------------------------
// Score of a complete block: (sum of the group's query heads) . (sum of the block's codes) * scale, in 64 bits.  The newest complete block is always
// taken.  A CTA per (sequence, kv head); 16 lanes take a block's sums, 8 dimensions each, four blocks in flight.  Bound by 64-bit products and the sums over
// lanes, then by the ranking: 64 sequences of up to 256 blocks, 8 heads, d = 128: 20 us (26 MB, 1.3 TB/s;
// 23 where nothing of them is in L2).
constexpr int kSelectThreads = 1024;   // at most
struct SelectArgs {
    Pages c;
    Sequences s;
    const void *q;       // [count][heads][d]
    int64_t batch, head;
    int group, wanted;
    int32_t *lists;      // [count][kv heads][wanted]
};
template <typename T> __global__ void __launch_bounds__(kSelectThreads) select_kernel(const SelectArgs a) {
    extern __shared__ double sm[];
    const int d = a.c.d, h = blockIdx.x % a.c.kv_heads, r = blockIdx.x / a.c.kv_heads;
    const int full = min(max(a.s.lengths[r], 0) / kBlock, a.s.max_blocks);
    const int tid = threadIdx.x, c = tid % 16 * 8;
    uint64_t *keys = reinterpret_cast<uint64_t *>(sm);
    uint32_t *taken = reinterpret_cast<uint32_t *>(keys + a.s.max_blocks);
    double sum[8] = {};
    if (c < d)
        for (int g = 0; g < a.group; ++g) {
            float f[8];
            load8(static_cast<const T *>(a.q) + r * a.batch + (h * a.group + g) * a.head + c, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += f[e];
        }
    constexpr int kFlight = 4;
    const int stride = blockDim.x / 16;
    for (int j0 = tid / 16; j0 - tid / 16 < full; j0 += kFlight * stride) {   // the same number of rounds for all lanes
        int page[kFlight];
        uint4 v[kFlight];
#pragma unroll
        for (int y = 0; y < kFlight; ++y) {
            const int j = j0 + y * stride;
            page[y] = j < full ? a.s.page(r, j, a.c.pages) : -1;
        }
#pragma unroll
        for (int y = 0; y < kFlight; ++y) {
            v[y] = make_uint4(0, 0, 0, 0);
            if (page[y] >= 0 && c < d) v[y] = *reinterpret_cast<const uint4 *>(a.c.sums + ((int64_t)page[y] * a.c.kv_heads + h) * d + c);
        }
#pragma unroll
        for (int y = 0; y < kFlight; ++y) {
            const int16_t *e16 = reinterpret_cast<const int16_t *>(&v[y]);
            double dot = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) dot = fma(sum[e], (double)e16[e], dot);
#pragma unroll
            for (int o = 8; o; o >>= 1) dot += __shfl_xor_sync(~0u, dot, o);
            const int j = j0 + y * stride;
            if (j < full && tid % 16 == 0)   // a block without a page cannot be had
                keys[j] = page[y] >= 0 ? blocks::sortable(dot * (double)a.c.scales[0][(int64_t)page[y] * a.c.kv_heads + h]) : 0ull;
        }
    }
    const int words = (a.s.max_blocks + 31) / 32;
    for (int x = tid; x < words; x += blockDim.x) taken[x] = full > 0 && (full - 1) / 32 == x ? 1u << ((full - 1) & 31) : 0u;
    __syncthreads();
    if (tid < 32) {
        blocks::take_best(keys, full - 1, a.wanted - 1, taken);
        __syncwarp();
        blocks::write_list(taken, words, a.wanted, a.lists + (int64_t)blockIdx.x * a.wanted);
    }
}

// ---- attention of single tokens ------------------------------------------------------------------------------------------
// A warp takes whole blocks: asynchronous copies bring a block's codes of one head (64 d bytes, contiguous) into its own ring in shared memory, two
// pieces ahead, and mma.sync multiplies the group's query rows (up to 16) with them.  Few rows against a stream of keys: bound by the reading of
// the cache, which tcgen05 tiles of 128 rows would not make quicker, while here codes go from bytes to fragments without another trip.  32 sequences of up to 128
// blocks, 8 heads, d = 128, groups of 4: 392 MB in 91 us, 4.3 TB/s; with the copies and no arithmetic 77.  4 sequences of 16 chosen blocks 14.5 us.
// Codes are exact in fp16 (below); the scale of a block of keys goes onto the scores, that of the values onto the block's
// product in fp32 before it joins the sums.  Probabilities are rounded to fp16 for the product (2^-11 relative; they are at most 1).  bf16 queries become
// fp16 without a rounding that counts: a row is multiplied by the power of two that brings its largest element to 1 .. 2, so what falls below fp16's
// normal range is off by less than 2^-24 of that element, fp32's own resolution.
//
// Fragments: a score product steps over 16 dimensions, and which 16 is free as long as both operands agree, so lane (key g, quad c) keeps the d / 4
// bytes from c d / 4 on of its key and uses four of them a step.  A value product steps over 16 keys in the order in which the scores' accumulators hold them;
// its columns are free: lane g keeps four consecutive dimensions 32 u + 4 g of every 32 (and two of the last 16), one column of each
// of the eight-wide tiles that they belong to.
constexpr int kWarps = 4, kDecodeThreads = kWarps * 32, kSlots = 3;

struct AttentionArgs {
    Pages c;
    Sequences s;
    const void *q;
    int64_t batch, head;
    int group, parts, pieces;   // query heads of a kv head, parts of 16 of them, pieces of a sequence's blocks
    const int32_t *lists;       // [count][kv heads][wanted] or null: all complete blocks
    int wanted;
    float scale;
    void *out;                  // [count][heads][d]
    float *partial;             // [count * kv heads * parts][pieces][16][d + 2] when pieces > 1
};

__device__ __forceinline__ uint32_t half2_bits(__half2 x) { return *reinterpret_cast<uint32_t *>(&x); }
// Codes as fp16 operands: code + 128 is a byte u, and the fp16 with the bits 0x00uu is u * 2^-24, exactly, so that spreading bytes is all the conversion there is.
// Products are taken of u; what 128 makes of them is where their sums start.
constexpr uint32_t kBias = 0x80808080u;
constexpr float kUnit = 0x1p24f, kStart = -0x1p-17f;   // 1 / 2^-24; -128 * 2^-24
__device__ __forceinline__ void key_codes(uint32_t word, uint32_t &lo, uint32_t &hi) {
    word ^= kBias;
    lo = __byte_perm(word, 0u, 0x4140);
    hi = __byte_perm(word, 0u, 0x4342);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack(float x, float y);
template <> __device__ __forceinline__ uint32_t pack<__half>(float x, float y) { return half2_bits(__floats2half2_rn(x, y)); }
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// dimension of accumulator column n (0 .. 7) of value tile t
template <int NK> __device__ __forceinline__ int value_dim(int t, int n) {
    const int full = NK / 2 * 4;   // tiles of the whole groups of 32
    return t < full ? t / 4 * 32 + n * 4 + t % 4 : NK / 2 * 32 + n * 2 + (t - full);
}

template <typename T, int NK> struct Rows {   // what a warp carries from block to block: rows g and g + 8
    float acc[2 * NK][4];
    float top[2], total[2];
};

// Scores of 64 keys (columns 8 n + 2 c, + 1 of rows g, g + 8) to probabilities, with the running maximum and sum; `n` keys are there.  factor: not negative.
template <typename T, int NK> __device__ __forceinline__ void softmax_step(Rows<T, NK> &r, float (&s)[8][4], const float (&factor)[2], int n) {
    const int c = threadIdx.x & 3;
    if (n < kBlock) {
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (x * 8 + 2 * c + (e & 1) >= n) s[x][e] = -INFINITY;
    }
    float shrink[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float m = -INFINITY;
#pragma unroll
        for (int x = 0; x < 8; ++x) m = fmaxf(m, fmaxf(s[x][2 * i], s[x][2 * i + 1]));
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 1));
        m = fmaxf(r.top[i], fmaxf(m, __shfl_xor_sync(~0u, m, 2)) * factor[i]);
        const float base = m == -INFINITY ? 0.f : m;
        shrink[i] = ex2(r.top[i] - base);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
            for (int e = 2 * i; e < 2 * i + 2; ++e) {
                s[x][e] = ex2(fmaf(s[x][e], factor[i], -base));
                sum[e & 1] += s[x][e];
            }
        r.total[i] = r.total[i] * shrink[i] + (sum[0] + sum[1]);   // this lane's part of the row: joined at the end
        r.top[i] = m;
    }
    if (__any_sync(~0u, shrink[0] != 1.f || shrink[1] != 1.f)) {   // seldom, once the first blocks have gone by
#pragma unroll
        for (int t = 0; t < 2 * NK; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) r.acc[t][e] *= shrink[e >> 1];
    }
}

// d / 4 bytes of a key, as wide as they lie aligned
template <int NK> __device__ __forceinline__ void key_words(const uint8_t *p, uint32_t (&w)[NK]) {
    if constexpr (NK % 4 == 0) {
#pragma unroll
        for (int x = 0; x < NK; x += 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(p + 4 * x);
            w[x] = v.x; w[x + 1] = v.y; w[x + 2] = v.z; w[x + 3] = v.w;
        }
    } else if constexpr (NK % 2 == 0) {
#pragma unroll
        for (int x = 0; x < NK; x += 2) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p + 4 * x);
            w[x] = v.x; w[x + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int x = 0; x < NK; ++x) w[x] = *reinterpret_cast<const uint32_t *>(p + 4 * x);
    }
}
// A piece in shared memory: 64 rows of d bytes, 16 apart, so that the lanes of a fragment, which read eight rows (keys) or every second one (values), meet different
// banks (bulk copies cannot leave a gap: 8 and 4 lanes to a bank).
template <int NK> constexpr int kPitch = NK * 16 + 16;
template <int NK> constexpr int kPieceBytes = kBlock * kPitch<NK>;
template <int NK> constexpr int decode_smem() {
    constexpr int pieces = kWarps * kSlots * kPieceBytes<NK>, join = kWarps * 16 * (NK * 16 + 2) * 4;
    return pieces > join ? pieces : join;
}

template <typename T, int NK> __global__ void __launch_bounds__(kDecodeThreads, 2) decode_kernel(const AttentionArgs a) {
    constexpr int D = NK * 16, P = kPitch<NK>;
    extern __shared__ __align__(128) uint8_t raw[];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int piece = blockIdx.x % a.pieces, item = blockIdx.x / a.pieces;
    const int part = item % a.parts, h = item / a.parts % a.c.kv_heads, r = item / a.parts / a.c.kv_heads;
    const int len = max(a.s.lengths[r], 0), full = min(len / kBlock, a.s.max_blocks), rest = len % kBlock;
    const int tail = a.s.tails[r];
    const int32_t *list = a.lists ? a.lists + ((int64_t)r * a.c.kv_heads + h) * a.wanted : nullptr;
    const int units = list ? a.wanted : full;
    const int lo = (int)((int64_t)units * piece / a.pieces), hi = (int)((int64_t)units * (piece + 1) / a.pieces);
    uint8_t *ring = raw + warp * kSlots * kPieceBytes<NK>;
    const uint32_t ring_at = tc::smem_u32(ring);

    // Page of unit u, or -1: a list's entry counts where it names a complete block with a page and the list has not named it before.
    auto page_of = [&](int u) {
        int j = u;
        if (list) {
            j = list[u];
            if (j < 0 || j >= full) return -1;
            bool again = false;
            for (int x = lane; x < u; x += 32) again |= list[x] == j;
            if (__any_sync(~0u, again)) return -1;
        }
        return a.s.page(r, j, a.c.pages);
    };
    struct Unit {
        int at, page;
        float sk, sv;
    };
    // the warp's next unit with a page, from u on, and its scales
    auto next = [&](int u) {
        Unit x = {hi, -1, 0.f, 0.f};
        for (; u < hi; u += kWarps)
            if ((x.page = page_of(u)) >= 0) {
                x.at = u;
                x.sk = a.c.scales[0][(int64_t)x.page * a.c.kv_heads + h];
                x.sv = a.c.scales[1][(int64_t)x.page * a.c.kv_heads + h];
                break;
            }
        return x;
    };
    uint32_t sent = 0, used = 0;   // pieces requested and used so far: keys and values of one block after another
    auto request = [&](int kv, const Unit &x) {   // one group of copies, an empty one where there is no unit
        if (x.at < hi) {
            const uint8_t *from = reinterpret_cast<const uint8_t *>(a.c.codes[kv]) + ((int64_t)x.page * a.c.kv_heads + h) * (kBlock * D);
            const uint32_t to = ring_at + sent % kSlots * kPieceBytes<NK>;
#pragma unroll
            for (int y = 0; y < 2 * NK; ++y) {   // 64 rows of NK chunks
                const int chunk = lane + 32 * y;
                tc::cp_async_16(to + chunk / NK * P + chunk % NK * 16, from + chunk * 16, 16);
            }
        }
        tc::cp_async_commit();
        ++sent;
    };
    auto arrived = [&]() -> const uint8_t * {   // the oldest piece; two younger ones may be on their way
        tc::cp_async_wait<2>();
        __syncwarp();
        return ring + used++ % kSlots * kPieceBytes<NK>;
    };

    // query rows: a[0] (row g, dimensions c D/4 + 4 s + 0, 1), a[1] row g + 8, a[2], a[3] dimensions + 2, + 3
    auto query = [&](uint32_t (&f)[NK][4]) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int x = part * 16 + g + 8 * i;
            const T *p = static_cast<const T *>(a.q) + r * a.batch + (int64_t)(h * a.group + x) * a.head + c * (D / 4);
#pragma unroll
            for (int s = 0; s < NK; ++s) {
                uint2 v = make_uint2(0, 0);
                if (x < a.group) v = *reinterpret_cast<const uint2 *>(p + 4 * s);
                f[s][i] = v.x;
                f[s][2 + i] = v.y;
            }
        }
    };
    uint32_t qf[NK][4];
    query(qf);
    const float factor = a.scale * blocks::kLog2e;
    float row_factor[2] = {factor, factor};
    if constexpr (!std::is_same<T, __half>::value) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float most = 0.f;
            auto pair = [](uint32_t w) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w)); };
#pragma unroll
            for (int s = 0; s < 2 * NK; ++s) {
                const float2 f = pair(qf[s / 2][i + s % 2 * 2]);
                most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
            most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
            most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
            const uint32_t e = min(max(__float_as_uint(most) >> 23, 1u), 253u);
            const float down = __uint_as_float((254u - e) << 23);
            row_factor[i] = factor * __uint_as_float(e << 23);
#pragma unroll
            for (int s = 0; s < 2 * NK; ++s) {
                uint32_t &w = qf[s / 2][i + s % 2 * 2];
                const float2 f = pair(w);
                w = pack<__half>(f.x * down, f.y * down);
            }
        }
    }
    float start[2];   // of the rows' sums with codes + 128
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float sum = 0.f;
#pragma unroll
        for (int s = 0; s < 2 * NK; ++s) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&qf[s / 2][i + s % 2 * 2]));
            sum += f.x + f.y;
        }
        sum += __shfl_xor_sync(~0u, sum, 1);
        sum += __shfl_xor_sync(~0u, sum, 2);
        start[i] = kStart * sum;
        row_factor[i] *= kUnit;
    }
    Rows<T, NK> rows;
#pragma unroll
    for (int t = 0; t < 2 * NK; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) rows.acc[t][e] = 0.f;
    rows.top[0] = rows.top[1] = -INFINITY;
    rows.total[0] = rows.total[1] = 0.f;

    // Pieces in the order K0 V0 K1 V1 ...; two are on their way ahead of the one in use.
    Unit now = next(lo + warp), then = {hi, -1, 0.f, 0.f};
    if (now.at < hi) {
        request(0, now);
        request(1, now);
        then = next(now.at + kWarps);
    }
    while (now.at < hi) {
        request(0, then);   // into the third slot
        const uint8_t *k = arrived();
        float s[8][4];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            s[x][0] = s[x][1] = start[0];
            s[x][2] = s[x][3] = start[1];
            uint32_t w[NK];
            key_words<NK>(k + (x * 8 + g) * P + c * (D / 4), w);
#pragma unroll
            for (int y = 0; y < NK; ++y) {
                uint32_t b0, b1;
                key_codes(w[y], b0, b1);
                mma<__half>(s[x], qf[y], b0, b1);
            }
        }
        __syncwarp();
        request(1, then);   // where the keys stood
        const Unit after = then.at < hi ? next(then.at + kWarps) : then;
        const float factors[2] = {row_factor[0] * now.sk, row_factor[1] * now.sk}, sv = now.sv * kUnit;
        softmax_step<T, NK>(rows, s, factors, kBlock);
        const uint8_t *v = arrived();
        uint32_t pf[4][4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            pf[y][0] = pack<__half>(s[2 * y][0], s[2 * y][1]);
            pf[y][1] = pack<__half>(s[2 * y][2], s[2 * y][3]);
            pf[y][2] = pack<__half>(s[2 * y + 1][0], s[2 * y + 1][1]);
            pf[y][3] = pack<__half>(s[2 * y + 1][2], s[2 * y + 1][3]);
        }
        float from[4] = {};   // what 128 makes of the values' sums: the probabilities, as they were rounded, times -128
#pragma unroll
        for (int y = 0; y < 4; ++y) mma<__half>(from, pf[y], 0x00800080u, 0x00800080u);
        auto values = [&](const int t0, const int tiles, const int dim, const bool half_word) {   // `tiles` tiles from t0 on: one word (half a word) per key
            float o[4][4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[x][e] = -from[e];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                uint32_t even[4], odd[4];   // bytes 0 and 2, 1 and 3 of four keys' words, a half each
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint8_t *vp = v + (16 * y + 2 * c + (e & 1) + 8 * (e >> 1)) * P + dim;
                    const uint32_t w = (half_word ? (uint32_t)*reinterpret_cast<const uint16_t *>(vp) : *reinterpret_cast<const uint32_t *>(vp)) ^ kBias;
                    even[e] = w & 0x00ff00ffu;
                    odd[e] = __byte_perm(w, 0u, 0x4341);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (x >= tiles) continue;
                    const uint32_t sel = x < 2 ? 0x5410 : 0x7632;   // halves of two keys side by side
                    const uint32_t(&w)[4] = x % 2 ? odd : even;
                    mma<__half>(o[x], pf[y], __byte_perm(w[0], w[1], sel), __byte_perm(w[2], w[3], sel));
                }
            }
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (x < tiles)
#pragma unroll
                    for (int e = 0; e < 4; ++e) rows.acc[t0 + x][e] = fmaf(sv, o[x][e], rows.acc[t0 + x][e]);
        };
#pragma unroll
        for (int y = 0; y < NK / 2; ++y) values(4 * y, 4, 32 * y + 4 * g, false);
        if constexpr (NK % 2 == 1) values(NK / 2 * 4, 2, NK / 2 * 32 + 2 * g, true);
        __syncwarp();
        now = then;
        then = after;
    }
    tc::cp_async_wait<0>();

    // the newest tokens, 16 bits, straight from the ring: one warp of the last piece
    if (rest > 0 && piece == a.pieces - 1 && warp == (hi - lo) % kWarps && tail >= 0 && tail < a.c.tails) {
        const int64_t first = (((int64_t)tail * a.c.kv_heads + h) * kRing + len / kBlock % 2 * kBlock) * D;
        const T *k = static_cast<const T *>(a.c.rings[0]) + first, *v = static_cast<const T *>(a.c.rings[1]) + first;
        if constexpr (!std::is_same<T, __half>::value) query(qf);   // bf16 as they are: so are the ring's keys
        float s[8][4];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
            if (x * 8 >= rest) continue;
            const bool here = x * 8 + g < rest;
#pragma unroll
            for (int y = 0; y < NK; ++y) {
                uint2 w = make_uint2(0, 0);
                if (here) w = *reinterpret_cast<const uint2 *>(k + (int64_t)(x * 8 + g) * D + c * (D / 4) + 4 * y);
                mma<T>(s[x], qf[y], w.x, w.y);
            }
        }
        const float factors[2] = {factor, factor};
        softmax_step<T, NK>(rows, s, factors, rest);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            if (y * 16 >= rest) continue;
            uint32_t pf[4];
            pf[0] = pack<T>(s[2 * y][0], s[2 * y][1]);
            pf[1] = pack<T>(s[2 * y][2], s[2 * y][3]);
            pf[2] = pack<T>(s[2 * y + 1][0], s[2 * y + 1][1]);
            pf[3] = pack<T>(s[2 * y + 1][2], s[2 * y + 1][3]);
#pragma unroll
            for (int z = 0; z < (NK + 1) / 2; ++z) {
                const bool whole = z < NK / 2;
                const int dim = whole ? 32 * z + 4 * g : 32 * z + 2 * g;
                uint2 w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = 16 * y + 2 * c + (e & 1) + 8 * (e >> 1);
                    w[e] = make_uint2(0, 0);
                    if (t < rest) {
                        const T *p = v + (int64_t)t * D + dim;
                        if (whole) w[e] = *reinterpret_cast<const uint2 *>(p);
                        else w[e].x = *reinterpret_cast<const uint32_t *>(p);
                    }
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (!whole && x >= 2) continue;
                    const uint32_t sel = x % 2 ? 0x7632 : 0x5410;
                    const uint32_t b0 = x < 2 ? __byte_perm(w[0].x, w[1].x, sel) : __byte_perm(w[0].y, w[1].y, sel);
                    const uint32_t b1 = x < 2 ? __byte_perm(w[2].x, w[3].x, sel) : __byte_perm(w[2].y, w[3].y, sel);
                    mma<T>(rows.acc[z * 4 + x < 2 * NK ? z * 4 + x : 0], pf, b0, b1);
                }
            }
        }
    }

    // join the warps: [warp][16][D + 2] in the shared memory that the pieces have left
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        rows.total[i] += __shfl_xor_sync(~0u, rows.total[i], 1);
        rows.total[i] += __shfl_xor_sync(~0u, rows.total[i], 2);
    }
    __syncthreads();
    float *joined = reinterpret_cast<float *>(raw);
    float *mine = joined + warp * 16 * (D + 2);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float *row = mine + (g + 8 * i) * (D + 2);
        if (c == 0) {
            row[D] = rows.top[i];
            row[D + 1] = rows.total[i];
        }
#pragma unroll
        for (int t = 0; t < 2 * NK; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) row[value_dim<NK>(t, 2 * c + e)] = rows.acc[t][2 * i + e];
    }
    __syncthreads();
    const int live = min(16, a.group - part * 16);
    for (int x = threadIdx.x; x < live * D; x += kDecodeThreads) {
        const int row = x / D, dim = x % D;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, joined[(w * 16 + row) * (D + 2) + D]);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f, total = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float *p = joined + (w * 16 + row) * (D + 2);
            const float f = ex2(p[D] - base);
            sum = fmaf(f, p[dim], sum);
            total = fmaf(f, p[D + 1], total);
        }
        if (a.pieces == 1) {
            static_cast<T *>(a.out)[((int64_t)r * a.c.kv_heads * a.group + h * a.group + part * 16 + row) * D + dim] = from_f32<T>(total == 0.f ? 0.f : sum / total);
        } else {
            float *p = a.partial + ((int64_t)blockIdx.x * 16 + row) * (D + 2);
            p[dim] = sum;
            if (dim == 0) {
                p[D] = top;
                p[D + 1] = total;
            }
        }
    }
}

// Joins the pieces of a sequence: a CTA per (sequence, kv head, part of 16 query heads).  A few us behind the kernel above, bound by its launch.
template <typename T> __global__ void __launch_bounds__(128) join_kernel(const AttentionArgs a) {
    pdl_wait();
    const int item = blockIdx.x, D = a.c.d;
    const int part = item % a.parts, h = item / a.parts % a.c.kv_heads, r = item / a.parts / a.c.kv_heads;
    const int live = min(16, a.group - part * 16);
    for (int x = threadIdx.x; x < live * D; x += 128) {
        const int row = x / D, dim = x % D;
        const float *p = a.partial + ((int64_t)item * a.pieces * 16 + row) * (D + 2);
        const int64_t step = 16 * (D + 2);
        float top = -INFINITY;
        for (int y = 0; y < a.pieces; ++y) top = fmaxf(top, __ldcg(p + y * step + D));
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f, total = 0.f;
        for (int y = 0; y < a.pieces; ++y) {
            const float f = ex2(__ldcg(p + y * step + D) - base);
            sum = fmaf(f, __ldcg(p + y * step + dim), sum);
            total = fmaf(f, __ldcg(p + y * step + D + 1), total);
        }
        static_cast<T *>(a.out)[((int64_t)r * a.c.kv_heads * a.group + h * a.group + part * 16 + row) * D + dim] = from_f32<T>(total == 0.f ? 0.f : sum / total);
    }
}

}  // namespace cache
}  // namespace vs
