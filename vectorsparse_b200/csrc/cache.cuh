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

// ---- appending ------------------------------------------------------------------------------------------------------
// One CTA takes one block of one sequence and head, keys or values: a block that becomes complete is gathered from ring and new tokens, reduced
// and rounded out of registers.  The CTA of a sequence's first block alone writes the ring, after it has read it.
constexpr int kAppendThreads = 256;
struct AppendArgs {
    Pages c;
    Sequences s;
    int tokens, touched;      // most new tokens of a sequence, most blocks they can touch
    const int32_t *counts;    // [count] or null: tokens each
    const void *at[2];        // new keys and values [count][tokens][kv heads][d]
    int64_t batch[2], token[2], head[2];
};
template <typename T> __global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
    __shared__ float most[kAppendThreads / 32];
    __shared__ int part[kAppendThreads * 8];   // [groups of tokens][d]
    const int kv = blockIdx.y, tid = threadIdx.x;
    const int64_t at = blockIdx.x;
    const int x = (int)(at % a.touched), h = (int)(at / a.touched % a.c.kv_heads), r = (int)(at / a.touched / a.c.kv_heads);
    const int before = max(a.s.lengths[r], 0), fresh = a.counts ? min(max(a.counts[r], 0), a.tokens) : a.tokens;
    const int total = min(before, 0x7fffffff - fresh) + fresh, j = before / kBlock + x;
    const int tail = a.s.tails[r], d = a.c.d;
    if (tail < 0 || tail >= a.c.tails || fresh == 0) return;
    T *ring = static_cast<T *>(a.c.rings[kv]) + ((int64_t)tail * a.c.kv_heads + h) * kRing * d;
    const T *news = static_cast<const T *>(a.at[kv]) + r * a.batch[kv] + h * a.head[kv];
    const int chunks = d / 8, groups = kAppendThreads / chunks, c = tid % chunks, g = tid / chunks;   // 8 dimensions to a thread
    const int page = total / kBlock > j ? a.s.page(r, j, a.c.pages) : -1;   // the same for all threads
    if (page >= 0) {
        constexpr int kPer = 4;   // tokens of a thread
        static_assert(kBlock * (blocks::kMaxD / 8) <= kPer * kAppendThreads, "threads for a block");
        float f[kPer][8];
        float top = 0.f;
#pragma unroll
        for (int y = 0; y < kPer; ++y) {
            const int o = g + y * groups, t = j * kBlock + o;
            const bool here = g < groups && o < kBlock;
#pragma unroll
            for (int e = 0; e < 8; ++e) f[y][e] = 0.f;
            if (here) load8(t < before ? ring + (int64_t)(t % kRing) * d + c * 8 : news + (int64_t)(t - before) * a.token[kv] + c * 8, f[y]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float m = fabsf(f[y][e]);
                if (m <= 3.402823466e38f) top = fmaxf(top, m);   // what is not finite does not set the scale
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        if (tid % 32 == 0) most[tid / 32] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kAppendThreads / 32; ++w) top = fmaxf(top, most[w]);
        const float scale = top * (1.f / 127.f);
        int8_t *codes = a.c.codes[kv] + ((int64_t)page * a.c.kv_heads + h) * kBlock * d;
        int sum[8] = {};
#pragma unroll
        for (int y = 0; y < kPer; ++y) {
            const int o = g + y * groups;
            if (g >= groups || o >= kBlock) continue;
            uint32_t word[2] = {};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float q = scale > 0.f ? rintf(__fdiv_rn(f[y][e], scale)) : 0.f;
                const int code = q == q ? (int)fminf(fmaxf(q, -127.f), 127.f) : 0;
                sum[e] += code;
                word[e / 4] |= (uint32_t)(code & 255) << (e % 4 * 8);
            }
            *reinterpret_cast<uint2 *>(codes + (int64_t)o * d + c * 8) = make_uint2(word[0], word[1]);
        }
        if (tid == 0) a.c.scales[kv][(int64_t)page * a.c.kv_heads + h] = scale;
        if (kv == 0) {
            if (g < groups)
#pragma unroll
                for (int e = 0; e < 8; ++e) part[g * d + c * 8 + e] = sum[e];
            __syncthreads();
            for (int e = tid; e < d; e += kAppendThreads) {
                int all = 0;
                for (int y = 0; y < groups; ++y) all += part[y * d + e];
                a.c.sums[((int64_t)page * a.c.kv_heads + h) * d + e] = (int16_t)all;
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
// taken.  A CTA per (sequence, kv head); 16 lanes take a block's sums, 8 dimensions each, four blocks in flight.
struct SelectArgs {
    Pages c;
    Sequences s;
    const void *q;       // [count][heads][d]
    int64_t batch, head;
    int group, wanted;
    int32_t *lists;      // [count][kv heads][wanted]
};
template <typename T> __global__ void select_kernel(const SelectArgs a) {
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
// A warp takes whole blocks: bulk copies bring a block's codes of one head (64 d bytes, contiguous) into its own ring in shared memory, two to three
// pieces ahead, and mma.sync multiplies the group's query rows (up to 16) with them.  Few rows against a stream of keys: bound by the reading of
// the cache, which tcgen05 tiles of 128 rows would not make quicker, while here codes go from bytes to fragments without another trip.
// Codes are whole numbers up to 127, exact in fp16; the scale of a block of keys goes onto the scores, that of the values onto the block's
// product in fp32 before it joins the sums.  Probabilities are rounded to fp16 for the product (2^-11 relative; they are at most 1).  bf16 queries become
// fp16 without a rounding that counts: a row is multiplied by the power of two that brings its largest element to 1 .. 2, so what falls below fp16's
// normal range is off by less than 2^-24 of that element, fp32's own resolution.
//
// Fragments: a score product steps over 16 dimensions, and which 16 is free as long as both operands agree, so lane (key g, quad c) keeps the d / 4
// bytes from c d / 4 on of its key and uses four of them a step.  A value product steps over 16 keys in the order in which the scores' accumulators hold them;
// its columns are free: lane g keeps four consecutive dimensions 32 u + 4 g of every 32 (and two of the last 16), one column of each
// of the eight-wide tiles that they belong to.
constexpr int kWarps = 4, kDecodeThreads = kWarps * 32, kSlots = 3;
constexpr uint32_t kStatusTimeout = 4096u;   // bit raised in the status word when a bounded wait ran out

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
    uint32_t *status;
};

__device__ __forceinline__ uint32_t half2_bits(__half2 x) { return *reinterpret_cast<uint32_t *>(&x); }
// bytes 0, 1 (2, 3) of a word of biased codes as two fp16: 0x6400 | x is 1024 + x
__device__ __forceinline__ uint32_t codes_f16(uint32_t biased_pair) {
    const __half2 off = __half2half2(__ushort_as_half((unsigned short)0x6480));   // 1024 + 128
    const uint32_t w = biased_pair;
    return half2_bits(__hsub2(*reinterpret_cast<const __half2 *>(&w), off));
}
__device__ __forceinline__ void key_codes(uint32_t word, uint32_t &lo, uint32_t &hi) {
    word ^= 0x80808080u;
    lo = codes_f16(__byte_perm(word, 0x64646464u, 0x4140));
    hi = codes_f16(__byte_perm(word, 0x64646464u, 0x4342));
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

// Scores of 64 keys (columns 8 n + 2 c, + 1 of rows g, g + 8) to probabilities, with the running maximum and sum; `n` keys are there.
template <typename T, int NK> __device__ __forceinline__ void softmax_step(Rows<T, NK> &r, float (&s)[8][4], const float (&factor)[2], int n) {
    const int c = threadIdx.x & 3;
#pragma unroll
    for (int x = 0; x < 8; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[x][e] = x * 8 + 2 * c + (e & 1) < n ? s[x][e] * factor[e >> 1] : -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float m = r.top[i];
#pragma unroll
        for (int x = 0; x < 8; ++x) m = fmaxf(m, fmaxf(s[x][2 * i], s[x][2 * i + 1]));
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 1));
        m = fmaxf(m, __shfl_xor_sync(~0u, m, 2));
        const float base = m == -INFINITY ? 0.f : m, shrink = exp2f(r.top[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
            for (int e = 2 * i; e < 2 * i + 2; ++e) {
                s[x][e] = exp2f(s[x][e] - base);
                sum += s[x][e];
            }
        r.total[i] = r.total[i] * shrink + sum;   // this lane's part of the row: joined at the end
        r.top[i] = m;
#pragma unroll
        for (int t = 0; t < 2 * NK; ++t) {
            r.acc[t][2 * i] *= shrink;
            r.acc[t][2 * i + 1] *= shrink;
        }
    }
}

template <typename T, int NK> __global__ void __launch_bounds__(kDecodeThreads, 2) decode_kernel(const AttentionArgs a) {
    constexpr int D = NK * 16, kPiece = kBlock * D;   // bytes of a block's codes
    extern __shared__ __align__(128) uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[kWarps][kSlots];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int piece = blockIdx.x % a.pieces, item = blockIdx.x / a.pieces;
    const int part = item % a.parts, h = item / a.parts % a.c.kv_heads, r = item / a.parts / a.c.kv_heads;
    const int len = max(a.s.lengths[r], 0), full = min(len / kBlock, a.s.max_blocks), rest = len % kBlock;
    const int tail = a.s.tails[r];
    const int32_t *list = a.lists ? a.lists + ((int64_t)r * a.c.kv_heads + h) * a.wanted : nullptr;
    const int units = list ? a.wanted : full;
    const int lo = (int)((int64_t)units * piece / a.pieces), hi = (int)((int64_t)units * (piece + 1) / a.pieces);
    uint8_t *ring = raw + warp * kSlots * kPiece;
    const uint32_t ring_at = tc::smem_u32(ring), bar = tc::smem_u32(&bars[warp][0]);
    if (lane < kSlots) tc::mbar_init(bar + 8 * lane, 1);
    tc::fence_mbar_init();
    __syncwarp();

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
    // the warp's next unit with a page, from u on
    auto next = [&](int u, int &page) {
        for (; u < hi; u += kWarps)
            if ((page = page_of(u)) >= 0) return u;
        return hi;
    };
    uint32_t sent = 0;   // pieces requested so far: keys and values of one block after another
    auto request = [&](int kv, int page) {
        const uint32_t slot = sent % kSlots;
        if (lane == 0) {
            tc::mbar_expect_tx(bar + 8 * slot, kPiece);
            tc::bulk_copy_g2s(ring_at + slot * kPiece, a.c.codes[kv] + ((int64_t)page * a.c.kv_heads + h) * kPiece, kPiece, bar + 8 * slot);
        }
        ++sent;
    };
    bool ok = true;
    uint32_t used = 0;
    auto arrived = [&]() -> const uint8_t * {   // the oldest piece
        const uint32_t slot = used % kSlots;
        ok = ok && tc::mbar_wait(bar + 8 * slot, (used / kSlots) & 1);
        return ring + slot * kPiece;
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
    Rows<T, NK> rows;
#pragma unroll
    for (int t = 0; t < 2 * NK; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) rows.acc[t][e] = 0.f;
    rows.top[0] = rows.top[1] = -INFINITY;
    rows.total[0] = rows.total[1] = 0.f;

    // Pieces in the order K0 V0 K1 V1 ...; two are on their way ahead of the one in use.
    int page = -1, page_next = -1, u = next(lo + warp, page);
    if (u < hi) {
        request(0, page);
        request(1, page);
    }
    while (u < hi && ok) {
        const int un = next(u + kWarps, page_next);
        const float sk = a.c.scales[0][(int64_t)page * a.c.kv_heads + h], sv = a.c.scales[1][(int64_t)page * a.c.kv_heads + h];
        if (un < hi) request(0, page_next);   // into the third slot
        const uint8_t *k = arrived();
        if (!ok) break;
        float s[8][4];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            s[x][0] = s[x][1] = s[x][2] = s[x][3] = 0.f;
            const uint8_t *kp = k + (x * 8 + g) * D + c * (D / 4);
#pragma unroll
            for (int y = 0; y < NK; ++y) {
                uint32_t b0, b1;
                key_codes(*reinterpret_cast<const uint32_t *>(kp + 4 * y), b0, b1);
                mma<__half>(s[x], qf[y], b0, b1);
            }
        }
        ++used;
        __syncwarp();
        if (un < hi) request(1, page_next);   // where the keys stood
        const float factors[2] = {row_factor[0] * sk, row_factor[1] * sk};
        softmax_step<T, NK>(rows, s, factors, kBlock);
        const uint8_t *v = arrived();
        if (!ok) break;
        uint32_t pf[4][4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            pf[y][0] = pack<__half>(s[2 * y][0], s[2 * y][1]);
            pf[y][1] = pack<__half>(s[2 * y][2], s[2 * y][3]);
            pf[y][2] = pack<__half>(s[2 * y + 1][0], s[2 * y + 1][1]);
            pf[y][3] = pack<__half>(s[2 * y + 1][2], s[2 * y + 1][3]);
        }
        auto values = [&](const int t0, const int tiles, const int dim, const bool half_word) {   // `tiles` tiles from t0 on: one word (half a word) per key
            float o[4][4] = {};
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint8_t *vp = v + (16 * y + 2 * c + (e & 1) + 8 * (e >> 1)) * D + dim;
                    w[e] = (half_word ? (uint32_t)*reinterpret_cast<const uint16_t *>(vp) : *reinterpret_cast<const uint32_t *>(vp)) ^ 0x80808080u;
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (x >= tiles) continue;
                    // byte x of two keys side by side, each under the 0x64 that makes it 1024 + x
                    const uint32_t sel = x | (4 + x) << 4;
                    const uint32_t p0 = __byte_perm(w[0], w[1], sel), p1 = __byte_perm(w[2], w[3], sel);
                    mma<__half>(o[x], pf[y], codes_f16(__byte_perm(p0, 0x64646464u, 0x4140)), codes_f16(__byte_perm(p1, 0x64646464u, 0x4140)));
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
        ++used;
        __syncwarp();
        u = un;
        page = page_next;
    }
    if (!ok && lane == 0) atomicOr(a.status, kStatusTimeout);
    // copies in flight end before the block's shared memory is reused or given back (a bounded wait gave up above: again bounded)
    for (; used < sent; ++used) (void)tc::mbar_wait(bar + 8 * (used % kSlots), (used / kSlots) & 1);

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
            const float f = exp2f(p[D] - base);
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

// Joins the pieces of a sequence: a CTA per (sequence, kv head, part of 16 query heads).
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
            const float f = exp2f(__ldcg(p + y * step + D) - base);
            sum = fmaf(f, __ldcg(p + y * step + dim), sum);
            total = fmaf(f, __ldcg(p + y * step + D + 1), total);
        }
        static_cast<T *>(a.out)[((int64_t)r * a.c.kv_heads * a.group + h * a.group + part * 16 + row) * D + dim] = from_f32<T>(total == 0.f ? 0.f : sum / total);
    }
}

}  // namespace cache
}  // namespace vs
