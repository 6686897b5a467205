// Attention over chosen blocks on the tensor cores (tcgen05).
//
// A tile is 128 rows: `tile` consecutive queries times the heads of a group, one head of keys.  It goes through the union of its queries' lists, a
// block of 64 keys at a time; a row that has not listed a block gets weights of 0 there.  Neighbouring queries choose mostly alike, so the union is not
// much longer than a list, and tiles of full height are what the tensor cores need: gathering each query's own blocks instead reads 32 KB of keys and values
// (d = 128) for a product of `group` rows, and is bound by L2 many times over.
//
// A multiplied tile knows nothing of single keys: 0 * Inf in it is a NaN that the operator does not have.  So a tile whose result is not finite says so in its
// word of `redo`, and the row kernels behind compute it again; they read only what a row attends to.  That is some 50 times the work: one Inf among the values of 8192 keys, lists
// without locality, 13 ms forward and 168 ms a training step against 0.5 and 2.9; NaN behind the ends of 4 sequences padded to 2048, a step 617 us against 343.
// A tile in which a bounded wait ran out has written nothing or a part: it goes the same way, besides the bit in the status word.
#pragma once
#include <cuda.h>

#include "blocks.cuh"
#include "common.cuh"
#include "tc_ptx.cuh"

namespace vs {
namespace blocks {
namespace tcore {

constexpr uint32_t kStatusForward = 512u, kStatusGradQ = 1024u, kStatusGradKV = 2048u;   // bits raised in the status word when a bounded wait ran out
constexpr int kRows = 128;
constexpr uint32_t kBf16Operands = (1u << 7) | (1u << 10);
template <typename T> __host__ __device__ constexpr uint32_t idesc(int n, int a_mn, int b_mn) {
    return tc::make_idesc_f16(kRows, n, a_mn, b_mn) | (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? kBf16Operands : 0u);
}

// Waits for a phase, or until another role of the CTA has given up; gives up itself after some seconds.  Polls without a time to be suspended for: those are quicker
// by a third where the phase is there already, as it mostly is, and that is 5 % of the forward kernel.
constexpr uint32_t kMaxPolls = 1u << 22;
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag) {
    for (uint32_t i = 0; i < kMaxPolls; ++i) {
        if (try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
    }
    *abort_flag = 1;
    return false;
}
// Whether phases are over, without waiting (try_wait may: it suspends the thread where the phase is not over).  Three at once, as bits: an answer takes some 300 cycles under the copies' and products' traffic, and they come together.
__device__ __forceinline__ uint32_t are_over(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1, uint32_t bar2, uint32_t parity2) {
    uint32_t bits;
    asm volatile(
        "{\n"
        ".reg .pred p, q, r;\n"
        ".reg .b32 x, y;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 q, [%3], %4;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 r, [%5], %6;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "selp.u32 x, 2, 0, q;\n"
        "selp.u32 y, 4, 0, r;\n"
        "or.b32 %0, %0, x;\n"
        "or.b32 %0, %0, y;\n"
        "}\n"
        : "=&r"(bits)
        : "r"(bar0), "r"(parity0), "r"(bar1), "r"(parity1), "r"(bar2), "r"(parity2)
        : "memory");
    return bits;
}
// Waits for three phases at once by a whole warp, which stays together: their answers come together, as above.  What the phases guard is read behind this alone: a load
// next to these instructions does not wait for their answers.
__device__ __forceinline__ bool wait_three(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1, uint32_t bar2, uint32_t parity2, volatile uint32_t *abort_flag) {
    bool ok = false;
    for (uint32_t i = 0; i < kMaxPolls && !ok; ++i) {
        uint32_t over;
        asm volatile(
            "{\n"
            ".reg .pred p, q, r;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 r, [%5], %6;\n"
            "and.pred p, p, q;\n"
            "and.pred p, p, r;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(over)
            : "r"(bar0), "r"(parity0), "r"(bar1), "r"(parity1), "r"(bar2), "r"(parity2)
            : "memory");
        ok = over != 0;
        if (!ok && *abort_flag) break;
    }
    if (!ok) *abort_flag = 1;
    return __all_sync(~0u, ok);
}
// wait() by a whole warp, which stays together.
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag) { return __all_sync(~0u, wait(bar, parity, abort_flag)); }
// One lane of a warp that is together.  The warp that issues products goes through its loop as a whole, and this lane issues: descriptors then come out of uniform
// registers; in a loop of one lane each of their halves is moved there first, and the products wait for that.
__device__ __forceinline__ bool elect_one() {
    uint32_t chosen;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(chosen));
    return chosen != 0;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// As fma2: two at a time.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 pair(uint32_t x, uint32_t y) { return make_float2(__uint_as_float(x), __uint_as_float(y)); }
template <typename T> __device__ __forceinline__ uint32_t pack2(float x, float y);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ bool finite(float x) { return x * 0.f == 0.f; }

// A block that a tile goes through: its number (-1: no more) and which of the tile's queries have listed it.
struct __align__(16) Entry {
    uint32_t rows[4];
    int32_t block;
    int32_t pad[3];
};
constexpr int kEntries = 8;   // in a ring: more than there are blocks between the loader and the softmax

// Sums in tensor memory are cut off, not rounded: one whose terms have one sign loses some 1.6 x 2^-23 of itself in every step of 16 terms.  After so many products of a tile or block
// (4 steps each in forward, 8 for dK and dV) a sum is put aside, added in fp32, and begun anew; what it has lost by then, 1.1e-4 and 2.0e-4, is less than half of fp16's own rounding.
constexpr uint32_t kRun = 256;

struct Tile {   // where a CTA's tile lies
    int b, kvh, i0;
    int64_t bh, index;   // index: among all tiles, in the order of the queries
};
__device__ __forceinline__ Tile tile_of(const Shape &s, int tile, int64_t index) {
    const int tiles = (s.queries + tile - 1) / tile;
    Tile t;
    t.bh = index / tiles;
    t.i0 = (tiles - 1 - (int)(index % tiles)) * tile;   // the last queries have most keys before them: they go first
    t.kvh = (int)(t.bh % s.kv_heads);
    t.b = (int)(t.bh / s.kv_heads);
    t.index = t.bh * tiles + t.i0 / tile;
    return t;
}

// A load that stays where it is written: left to itself the compiler moves it to each use of its word, into the loop over a word's bits, and every step of
// the loader waits for L2.
__device__ __forceinline__ uint32_t load_here(const uint32_t *p) {
    uint32_t v;
    asm volatile("ld.global.cg.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
// The blocks that a tile of queries has listed, in ascending order, found by a warp 32 at a time.
struct Scan {
    const uint32_t *bits;
    int blocks, end, words, shift;
    uint32_t mask;
    int base = 0;
    uint32_t then[4];

    __device__ __forceinline__ void fetch(int from, uint32_t (&to)[4]) const {
        const int j = from + (threadIdx.x & 31);
#pragma unroll
        for (int k = 0; k < 4; ++k) to[k] = k < words && j < end ? (load_here(bits + (int64_t)k * blocks + j) >> shift) & mask : 0u;
    }
    __device__ __forceinline__ Scan(const Shape &s, const uint32_t *all, const Tile &t, int tile) {
        blocks = s.blocks;
        const int w = t.i0 >> 5;
        bits = all + (t.bh * s.words + w) * s.blocks;
        words = tile <= 32 ? 1 : min(tile / 32, s.words - w);
        shift = t.i0 & 31;
        mask = tile >= 32 ? ~0u : (1u << tile) - 1;
        const int last = min(t.i0 + tile, s.queries) - 1, len = s.length(t.b);
        end = min(s.blocks, (s.end(last, len) + kBlock - 1) / kBlock);
        fetch(0, then);
    }
    // The next 32 blocks' words go to `to` (a row of 32 for each of four words); false where there are no more.  What goes through the chunk then
    // needs no shuffles: between waits of a single lane those cost the warp a thousand cycles an entry.
    __device__ __forceinline__ bool next(uint32_t (*to)[32], uint32_t &some) {
        if (base >= end) return false;
        const int lane = threadIdx.x & 31;
        __syncwarp();   // the chunk before has been gone through
#pragma unroll
        for (int k = 0; k < 4; ++k) to[k][lane] = then[k];
        some = __ballot_sync(~0u, (then[0] | then[1] | then[2] | then[3]) != 0);
        fetch(base + 32, then);
        base += 32;
        __syncwarp();
        return true;
    }
};

// Writes 32 rows of the warp, one to a lane, so that a row's bytes leave together: `value(g, v)` gives the lane's elements 32 g .. 32 g + 31 as
// four 16-byte pieces.  They pass through `stage`, 32 rows of 128 bytes in each of DP / 64 slabs `slab` bytes apart, the pieces swizzled by the row.
// `first`: 0 or 1, the half of the slab that the first 32 elements take.
template <typename T, int DP, typename F> __device__ __forceinline__ void write_rows(uint8_t *stage, int slab, T *out, int64_t row_at, bool there, int d, int first, F value) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int g = 0; g < DP / 32; ++g) {
        uint4 v[4];
        value(g, v);
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4 *>(stage + (g + first) / 2 * slab + lane * 128 + ((((g + first) % 2 * 4 + c) ^ (lane & 7)) << 4)) = v[c];
    }
    __syncwarp();
    constexpr int kLanes = DP / 8;   // to a row
#pragma unroll 4
    for (int r0 = 0; r0 < 32; r0 += 32 / kLanes) {
        const int r = r0 + lane / kLanes, c = lane % kLanes, at_slab = c + first * 4;
        const int64_t at = __shfl_sync(~0u, row_at, r);
        const bool live = __shfl_sync(~0u, (int)there, r);
        if (live && c * 8 < d)
            *reinterpret_cast<uint4 *>(out + at + c * 8) = *reinterpret_cast<const uint4 *>(stage + at_slab / 8 * slab + r * 128 + (((at_slab % 8) ^ (r & 7)) << 4));
    }
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t x) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&x));
    else return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
// The two warps of a quarter of the rows meet (64 threads, barriers 1 .. 4).
__device__ __forceinline__ void bar_pair(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
template <typename T> __device__ __forceinline__ uint4 pack8(const float *f) {
    return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

// ---- forward ----------------------------------------------------------------------------------------------------------
// A barrier tells a phase from the next but not from the one after that, so what may be two products ahead or behind has two barriers, one for either buffer of S.
// Per block: S[128 x 64] = Q K^T (operands in shared memory), the softmax's step by two threads per row, 32 keys each, out of tensor memory, P (16 bits) back into S's place,
// O[128 x d] += P V with P as the operand in tensor memory.  S is double buffered; 256 columns of tensor memory and ~100 KB of shared memory, so that
// two CTAs share an SM and one's products run under the other's exponentials.
// The maximum that weights are taken relative to follows the true one only when that has grown by 2^8: weights then stay below 256, exact enough in
// either type, and O is seldom rescaled.
// Bound by the hand-overs between its roles: with one multiplication to a product and no exponentials an earlier form took 635 us of its 810 at 16384 x 16384,
// 32 heads on 4, d = 128, 16 blocks each (158 000 tiles of 128 x 64).  Now 637 us: 1.04 PFLOP/s on the tiles, 0.41 on the pairs that the lists name, the unions being
// 2.5 times as long as a list.  The waits of a step's products taken together: 652 before.  Two blocks to a step, and a loader that stays together as a warp, were slower.
constexpr float kSlack = 8.f;
// kLong: lists of more than kRun blocks.  O is put aside in tensor memory every kRun blocks of the union: without it results were 4.3e-4 too small by 1024 blocks and 6.9e-3 by 16384, and
// the gradients of q, which read them, off by 0.17 and 11 %.  d > 64: that takes the columns of both CTAs, so one to an SM.  2048 queries, 8 heads on
// 2, 1024 blocks each: d = 128 1040 us (1037 without), d = 64 856 (826).
template <int DP, bool kLong> struct ForwardSmem {
    static constexpr int kSlots = DP == 128 ? 4 : 6;
    static constexpr int kSlotBytes = kBlock * DP * 2, kQBytes = kRows * DP * 2;
    static constexpr int kQ = 3 * 1024, kRing = kQ + kQBytes, kUsed = kRing + kSlots * kSlotBytes;   // ahead: entries, barriers, a chunk of the scan, 2 KB for the rows' threads
    static constexpr uint32_t kColumns = kLong && DP == 128 ? 512 : 256;   // of tensor memory: S twice, O, and what is put aside
    static constexpr int kBytes = kColumns > 256 ? 120 * 1024 : kUsed;     // no second CTA that would wait for the first one's columns
    static constexpr int kEntriesAt = 0, kBars = kEntries * sizeof(Entry);
    static constexpr int kBarQ = kBars, kFull = kBarQ + 8, kEmpty = kFull + 8 * kSlots, kS = kEmpty + 8 * kSlots, kP = kS + 16, kPv = kP + 16, kDrain = kPv + 16, kAbort = kDrain + 8,
                         kHolder = kAbort + 4;
    static constexpr int kChunk = 512, kMeet = 1024;
    static_assert(kHolder + 4 <= kChunk && kMeet + 4 * kRows * 4 <= kQ, "head");
    static_assert(2 * (kUsed + 2048) <= 228 * 1024 && kUsed <= kBytes && (kColumns > 256) == (2 * (kBytes + 2048) > 228 * 1024), "two CTAs an SM, or one");
};
constexpr int kForwardThreads = 320;

template <typename T, int DP, bool kLong>
__global__ void __launch_bounds__(kForwardThreads, 2) forward_kernel(const Args a, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                     const __grid_constant__ CUtensorMap map_v, uint32_t *redo, uint32_t *status) {
    using M = ForwardSmem<DP, kLong>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t raw = tc::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *sm = smem_raw + (base - raw);
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(sm + M::kAbort);
    const Shape &s = a.s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Tile t = tile_of(s, a.tile, blockIdx.x);
    const int len = s.length(t.b);

    if (threadIdx.x == 0) {
        tc::mbar_init(base + M::kBarQ, 1);
        for (int i = 0; i < M::kSlots; ++i) {
            tc::mbar_init(base + M::kFull + 8 * i, 1);
            tc::mbar_init(base + M::kEmpty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(base + M::kS + 8 * i, 2);   // the product, and the word of the thread that issued it on the entry
            tc::mbar_init(base + M::kP + 8 * i, 8);
            tc::mbar_init(base + M::kPv + 8 * i, 1);
        }
        tc::mbar_init(base + M::kDrain, 1);
        *abort_flag = 0;
        tc::fence_mbar_init();
    }
    if (warp == 9) {
        tc::tmem_alloc(base + M::kHolder, M::kColumns);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + M::kHolder);
    const uint32_t tmem_o = tmem + 128;
    bool bad = false;
    pdl_launch_dependents();   // behind the allocation, as in the kernels below

    pdl_wait();   // all roles: the bounded waits below are for this kernel's own work, not for that of kernels before it
    if (warp == 8) {
        // loader: position 2 x holds the keys, 2 x + 1 the values of the x-th block
        const uint32_t q_bytes = (uint32_t)(a.tile * s.group * 128 * (DP / 64));
        if (lane == 0) {
            tc::mbar_expect_tx(base + M::kBarQ, q_bytes);
            for (int x = 0; x < DP / 64; ++x) tc::tma_load_4d(base + M::kQ + x * kRows * 128, &map_q, base + M::kBarQ, x * 64, t.kvh * s.group, t.i0, t.b);
        }
        uint32_t at = 0;
        bool ok = true;
        auto slot_free = [&]() {   // lane 0: the slot of position `at`
            return at < (uint32_t)M::kSlots || wait(base + M::kEmpty + 8 * (at % M::kSlots), (at / M::kSlots - 1) & 1, abort_flag);
        };
        auto load = [&](const CUtensorMap *map, int j) {
            const uint32_t slot = at % M::kSlots, bar = base + M::kFull + 8 * slot;
            tc::mbar_expect_tx(bar, M::kSlotBytes);
            for (int x = 0; x < DP / 64; ++x) tc::tma_load_4d(base + M::kRing + slot * M::kSlotBytes + x * kBlock * 128, map, bar, x * 64, t.kvh, j * kBlock, t.b);
            ++at;
        };
        Scan scan(s, a.bits, t, a.tile);
        uint32_t(*chunk)[32] = reinterpret_cast<uint32_t(*)[32]>(sm + M::kChunk);
        uint32_t some;
        while (scan.next(chunk, some))
            if (lane == 0)
                for (; some && ok; some &= some - 1) {
                    const int x = __ffs(some) - 1, block = scan.base - 32 + x;
                    ok = slot_free();
                    if (!ok) break;
                    Entry *to = reinterpret_cast<Entry *>(sm + M::kEntriesAt) + (at / 2) % kEntries;
                    *reinterpret_cast<uint4 *>(to->rows) = make_uint4(chunk[0][x], chunk[1][x], chunk[2][x], chunk[3][x]);
                    to->block = block;
                    load(&map_k, block);
                    ok = slot_free();
                    if (ok) load(&map_v, block);
                }
        if (lane == 0) {
            if (ok && slot_free()) {
                reinterpret_cast<Entry *>(sm + M::kEntriesAt)[(at / 2) % kEntries].block = -1;
                tc::mbar_arrive(base + M::kFull + 8 * (at % M::kSlots));
            }
            if (*abort_flag) {   // copies in flight end before the shared memory is given back
                for (uint32_t y = 0; y < 1024 && !tc::mbar_try_wait(base + M::kBarQ, 0); ++y) {}
                for (uint32_t x = at > (uint32_t)M::kSlots ? at - M::kSlots : 0; x < at; ++x)
                    for (uint32_t y = 0; y < 1024 && !tc::mbar_try_wait(base + M::kFull + 8 * (x % M::kSlots), (x / M::kSlots) & 1); ++y) {}
            }
        }
    } else if (warp == 9) {
        constexpr uint32_t kIdescS = idesc<T>(kBlock, 0, 0), kIdescO = idesc<T>(DP, 0, 1);
        const uint32_t hi = tc::smem_desc_hi(1024, (uint32_t)tc::kSwizzle128B);
        const uint32_t q_lo = tc::smem_desc_lo(base + M::kQ, 16), k_lo = tc::smem_desc_lo(base + M::kRing, 16);
        const uint32_t v_lo = tc::smem_desc_lo(base + M::kRing, kBlock * 128);   // 64-dimension slabs
        const bool leader = elect_one();
        bool ok = wait_all(base + M::kBarQ, 0, abort_flag);
        uint32_t x = 0;
        auto values = [&](uint32_t y) {   // O += P V of the y-th block
            const uint32_t at = 2 * y + 1, slot = at % M::kSlots;
            const uint32_t p_bar = base + M::kP + 8 * (y & 1), p_phase = (y >> 1) & 1;
            ok = ok && wait_three(base + M::kFull + 8 * slot, (at / M::kSlots) & 1, p_bar, p_phase, p_bar, p_phase, abort_flag);
            if (!ok) return;
            tc::tc_fence_after_sync();
            if (leader) {
#pragma unroll
                for (int k = 0; k < kBlock / 16; ++k)
                    tc::mma_f16_ts(tmem_o, tmem + (y & 1) * 64 + 8 * k, tc::desc64(v_lo + slot * (M::kSlotBytes >> 4) + 128 * k, hi), kIdescO, (kLong ? y % kRun : y) > 0 || k > 0);
                tc::mma_commit(base + M::kPv + 8 * (y & 1));
                tc::mma_commit(base + M::kEmpty + 8 * slot);
            }
            __syncwarp();
        };
        for (; ok; ++x) {
            const uint32_t at = 2 * x, slot = at % M::kSlots;
            // S goes where the P of two blocks ago stood: its product has ended (of a barrier without a phase yet the one before its first is over)
            const uint32_t pv_bar = base + M::kPv + 8 * (x & 1), pv_phase = ((x - 2) >> 1) & 1;
            ok = wait_three(base + M::kFull + 8 * slot, (at / M::kSlots) & 1, pv_bar, pv_phase, pv_bar, pv_phase, abort_flag);
            if (!ok) break;
            if (__any_sync(~0u, reinterpret_cast<volatile Entry *>(sm + M::kEntriesAt)[x % kEntries].block < 0)) {
                if (leader) {
                    tc::mbar_arrive(base + M::kS + 8 * (x & 1));
                    tc::mbar_arrive(base + M::kS + 8 * (x & 1));
                }
                break;
            }
            tc::tc_fence_after_sync();
            if (leader) {
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
                    tc::mma_f16_ss(tmem + (x & 1) * 64, tc::desc64(q_lo + (k / 4) * (kRows * 128 >> 4) + (k % 4) * 2, hi),
                                   tc::desc64(k_lo + slot * (M::kSlotBytes >> 4) + (k / 4) * (kBlock * 128 >> 4) + (k % 4) * 2, hi), kIdescS, k > 0);
                tc::mma_commit(base + M::kS + 8 * (x & 1));
                tc::mbar_arrive(base + M::kS + 8 * (x & 1));
                tc::mma_commit(base + M::kEmpty + 8 * slot);
            }
            __syncwarp();
            if (x > 0) values(x - 1);
        }
        if (ok && x > 0) values(x - 1);
        // what was issued ends before tensor memory is given back; normally the softmax has waited for it already
        if (leader) {
            tc::mma_commit(base + M::kDrain);
            for (uint32_t y = 0; y < 4096 && !tc::mbar_try_wait(base + M::kDrain, 0); ++y) {}
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, half = warp >> 2, r = quarter * 32 + lane, qx = r / s.group, i = t.i0 + qx;
        float *meet = reinterpret_cast<float *>(sm + M::kMeet);   // [2][2][128]: what the two threads of a row tell each other
        const bool there = r < a.tile * s.group && i < s.queries, alive = there && i < s.rows(t.b);   // rows behind a sequence's end have zeros, whatever stands there
        const int h = t.kvh * s.group + r % s.group, end = there ? s.end(i, len) : 0;
        const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
        const float c = a.scale * kLog2e;
        float top = -INFINITY, total = 0.f;   // what the weights are relative to, and the sum of this thread's
        float aside_top = -INFINITY;          // what those of the sums put aside were relative to
        auto aside_scale = [&] { return aside_top == -INFINITY ? 0.f : ex2(aside_top - top); };
        uint32_t x = 0;
        bool ok = true;
        for (;; ++x) {
            ok = __all_sync(~0u, wait(base + M::kS + 8 * (x & 1), (x >> 1) & 1, abort_flag));
            if (!ok) break;
            const volatile Entry &e = reinterpret_cast<volatile Entry *>(sm + M::kEntriesAt)[x % kEntries];
            const int block = e.block;
            if (block < 0) break;
            const bool listed = alive && (e.rows[qx >> 5] >> (qx & 31) & 1u);
            const int n = listed ? min(kBlock, end - block * kBlock) : 0;   // keys of the row
            tc::tc_fence_after_sync();
            if (kLong && x > 0 && x % kRun == 0) {   // this block's product, which begins anew, waits for this warp's weights
                ok = __all_sync(~0u, wait(base + M::kPv + 8 * ((x - 1) & 1), ((x - 1) >> 1) & 1, abort_flag));
                if (!ok) break;
                tc::tc_fence_after_sync();
                const float shrink = aside_scale();
#pragma unroll 1
                for (int k = half * (DP / 2); k < (half + 1) * (DP / 2); k += 32) {
                    uint32_t o[32], before[32];
                    tc::tmem_ld_x32(mine + 128 + k, o);
                    if (x > kRun) {
                        tc::tmem_ld_x32(mine + 128 + DP + k, before);
#pragma unroll
                        for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(fmaf(__uint_as_float(before[y]), shrink, __uint_as_float(o[y])));
                    }
                    tc::tmem_st_x32(mine + 128 + DP + k, o);
                }
                tc::tmem_st_wait();
                aside_top = top;
            }
            uint32_t u[32];
            tc::tmem_ld_x32(mine + (x & 1) * 64 + 32 * half, u);
            if (__any_sync(~0u, n > 0 && n < kBlock)) {   // a block that ends inside: the queries' own, mostly
#pragma unroll
                for (int k = 0; k < 32; ++k)
                    if (32 * half + k >= n) u[k] = __float_as_uint(-INFINITY);
            }
            float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 32; k += 2) m[k / 2 % 4] = max3(m[k / 2 % 4], __uint_as_float(u[k]), __uint_as_float(u[k + 1]));
            m[0] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            float *here = meet + (x & 1) * 2 * kRows + r;
            here[half * kRows] = m[0];
            bar_pair(1 + quarter);   // also: both have read their scores, P may go where the first half's stood
            const float high = n > 0 ? fmaxf(m[0], here[(half ^ 1) * kRows]) * c : -INFINITY;
            if (__any_sync(~0u, high > top + kSlack)) {
                const float to = fmaxf(top, high), shrink = to == -INFINITY ? 1.f : ex2(top - to);
                top = to;
                total *= shrink;
                if (x > 0) {
                    ok = __all_sync(~0u, wait(base + M::kPv + 8 * ((x - 1) & 1), ((x - 1) >> 1) & 1, abort_flag));
                    if (!ok) break;
                    tc::tc_fence_after_sync();
#pragma unroll 1
                    for (int k = half * (DP / 2); k < (half + 1) * (DP / 2); k += 32) {
                        uint32_t o[32];
                        tc::tmem_ld_x32(mine + 128 + k, o);
#pragma unroll
                        for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * shrink);
                        tc::tmem_st_x32(mine + 128 + k, o);
                    }
                }
            }
            // a row that has not listed the block has no weight there: its scores, finite ones, all end at -inf
            const float off = n <= 0 ? -INFINITY : top == -INFINITY ? 0.f : -top;
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            uint32_t p[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                float2 y = fma2(pair(u[2 * k], u[2 * k + 1]), make_float2(c, c), make_float2(off, off));
                y.x = ex2(y.x);
                y.y = ex2(y.y);
                sum[k % 2] = add2(sum[k % 2], y);
                p[k] = pack2<T>(y.x, y.y);
            }
            sum[0] = add2(sum[0], sum[1]);
            total += sum[0].x + sum[0].y;
            tc::tmem_st_x16(mine + (x & 1) * 64 + 16 * half, p);
            tc::tmem_st_wait();
            tc::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(base + M::kP + 8 * (x & 1));
        }
        // the last product, and with it all before it; without any, the copy of Q ends before its place takes the result
        if (ok) ok = __all_sync(~0u, x > 0 ? wait(base + M::kPv + 8 * ((x - 1) & 1), ((x - 1) >> 1) & 1, abort_flag) : wait(base + M::kBarQ, 0, abort_flag));
        if (ok) {
            tc::tc_fence_after_sync();
            const int64_t row = (((int64_t)t.b * s.queries + i) * s.heads + h) * s.d;
            float *here = meet + (x & 1) * 2 * kRows + r;
            here[half * kRows] = total;
            bar_pair(1 + quarter);
            total = meet[(x & 1) * 2 * kRows + r] + meet[((x & 1) * 2 + 1) * kRows + r];   // in the same order in both
            const float inv = total == 0.f ? 0.f : 1.f / total;
            auto result = [&](int g, float (&f)[32]) {
                uint32_t o[32];
                if (x > 0) tc::tmem_ld_x32(mine + 128 + half * (DP / 2) + 32 * g, o);
                if (kLong && x > kRun) {
                    const float shrink = aside_scale();
                    uint32_t before[32];
                    tc::tmem_ld_x32(mine + 128 + DP + half * (DP / 2) + 32 * g, before);
#pragma unroll
                    for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(fmaf(__uint_as_float(before[y]), shrink, __uint_as_float(o[y])));
                }
#pragma unroll
                for (int y = 0; y < 32; ++y) f[y] = x > 0 && alive && total != 0.f ? __uint_as_float(o[y]) * inv : 0.f;
            };
            // the two warps of a quarter take a half of the dimensions each
            uint8_t *stage = sm + M::kQ + quarter * 32 * 128 + (DP == 128 ? half * kRows * 128 : 0);
            const int first = half * (DP / 2);
            write_rows<T, DP / 2>(stage, kRows * 128, static_cast<T *>(a.result) + first, row, there, s.d - first, half * (DP == 64), [&](int g, uint4 (&v)[4]) {
                float f[32];
                result(g, f);
#pragma unroll
                for (int y = 0; y < 32; ++y) bad |= alive && !finite(f[y]);
#pragma unroll
                for (int y = 0; y < 4; ++y) v[y] = pack8<T>(f + 8 * y);
            });
            if (a.result_low)
                write_rows<T, DP / 2>(stage, kRows * 128, static_cast<T *>(a.result_low) + first, row, there, s.d - first, half * (DP == 64), [&](int g, uint4 (&v)[4]) {
                    float f[32];
                    result(g, f);
#pragma unroll
                    for (int y = 0; y < 32; ++y) f[y] -= to_f32(from_f32<T>(f[y]));
#pragma unroll
                    for (int y = 0; y < 4; ++y) v[y] = pack8<T>(f + 8 * y);
                });
            bad |= alive && total != total;
            if (there && half == 0) a.lse[((int64_t)t.b * s.heads + h) * s.queries + i] = !alive || total == 0.f ? INFINITY : top + log2f(total);
        }
    }
    tc::tc_fence_before_sync();
    const bool again = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
        const bool gave_up = *abort_flag != 0;
        redo[t.index] = again || gave_up;
        if (gave_up) atomicOr(status, kStatusForward);
    }
    if (warp == 9) {
        tc::tc_fence_after_sync();
        tc::tmem_dealloc(tmem, M::kColumns);
    }
}

// ---- backward ---------------------------------------------------------------------------------------------------------
// Weights and the scores' gradients are rounded to 16 bits for their products.  fp16 keeps its precision only above 2^-14, so there both are multiplied by powers of
// two first: the weights, at most 1, by 2^14; the gradients by the one that brings the largest finite element of grad_out to 32 .. 64: for dQ the largest of the row, for dK, whose
// sums join rows, that of the rows that have listed the block.  So no row's gradients depend on how large another's are where the two do not meet in a sum.
template <typename T> struct Lift {
    static constexpr float kWeight = std::is_same<T, __half>::value ? 14.f : 0.f;   // exponent
    static __device__ __forceinline__ float grad(const uint32_t *most) {
        if constexpr (!std::is_same<T, __half>::value) return 1.f;
        const uint32_t e = __ldcg(most) >> 23;
        return e < 6 || e >= 253 ? 1.f : __uint_as_float((259u - e) << 23);   // 2^(5 - (e - 127))
    }
};
__device__ __forceinline__ float exp2i(float e) { return __uint_as_float((uint32_t)((int)e + 127) << 23); }   // a whole exponent

// dQ: a tile of queries through the union of its lists, as forward.  Per block S = Q K^T and dP = dO V^T, dS = P (dP - delta) back into S's place as an operand,
// dQ += dS K with the same keys, now contracted over.  A row's dS sum to 0, so its products with the keys cancel and a
// rounding of dS counts more than one of the result (1.5 times its error): dS goes in as two words, itself and what its rounding left over.  Keys are double buffered, values not: their place is free once dP is there, long before the
// next ones are needed.  256 columns of tensor memory, 113 KB of shared memory (d = 128): two CTAs an SM, one's products under the other's exponentials.
// Bound by its chain of products and softmax, single buffered: 8192 x 8192, 32 heads on 4, d = 128, 16 blocks each, 70 900 tiles of 128 x 64: 528 us
// (476 without the second word).
// kLong: as in forward, dQ put aside every kRun blocks: without it sums of one sign were 9.8e-4 too small by 8000 blocks and 1.8e-3 by 16000, with it 4e-5.  The backward pass of the
// queries named there: d = 128 3310 us (3235 without), d = 64 2530 (2500).
template <int DP, bool kLong> struct GradQSmem {
    static constexpr int kSlotBytes = kBlock * DP * 2, kQBytes = kRows * DP * 2;
    static constexpr int kQ = 1024, kG = kQ + kQBytes, kK = kG + kQBytes, kV = kK + 2 * kSlotBytes, kUsed = kV + kSlotBytes;
    static constexpr uint32_t kColumns = kLong && DP == 128 ? 512 : 256;   // of tensor memory: S, dP, dQ, and what is put aside
    static constexpr int kBytes = kColumns > 256 ? 120 * 1024 : kUsed;
    static constexpr int kBars = kEntries * sizeof(Entry);
    static constexpr int kBarQ = kBars, kKFull = kBarQ + 8, kKEmpty = kKFull + 16, kVFull = kKEmpty + 16, kVEmpty = kVFull + 8, kSP = kVEmpty + 8, kDs = kSP + 8, kDq = kDs + 8,
                         kE = kDq + 8, kDrain = kE + 8 * kEntries, kAbort = kDrain + 8, kHolder = kAbort + 4;
    static constexpr int kChunk = 512;
    static_assert(kHolder + 4 <= kChunk, "head");
    static_assert(2 * (kUsed + 1024) <= 228 * 1024 && kUsed <= kBytes && (kColumns > 256) == (2 * (kBytes + 1024) > 228 * 1024), "two CTAs an SM, or one");
};
constexpr int kGradQThreads = 320;
template <typename T, int DP, bool kLong>
__global__ void __launch_bounds__(kGradQThreads, 2) grad_q_kernel(const Args a, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_g,
                                                                    const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, uint32_t *redo,
                                                                    uint32_t *status) {
    using M = GradQSmem<DP, kLong>;
    extern __shared__ __align__(1024) uint8_t sm[];
    const uint32_t base = tc::smem_u32(sm);
    const Shape &s = a.s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Tile t = tile_of(s, a.tile, blockIdx.x);
    if (base & 1023u) {   // there is no room for a margin: a tile whose memory does not start where the swizzle needs it is left to the kernel behind
        pdl_wait();
        if (threadIdx.x == 0) redo[t.index] = 1;
        return;
    }
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(sm + M::kAbort);
    const int len = s.length(t.b);

    if (threadIdx.x == 0) {
        for (int bar : {M::kBarQ, M::kKFull, M::kKFull + 8, M::kKEmpty, M::kKEmpty + 8, M::kVFull, M::kVEmpty, M::kSP, M::kDq, M::kDrain}) tc::mbar_init(base + bar, 1);
        tc::mbar_init(base + M::kDs, 8);
        for (int i = 0; i < kEntries; ++i) tc::mbar_init(base + M::kE + 8 * i, 1);
        *abort_flag = 0;
        tc::fence_mbar_init();
    }
    if (warp == 9) {
        tc::tmem_alloc(base + M::kHolder, M::kColumns);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + M::kHolder);
    bool bad = false;
    // Behind the allocation: the next kernel's CTAs take tensor memory before they wait for this one, and an allocation here must not wait for theirs.
    pdl_launch_dependents();

    pdl_wait();   // all roles: the bounded waits below are for this kernel's own work, not for that of kernels before it
    if (warp == 8) {
        const uint32_t q_bytes = (uint32_t)(a.tile * s.group * 128 * (DP / 64));
        if (lane == 0) {
            tc::mbar_expect_tx(base + M::kBarQ, 2 * q_bytes);
            for (int x = 0; x < DP / 64; ++x) {
                tc::tma_load_4d(base + M::kQ + x * kRows * 128, &map_q, base + M::kBarQ, x * 64, t.kvh * s.group, t.i0, t.b);
                tc::tma_load_4d(base + M::kG + x * kRows * 128, &map_g, base + M::kBarQ, x * 64, t.kvh * s.group, t.i0, t.b);
            }
        }
        const bool leader = elect_one();
        uint32_t x = 0;
        bool ok = true;
        auto load = [&](const CUtensorMap *map, uint32_t to, uint32_t bar, int j) {
            tc::mbar_expect_tx(bar, M::kSlotBytes);
            for (int y = 0; y < DP / 64; ++y) tc::tma_load_4d(to + y * kBlock * 128, map, bar, y * 64, t.kvh, j * kBlock, t.b);
        };
        Scan scan(s, a.bits, t, a.tile);
        uint32_t(*chunk)[32] = reinterpret_cast<uint32_t(*)[32]>(sm + M::kChunk);
        uint32_t some;
        while (scan.next(chunk, some))
            for (; some && ok; some &= some - 1, ++x) {
                const int y = __ffs(some) - 1, block = scan.base - 32 + y;
                if (!(ok = x < 2 || wait_all(base + M::kKEmpty + 8 * (x & 1), ((x - 2) >> 1) & 1, abort_flag))) break;
                if (leader) {
                    Entry *to = reinterpret_cast<Entry *>(sm) + x % kEntries;
                    *reinterpret_cast<uint4 *>(to->rows) = make_uint4(chunk[0][y], chunk[1][y], chunk[2][y], chunk[3][y]);
                    to->block = block;
                    tc::mbar_arrive(base + M::kE + 8 * (x % kEntries));
                    load(&map_k, base + M::kK + (x & 1) * M::kSlotBytes, base + M::kKFull + 8 * (x & 1), block);
                }
                __syncwarp();
                if (!(ok = x < 1 || wait_all(base + M::kVEmpty, (x - 1) & 1, abort_flag))) break;
                if (leader) load(&map_v, base + M::kV, base + M::kVFull, block);
                __syncwarp();
            }
        if (leader) {
            if (ok && (x < 2 || wait(base + M::kKEmpty + 8 * (x & 1), ((x - 2) >> 1) & 1, abort_flag)) && (x < 1 || wait(base + M::kVEmpty, (x - 1) & 1, abort_flag))) {
                reinterpret_cast<Entry *>(sm)[x % kEntries].block = -1;
                tc::mbar_arrive(base + M::kE + 8 * (x % kEntries));
                tc::mbar_arrive(base + M::kKFull + 8 * (x & 1));
                tc::mbar_arrive(base + M::kVFull);
            }
            if (*abort_flag) {   // copies in flight end before the shared memory is given back
                for (uint32_t y = 0; y < 1024 && !tc::mbar_try_wait(base + M::kBarQ, 0); ++y) {}
                for (uint32_t z = x > 2 ? x - 2 : 0; z < x; ++z) {
                    for (uint32_t y = 0; y < 1024 && !tc::mbar_try_wait(base + M::kKFull + 8 * (z & 1), (z >> 1) & 1); ++y) {}
                    for (uint32_t y = 0; y < 1024 && !tc::mbar_try_wait(base + M::kVFull, z & 1); ++y) {}
                }
            }
        }
    } else if (warp == 9) {
        constexpr uint32_t kIdescS = idesc<T>(kBlock, 0, 0), kIdescQ = idesc<T>(DP, 0, 1);
        const uint32_t hi = tc::smem_desc_hi(1024, (uint32_t)tc::kSwizzle128B);
        const uint32_t q_lo = tc::smem_desc_lo(base + M::kQ, 16), g_lo = tc::smem_desc_lo(base + M::kG, 16), k_lo = tc::smem_desc_lo(base + M::kK, 16);
        const uint32_t v_lo = tc::smem_desc_lo(base + M::kV, 16), kt_lo = tc::smem_desc_lo(base + M::kK, kBlock * 128);
        const bool leader = elect_one();
        bool ok = wait_all(base + M::kBarQ, 0, abort_flag);
        for (uint32_t x = 0; ok; ++x) {
            const uint32_t slot = x & 1, at = slot * (M::kSlotBytes >> 4);
            // S goes where dS stood (of a barrier without a phase yet the one before its first is over)
            ok = wait_three(base + M::kKFull + 8 * slot, (x >> 1) & 1, base + M::kDq, (x - 1) & 1, base + M::kVFull, x & 1, abort_flag);
            if (!ok || __any_sync(~0u, reinterpret_cast<volatile Entry *>(sm)[x % kEntries].block < 0)) break;
            tc::tc_fence_after_sync();
            if (leader) {
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
                    tc::mma_f16_ss(tmem, tc::desc64(q_lo + (k / 4) * (kRows * 128 >> 4) + (k % 4) * 2, hi),
                                   tc::desc64(k_lo + at + (k / 4) * (kBlock * 128 >> 4) + (k % 4) * 2, hi), kIdescS, k > 0);
#pragma unroll
                for (int k = 0; k < DP / 16; ++k)
                    tc::mma_f16_ss(tmem + 64, tc::desc64(g_lo + (k / 4) * (kRows * 128 >> 4) + (k % 4) * 2, hi),
                                   tc::desc64(v_lo + (k / 4) * (kBlock * 128 >> 4) + (k % 4) * 2, hi), kIdescS, k > 0);
                tc::mma_commit(base + M::kSP);
                tc::mma_commit(base + M::kVEmpty);
            }
            __syncwarp();
            if (!(ok = wait_all(base + M::kDs, x & 1, abort_flag))) break;
            tc::tc_fence_after_sync();
            if (leader) {
#pragma unroll
                for (int k = 0; k < kBlock / 16; ++k)
                    tc::mma_f16_ts(tmem + 128, tmem + 8 * k, tc::desc64(kt_lo + at + 128 * k, hi), kIdescQ, (kLong ? x % kRun : x) > 0 || k > 0);
#pragma unroll
                for (int k = 0; k < kBlock / 16; ++k)   // what the rounding of dS left over
                    tc::mma_f16_ts(tmem + 128, tmem + 32 + 8 * k, tc::desc64(kt_lo + at + 128 * k, hi), kIdescQ, true);
                tc::mma_commit(base + M::kDq);
                tc::mma_commit(base + M::kKEmpty + 8 * slot);
            }
            __syncwarp();
        }
        if (leader) {
            tc::mma_commit(base + M::kDrain);
            for (uint32_t y = 0; y < 4096 && !tc::mbar_try_wait(base + M::kDrain, 0); ++y) {}
        }
        __syncwarp();
    } else {
        const int quarter = warp & 3, half = warp >> 2;   // two warps to a quarter of the rows, 32 keys each
        const int r = quarter * 32 + lane, qx = r / s.group, i = t.i0 + qx;
        const bool there = r < a.tile * s.group && i < s.queries, alive = there && i < s.rows(t.b);   // rows behind a sequence's end have zeros, whatever stands there
        const int h = t.kvh * s.group + r % s.group, end = there ? s.end(i, len) : 0;
        const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
        const float c = a.scale * kLog2e;
        float lse = INFINITY, lift = 1.f, minus_delta = 0.f;
        uint32_t x = 0;
        bool ok = true;
        for (;; ++x) {
            ok = __all_sync(~0u, wait(base + M::kE + 8 * (x % kEntries), (x / kEntries) & 1, abort_flag));
            if (!ok) break;
            const volatile Entry &e = reinterpret_cast<volatile Entry *>(sm)[x % kEntries];
            const int block = e.block;
            if (block < 0) break;
            const bool listed = alive && (e.rows[qx >> 5] >> (qx & 31) & 1u);
            const int n = listed ? min(kBlock, end - block * kBlock) : 0;   // keys of the row
            if (x == 0 && there) {
                const int64_t row = ((int64_t)t.b * s.heads + h) * s.queries + i;
                lift = Lift<T>::grad(a.most + row);
                lse = __ldcg(a.lse + row);
                minus_delta = -__ldcg(a.delta + row) * lift;
            }
            ok = __all_sync(~0u, wait(base + M::kSP, x & 1, abort_flag));
            if (!ok) break;
            tc::tc_fence_after_sync();
            if (kLong && x > 0 && x % kRun == 0) {   // the scores have been issued behind the end of the products before
#pragma unroll 1
                for (int k = half * (DP / 2); k < (half + 1) * (DP / 2); k += 32) {
                    uint32_t o[32], before[32];
                    tc::tmem_ld_x32(mine + 128 + k, o);
                    if (x > kRun) {
                        tc::tmem_ld_x32(mine + 128 + DP + k, before);
#pragma unroll
                        for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) + __uint_as_float(before[y]));
                    }
                    tc::tmem_st_x32(mine + 128 + DP + k, o);
                }
                tc::tmem_st_wait();
            }
            const bool whole = __all_sync(~0u, n <= 0 || n == kBlock);
            const float off = n > 0 ? -lse : -INFINITY;   // a row that has not listed the block has no weight there
            uint32_t u[32], d[32], ds[16], low[16];
            tc::tmem_ld_x32_issue(mine + 32 * half, u);
            tc::tmem_ld_x32_issue(mine + 64 + 32 * half, d);
            tc::tmem_ld_x32_wait(u);
            tc::tmem_ld_x32_wait(d);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                float2 w = fma2(pair(u[2 * k], u[2 * k + 1]), make_float2(c, c), make_float2(off, off));
                w.x = ex2(w.x);
                w.y = ex2(w.y);
                float2 f = mul2(w, fma2(pair(d[2 * k], d[2 * k + 1]), make_float2(lift, lift), make_float2(minus_delta, minus_delta)));
                if (!whole) {
                    if (32 * half + 2 * k >= n) f.x = 0.f;
                    if (32 * half + 2 * k + 1 >= n) f.y = 0.f;
                }
                ds[k] = pack2<T>(f.x, f.y);
                const float2 left = fma2(unpack2<T>(ds[k]), make_float2(-1.f, -1.f), f);
                low[k] = pack2<T>(left.x, left.y);
            }
            // dS goes where the scores stood, which both warps of a quarter have read before they come here
            bar_pair(1 + quarter);
            tc::tmem_st_x16(mine + 16 * half, ds);
            tc::tmem_st_x16(mine + 32 + 16 * half, low);
            tc::tmem_st_wait();
            tc::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(base + M::kDs);
        }
        if (ok) ok = __all_sync(~0u, x > 0 ? wait(base + M::kDq, (x - 1) & 1, abort_flag) : wait(base + M::kBarQ, 0, abort_flag));
        if (ok) {
            tc::tc_fence_after_sync();
            const int64_t row = (((int64_t)t.b * s.queries + i) * s.heads + h) * s.d;
            const float back = a.scale / lift;
            // the two warps of a quarter take a half of the dimensions each
            write_rows<T, DP / 2>(sm + M::kQ + quarter * 32 * 128 + (DP == 128 ? half * kRows * 128 : 0), kRows * 128, static_cast<T *>(a.result) + half * (DP / 2), row, there,
                                  s.d - half * (DP / 2), half * (DP == 64), [&](int g, uint4 (&v)[4]) {
                uint32_t o[32];
                float f[32];
                if (x > 0) tc::tmem_ld_x32(mine + 128 + half * (DP / 2) + 32 * g, o);
                if (kLong && x > kRun) {
                    uint32_t before[32];
                    tc::tmem_ld_x32(mine + 128 + DP + half * (DP / 2) + 32 * g, before);
#pragma unroll
                    for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) + __uint_as_float(before[y]));
                }
#pragma unroll
                for (int y = 0; y < 32; ++y) {
                    f[y] = x > 0 && alive ? __uint_as_float(o[y]) * back : 0.f;
                    bad |= alive && !finite(f[y]);
                }
#pragma unroll
                for (int y = 0; y < 4; ++y) v[y] = pack8<T>(f + 8 * y);
            });
        }
    }
    tc::tc_fence_before_sync();
    const bool again = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
        const bool gave_up = *abort_flag != 0;
        redo[t.index] = again || gave_up;
        if (gave_up) atomicOr(status, kStatusGradQ);
    }
    if (warp == 9) {
        tc::tc_fence_after_sync();
        tc::tmem_dealloc(tmem, M::kColumns);
    }
}

// dK, dV: a block of 64 keys of one head through the tiles of queries in which any has listed it.  Per tile S = Q K^T and dP = dO V^T as above, rows in lanes;
// P and dS go to shared memory, where they are the operands of dV^T[d x 64] += dO^T P and dK^T += Q^T dS: contracted over the rows, all heads of the group
// summed on the way, in the order of the tiles.  d <= 64: both at once, [dO Q]^T [P dS], whose other two quarters are not used.
// d > 64: 225 KB of shared memory, one CTA an SM, five places for copies of Q and dO, which come one by one; S and dP double buffered in tensor memory, so that the
// products of the next tile run under this one's exponentials, and two groups of softmax warps that take tiles in turn.  d <= 64: two CTAs an SM with one buffer and
// one group each, so that one begins and ends under the other's work; few tiles have listed a block where a tile is 128 queries.  A group has eight warps, two to a
// quarter of the rows, 32 keys each.
// Bound by shared memory and hand-overs: a tile's products read 192 KB of operands there (1540 cycles), its copies and P, dS write 96 KB (770), and it takes 3200: the
// tiles above 851 us, 0.70 PFLOP/s on them (938 with four places, one group and one wait after another; 837 before sums were put aside).  A block that most later queries have listed (up to 392
// tiles there, 138 on average) is one CTA's work and starts first.
//
// After kRun tiles the first group puts the sums aside, in the workspace, where they are added in fp32: without it dV was 7.9e-4 too small by 1024 tiles and 4.6 % by 60 000, with it
// 2.0e-4 however many there are.  The tiles above take 17 us more; runs of 128 lose 1.0e-4 and take 57.
template <int DP> struct GradKVSmem {
    static constexpr int kBuffers = DP == 64 ? 1 : 2, kCtas = DP == 64 ? 2 : 1;   // of S and dP; CTAs an SM
    // Q and dO of tile x are copies 2 x and 2 x + 1, copy n in place n % kPlaces; d <= 64: always Q in an even one, dO behind it
    static constexpr uint32_t kPlaces = DP == 64 ? 4 : 5;
    static constexpr int kGroups = DP == 64 ? 1 : 2, kThreads = 64 + 256 * kGroups;   // of eight softmax warps, which take turns
    static constexpr uint32_t kColumns = kBuffers * 128 + 128;   // of tensor memory: S and dP, the gradients
    static constexpr uint32_t kAlloc = kColumns > 256 ? 512 : 256;
    static constexpr int kSlotBytes = kBlock * DP * 2, kQBytes = kRows * DP * 2, kPBytes = kRows * kBlock * 2;
    static constexpr int kK = 1024, kV = kK + kSlotBytes, kP = kV + kSlotBytes, kStage = kP + 2 * kPBytes,   // P, dS; places for Q and dO
                         kBytes = kStage + kPlaces * kQBytes;
    static constexpr int kBars = kEntries * sizeof(Entry);
    static constexpr int kKV = kBars, kFull = kKV + 8, kEmpty = kFull + 8 * kPlaces, kSP = kEmpty + 8 * kPlaces, kPds = kSP + 16, kDone = kPds + 8, kE = kDone + 16, kDrain = kE + 8 * kEntries,
                         kAbort = kDrain + 8, kHolder = kAbort + 4;
    static constexpr int kChunk = 512;
    static_assert(kHolder + 4 <= kChunk && kCtas * (kBytes + 1024) <= 228 * 1024, "shared memory");
    static_assert(kRun % kGroups == 0, "the first group's tile begins a run");
    static constexpr int kAside = 2 * kBlock * DP;   // sums of a block
};
template <typename T, int DP>
__global__ void __launch_bounds__(GradKVSmem<DP>::kThreads, GradKVSmem<DP>::kCtas) grad_kv_kernel(const Args a, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_g,
                                                                    const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, uint32_t *redo,
                                                                    uint32_t *status) {
    using M = GradKVSmem<DP>;
    extern __shared__ __align__(1024) uint8_t sm[];
    const uint32_t base = tc::smem_u32(sm);
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(sm + M::kAbort);
    const Shape &s = a.s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t bh = blockIdx.x % ((int64_t)s.batch * s.kv_heads);   // the first blocks have most queries behind them: they go first, of all heads
    const int j = (int)(blockIdx.x / ((int64_t)s.batch * s.kv_heads)), kvh = (int)(bh % s.kv_heads), b = (int)(bh / s.kv_heads);
    const int len = s.length(b), live = a.tile * s.group;
    if (base & 1023u) {   // as in the kernel above
        pdl_wait();
        if (threadIdx.x == 0) redo[bh * s.blocks + j] = 1;
        return;
    }

    if (threadIdx.x == 0) {
        for (int bar : {M::kKV, M::kSP, M::kSP + 8, M::kDone, M::kDone + 8, M::kDrain}) tc::mbar_init(base + bar, 1);
        for (uint32_t i = 0; i < 2 * M::kPlaces; ++i) tc::mbar_init(base + M::kFull + 8 * i, 1);   // and kEmpty, behind it
        tc::mbar_init(base + M::kPds, 8);
        for (int i = 0; i < kEntries; ++i) tc::mbar_init(base + M::kE + 8 * i, 1);
        *abort_flag = 0;
        tc::fence_mbar_init();
    }
    if (warp == 9) {
        tc::tmem_alloc(base + M::kHolder, M::kAlloc);
        tc::tmem_relinquish();
    }
    // rows of the last places, which no copy fills, are contracted over too: zeros
    for (int x = threadIdx.x; x < (kRows - live) * 8 * (int)M::kPlaces * (DP / 64); x += M::kThreads)
        *reinterpret_cast<uint4 *>(sm + M::kStage + x / ((kRows - live) * 8) * (kRows * 128) + live * 128 + x % ((kRows - live) * 8) * 16) = make_uint4(0, 0, 0, 0);
    tc::fence_proxy_async();
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(sm + M::kHolder), tmem_acc = tmem + M::kBuffers * 128;
    bool bad = false;
    pdl_launch_dependents();

    pdl_wait();   // all roles: the bounded waits below are for this kernel's own work, not for that of kernels before it
    if (warp == 8) {
        if (lane == 0) {
            tc::mbar_expect_tx(base + M::kKV, 2 * M::kSlotBytes);
            for (int y = 0; y < DP / 64; ++y) {
                tc::tma_load_4d(base + M::kK + y * kBlock * 128, &map_k, base + M::kKV, y * 64, kvh, j * kBlock, b);
                tc::tma_load_4d(base + M::kV + y * kBlock * 128, &map_v, base + M::kKV, y * 64, kvh, j * kBlock, b);
            }
        }
        const uint32_t q_bytes = (uint32_t)(live * 128 * (DP / 64));
        const int tiles = (s.queries + a.tile - 1) / a.tile;
        const int shown = j * kBlock >= len ? tiles : s.causal ? max(0, j * kBlock - (s.keys - s.queries)) / a.tile : 0;   // no tile before can have the block
        const uint32_t mask = a.tile >= 32 ? ~0u : (1u << a.tile) - 1;
        const uint32_t *bits = a.bits + bh * s.words * s.blocks + j;
        uint32_t then[4];
        auto fetch = [&](int from) {
            const int i0 = (from + lane) * a.tile;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                then[k] = from + lane < tiles && (k == 0 || 32 * k < a.tile) && (i0 >> 5) + k < s.words
                              ? (load_here(bits + (int64_t)((i0 >> 5) + k) * s.blocks) >> (i0 & 31)) & mask
                              : 0u;
        };
        uint32_t(*chunk)[32] = reinterpret_cast<uint32_t(*)[32]>(sm + M::kChunk);
        uint32_t x = 0, copies = 0;
        bool ok = true;
        auto free = [&](uint32_t n) { return n < M::kPlaces || wait(base + M::kEmpty + 8 * (n % M::kPlaces), (n / M::kPlaces - 1) & 1, abort_flag); };
        fetch(shown);
        for (int from = shown; from < tiles; from += 32) {   // as Scan::next
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) chunk[k][lane] = then[k];
            uint32_t some = __ballot_sync(~0u, (then[0] | then[1] | then[2] | then[3]) != 0);
            fetch(from + 32);
            __syncwarp();
            if (lane == 0)
                for (; some && ok; some &= some - 1, ++x) {
                    const int src = __ffs(some) - 1;
                    const int i0 = (from + src) * a.tile;
                    auto copy = [&](const CUtensorMap *map, uint32_t n) {
                        const uint32_t bar = base + M::kFull + 8 * (n % M::kPlaces), at = base + M::kStage + n % M::kPlaces * M::kQBytes;
                        tc::mbar_expect_tx(bar, q_bytes);
                        for (int y = 0; y < DP / 64; ++y) tc::tma_load_4d(at + y * kRows * 128, map, bar, y * 64, kvh * s.group, i0, b);
                    };
                    if (!(ok = free(2 * x))) break;
                    Entry *to = reinterpret_cast<Entry *>(sm) + x % kEntries;
                    *reinterpret_cast<uint4 *>(to->rows) = make_uint4(chunk[0][src], chunk[1][src], chunk[2][src], chunk[3][src]);
                    to->block = i0;
                    tc::mbar_arrive(base + M::kE + 8 * (x % kEntries));
                    copy(&map_q, 2 * x);
                    copies = 2 * x + 1;
                    if (!(ok = free(2 * x + 1))) break;
                    copy(&map_g, 2 * x + 1);
                    copies = 2 * x + 2;
                }
        }
        if (lane == 0) {
            if (ok && free(2 * x) && free(2 * x + 1)) {
                for (uint32_t y = x; y < x + M::kGroups; ++y) {   // the end, for each group, with the number of tiles
                    Entry *to = reinterpret_cast<Entry *>(sm) + y % kEntries;
                    to->rows[0] = x;
                    to->block = -1;
                    tc::mbar_arrive(base + M::kE + 8 * (y % kEntries));
                }
                tc::mbar_arrive(base + M::kFull + 8 * (2 * x % M::kPlaces));
                tc::mbar_arrive(base + M::kFull + 8 * ((2 * x + 1) % M::kPlaces));
            }
            if (*abort_flag)   // copies in flight end before the shared memory is given back
                for (uint32_t n = copies > M::kPlaces ? copies - M::kPlaces : 0; n < copies; ++n)
                    for (uint32_t y = 0; y < 1024 && !tc::mbar_try_wait(base + M::kFull + 8 * (n % M::kPlaces), (n / M::kPlaces) & 1); ++y) {}
            for (uint32_t y = 0; y < tc::kMaxPolls && !tc::mbar_try_wait(base + M::kKV, 0); ++y) {}   // nobody else waits for these where no tile has the block
        }
    } else if (warp == 9) {
        constexpr uint32_t kIdescS = idesc<T>(kBlock, 0, 0), kIdescG = idesc<T>(DP == 64 ? 2 * kBlock : kBlock, 1, 1);
        const uint32_t hi = tc::smem_desc_hi(1024, (uint32_t)tc::kSwizzle128B);
        const uint32_t k_lo = tc::smem_desc_lo(base + M::kK, 16), v_lo = tc::smem_desc_lo(base + M::kV, 16);
        const uint32_t q_lo = tc::smem_desc_lo(base + M::kStage, 16);
        // contracted over the rows: 64-dimension slabs; at d <= 64 Q's slab and dO's are the two halves of one operand, P and dS of the other
        const uint32_t qt_lo = tc::smem_desc_lo(base + M::kStage, kRows * 128);
        const uint32_t p_lo = tc::smem_desc_lo(base + M::kP, M::kPBytes), ds_lo = tc::smem_desc_lo(base + M::kP + M::kPBytes, M::kPBytes);
        const bool leader = elect_one();
        bool ok = wait_all(base + M::kKV, 0, abort_flag);
        uint32_t scored = 0, summed = 0, idle = 0;   // tiles whose scores, and whose gradients, have been issued
        bool last = false;
        struct Turn {   // place and phase of a copy: counted on, not divided, so that they and the descriptors made of them stay in uniform registers
            uint32_t place, phase;
            __device__ void next() {
                place += 2;
                if (place >= M::kPlaces) place -= M::kPlaces, phase ^= 1;
            }
        } q_turn = {0, 0}, g_turn = {1, 0}, q_sum = {0, 0}, g_sum = {1, 0};
        auto product = [&](uint32_t at, uint32_t to, uint32_t with) {   // S or dP: rows of a copy times the keys or values
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
                tc::mma_f16_ss(to, tc::desc64(at + (k / 4) * (kRows * 128 >> 4) + (k % 4) * 2, hi), tc::desc64(with + (k / 4) * (kBlock * 128 >> 4) + (k % 4) * 2, hi),
                               kIdescS, k > 0);
        };
        // Whichever can go goes: gradients first, for they free places.  S and dP go where those of kBuffers tiles ago stood, which were read before P and dS were
        // said to be there.
        while (ok && !(last && summed == scored)) {
            const uint32_t over = __reduce_and_sync(~0u, are_over(base + M::kPds, summed & 1, base + M::kFull + 8 * q_turn.place, q_turn.phase,
                                                                  base + M::kFull + 8 * g_turn.place, g_turn.phase));
            if (summed < scored && (over & 1)) {
                tc::tc_fence_after_sync();
                if (leader) {
                    const uint32_t q_at = qt_lo + q_sum.place * (M::kQBytes >> 4), g_at = qt_lo + g_sum.place * (M::kQBytes >> 4);
                    if constexpr (DP == 64) {   // rows of the result: Q's dimensions, then dO's; columns: with P, then with dS
#pragma unroll
                        for (int k = 0; k < kRows / 16; ++k)
                            tc::mma_f16_ss(tmem_acc, tc::desc64(q_at + 128 * k, hi), tc::desc64(p_lo + 128 * k, hi), kIdescG, summed % kRun > 0 || k > 0);
                    } else {
#pragma unroll
                        for (int k = 0; k < kRows / 16; ++k)
                            tc::mma_f16_ss(tmem_acc + 64, tc::desc64(q_at + 128 * k, hi), tc::desc64(ds_lo + 128 * k, hi), kIdescG, summed % kRun > 0 || k > 0);
                        tc::mma_commit(base + M::kEmpty + 8 * q_sum.place);
#pragma unroll
                        for (int k = 0; k < kRows / 16; ++k)
                            tc::mma_f16_ss(tmem_acc, tc::desc64(g_at + 128 * k, hi), tc::desc64(p_lo + 128 * k, hi), kIdescG, summed % kRun > 0 || k > 0);
                    }
                    tc::mma_commit(base + M::kDone + 8 * (summed & 1));
                    if (DP == 64) tc::mma_commit(base + M::kEmpty + 8 * q_sum.place);
                    tc::mma_commit(base + M::kEmpty + 8 * g_sum.place);
                }
                __syncwarp();
                ++summed;
                q_sum.next();
                g_sum.next();
            } else if (!last && scored < summed + M::kBuffers && over >= 6) {
                last = __any_sync(~0u, reinterpret_cast<volatile Entry *>(sm)[scored % kEntries].block < 0);
                if (!last) {
                    tc::tc_fence_after_sync();
                    if (leader) {
                        product(q_lo + q_turn.place * (M::kQBytes >> 4), tmem + scored % M::kBuffers * 128, k_lo);
                        product(q_lo + g_turn.place * (M::kQBytes >> 4), tmem + scored % M::kBuffers * 128 + 64, v_lo);
                        tc::mma_commit(base + M::kSP + 8 * (scored % M::kBuffers));
                    }
                    __syncwarp();
                    ++scored;
                    q_turn.next();
                    g_turn.next();
                }
            } else {
                if (++idle == kMaxPolls) *abort_flag = 1;
                ok = !__any_sync(~0u, *abort_flag != 0);
                continue;
            }
            idle = 0;
        }
        if (leader) {   // the results are read behind this; and tensor memory is given back
            tc::mma_commit(base + M::kDrain);
            for (uint32_t y = 0; y < 4096 && !tc::mbar_try_wait(base + M::kDrain, 0); ++y) {}
        }
        __syncwarp();
    } else {
        const int group = warp > 9, quarter = warp & 3, half = (group ? warp - 10 : warp) >> 2;
        const int r = quarter * 32 + lane, qx = r / s.group, g = r % s.group, h = kvh * s.group + g;
        const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16) + 32 * half;
        const float c = a.scale * kLog2e;
        float lift = 1.f;
        uint32_t x = group, total = 0;
        bool ok = true;
        // what a row has in a tile; its two numbers come from L2 and are asked for before its scores are waited for
        struct Row {
            bool listed;
            int n;   // keys of the row from this warp's first on
            float lse, delta;
        } next;
        bool more = false;
        auto look = [&](uint32_t y) {   // the row of tile y into `next`
            ok = __all_sync(~0u, wait(base + M::kE + 8 * (y % kEntries), (y / kEntries) & 1, abort_flag));
            if (!ok) return;
            const volatile Entry &e = reinterpret_cast<volatile Entry *>(sm)[y % kEntries];
            const int i0 = e.block, i = i0 + qx;
            more = i0 >= 0;
            if (!more) {
                total = e.rows[0];
                return;
            }
            next.listed = r < live && i < s.queries && (e.rows[qx >> 5] >> (qx & 31) & 1u);
            next.n = next.listed ? min(kBlock, s.end(i, len) - j * kBlock) - 32 * half : 0;
            next.lse = INFINITY;
            next.delta = 0.f;
            if (next.listed) {
                const int64_t row = ((int64_t)b * s.heads + h) * s.queries + i;
                next.lse = __ldcg(a.lse + row);
                next.delta = __ldcg(a.delta + row);
            }
        };
        // accumulators: a dimension to a lane, keys in columns.  d > 64: dV in columns 0 .. 63, dK in 64 ..; d <= 64: dK in lanes 0 .. 63 of columns 64 ..,
        // dV in lanes 64 .. of columns 0 ..  The two halves of the first group's warps take one of the two each, or 32 keys each.
        const bool is_k = DP == 64 ? quarter < 2 : half == 1;
        constexpr int kParts = DP == 64 ? 1 : 2;
        const uint32_t sums_at = tmem_acc + ((uint32_t)(quarter * 32) << 16) + (is_k ? 64 : 0) + (DP == 64 ? 32 * half : 0);
        float *aside = a.aside + (bh * s.blocks + j) * M::kAside + threadIdx.x;
        look(x);
        if (ok && more) lift = Lift<T>::grad(a.peak + bh * s.blocks + j) * exp2i(-Lift<T>::kWeight);
        for (; ok && more; x += M::kGroups) {
            if (x > 0 && x % kRun == 0) {   // the first group: its P and dS, without which the next product does not start, are not there yet
                if (!(ok = __all_sync(~0u, wait(base + M::kDone + 8 * ((x - 1) & 1), ((x - 1) >> 1) & 1, abort_flag)))) break;
                tc::tc_fence_after_sync();
#pragma unroll 1
                for (int part = 0; part < kParts; ++part) {
                    uint32_t o[32];
                    tc::tmem_ld_x32(sums_at + 32 * part, o);
#pragma unroll
                    for (int y = 0; y < 32; ++y) {
                        float *to = aside + (part * 32 + y) * 256;
                        *to = x > kRun ? *to + __uint_as_float(o[y]) : __uint_as_float(o[y]);
                    }
                }
            }
            const bool listed = next.listed;
            const int n = next.n;
            const float base2 = next.lse - Lift<T>::kWeight, minus_delta = -next.delta * lift;
            ok = __all_sync(~0u, wait(base + M::kSP + 8 * (x % M::kBuffers), (x / M::kBuffers) & 1, abort_flag));
            if (!ok) break;
            tc::tc_fence_after_sync();
            const bool whole = __all_sync(~0u, !listed || n >= 32);   // a row that has not listed the block has no weight there: base2
            uint32_t u[32], d[32], p[16], ds[16];
            tc::tmem_ld_x32_issue(mine + x % M::kBuffers * 128, u);
            tc::tmem_ld_x32_issue(mine + x % M::kBuffers * 128 + 64, d);
            tc::tmem_ld_x32_wait(u);
            tc::tmem_ld_x32_wait(d);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                float2 w = fma2(pair(u[2 * k], u[2 * k + 1]), make_float2(c, c), make_float2(-base2, -base2));
                w.x = ex2(w.x);
                w.y = ex2(w.y);
                float2 f = mul2(w, fma2(pair(d[2 * k], d[2 * k + 1]), make_float2(lift, lift), make_float2(minus_delta, minus_delta)));
                if (!whole) {
                    if (2 * k >= n) w.x = f.x = 0.f;
                    if (2 * k + 1 >= n) w.y = f.y = 0.f;
                }
                p[k] = pack2<T>(w.x, w.y);
                ds[k] = pack2<T>(f.x, f.y);
            }
            // P and dS of the tile before have been read.  A barrier for every second tile: the phase before this one, of tile x - 3, is over, for this group has waited for it
            // ahead of tile x - 2 (one group: likewise).
            if (x > 0 && !(ok = __all_sync(~0u, wait(base + M::kDone + 8 * ((x - 1) & 1), ((x - 1) >> 1) & 1, abort_flag)))) break;
            uint8_t *to = sm + M::kP + r * 128;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int at = ((4 * half + y) ^ (r & 7)) << 4;
                *reinterpret_cast<uint4 *>(to + at) = make_uint4(p[4 * y], p[4 * y + 1], p[4 * y + 2], p[4 * y + 3]);
                *reinterpret_cast<uint4 *>(to + M::kPBytes + at) = make_uint4(ds[4 * y], ds[4 * y + 1], ds[4 * y + 2], ds[4 * y + 3]);
            }
            tc::fence_proxy_async();
            tc::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(base + M::kPds);
            look(x + M::kGroups);
        }
        // All products, of this group's tiles and of the other's.  The last tile may be the other group's, and the end is posted when the place of Q of the tile before it is
        // free, ahead of that tile's kDone: a wait for kDone could take an earlier phase for the last one.  kDrain has one phase, behind the last product.
        if (ok && total > 0) ok = __all_sync(~0u, wait(base + M::kDrain, 0, abort_flag));
        if (ok && group == 0) {
            tc::tc_fence_after_sync();
            const float back_v = exp2i(-Lift<T>::kWeight), back_k = total > 0 ? a.scale / (lift * exp2i(Lift<T>::kWeight)) : 0.f;
            const int dim = (DP == 64 ? quarter % 2 : quarter) * 32 + lane;
            const float back = is_k ? back_k : back_v;
            T *out = static_cast<T *>(is_k ? a.grad_k : a.grad_v) + (((int64_t)b * s.keys + j * kBlock) * s.kv_heads + kvh) * s.d + dim;
            const int64_t pitch = (int64_t)s.kv_heads * s.d;
            const int keys = min(kBlock, s.keys - j * kBlock);
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                const int first = DP == 64 ? 32 * half : 32 * part;
                uint32_t o[32];
                if (total > 0) tc::tmem_ld_x32(sums_at + 32 * part, o);
#pragma unroll
                for (int y = 0; y < 32; ++y) {
                    const float sum = total > kRun ? __uint_as_float(o[y]) + aside[(part * 32 + y) * 256] : __uint_as_float(o[y]);
                    const float f = total > 0 ? sum * back : 0.f;
                    if (dim < s.d && first + y < keys) {
                        bad |= !finite(f);
                        out[(first + y) * pitch] = from_f32<T>(f);
                    }
                }
            }
        }
    }
    tc::tc_fence_before_sync();
    const bool again = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
        const bool gave_up = *abort_flag != 0;
        redo[bh * s.blocks + j] = again || gave_up;
        if (gave_up) atomicOr(status, kStatusGradKV);
    }
    if (warp == 9) {
        tc::tc_fence_after_sync();
        tc::tmem_dealloc(tmem, M::kAlloc);
    }
}

}  // namespace tcore
}  // namespace blocks
}  // namespace vs
