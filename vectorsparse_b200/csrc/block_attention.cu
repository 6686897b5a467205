// extern "C" entry points of attention over chosen blocks and of the 8-bit cache: argument validation and launches.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <type_traits>
#include <utility>

#include "vsparse_b200.h"
#include "common.cuh"
#include "host.h"
#include "smem_limit.h"
#include "blocks.cuh"
#include "blocks_tc.cuh"
#include "cache.cuh"

#define VS_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

using namespace vs;

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
constexpr int64_t kMaxGrid = 0x7fffffff;
constexpr int kMaxSmem = 227 * 1024;

template <typename... Exp, typename... Act>
cudaError_t launch_behind(void (*kernel)(Exp...), unsigned grid, unsigned block, size_t smem, cudaStream_t s, Act &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Act>(args)...);
}
// The most shared memory that a kernel may ask for, told to the runtime where it grows (the kernel's address is the key).
template <auto kKernel> int allow_smem(int bytes) {
    static SmemLimit limit;
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= SmemLimit::kDevices) return VS_ERR_ARG;
    return limit.raise(dev, bytes, [&] { return (int)cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
}

// ---- attention over chosen blocks -----------------------------------------------------------------------------------

// Sizes and types of a call; nothing of it needs a device.
int check_shape(int dtype, int batch, int queries, int keys, int heads, int kv_heads, int d, int count, int causal, const int32_t *lengths, blocks::Shape &s) {
    if (dtype != VS_F16 && dtype != VS_BF16) return VS_ERR_DTYPE;
    if (batch < 0 || queries < 0 || keys < 0) return VS_ERR_SHAPE;
    if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads / kv_heads > 128) return VS_ERR_SHAPE;
    if (d < 8 || d > blocks::kMaxD || d % 8 != 0) return VS_ERR_SHAPE;
    if (count < 1 || count > blocks::kMaxCount || queries > blocks::kMaxQueries || keys > blocks::kMaxBlocks * blocks::kBlock) return VS_ERR_SHAPE;
    if (causal != 0 && causal != 1) return VS_ERR_ARG;
    if (causal && queries > keys) return VS_ERR_SHAPE;
    if (lengths && queries != keys) return VS_ERR_SHAPE;
    if (lengths && !aligned4(lengths)) return VS_ERR_ALIGN;
    s.batch = batch; s.queries = queries; s.keys = keys; s.heads = heads; s.kv_heads = kv_heads; s.d = d; s.count = count; s.causal = causal;
    s.group = heads / kv_heads;
    s.blocks = (keys + blocks::kBlock - 1) / blocks::kBlock;
    s.words = (queries + 31) / 32;
    s.lengths = lengths;
    const int64_t pairs = (int64_t)batch * kv_heads;
    // CTAs of any launch: a word, a query (tiles of one) or a block of keys each
    if (pairs * std::max<int64_t>(queries, s.blocks) > kMaxGrid || (int64_t)batch * heads > kMaxGrid || (int64_t)batch * heads * queries > kMaxGrid * 16) return VS_ERR_SHAPE;
    return VS_OK;
}
int operand(blocks::Operand &o, const void *at, const int64_t *strides, int batch, int tokens, int heads) {
    if (!at || !strides) return VS_ERR_NULL;
    if (!aligned16(at)) return VS_ERR_ALIGN;
    const int extent[3] = {batch, tokens, heads};
    for (int i = 0; i < 3; ++i) {
        if (strides[i] < 0 || (strides[i] == 0 && extent[i] > 1)) return VS_ERR_SHAPE;
        if (strides[i] % 8 != 0) return VS_ERR_ALIGN;
    }
    o.at = at; o.batch = strides[0]; o.token = strides[1]; o.head = strides[2];
    return VS_OK;
}
void contiguous(blocks::Operand &o, const void *at, int64_t tokens, int64_t heads, int64_t d) {
    o.at = at; o.batch = tokens * heads * d; o.token = heads * d; o.head = d;
}
inline int64_t up256(int64_t bytes) { return (bytes + 255) & ~255ll; }
inline int64_t bits_bytes(const blocks::Shape &s) { return up256((int64_t)s.batch * s.kv_heads * s.words * s.blocks * 4); }

inline int64_t rows_bytes(const blocks::Shape &s) { return up256((int64_t)s.batch * s.heads * s.queries * 4); }
// Queries of a tile: the largest power of two whose rows (queries x heads of the group) fit 128.
inline int tile_queries(int group) {
    int t = 128;
    while (t * group > 128) t /= 2;
    return t;
}
// Where a block can have more tiles than are summed at a stretch: what is put aside.
inline int64_t aside_bytes(const blocks::Shape &s) {
    const int tile = tile_queries(s.group);
    return s.queries / tile < (int)blocks::tcore::kRun ? 0 : (int64_t)s.batch * s.kv_heads * s.blocks * 4 * (s.d <= 64 ? blocks::tcore::GradKVSmem<64>::kAside : blocks::tcore::GradKVSmem<128>::kAside);
}
inline int64_t redo_bytes(const blocks::Shape &s) { return up256((int64_t)s.batch * s.kv_heads * ((int64_t)s.queries + s.blocks) * 4); }   // a word per tile and block

template <typename T, int QT> int launch_scores(const blocks::Shape &s, const blocks::Operand &q, const double *means, int32_t *lists, cudaStream_t st) {
    const int smem = (int)blocks::score_bytes<QT>(s.blocks, s.d);
    const int rc = allow_smem<blocks::score_kernel<T, QT>>(smem);
    if (rc != VS_OK) return rc;
    const int64_t grid = (int64_t)s.batch * s.kv_heads * ((s.queries + QT - 1) / QT);
    blocks::score_kernel<T, QT><<<(unsigned)grid, blocks::kScoreThreads, smem, st>>>(s, q, means, lists);
    return (int)cudaGetLastError();
}
// The workspace of a choice: means in 64 and in 32 bits and the norms of the latter, then the scores of a slab and the error bounds of its queries.  Slabs of 48 MB stay in
// L2 between the two kernels that share them.
struct SelectSpace {
    int64_t means, blocks, tiles, slab;   // elements of the means, blocks of keys, tiles of queries, tiles of a slab
    bool fast;
    int64_t bytes() const { return up256(means * 8) + up256(means * 4) + up256(blocks * 4) + slab * blocks::kFastQueries * 4 * (per_query + 1); }
    int64_t per_query;
    SelectSpace(int64_t pairs, int64_t queries, int64_t keys, int64_t d) {
        per_query = (keys + blocks::kBlock - 1) / blocks::kBlock;
        blocks = pairs * per_query;
        means = blocks * d;
        tiles = pairs * ((queries + blocks::kFastQueries - 1) / blocks::kFastQueries);
        fast = per_query > 0 && per_query <= blocks::kFastMost;
        slab = fast ? std::max<int64_t>(1, std::min(tiles, (int64_t(48) << 20) / (blocks::kFastQueries * 4 * per_query))) : 0;
    }
};
template <typename T> int select(const blocks::Shape &s, const blocks::Operand &q, const blocks::Operand &k, int32_t *lists, void *workspace, cudaStream_t st) {
    const SelectSpace space((int64_t)s.batch * s.kv_heads, s.queries, s.keys, s.d);
    char *at = static_cast<char *>(workspace);
    double *means = reinterpret_cast<double *>(at);
    float *means32 = reinterpret_cast<float *>(at += up256(space.means * 8)), *norms = reinterpret_cast<float *>(at += up256(space.means * 4));
    if (s.blocks > 0) {
        blocks::means_kernel<T><<<(unsigned)space.blocks, blocks::kMeanThreads, 0, st>>>(s, k, means, means32, norms);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return (int)e;
    }
    if (space.fast && s.count <= blocks::kFastCount) {
        const int smem = blocks::fast_bytes(s.d);
        const int rc = allow_smem<blocks::fast_score_kernel<T>>(smem);
        if (rc != VS_OK) return rc;
        blocks::Slab slab;
        slab.scores = reinterpret_cast<float *>(at + up256(space.blocks * 4));
        slab.errors = slab.scores + space.slab * blocks::kFastQueries * s.blocks;
        for (slab.first = 0; slab.first < space.tiles; slab.first += space.slab) {
            slab.tiles = std::min(space.slab, space.tiles - slab.first);
            cudaError_t e = launch_behind(blocks::fast_score_kernel<T>, (unsigned)slab.tiles, blocks::kFastThreads, smem, st, s, q, (const float *)means32, slab);
            if (e == cudaSuccess)
                e = launch_behind(blocks::fast_rank_kernel<T>, (unsigned)(slab.tiles * blocks::kFastQueries / (blocks::kFastThreads / 32)), blocks::kFastThreads, 0, st, s, q,
                                  (const double *)means, (const float *)norms, slab, lists);
            if (e != cudaSuccess) return (int)e;
        }
        return VS_OK;
    }
    // as many queries to a CTA as their scores leave room for
    if (blocks::score_bytes<32>(s.blocks, s.d) <= kMaxSmem) return launch_scores<T, 32>(s, q, means, lists, st);
    if (blocks::score_bytes<8>(s.blocks, s.d) <= kMaxSmem) return launch_scores<T, 8>(s, q, means, lists, st);
    return launch_scores<T, 1>(s, q, means, lists, st);
}
static_assert(2 * (blocks::fast_bytes(blocks::kMaxD) + 1024) <= 228 * 1024, "two CTAs an SM");
static_assert(blocks::score_bytes<1>(blocks::kMaxBlocks, blocks::kMaxD) <= kMaxSmem, "scores of one query");

int make_bits(const blocks::Shape &s, const int32_t *lists, uint32_t *bits, uint32_t *zero, cudaStream_t st) {
    if (s.blocks == 0) return VS_OK;
    blocks::bits_kernel<<<(unsigned)((int64_t)s.batch * s.kv_heads * s.words), blocks::kBitsThreads, 0, st>>>(s, lists, bits, zero);
    return (int)cudaGetLastError();
}

// {d, heads, tokens, batch} of an operand, for copies of 64 dimensions of `heads` heads of `tokens` tokens, 128-byte swizzle; zeros outside.
template <typename T> int make_map(CUtensorMap *map, const blocks::Operand &o, int64_t batch, int64_t tokens, int64_t heads, int64_t d, int box_heads, int box_tokens) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return VS_ERR_DEVICE;
    auto bytes = [](int64_t stride, int64_t extent) { return (cuuint64_t)(extent > 1 ? stride * 2 : 16); };   // of one, any will do
    const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)batch};
    const cuuint64_t strides[3] = {bytes(o.head, heads), bytes(o.token, tokens), bytes(o.batch, batch)};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens, 1}, unit[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return fn(map, type, 4, const_cast<void *>(o.at), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? VS_OK
               : VS_ERR_ARG;
}
// Tiles of a call and the words that say which of them are to be computed again, one by one.
inline int64_t query_tiles(const blocks::Shape &s) {
    const int tile = tile_queries(s.group);
    return (int64_t)s.batch * s.kv_heads * ((s.queries + tile - 1) / tile);
}
inline unsigned again_grid(int64_t tiles) { return (unsigned)std::min<int64_t>(tiles, 4 * 148); }

// A handful of products, a prompt's first tokens: the row kernels alone, in fp32 throughout.  Nothing averages the 16-bit roundings of a tile's weights there, and it is no slower: 5 rows of 4 keys 8.4
// us and 21.1 backward against 8.2 and 21.6 by tiles, 32 rows of 2 keys 6.0 and 10.5 against 7.2 and 16.7; 64 rows of 8 keys 22 and 23 against 6.9 and 15.3.
inline bool few(const blocks::Shape &s) {
    return (int64_t)s.batch * s.queries * s.heads <= 64 && (int64_t)s.batch * s.queries * s.heads * std::min<int64_t>(s.keys, (int64_t)s.count * blocks::kBlock) <= 64;
}

// Lists that can hold more blocks than are summed at a stretch.
inline bool long_lists(const blocks::Shape &s) { return std::min(s.count, s.blocks) > (int)blocks::tcore::kRun; }

template <typename T, int DP, bool kLong> int forward(blocks::Args a, uint32_t *redo, uint32_t *status, cudaStream_t st) {
    const blocks::Shape &s = a.s;
    using Smem = blocks::tcore::ForwardSmem<DP, kLong>;
    CUtensorMap q, k, v;
    a.tile = tile_queries(s.group);
    int rc = make_map<T>(&q, a.q, s.batch, s.queries, s.heads, s.d, s.group, a.tile);
    if (rc == VS_OK) rc = make_map<T>(&k, a.k, s.batch, s.keys, s.kv_heads, s.d, 1, blocks::kBlock);
    if (rc == VS_OK) rc = make_map<T>(&v, a.v, s.batch, s.keys, s.kv_heads, s.d, 1, blocks::kBlock);
    if (rc == VS_OK) rc = allow_smem<blocks::tcore::forward_kernel<T, DP, kLong>>(Smem::kBytes + 1024);
    if (rc != VS_OK) return rc;
    const int64_t tiles = query_tiles(s);
    cudaError_t e = launch_behind(blocks::tcore::forward_kernel<T, DP, kLong>, (unsigned)tiles, blocks::tcore::kForwardThreads, Smem::kBytes + 1024, st, a, q, k, v, redo, status);
    if (e != cudaSuccess) return (int)e;
    a.redo = redo;
    return (int)launch_behind(blocks::rows_kernel<T, false>, again_grid(tiles), blocks::kRowThreads, 0, st, a);
}
template <typename T> int attention(blocks::Args a, uint32_t *redo, cudaStream_t st) {
    const blocks::Shape &s = a.s;
    if (s.keys == 0 || few(s)) {
        a.tile = 1;
        blocks::rows_kernel<T, false><<<again_grid((int64_t)s.batch * s.kv_heads * s.queries), blocks::kRowThreads, 0, st>>>(a);
        return (int)cudaGetLastError();
    }
    int sms = 0;
    uint32_t *status = nullptr;
    const int rc = current_device(&sms, &status);
    if (rc != VS_OK) return rc;
    if (long_lists(s)) return s.d <= 64 ? forward<T, 64, true>(a, redo, status, st) : forward<T, 128, true>(a, redo, status, st);
    return s.d <= 64 ? forward<T, 64, false>(a, redo, status, st) : forward<T, 128, false>(a, redo, status, st);
}
template <typename T, int DP, bool kLong> int backward(blocks::Args a, uint32_t *redo, uint32_t *status, cudaStream_t st) {
    const blocks::Shape &s = a.s;
    using SmemQ = blocks::tcore::GradQSmem<DP, kLong>;
    using SmemKV = blocks::tcore::GradKVSmem<DP>;
    CUtensorMap q, g, k, v;
    a.tile = tile_queries(s.group);
    int rc = make_map<T>(&q, a.q, s.batch, s.queries, s.heads, s.d, s.group, a.tile);
    if (rc == VS_OK) rc = make_map<T>(&g, a.grad_out, s.batch, s.queries, s.heads, s.d, s.group, a.tile);
    if (rc == VS_OK) rc = make_map<T>(&k, a.k, s.batch, s.keys, s.kv_heads, s.d, 1, blocks::kBlock);
    if (rc == VS_OK) rc = make_map<T>(&v, a.v, s.batch, s.keys, s.kv_heads, s.d, 1, blocks::kBlock);
    if (rc == VS_OK) rc = allow_smem<blocks::tcore::grad_q_kernel<T, DP, kLong>>(SmemQ::kBytes);
    if (rc == VS_OK) rc = allow_smem<blocks::tcore::grad_kv_kernel<T, DP>>(SmemKV::kBytes);
    if (rc != VS_OK) return rc;
    const int64_t rows = (int64_t)s.batch * s.queries * s.heads, tiles = query_tiles(s), blocks_all = (int64_t)s.batch * s.kv_heads * s.blocks;
    uint32_t *redo_kv = redo + tiles;
    cudaError_t e = launch_behind(blocks::delta_kernel<T>, (unsigned)((rows + 15) / 16), 256, 0, st, a);
    if (std::is_same<T, __half>::value && e == cudaSuccess)
        e = launch_behind(blocks::peaks_kernel, (unsigned)((int64_t)s.batch * s.kv_heads * s.words), blocks::kBitsThreads, 0, st, a);
    if (e == cudaSuccess)
        e = launch_behind(blocks::tcore::grad_q_kernel<T, DP, kLong>, (unsigned)tiles, blocks::tcore::kGradQThreads, SmemQ::kBytes, st, a, q, g, k, v, redo, status);
    if (e == cudaSuccess)
        e = launch_behind(blocks::tcore::grad_kv_kernel<T, DP>, (unsigned)blocks_all, SmemKV::kThreads, SmemKV::kBytes, st, a, q, g, k, v, redo_kv, status);
    if (e != cudaSuccess) return (int)e;
    a.redo = redo;
    e = launch_behind(blocks::rows_kernel<T, true>, again_grid(tiles), blocks::kRowThreads, 0, st, a);
    if (e != cudaSuccess) return (int)e;
    a.redo = redo_kv;
    return (int)launch_behind(blocks::keys_kernel<T>, again_grid(blocks_all), blocks::kRowThreads, 0, st, a);
}
template <typename T> int attention_backward(blocks::Args a, uint32_t *redo, cudaStream_t st) {
    int sms = 0;
    uint32_t *status = nullptr;
    const int rc = current_device(&sms, &status);
    if (rc != VS_OK) return rc;
    if (few(a.s)) {
        a.tile = 1;
        const int64_t rows = (int64_t)a.s.batch * a.s.queries * a.s.heads;
        cudaError_t e = launch_behind(blocks::delta_kernel<T>, (unsigned)((rows + 15) / 16), 256, 0, st, a);
        if (e == cudaSuccess) e = launch_behind(blocks::rows_kernel<T, true>, again_grid((int64_t)a.s.batch * a.s.kv_heads * a.s.queries), blocks::kRowThreads, 0, st, a);
        if (e == cudaSuccess) e = launch_behind(blocks::keys_kernel<T>, again_grid((int64_t)a.s.batch * a.s.kv_heads * a.s.blocks), blocks::kRowThreads, 0, st, a);
        return (int)e;
    }
    if (long_lists(a.s)) return a.s.d <= 64 ? backward<T, 64, true>(a, redo, status, st) : backward<T, 128, true>(a, redo, status, st);
    return a.s.d <= 64 ? backward<T, 64, false>(a, redo, status, st) : backward<T, 128, false>(a, redo, status, st);
}

inline bool scale_ok(float scale) { return scale > 0.f && std::isfinite(scale); }

}  // namespace

VS_EXPORT int64_t vs_select_blocks_workspace_bytes(int batch, int queries, int keys, int kv_heads, int d) {
    if (batch < 1 || queries < 1 || keys < 1 || kv_heads < 1 || d < 1) return 0;
    return SelectSpace((int64_t)batch * kv_heads, queries, keys, d).bytes();
}

VS_EXPORT int vs_select_blocks(int dtype, int batch, int queries, int keys, int heads, int kv_heads, int d, int count, int causal, const void *q,
                               const int64_t *q_strides, const void *k, const int64_t *k_strides, const int32_t *lengths, int32_t *lists, void *workspace,
                               int64_t workspace_bytes, void *stream) {
    blocks::Shape s;
    int rc = check_shape(dtype, batch, queries, keys, heads, kv_heads, d, count, causal, lengths, s);
    if (rc != VS_OK) return rc;
    if (batch == 0 || queries == 0) return VS_OK;
    blocks::Operand oq, ok = {};
    if ((rc = operand(oq, q, q_strides, batch, queries, heads)) != VS_OK) return rc;
    if (keys > 0 && (rc = operand(ok, k, k_strides, batch, keys, kv_heads)) != VS_OK) return rc;
    if (!lists || (keys > 0 && !workspace)) return VS_ERR_NULL;
    if (!aligned16(workspace) || !aligned4(lists)) return VS_ERR_ALIGN;
    if (workspace_bytes < vs_select_blocks_workspace_bytes(batch, queries, keys, kv_heads, d)) return VS_ERR_SHAPE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == VS_F16 ? select<__half>(s, oq, ok, lists, workspace, st) : select<__nv_bfloat16>(s, oq, ok, lists, workspace, st);
}

VS_EXPORT int64_t vs_selected_attention_workspace_bytes(int batch, int queries, int keys, int heads, int kv_heads, int d, int backward) {
    blocks::Shape s;
    if (check_shape(VS_F16, batch, queries, keys, heads, kv_heads, d, 1, 0, nullptr, s) != VS_OK) return 0;
    return bits_bytes(s) + redo_bytes(s) + (backward ? 2 * rows_bytes(s) + up256((int64_t)batch * kv_heads * s.blocks * 4) + aside_bytes(s) : 0);   // two words of a row, one of a block
}

VS_EXPORT int vs_selected_attention(int dtype, int batch, int queries, int keys, int heads, int kv_heads, int d, int count, int causal, const void *q,
                                    const int64_t *q_strides, const void *k, const int64_t *k_strides, const void *v, const int64_t *v_strides,
                                    const int32_t *lengths, const int32_t *lists, void *out, void *out_low, float *lse, float scale, void *workspace,
                                    int64_t workspace_bytes, void *stream) {
    blocks::Args a = {};
    int rc = check_shape(dtype, batch, queries, keys, heads, kv_heads, d, count, causal, lengths, a.s);
    if (rc != VS_OK) return rc;
    if (!scale_ok(scale)) return VS_ERR_ARG;
    if (batch == 0 || queries == 0) return VS_OK;
    if ((rc = operand(a.q, q, q_strides, batch, queries, heads)) != VS_OK) return rc;
    if (keys > 0 && ((rc = operand(a.k, k, k_strides, batch, keys, kv_heads)) != VS_OK || (rc = operand(a.v, v, v_strides, batch, keys, kv_heads)) != VS_OK)) return rc;
    if (!lists || !out || !lse || (keys > 0 && !workspace)) return VS_ERR_NULL;
    if (!aligned16(out) || !aligned16(out_low) || !aligned16(workspace) || !aligned4(lists) || !aligned4(lse)) return VS_ERR_ALIGN;
    if (workspace_bytes < vs_selected_attention_workspace_bytes(batch, queries, keys, heads, kv_heads, d, 0)) return VS_ERR_SHAPE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint32_t *bits = static_cast<uint32_t *>(workspace);
    if ((rc = make_bits(a.s, lists, bits, nullptr, st)) != VS_OK) return rc;
    a.bits = bits; a.lse = lse; a.result = out; a.result_low = out_low; a.scale = scale;
    uint32_t *redo = reinterpret_cast<uint32_t *>(static_cast<char *>(workspace) + bits_bytes(a.s));
    return dtype == VS_F16 ? attention<__half>(a, redo, st) : attention<__nv_bfloat16>(a, redo, st);
}

VS_EXPORT int vs_selected_attention_backward(int dtype, int batch, int queries, int keys, int heads, int kv_heads, int d, int count, int causal,
                                             const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides, const void *v,
                                             const int64_t *v_strides, const int32_t *lengths, const int32_t *lists, const void *out, const void *out_low, const float *lse,
                                             const void *grad_out, const int64_t *grad_out_strides, void *grad_q, void *grad_k, void *grad_v, float scale,
                                             void *workspace, int64_t workspace_bytes, void *stream) {
    blocks::Args a = {};
    int rc = check_shape(dtype, batch, queries, keys, heads, kv_heads, d, count, causal, lengths, a.s);
    if (rc != VS_OK) return rc;
    if (!scale_ok(scale)) return VS_ERR_ARG;
    if (batch == 0) return VS_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (queries == 0 || keys == 0) {   // no query attends to a key
        const size_t q_bytes = (size_t)batch * queries * heads * d * 2, k_bytes = (size_t)batch * keys * kv_heads * d * 2;
        if ((q_bytes && !grad_q) || (k_bytes && (!grad_k || !grad_v))) return VS_ERR_NULL;
        cudaError_t e = cudaSuccess;
        if (q_bytes) e = cudaMemsetAsync(grad_q, 0, q_bytes, st);
        if (e == cudaSuccess && k_bytes) e = cudaMemsetAsync(grad_k, 0, k_bytes, st);
        if (e == cudaSuccess && k_bytes) e = cudaMemsetAsync(grad_v, 0, k_bytes, st);
        return (int)e;
    }
    if ((rc = operand(a.q, q, q_strides, batch, queries, heads)) != VS_OK || (rc = operand(a.k, k, k_strides, batch, keys, kv_heads)) != VS_OK || (rc = operand(a.v, v, v_strides, batch, keys, kv_heads)) != VS_OK ||
        (rc = operand(a.grad_out, grad_out, grad_out_strides, batch, queries, heads)) != VS_OK)
        return rc;
    if (!lists || !out || !lse || !grad_q || !grad_k || !grad_v || !workspace) return VS_ERR_NULL;
    if (!aligned16(out) || !aligned16(out_low) || !aligned16(grad_q) || !aligned16(grad_k) || !aligned16(grad_v) || !aligned16(workspace) || !aligned4(lists) || !aligned4(lse)) return VS_ERR_ALIGN;
    if (workspace_bytes < vs_selected_attention_workspace_bytes(batch, queries, keys, heads, kv_heads, d, 1)) return VS_ERR_SHAPE;
    contiguous(a.out, out, queries, heads, d);
    a.out_low = out_low;
    char *at = static_cast<char *>(workspace);
    uint32_t *bits = reinterpret_cast<uint32_t *>(at), *redo = reinterpret_cast<uint32_t *>(at + bits_bytes(a.s));
    a.bits = bits; a.lse = const_cast<float *>(lse); a.scale = scale; a.result = grad_q; a.grad_k = grad_k; a.grad_v = grad_v;
    at += bits_bytes(a.s) + redo_bytes(a.s);
    a.delta = reinterpret_cast<float *>(at);
    a.most = reinterpret_cast<uint32_t *>(at + rows_bytes(a.s));
    a.peak = reinterpret_cast<uint32_t *>(at + 2 * rows_bytes(a.s));
    a.aside = reinterpret_cast<float *>(at + 2 * rows_bytes(a.s) + up256((int64_t)batch * kv_heads * a.s.blocks * 4));
    if ((rc = make_bits(a.s, lists, bits, a.peak, st)) != VS_OK) return rc;
    return dtype == VS_F16 ? attention_backward<__half>(a, redo, st) : attention_backward<__nv_bfloat16>(a, redo, st);
}

// ---- the cache ----------------------------------------------------------------------------------------------------------

namespace {

int check_cache(int dtype, int pages, int tails, int kv_heads, int d, int sequences, int max_blocks) {
    if (dtype != VS_F16 && dtype != VS_BF16) return VS_ERR_DTYPE;
    if (pages < 0 || tails < 0 || sequences < 0 || kv_heads < 1 || max_blocks < 0) return VS_ERR_SHAPE;
    if (d < 16 || d > blocks::kMaxD || d % 16 != 0) return VS_ERR_SHAPE;
    if ((int64_t)sequences * kv_heads > kMaxGrid) return VS_ERR_SHAPE;
    return VS_OK;
}

template <typename T, int NK> int launch_decode(const cache::AttentionArgs &a, int items, cudaStream_t st) {
    const int smem = cache::decode_smem<NK>();
    const int rc = allow_smem<cache::decode_kernel<T, NK>>(smem);
    if (rc != VS_OK) return rc;
    cache::decode_kernel<T, NK><<<(unsigned)(items * a.pieces), cache::kDecodeThreads, smem, st>>>(a);
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && a.pieces > 1) e = launch_behind(cache::join_kernel<T>, (unsigned)items, 128u, 0, st, a);
    return (int)e;
}
template <typename T> int decode(const cache::AttentionArgs &a, int items, cudaStream_t st) {
    switch (a.c.d / 16) {
        case 1: return launch_decode<T, 1>(a, items, st);
        case 2: return launch_decode<T, 2>(a, items, st);
        case 3: return launch_decode<T, 3>(a, items, st);
        case 4: return launch_decode<T, 4>(a, items, st);
        case 5: return launch_decode<T, 5>(a, items, st);
        case 6: return launch_decode<T, 6>(a, items, st);
        case 7: return launch_decode<T, 7>(a, items, st);
        default: return launch_decode<T, 8>(a, items, st);
    }
}

// Pieces that the blocks of a sequence and head are shared out in: so many that the GPU is full once (two CTAs an SM), but at least four blocks to a warp.  More even out
// sequences of unlike lengths, but each begins and ends anew: 256 heads of up to 128 blocks in 2 / 3 / 5 pieces 92 / 98 / 106 us; 32 heads with 16 blocks in 1 / 2 pieces
// 14.4 / 16.4 us.
int decode_pieces(int64_t items, int units) {
    constexpr int kCtas = 148 * 2;
    const int64_t want = (kCtas + items - 1) / items, most = std::max(1, units / (4 * cache::kWarps));
    return (int)std::min<int64_t>({want, most, 64});
}

}  // namespace

VS_EXPORT int vs_cache_append(int dtype, int pages, int tails, int kv_heads, int d, int8_t *k_codes, int8_t *v_codes, float *k_scales, float *v_scales,
                              int16_t *k_sums, void *k_ring, void *v_ring, int sequences, int tokens, const void *k, const int64_t *k_strides,
                              const void *v, const int64_t *v_strides, const int32_t *table, int max_blocks, const int32_t *tail_indices,
                              const int32_t *lengths, const int32_t *counts, void *stream) {
    int rc = check_cache(dtype, pages, tails, kv_heads, d, sequences, max_blocks);
    if (rc != VS_OK) return rc;
    if (tokens < 0) return VS_ERR_SHAPE;
    if (sequences == 0 || tokens == 0) return VS_OK;
    blocks::Operand n[2];
    if ((rc = operand(n[0], k, k_strides, sequences, tokens, kv_heads)) != VS_OK || (rc = operand(n[1], v, v_strides, sequences, tokens, kv_heads)) != VS_OK) return rc;
    if ((pages > 0 && (!k_codes || !v_codes || !k_scales || !v_scales || !k_sums)) || (tails > 0 && (!k_ring || !v_ring)) || (max_blocks > 0 && !table) ||
        !tail_indices || !lengths)
        return VS_ERR_NULL;
    for (const void *p : {(const void *)k_codes, (const void *)v_codes, (const void *)k_ring, (const void *)v_ring, (const void *)k_sums})
        if (!aligned16(p)) return VS_ERR_ALIGN;
    for (const void *p : {(const void *)table, (const void *)tail_indices, (const void *)lengths, (const void *)counts, (const void *)k_scales, (const void *)v_scales})
        if (!aligned4(p)) return VS_ERR_ALIGN;
    cache::AppendArgs a;
    a.c = {pages, tails, kv_heads, d, {k_codes, v_codes}, {k_scales, v_scales}, k_sums, {k_ring, v_ring}};
    a.s = {sequences, table, max_blocks, tail_indices, lengths};
    a.tokens = tokens;
    a.touched = (int)(((int64_t)tokens + blocks::kBlock - 2) / blocks::kBlock + 1);
    a.counts = counts;
    for (int i = 0; i < 2; ++i) {
        a.at[i] = n[i].at; a.batch[i] = n[i].batch; a.token[i] = n[i].token; a.head[i] = n[i].head;
    }
    const int64_t grid = (int64_t)sequences * kv_heads * a.touched;
    if (grid > kMaxGrid) return VS_ERR_SHAPE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == VS_F16) cache::append_kernel<__half><<<dim3((unsigned)grid, 2), cache::kAppendThreads, blocks::kBlock * d * 2, st>>>(a);
    else cache::append_kernel<__nv_bfloat16><<<dim3((unsigned)grid, 2), cache::kAppendThreads, blocks::kBlock * d * 2, st>>>(a);
    return (int)cudaGetLastError();
}

VS_EXPORT int vs_cache_select(int dtype, int pages, int heads, int kv_heads, int d, const float *k_scales, const int16_t *k_sums, int sequences,
                              const void *q, const int64_t *q_strides, const int32_t *table, int max_blocks, const int32_t *lengths, int count,
                              int32_t *lists, void *stream) {
    int rc = check_cache(dtype, pages, 0, kv_heads, d, sequences, max_blocks);
    if (rc != VS_OK) return rc;
    if (heads < kv_heads || heads % kv_heads != 0 || count < 1 || count > blocks::kMaxCount || max_blocks > blocks::kMaxBlocks) return VS_ERR_SHAPE;
    if (sequences == 0) return VS_OK;
    if (!q || !q_strides || !lengths || !lists || (max_blocks > 0 && !table) || (pages > 0 && (!k_scales || !k_sums))) return VS_ERR_NULL;
    if (!aligned16(q) || !aligned16(k_sums)) return VS_ERR_ALIGN;
    for (const void *p : {(const void *)table, (const void *)lengths, (const void *)lists, (const void *)k_scales})
        if (!aligned4(p)) return VS_ERR_ALIGN;
    for (int i = 0; i < 2; ++i) {
        if (q_strides[i] < 0) return VS_ERR_SHAPE;
        if (q_strides[i] % 8 != 0) return VS_ERR_ALIGN;
    }
    cache::SelectArgs a = {};
    a.c.pages = pages; a.c.kv_heads = kv_heads; a.c.d = d; a.c.scales[0] = const_cast<float *>(k_scales); a.c.sums = const_cast<int16_t *>(k_sums);
    a.s = {sequences, table, max_blocks, nullptr, lengths};
    a.q = q; a.batch = q_strides[0]; a.head = q_strides[1];
    a.group = heads / kv_heads; a.wanted = count; a.lists = lists;
    const int smem = (int)((int64_t)max_blocks * 8 + (max_blocks + 31) / 32 * 4), threads = max_blocks > 256 ? cache::kSelectThreads : 256;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == VS_F16) {
        if ((rc = allow_smem<cache::select_kernel<__half>>(smem)) != VS_OK) return rc;
        cache::select_kernel<__half><<<(unsigned)(sequences * kv_heads), threads, smem, st>>>(a);
    } else {
        if ((rc = allow_smem<cache::select_kernel<__nv_bfloat16>>(smem)) != VS_OK) return rc;
        cache::select_kernel<__nv_bfloat16><<<(unsigned)(sequences * kv_heads), threads, smem, st>>>(a);
    }
    return (int)cudaGetLastError();
}

VS_EXPORT int64_t vs_cache_attention_workspace_bytes(int sequences, int heads, int kv_heads, int d, int units) {
    if (sequences < 1 || kv_heads < 1 || heads < kv_heads || d < 1 || units < 0) return 0;
    const int64_t items = (int64_t)sequences * kv_heads * ((heads / kv_heads + 15) / 16);
    const int pieces = decode_pieces(items, units);
    return pieces > 1 ? up256(items * pieces * 16 * (d + 2) * 4) : 0;
}

VS_EXPORT int vs_cache_attention(int dtype, int pages, int tails, int heads, int kv_heads, int d, const int8_t *k_codes, const int8_t *v_codes,
                                 const float *k_scales, const float *v_scales, const void *k_ring, const void *v_ring, int sequences, const void *q,
                                 const int64_t *q_strides, const int32_t *table, int max_blocks, const int32_t *tail_indices, const int32_t *lengths,
                                 const int32_t *lists, int count, void *out, float scale, void *workspace, int64_t workspace_bytes, void *stream) {
    int rc = check_cache(dtype, pages, tails, kv_heads, d, sequences, max_blocks);
    if (rc != VS_OK) return rc;
    if (heads < kv_heads || heads % kv_heads != 0 || (lists && (count < 1 || count > blocks::kMaxCount))) return VS_ERR_SHAPE;
    if (!scale_ok(scale)) return VS_ERR_ARG;
    if (sequences == 0) return VS_OK;
    if (!q || !q_strides || !lengths || !out || !tail_indices || (max_blocks > 0 && !table) || (pages > 0 && (!k_codes || !v_codes || !k_scales || !v_scales)) ||
        (tails > 0 && (!k_ring || !v_ring)))
        return VS_ERR_NULL;
    for (const void *p : {q, (const void *)k_codes, (const void *)v_codes, k_ring, v_ring, (const void *)out, (const void *)workspace})
        if (!aligned16(p)) return VS_ERR_ALIGN;
    for (const void *p : {(const void *)table, (const void *)tail_indices, (const void *)lengths, (const void *)lists, (const void *)k_scales, (const void *)v_scales})
        if (!aligned4(p)) return VS_ERR_ALIGN;
    for (int i = 0; i < 2; ++i) {
        if (q_strides[i] < 0) return VS_ERR_SHAPE;
        if (q_strides[i] % 8 != 0) return VS_ERR_ALIGN;
    }
    const int units = lists ? count : max_blocks;
    cache::AttentionArgs a = {};
    a.parts = (heads / kv_heads + 15) / 16;
    const int64_t items = (int64_t)sequences * kv_heads * a.parts;
    a.pieces = decode_pieces(items, units);
    if (items * a.pieces > kMaxGrid) return VS_ERR_SHAPE;
    if (workspace_bytes < vs_cache_attention_workspace_bytes(sequences, heads, kv_heads, d, units)) return VS_ERR_SHAPE;
    if (a.pieces > 1 && !workspace) return VS_ERR_NULL;
    a.c = {pages, tails, kv_heads, d, {const_cast<int8_t *>(k_codes), const_cast<int8_t *>(v_codes)}, {const_cast<float *>(k_scales), const_cast<float *>(v_scales)},
           nullptr, {const_cast<void *>(k_ring), const_cast<void *>(v_ring)}};
    a.s = {sequences, table, max_blocks, tail_indices, lengths};
    a.q = q; a.batch = q_strides[0]; a.head = q_strides[1];
    a.group = heads / kv_heads; a.lists = lists; a.wanted = count; a.scale = scale; a.out = out;
    a.partial = static_cast<float *>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == VS_F16 ? decode<__half>(a, (int)items, st) : decode<__nv_bfloat16>(a, (int)items, st);
}
