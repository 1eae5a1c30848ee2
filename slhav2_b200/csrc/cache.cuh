// Exact attention over a cache of key and value rows: what its kernels share (cache_attend.cu, cache_observe.cu, cache_evict.cu) and the
// launchers that the C ABI calls (capi_cache.cuh).
#pragma once

#include <atomic>
#include <vector>

#include "runtime.cuh"

namespace slha {

constexpr uint32_t CACHE_TABLE = 64;         // segments whose table travels in a kernel's parameters
constexpr uint32_t TREE_MOST = 256;          // drafted tokens of a segment
constexpr uint32_t CACHE_DIM_MOST = 256;
// Bytes of the parts of split segments that a launch may leave to be joined (the sums of a block of query rows of all KV heads may be more): a segment that can be left whole is, beyond
// it, and one that cannot is worked off in several launches.
constexpr uint64_t CACHE_PARTS_MOST = 512ull << 20;

// A segment and its share of a launch's work.
struct CacheSeg {
    uint64_t row_begin;
    uint32_t n_rows, query_begin, n_queries, base;
    uint32_t item_begin;   // first work item
    uint32_t block_begin;  // first block of query rows, of the segments whose rows are split
    uint32_t chunk_tiles;  // key tiles of an item
    uint32_t n_chunks;     // items of a block of query rows
    uint32_t seg;          // its number in the caller's table
    uint32_t pad;
    union {
        uint64_t to_begin;  // removal: its first row's place where rows go to
        struct {
            uint32_t block_first, n_blocks;  // attention: the first of the segment's blocks of query rows that a launch takes, and how many it does
        };
    };
};
struct CacheTable {
    CacheSeg s[CACHE_TABLE];
};
struct CacheArgs {
    const void *keys, *values, *q;
    void* out;
    float* lse;
    uint64_t krs, khs, vrs, vhs, qts, qhs, ots, ohs;  // strides in elements
    const uint32_t *row_pos, *row_doc;
    uint64_t entry_hs;
    const uint32_t *rows, *q_pos, *q_doc, *prefix, *parents;
    const float* slopes;
    const CacheSeg* table;  // null: in the parameters
    float *part_o, *part_ml;
    const float *lse_in, *w_in;  // observe
    float* w_out;
    uint64_t w_hs;
    float decay;
    uint32_t n_segs, n_kv, group, d, n_heads, n_tokens;
    float scale, cap;
    uint32_t window_last;  // the largest distance that is seen
    int32_t causal;
    int32_t tree;
    uint32_t cluster;  // CTAs that share a block of query rows and join their sums themselves (every segment has so many runs), or 0
};
struct EvictArgs {
    const void *keys, *values;
    void *to_keys, *to_values;
    uint64_t krs, khs, vrs, vhs, tkrs, tkhs, tvrs, tvhs;  // strides in bytes
    const uint32_t *pos, *doc;
    uint32_t *to_pos, *to_doc;
    uint64_t entry_hs, to_entry_hs;
    const float* w;
    float* to_w;
    uint64_t w_hs, to_w_hs;
    const unsigned char* tiles;
    unsigned char* to_tiles;
    uint64_t tile_hs, to_tile_hs;
    const uint32_t* rows;
    uint32_t *rows_out, *source, *places, *holes, *stay;
    const CacheSeg* table;
    uint32_t n_segs, n_kv, row_bytes, budget, room, sink, recent, in_place;
};

#ifdef __CUDACC__
// the segment that work item `item` belongs to: the last one that begins at or before it
template <typename F>
__device__ __forceinline__ uint32_t cache_find(uint32_t n, uint32_t item, F begin) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (begin(mid) <= item) lo = mid;
        else hi = mid;
    }
    return lo;
}
// tanh.  Up to 1 a polynomial in x^2, the minimax one of tanh(x) / x (found by exchange of extrema in 40 digits): 5e-8 relative in exact arithmetic, 1.2e-7 of 1 in
// float32; beyond, CUDA's.
constexpr float TANH_0 = 9.999999502407769e-1f, TANH_1 = -3.3332839153106564e-1f, TANH_2 = 1.3325204076281205e-1f, TANH_3 = -5.345702958893045e-2f,
                TANH_4 = 2.028998046010164e-2f, TANH_5 = -6.203379131937655e-3f, TANH_6 = 1.041022640341338e-3f;
__device__ __forceinline__ float tanh_small(float x) {
    const float u = x * x;
    float p = fmaf(u, TANH_6, TANH_5);
    p = fmaf(u, p, TANH_4);
    p = fmaf(u, p, TANH_3);
    p = fmaf(u, p, TANH_2);
    p = fmaf(u, p, TANH_1);
    return x * fmaf(u, p, TANH_0);
}
__device__ __forceinline__ float cache_tanh(float x) { return fabsf(x) <= 1.0f ? tanh_small(x) : tanhf(x); }
// Whether a token sees a row.
struct CacheSight {
    uint32_t window_last, prefix;
    int causal;
    __device__ __forceinline__ bool sees(uint32_t qp, uint32_t kp) const {
        const bool past = kp <= qp;
        const uint32_t away = past ? qp - kp : kp - qp;
        return ((past || !causal) && away <= window_last) || kp < prefix;
    }
};
// The distance of two positions.  Where many are taken from one token, as the difference of two float32, either position counted from one nearby: that costs no conversion. With the
// token within 2^23 of where it is counted from, its own is exact, and the row's rounding is at most twice that of the distance; tokens further away take their distances in integers.
constexpr uint32_t DISTANCE_NEAR = 1u << 23;
__device__ __forceinline__ float cache_distance(uint32_t a, uint32_t b) { return (float)(a <= b ? b - a : a - b); }
// Positions and documents of a tile's rows, or of a block's query rows.
struct CacheRanges {
    uint32_t pmin, pmax, dmin, dmax;
};
// 0: none of a tile's rows is seen by any of a block's query rows, 2: all are by all, 1: otherwise.  drafts: the tile holds drafted rows; inside: it ends before the last row does.
__device__ __forceinline__ int cache_tile_class(const CacheRanges& k, const CacheRanges& q, const CacheSight& sight, bool drafts, bool inside) {
    if (k.dmin > q.dmax || k.dmax < q.dmin) return 0;
    const uint32_t near_ = k.pmax < q.pmin ? q.pmin - k.pmax : k.pmin > q.pmax ? k.pmin - q.pmax : 0u;
    const uint32_t far_ = max(q.pmax > k.pmin ? q.pmax - k.pmin : 0u, k.pmax > q.pmin ? k.pmax - q.pmin : 0u);
    if (!drafts && k.pmin >= sight.prefix && ((sight.causal && k.pmin > q.pmax) || near_ > sight.window_last)) return 0;
    const bool all = k.pmax < sight.prefix || ((!sight.causal || k.pmax <= q.pmin) && far_ <= sight.window_last);
    return all && !drafts && inside && k.dmin == k.dmax && q.dmin == q.dmax && k.dmin == q.dmin ? 2 : 1;
}
#endif

// Work items: every segment's tiles in runs of at most `most`.
struct CacheWork {
    std::vector<CacheSeg> segs;
    uint64_t items = 0, blocks = 0;  // blocks: of query rows whose segments are split
    uint32_t chunks = 1;             // the most runs of one segment
};

// Working memory of one call: the thread's, or under capture memory that the graph allocates and frees with every run, so that graphs share none.
struct CacheMemory {
    Ctx* c;
    void* graph = nullptr;
    Status get(size_t bytes, void** out) {
        if (!ctx_capturing(c)) return ctx_device_scratch(c, bytes, out);
        SLHA_CUDA(cudaMallocAsync(&graph, bytes, c->stream));
        *out = graph;
        return Status();
    }
    Status done() {
        if (graph) SLHA_CUDA(cudaFreeAsync(graph, c->stream));
        return Status();
    }
};
// launch_behind with clusters of `size` CTAs
template <typename... P, typename... A>
inline cudaError_t launch_cluster(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, uint32_t size, A&&... args) {
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {size, 1, 1};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = size > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}
// Which kernels the calling thread's latest call on a cache of rows launched (SLHA_B200_CACHE_*).
extern thread_local uint32_t g_cache_kernels;
// The table of a launch: in the kernel's parameters, or uploaded where it is longer.
Status cache_table(Ctx* c, const std::vector<CacheSeg>& segs, CacheTable* inl, const CacheSeg** dev);
// Raises a kernel's limit of dynamic shared memory, once per kernel and device.
template <auto KERNEL>
Status cache_smem(Ctx* c, size_t bytes) {
    static std::atomic<uint32_t> raised{0};
    const uint32_t bit = 1u << c->device;
    if (raised.load(std::memory_order_relaxed) & bit) return Status();
    SLHA_CUDA(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    raised.fetch_or(bit, std::memory_order_relaxed);
    return Status();
}

inline uint64_t cache_part_bytes(uint64_t items, uint32_t n_kv, uint32_t mb, uint32_t d) { return items * n_kv * mb * (d * 4ull + 8); }
Status cache_part_memory(CacheArgs* a, uint64_t items, uint32_t mb, CacheMemory* mem);  // where the parts of split segments go
Status launch_cache_join(Ctx* c, CacheArgs a, int dtype, const CacheWork& w, uint32_t mb);
Status launch_attend_wide(Ctx* c, CacheArgs a, CacheWork w, bool* taken);
Status launch_attend_cache(Ctx* c, CacheArgs a, int dtype, const std::vector<SlhaB200Segment>& segs);
Status launch_observe_wide(Ctx* c, CacheArgs a, std::vector<CacheSeg> segs, uint64_t most_rows, bool* taken);
Status launch_observe_cache(Ctx* c, CacheArgs a, int dtype, const std::vector<SlhaB200Segment>& segs);
Status launch_evict_cache(Ctx* c, EvictArgs a, const std::vector<SlhaB200Segment>& segs, const std::vector<SlhaB200Segment>& to_segs);

}  // namespace slha
