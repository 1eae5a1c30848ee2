// Exact attention of many query rows over a cache of bfloat16 rows: prompts, chunks of prompts, trees of drafted tokens (the arithmetic is that of cache_attend.cu).
//
// A CTA takes 256 query rows of one KV head, as two tiles of 128, and a run of the segment's rows in tiles of 128 keys.  Both products run on tcgen05:
// S = Q K^T (128 x 128, both operands in shared memory) into TMEM, O += P V with P in TMEM, where it takes the place of the S it was made from, and V as it lies
// (its rows along the contraction).  Four warps a tile of query rows turn S into P, a row a thread; while one tile's scores are turned the other tile's products run.  One
// thread issues the products, three warps fetch (cp.async, so that rows may lie at any stride of 16 bytes), two key and two value tiles ahead.
//
// O is not scaled with every growth of a row's maximum: weights are taken against the maximum of an earlier tile until a score exceeds it by 2^8 (P then holds up to 256, as
// exact as below 1), which hardly ever happens after the first tiles.
#include <cuda_bf16.h>

#include <algorithm>

#include "cache.cuh"
#include "cache_mma.cuh"

namespace slha {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int THREADS = 384, WARPS = THREADS / 32, KT = 128, MB = 256, FETCHERS = 96, MMA_WARP = 8;
constexpr uint32_t RUN_MOST = 1024;           // key tiles of an item
constexpr uint32_t HALF = 128 * 128;          // bytes of 128 rows x 64 elements
constexpr uint32_t SPINS = 1u << 22;          // polls of a wait before it gives up (a fraction of a second)
constexpr float LAZY = 8.0f;

template <int D>
struct Wide {
    static constexpr int HALVES = D / 64;
    static constexpr uint32_t TILE = HALVES * HALF;
    static constexpr uint32_t K_AT = 2 * TILE, V_AT = 4 * TILE, META_AT = 6 * TILE;   // META: 4 x (positions, documents) of a key tile
    static constexpr uint32_t LIST_AT = META_AT + 4 * 2 * KT * 4, CLS_AT = LIST_AT + RUN_MOST * 2, ROWS_AT = CLS_AT + RUN_MOST;  // ROWS: position, document, slope, token
    static constexpr uint32_t RANGE_AT = ROWS_AT + 4 * MB * 4, BAR_AT = RANGE_AT + 64, TREE_AT = BAR_AT + 256;
    static constexpr uint32_t SMEM = TREE_AT + 1024, SMEM_TREE = SMEM + TREE_MOST * 8 + MB * (TREE_MOST / 8);
    static_assert(SMEM_TREE <= 227 * 1024, "shared memory of an SM");
};
// barriers, 8 bytes each
enum { K_FULL = 0, V_FULL = 2, K_FREE = 4, V_FREE = 6, S_FULL = 8, P_FULL = 10, O_FULL = 12, TMEM_WORD = 13, ODD_WORD = 14, META_FULL = 16 };

__device__ __forceinline__ void bar_init(uint32_t addr, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(addr), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t addr) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(addr) : "memory"); }
__device__ __forceinline__ bool bar_wait(uint32_t addr, uint32_t parity) {
    for (uint32_t i = 0; i < SPINS; ++i) {
        uint32_t ok;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
        if (ok) return true;
        if (i > 64) __nanosleep(32);
    }
    return false;
}
__device__ __forceinline__ void tc_commit_to(uint32_t addr) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// Shared-memory operands, 128-byte swizzle.  Contraction along the 128-byte lines (Q, K): groups of eight lines 1024 bytes apart.  Contraction across the lines (V): eight lines
// 1024 bytes apart likewise, the next 64 elements of a line one HALF further.
__device__ __forceinline__ uint64_t desc_along(uint32_t s) {
    return (uint64_t)((s & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t desc_across(uint32_t s) {
    return (uint64_t)((s & 0x3FFFFu) >> 4) | (uint64_t)(HALF >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D float32, A and B bfloat16, M = 128, N columns; across: B's contraction runs across its lines
__host__ __device__ constexpr uint32_t wide_idesc(uint32_t n, bool across) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (across ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
#define R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define W8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])
// Columns of this thread's TMEM lane; to be waited for (tmem_wait) and held before they are used.
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t* x) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : R8(x, 0), R8(x, 8), R8(x, 16), R8(x, 24) : "r"(t) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t t, uint32_t* x) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\ntcgen05.wait::ld.sync.aligned;\n"
                 : "=&r"(x[0]), "=&r"(x[1]), "=&r"(x[2]), "=&r"(x[3]), "=&r"(x[4]), "=&r"(x[5]), "=&r"(x[6]), "=&r"(x[7]), "=&r"(x[8]), "=&r"(x[9]), "=&r"(x[10]), "=&r"(x[11]),
                   "=&r"(x[12]), "=&r"(x[13]), "=&r"(x[14]), "=&r"(x[15]) : "r"(t) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t* x) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(t), W8(x, 0), W8(x, 8) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ bool odd_pair(uint32_t w) { return (w & 0x7F800000u) == 0x7F800000u || (w & 0x00007F80u) == 0x00007F80u; }

// What a CTA works on.
struct Item {
    CacheSeg sg;
    uint32_t head, item, row0, q_rows, n, ctx, first_tile, end_tile;
    CacheSight sight;
    uint64_t entry;
};

// A query row's result: to the outputs, or as the part of a split segment.
struct RowOut {
    unsigned char* out;  // bfloat16 row of the output, or null
    float* part;
    __device__ __forceinline__ void statistics(const CacheArgs& a, const Item& w, uint32_t r, float m, float l) const {
        if (out) {
            const uint32_t row = w.row0 + r;
            if (a.lse) a.lse[(uint64_t)(w.sg.query_begin + row / a.group) * a.n_heads + w.head * a.group + row % a.group] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
        } else {
            const uint64_t at = ((uint64_t)w.item * a.n_kv + w.head) * MB + r;
            a.part_ml[at * 2] = l == 0.0f ? -INFINITY : m;
            a.part_ml[at * 2 + 1] = l;
        }
    }
};
__device__ __forceinline__ RowOut row_out(const CacheArgs& a, const Item& w, uint32_t r) {
    const uint32_t row = w.row0 + r;
    RowOut o{nullptr, nullptr};
    if (w.sg.n_chunks == 1) o.out = static_cast<unsigned char*>(a.out) + ((uint64_t)(w.sg.query_begin + row / a.group) * a.ots + (uint64_t)(w.head * a.group + row % a.group) * a.ohs) * 2;
    else o.part = a.part_o + (((uint64_t)w.item * a.n_kv + w.head) * MB + r) * a.d;
    return o;
}

// The item again on the CUDA cores, a warp a query row and a row of the cache at a time, where only what is seen is read: for values that are not finite in a tile that not all see
// (a weight of zero would not keep them out of the sums), and where a wait ran out.
__device__ __noinline__ void by_rows(const CacheArgs& a, const Item& w, const uint32_t* s_qp, const uint32_t* s_qd, const float* s_slope, const uint32_t* s_tok, const uint32_t* s_depth,
                                     const uint32_t* s_anc) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q);
    const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(a.keys) + w.sg.row_begin * a.krs + w.head * a.khs;
    const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.values) + w.sg.row_begin * a.vrs + w.head * a.vhs;
    const uint32_t c = lane * 4;
    const bool mine = c < a.d;
    for (uint32_t r = warp; r < min((uint32_t)MB, w.q_rows - w.row0); r += WARPS) {
        const uint32_t row = w.row0 + r;
        const __nv_bfloat16* qr = q + (uint64_t)(w.sg.query_begin + row / a.group) * a.qts + (uint64_t)(w.head * a.group + row % a.group) * a.qhs;
        float x[4] = {0, 0, 0, 0}, o[4] = {0, 0, 0, 0}, m = -INFINITY, l = 0.0f;
        if (mine)
            for (int e = 0; e < 4; ++e) x[e] = __bfloat162float(qr[c + e]);
        for (uint32_t i = w.first_tile * KT; i < min(w.end_tile * KT, w.n); ++i) {
            const bool drafted = a.tree && i >= w.ctx;
            const uint32_t kp = a.row_pos ? a.row_pos[w.entry + i] : drafted ? w.sg.base + w.ctx + s_depth[i - w.ctx] : w.sg.base + i;
            if (!w.sight.sees(s_qp[r], kp) || (a.row_doc && a.row_doc[w.entry + i] != s_qd[r])) continue;
            if (drafted && !(s_anc[s_tok[r] * (TREE_MOST / 32) + ((i - w.ctx) >> 5)] >> ((i - w.ctx) & 31) & 1u)) continue;
            float s = 0.0f;
            if (mine)
                for (int e = 0; e < 4; ++e) s = fmaf(x[e], __bfloat162float(k[(uint64_t)i * a.krs + c + e]), s);
            for (int b = 16; b; b >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, b);
            s = a.cap > 0.0f ? a.cap * LOG2E * cache_tanh(s * a.scale / a.cap) : s * a.scale * LOG2E;
            const uint32_t away = kp <= s_qp[r] ? s_qp[r] - kp : kp - s_qp[r];
            s = fmaf(-s_slope[r], (float)away, s);
            const float top = fmaxf(m, s), use = top == -INFINITY ? 0.0f : top, f = exp2_fast(m - use), p = exp2_fast(s - use);
            m = top;
            l = fmaf(l, f, p);
            for (int e = 0; e < 4; ++e) {
                o[e] *= f;
                if (mine && p != 0.0f) o[e] = fmaf(p, __bfloat162float(v[(uint64_t)i * a.vrs + c + e]), o[e]);
            }
        }
        const RowOut to = row_out(a, w, r);
        if (mine) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            if (to.out) *reinterpret_cast<uint2*>(to.out + c * 2) = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
            else *reinterpret_cast<float4*>(to.part + c) = make_float4(o[0], o[1], o[2], o[3]);
        }
        if (lane == 0) to.statistics(a, w, r, m, l);
    }
}

template <int D>
__global__ void __launch_bounds__(THREADS, 1) cache_attend_wide_kernel(const __grid_constant__ CacheArgs a, const __grid_constant__ CacheTable tab) {
    using S = Wide<D>;
    dep_wait();
    extern __shared__ unsigned char raw[];
    const uint32_t sb = (smem_addr(raw) + 1023u) & ~1023u;
    unsigned char* sm = raw + (sb - smem_addr(raw));
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    Item w;
    w.head = blockIdx.x % a.n_kv;
    w.item = blockIdx.x / a.n_kv;
    {
        const CacheSeg* table = a.table ? a.table : tab.s;
        w.sg = table[cache_find(a.n_segs, w.item, [&](uint32_t i) { return table[i].item_begin; })];
    }
    w.n = a.rows ? min(a.rows[w.sg.seg], w.sg.n_rows) : w.sg.n_rows;
    w.ctx = w.n - min(w.n, w.sg.n_queries);
    w.q_rows = w.sg.n_queries * a.group;
    w.row0 = (w.item - w.sg.item_begin) / w.sg.n_chunks * MB;
    {
        const uint32_t chunk = (w.item - w.sg.item_begin) % w.sg.n_chunks, tiles = (w.n + KT - 1) / KT;
        w.first_tile = min(tiles, chunk * w.sg.chunk_tiles);
        w.end_tile = min(tiles, w.first_tile + w.sg.chunk_tiles);
    }
    w.sight = CacheSight{a.window_last, a.prefix ? a.prefix[w.sg.seg] : 0u, a.causal};
    w.entry = w.head * a.entry_hs + w.sg.row_begin;
    const bool has_pos = a.row_pos, has_doc = a.row_doc, has_slope = a.slopes, has_cap = a.cap > 0.0f;
    const uint32_t used = min((uint32_t)MB, w.q_rows - w.row0);
    const bool two = used > 128;

    uint32_t* s_meta = reinterpret_cast<uint32_t*>(sm + S::META_AT);
    uint16_t* s_list = reinterpret_cast<uint16_t*>(sm + S::LIST_AT);
    unsigned char* s_cls = sm + S::CLS_AT;
    uint32_t* s_qp = reinterpret_cast<uint32_t*>(sm + S::ROWS_AT);
    uint32_t* s_qd = s_qp + MB;
    float* s_slope = reinterpret_cast<float*>(s_qd + MB);
    uint32_t* s_tok = reinterpret_cast<uint32_t*>(s_slope + MB);
    uint32_t* s_range = reinterpret_cast<uint32_t*>(sm + S::RANGE_AT);
    uint32_t* s_par = reinterpret_cast<uint32_t*>(sm + S::TREE_AT);
    uint32_t* s_depth = s_par + TREE_MOST;
    uint32_t* s_anc = s_depth + TREE_MOST;
    const uint32_t bars = sb + S::BAR_AT;
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(sm + S::BAR_AT + TMEM_WORD * 8);
    volatile uint32_t* s_odd = reinterpret_cast<volatile uint32_t*>(sm + S::BAR_AT + ODD_WORD * 8);
    const auto bar = [&](int which) { return bars + which * 8; };
    const uint32_t tok0 = w.row0 / a.group;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(bar(K_FULL + i), FETCHERS);
            bar_init(bar(V_FULL + i), FETCHERS);
            bar_init(bar(K_FREE + i), 1);
            bar_init(bar(V_FREE + i), 1);
            bar_init(bar(S_FULL + i), 1);
            bar_init(bar(P_FULL + i), 128);
        }
        bar_init(bar(O_FULL), 1);
        for (int i = 0; i < 4; ++i) bar_init(bar(META_FULL + i), FETCHERS);
        *s_odd = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(bar(TMEM_WORD)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (a.tree) {
        for (uint32_t j = tid; j < w.sg.n_queries; j += THREADS) {
            const uint32_t p = a.parents[w.sg.query_begin + j];
            s_par[j] = p < j ? p : 0xFFFFFFFFu;
        }
        for (uint32_t i = tid; i < MB * (TREE_MOST / 32); i += THREADS) s_anc[i] = 0;
        __syncthreads();
        for (uint32_t j = tid; j < w.sg.n_queries; j += THREADS) {  // (parents are smaller than their children: every walk ends)
            const uint32_t mine = j - tok0;
            uint32_t depth = 0, at = j;
            while (true) {
                if (mine < MB) s_anc[mine * (TREE_MOST / 32) + (at >> 5)] |= 1u << (at & 31);
                if (s_par[at] == 0xFFFFFFFFu) break;
                at = s_par[at];
                ++depth;
            }
            s_depth[j] = depth;
        }
        __syncthreads();
    }
    {
        const unsigned char* q = static_cast<const unsigned char*>(a.q);
        for (int i = tid; i < (two ? MB : 128) * S::HALVES * 8; i += THREADS) {
            const uint32_t r = i / (S::HALVES * 8), c = i % (S::HALVES * 8), row = w.row0 + r;
            const bool there = row < w.q_rows && c * 8 < a.d;
            const uint64_t at = there ? (uint64_t)(w.sg.query_begin + row / a.group) * a.qts + (uint64_t)(w.head * a.group + row % a.group) * a.qhs + c * 8 : 0;
            copy16(sb + (r >> 7) * S::TILE + (c >> 3) * HALF + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4), q + at * 2, there);
        }
        copy_commit();
    }
    for (uint32_t r = tid; r < MB; r += THREADS) {
        const uint32_t row = min(w.row0 + r, w.q_rows - 1), tok = row / a.group;
        s_qp[r] = a.q_pos ? a.q_pos[w.sg.query_begin + tok] : w.sg.base + w.ctx + (a.tree ? s_depth[tok] : tok);
        s_qd[r] = has_doc ? a.q_doc[w.sg.query_begin + tok] : 0u;
        s_slope[r] = has_slope ? a.slopes[w.head * a.group + row % a.group] * LOG2E : 0.0f;
        s_tok[r] = tok - tok0;
    }
    __syncthreads();
    if (warp < 2) {  // positions and documents of either tile of query rows
        CacheRanges q{0xFFFFFFFFu, 0u, 0xFFFFFFFFu, 0u};
        for (int r = warp * 128 + lane; r < warp * 128 + 128; r += 32) {
            q.pmin = min(q.pmin, s_qp[r]);
            q.pmax = max(q.pmax, s_qp[r]);
            q.dmin = min(q.dmin, s_qd[r]);
            q.dmax = max(q.dmax, s_qd[r]);
        }
        q.pmin = __reduce_min_sync(0xFFFFFFFFu, q.pmin);
        q.pmax = __reduce_max_sync(0xFFFFFFFFu, q.pmax);
        q.dmin = __reduce_min_sync(0xFFFFFFFFu, q.dmin);
        q.dmax = __reduce_max_sync(0xFFFFFFFFu, q.dmax);
        if (lane == 0) s_range[warp * 4] = q.pmin, s_range[warp * 4 + 1] = q.pmax, s_range[warp * 4 + 2] = q.dmin, s_range[warp * 4 + 3] = q.dmax;
    }
    __syncthreads();
    const uint32_t in_run = w.end_tile - w.first_tile;
    {   // which tiles are visited, and which of them either tile of query rows sees as a whole
        const CacheRanges qa{s_range[0], s_range[1], s_range[2], s_range[3]}, qb{s_range[4], s_range[5], s_range[6], s_range[7]};
        const auto classes = [&](const CacheRanges& k, uint32_t last) {
            const bool drafts = a.tree && last >= w.ctx, inside = last < w.n;
            const int x = cache_tile_class(k, qa, w.sight, drafts, inside), y = cache_tile_class(k, qb, w.sight, drafts, inside);
            return (x || y ? 1 : 0) | (x == 2 ? 2 : 0) | (y == 2 ? 4 : 0);
        };
        if (has_pos || has_doc) {
            for (uint32_t j = warp; j < in_run; j += WARPS) {
                const uint32_t first = (w.first_tile + j) * KT;
                CacheRanges k{0xFFFFFFFFu, 0u, has_doc ? 0xFFFFFFFFu : 0u, 0u};
#pragma unroll
                for (int e = 0; e < KT / 32; ++e) {
                    const uint32_t i = min(first + lane + e * 32, w.n - 1);
                    const uint32_t p = has_pos ? a.row_pos[w.entry + i] : w.sg.base + i;
                    k.pmin = min(k.pmin, p);
                    k.pmax = max(k.pmax, p);
                    if (has_doc) {
                        const uint32_t d = a.row_doc[w.entry + i];
                        k.dmin = min(k.dmin, d);
                        k.dmax = max(k.dmax, d);
                    }
                }
                k.pmin = __reduce_min_sync(0xFFFFFFFFu, k.pmin);
                k.pmax = __reduce_max_sync(0xFFFFFFFFu, k.pmax);
                k.dmin = __reduce_min_sync(0xFFFFFFFFu, k.dmin);
                k.dmax = __reduce_max_sync(0xFFFFFFFFu, k.dmax);
                if (lane == 0) s_cls[j] = (unsigned char)classes(k, first + KT - 1);
            }
        } else {
            for (uint32_t j = tid; j < in_run; j += THREADS) {
                const uint32_t first = (w.first_tile + j) * KT, last = first + KT - 1;
                s_cls[j] = (unsigned char)classes(CacheRanges{w.sg.base + first, w.sg.base + min(last, w.n - 1), 0u, 0u}, last);
            }
        }
    }
    copy_wait<0>();
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // (the queries, read by the products)
    __syncthreads();
    uint32_t cnt = 0;
    for (uint32_t j0 = 0; j0 < in_run; j0 += 32) {  // (every warp counts, the first one writes)
        const int cls = j0 + lane < in_run ? s_cls[j0 + lane] : 0;
        const uint32_t mask = __ballot_sync(0xFFFFFFFFu, cls != 0);
        if (warp == 0 && cls) s_list[cnt + __popc(mask & ((1u << lane) - 1u))] = (uint16_t)((j0 + lane) << 2 | cls >> 1);
        cnt += __popc(mask);
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *s_tmem;
    bool fail = false;

    if (warp < 8) {
        // ---- scores to weights: a query row a thread
        const uint32_t t = warp >> 2, r = tid;
        if (t == 0 || two) {
            const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21), ts = lanes + t * 128, to = lanes + 256 + t * 128;
            const float to_log2 = has_cap ? a.scale / a.cap : a.scale * LOG2E, cap2 = a.cap * LOG2E;
            const uint32_t qp = s_qp[r], qd = s_qd[r];
            const float slope = s_slope[r];
            float m = -INFINITY, l = 0.0f;
            for (uint32_t li = 0; li < cnt; ++li) {
                if (!__all_sync(0xFFFFFFFFu, bar_wait(bar(S_FULL + t), li & 1))) {
                    fail = true;
                    break;
                }
                tc_after();
                const uint32_t what = s_list[li];
                const bool all = what >> t & 1;
                uint32_t u[128];
                float* s = reinterpret_cast<float*>(u);
#pragma unroll
                for (int c = 0; c < 128; c += 32) tmem_ld32(ts + c, u + c);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 128; ++c) asm volatile("" : "+r"(u[c]));
                float mul = to_log2, top = -INFINITY;
                if (!all || has_slope || has_cap) {
                    mul = 1.0f;
                    if (has_cap) {
                        float big = 0.0f;
#pragma unroll
                        for (int c = 0; c < 128; ++c) big = fmaxf(big, fabsf(s[c]));
                        if (__any_sync(0xFFFFFFFFu, !(big * to_log2 <= 1.0f))) {
#pragma unroll
                            for (int c = 0; c < 128; ++c) {  // tanh x = 1 - 2 / (exp(2 x) + 1)
                                const float e = exp2_fast(s[c] * to_log2 * (2.0f * LOG2E));
                                s[c] = fmaf(-2.0f * cap2, __frcp_rn(e + 1.0f), cap2);
                            }
                        } else {
#pragma unroll
                            for (int c = 0; c < 128; ++c) s[c] = cap2 * tanh_small(s[c] * to_log2);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 128; ++c) s[c] *= to_log2;
                    }
                    if (!all || has_slope) {
                        if (!__all_sync(0xFFFFFFFFu, bar_wait(bar(META_FULL + (li & 3)), li >> 2 & 1))) {
                            fail = true;
                            break;
                        }
                        const uint4* kp4 = reinterpret_cast<const uint4*>(s_meta + (li & 3) * 2 * KT);
                        const uint32_t first = (w.first_tile + (what >> 2)) * KT;
#pragma unroll
                        for (int c = 0; c < 128; c += 4) {
                            const uint4 p4 = kp4[c / 4], d4 = has_doc ? kp4[KT / 4 + c / 4] : make_uint4(0u, 0u, 0u, 0u);
                            const uint32_t kp[4] = {p4.x, p4.y, p4.z, p4.w}, kd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t away = kp[e] <= qp ? qp - kp[e] : kp[e] - qp;
                                if (has_slope) s[c + e] = fmaf(-slope, (float)away, s[c + e]);
                                if (!all) {
                                    const uint32_t row = first + c + e;
                                    bool seen = row < w.n && w.sight.sees(qp, kp[e]) && kd[e] == qd;
                                    if (a.tree && row >= w.ctx && row < w.n) seen = seen && (s_anc[s_tok[r] * (TREE_MOST / 32) + ((row - w.ctx) >> 5)] >> ((row - w.ctx) & 31) & 1u);
                                    if (!seen) s[c + e] = -INFINITY;
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < 128; ++c) top = fmaxf(top, s[c]);
                top *= mul;
                if (__any_sync(0xFFFFFFFFu, top > m + LAZY)) {
                    const float now = fmaxf(m, top), f = m == -INFINITY ? 0.0f : exp2_fast(m - now);
                    m = now;
                    l *= f;
                    if (li > 0) {  // (the scores are there, so the products before them are done)
#pragma unroll
                        for (int c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(to + c, o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16(to + c, o);
                        }
                    }
                }
                const float use = m == -INFINITY ? 0.0f : m;
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float x = exp2_fast(fmaf(s[c + e], mul, -use)), y = exp2_fast(fmaf(s[c + e + 1], mul, -use));
                        sum[e & 2] += x;
                        sum[(e & 2) + 1] += y;
                        p[e / 2] = pack_bf16(x, y);
                    }
                    tmem_st16(ts + c / 2, p);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
                tc_before();
                bar_arrive(bar(P_FULL + t));
            }
            if (cnt && !fail) {
                fail = !__all_sync(0xFFFFFFFFu, bar_wait(bar(O_FULL), 0));
                tc_after();
            }
            // (TMEM is read by the whole warp, behind the rows' end too)
            const bool there = r < used;
            const RowOut out = row_out(a, w, there ? r : 0);
            const float inv = out.out ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
#pragma unroll
            for (int c = 0; c < D; c += 16) {
                __syncwarp();
                uint32_t o[16];
                tmem_ld16(to + c, o);
                float x[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = cnt && l != 0.0f ? __uint_as_float(o[e]) * inv : 0.0f;
#pragma unroll
                for (int h = 0; h < 16; h += 8) {
                    if (!there || c + h >= (int)a.d) continue;
                    if (out.out) {
                        *reinterpret_cast<uint4*>(out.out + (c + h) * 2) =
                            make_uint4(pack_bf16(x[h], x[h + 1]), pack_bf16(x[h + 2], x[h + 3]), pack_bf16(x[h + 4], x[h + 5]), pack_bf16(x[h + 6], x[h + 7]));
                    } else {
                        *reinterpret_cast<float4*>(out.part + c + h) = make_float4(x[h], x[h + 1], x[h + 2], x[h + 3]);
                        *reinterpret_cast<float4*>(out.part + c + h + 4) = make_float4(x[h + 4], x[h + 5], x[h + 6], x[h + 7]);
                    }
                }
            }
            if (there) out.statistics(a, w, r, m, l);
        }
    } else if (warp == MMA_WARP) {
        // ---- the products
        uint32_t lead;
        asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(lead));
        if (lead && cnt) {
            const auto scores = [&](uint32_t li, uint32_t t) {
                const uint32_t k = sb + S::K_AT + (li & 1) * S::TILE, q = sb + t * S::TILE;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t at = (kk >> 2) * HALF + (kk & 3) * 32;
                    mma_shared(tmem + t * 128, desc_along(q + at), desc_along(k + at), wide_idesc(KT, false), kk > 0);
                }
                tc_commit_to(bar(S_FULL + t));
            };
            const auto values = [&](uint32_t li, uint32_t t) {
                const uint32_t v = sb + S::V_AT + (li & 1) * S::TILE;
#pragma unroll
                for (int kk = 0; kk < KT / 16; ++kk) mma_tmem(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, desc_across(v + kk * 2048), wide_idesc(D, true), li > 0 || kk > 0);
            };
            fail = !bar_wait(bar(K_FULL), 0);
            if (!fail) {
                scores(0, 0);
                if (two) scores(0, 1);
                tc_commit_to(bar(K_FREE));
            }
            for (uint32_t li = 0; li < cnt && !fail; ++li) {
                const bool more = li + 1 < cnt;
                if (!bar_wait(bar(V_FULL + (li & 1)), li >> 1 & 1) || !bar_wait(bar(P_FULL), li & 1)) {
                    fail = true;
                    break;
                }
                tc_after();
                values(li, 0);
                if (more) {
                    if (!bar_wait(bar(K_FULL + (li + 1 & 1)), (li + 1) >> 1 & 1)) {
                        fail = true;
                        break;
                    }
                    scores(li + 1, 0);
                }
                if (two) {
                    if (!bar_wait(bar(P_FULL + 1), li & 1)) {
                        fail = true;
                        break;
                    }
                    tc_after();
                    values(li, 1);
                }
                tc_commit_to(bar(V_FREE + (li & 1)));
                if (more) {
                    if (two) scores(li + 1, 1);
                    tc_commit_to(bar(K_FREE + (li + 1 & 1)));
                }
            }
            tc_commit_to(bar(O_FULL));
        }
        __syncwarp();
    } else {
        // ---- rows into shared memory.  A tile's copies are announced when the next ones have been issued.
        const uint32_t x0 = tid - 288;
        const unsigned char* kb = static_cast<const unsigned char*>(a.keys) + (w.sg.row_begin * a.krs + w.head * a.khs) * 2;
        const unsigned char* vb = static_cast<const unsigned char*>(a.values) + (w.sg.row_begin * a.vrs + w.head * a.vhs) * 2;
        constexpr int PIECES = S::HALVES * 8;
        const auto fetch = [&](uint32_t dst, const unsigned char* from, uint64_t stride, uint32_t first) {
            for (uint32_t i = x0; i < KT * PIECES; i += FETCHERS) {
                const uint32_t r = i / PIECES, c = i % PIECES, row = first + r;
                const bool there = row < w.n && c * 8 < a.d;
                copy16(dst + (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4), there ? from + row * stride * 2 + c * 16 : from, there);
            }
            copy_commit();
        };
        const auto say = [&](int which) {
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            bar_arrive(bar(which));
        };
        // values of a tile that not all see: a thread looks at the pieces that it has fetched
        const auto look = [&](uint32_t li) {
            if ((s_list[li] & 3u) == (two ? 3u : 1u) || (!two && (s_list[li] & 1u))) return;
            bool odd = false;
            for (uint32_t i = x0; i < KT * PIECES; i += FETCHERS) {
                const uint32_t r = i / PIECES, c = i % PIECES;
                const uint4 v = *reinterpret_cast<const uint4*>(sm + S::V_AT + (li & 1) * S::TILE + (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                odd |= odd_pair(v.x) || odd_pair(v.y) || odd_pair(v.z) || odd_pair(v.w);
            }
            if (odd) *s_odd = 1u;
        };
        for (uint32_t li = 0; li < cnt; ++li) {
            const uint32_t slot = li & 1, first = (w.first_tile + (s_list[li] >> 2)) * KT;
            if (li >= 2 && !bar_wait(bar(K_FREE + slot), (li >> 1) - 1 & 1)) {
                fail = true;
                break;
            }
            // (the tile four before this one has been turned into weights: its positions are no longer read)
            for (uint32_t i = x0; i < KT; i += FETCHERS) {
                const uint32_t row = min(first + i, w.n - 1);
                uint32_t* at = s_meta + (li & 3) * 2 * KT + i;
                at[0] = has_pos ? a.row_pos[w.entry + row] : a.tree && row >= w.ctx ? w.sg.base + w.ctx + s_depth[row - w.ctx] : w.sg.base + row;
                if (has_doc) at[KT] = a.row_doc[w.entry + row];
            }
            bar_arrive(bar(META_FULL + (li & 3)));
            fetch(sb + S::K_AT + slot * S::TILE, kb, a.krs, first);
            if (li > 0) {
                copy_wait<1>();
                look(li - 1);
                say(V_FULL + (slot ^ 1));
            }
            if (li >= 2 && !bar_wait(bar(V_FREE + slot), (li >> 1) - 1 & 1)) {
                fail = true;
                break;
            }
            fetch(sb + S::V_AT + slot * S::TILE, vb, a.vrs, first);
            copy_wait<1>();
            say(K_FULL + slot);
        }
        copy_wait<0>();
        if (cnt && !fail) {
            look(cnt - 1);
            say(V_FULL + (cnt - 1 & 1));
        }
    }
    if (fail) *s_odd = 1u;
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
    if (*s_odd) by_rows(a, w, s_qp, s_qd, s_slope, s_tok, s_depth, s_anc);
}

template <int D>
Status launch_wide(Ctx* c, CacheArgs a, CacheWork w) {
    using S = Wide<D>;
    cache_cut(&w, a.group, MB, KT, std::min(RUN_MOST, cache_longest_run(w, a.group, MB, KT, a.n_kv, (uint32_t)sm_count(c->device))));
    if (w.items * a.n_kv > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "attention over a cache: too many blocks of query rows");
    CacheTable tab;
    SLHA_TRY(cache_table(c, w.segs, &tab, &a.table));
    a.n_segs = (uint32_t)w.segs.size();
    CacheMemory mem{c};
    SLHA_TRY(cache_part_memory(&a, w, MB, &mem));
    SLHA_TRY((cache_smem<cache_attend_wide_kernel<D>>(c, S::SMEM_TREE)));
    SLHA_CUDA(launch_behind(cache_attend_wide_kernel<D>, dim3((uint32_t)(w.items * a.n_kv)), dim3(THREADS), a.tree ? S::SMEM_TREE : S::SMEM, c->stream, a, tab));
    count_launch();
    if (w.blocks) SLHA_TRY(launch_cache_join(c, a, SLHA_B200_BF16, w, MB));
    return mem.done();
}

}  // namespace

Status launch_attend_wide(Ctx* c, CacheArgs a, CacheWork w) { return a.d <= 64 ? launch_wide<64>(c, a, std::move(w)) : launch_wide<128>(c, a, std::move(w)); }

}  // namespace slha
