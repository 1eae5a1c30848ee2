// Exact attention of many query rows over a cache of bfloat16 rows: prompts, chunks of prompts, trees of drafted tokens (the arithmetic is that of cache_attend.cu).
//
// A CTA takes 256 query rows of one KV head, as two tiles of 128, and a run of the segment's rows in tiles of 128 keys.  Both products run on tcgen05:
// S = Q K^T (128 x 128, both operands in shared memory) into TMEM, O += P V with P in TMEM, where it takes the place of the S it was made from, and V as it lies
// (its rows along the contraction).  Four warps a tile of query rows turn S into P, a row a thread; while one tile's scores are turned the other tile's products run.  One
// thread issues the products, one warp fetches, two key and two value tiles ahead: whole tiles by TMA (one map of all rows and KV heads), the tile behind which a segment
// ends by cp.async, which reads nothing beyond the end and leaves zeros there.
//
// Bound by the softmax beside the products (a row a thread, 128 columns: one exponential, two multiply-adds and half a conversion a score, TMEM loads and stores): 8192 tokens x 32
// heads x 8192 rows, nothing masked, 846 us = 1300 TFLOP/s, 79 % of what a library's matrix product reaches; causal 456 us (1206, of the half that is seen; up to 510 where the power limit lowers the clock; tiles on the diagonal are
// worked in full); 4096 x 4096 under a cap 370 us, where the hyperbolic tangent's polynomial is eight more multiply-adds a score; with the rows' own kernel of 64 (cache_attend.cu) the
// prompts below took 3.6 to 3.9 times as long.  Two tiles of query rows a CTA, because one tile's softmax then hides behind the other's products, and because 256 rows of sums
// fill half of TMEM and the two tiles' scores the other.
//
// O is not scaled with every growth of a row's maximum: weights are taken against the maximum of an earlier tile until a score exceeds it by 2^8 (P then holds up to 256, as
// exact as below 1), which hardly ever happens after the first tiles.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "cache.cuh"
#include "cache_tc.cuh"

namespace slha {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int THREADS = 384, WARPS = THREADS / 32, KT = 128, MB = 256, MMA_WARP = 8, FETCH_WARP = 9;  // (the last two look over values)
// Registers a thread: 168 for all at the launch; the two warpgroups that hold a row of scores take 200, the third gives them up: 2 x 200 + 104 = 3 x 168.
constexpr int REGS_ALL = 168, REGS_ROWS = 200, REGS_REST = 104;
constexpr uint32_t RUN_MOST = 1024;           // key tiles of an item
constexpr float LAZY = 8.0f;

template <int D>
struct Wide {
    static constexpr int HALVES = D / 64;
    static constexpr uint32_t TILE = HALVES * HALF;
    static constexpr uint32_t K_AT = 2 * TILE, V_AT = 4 * TILE, META_AT = 6 * TILE;   // META: 4 x (positions, documents, distances) of a key tile
    static constexpr uint32_t LIST_AT = META_AT + 4 * 3 * KT * 4, CLS_AT = LIST_AT + RUN_MOST * 4, ROWS_AT = CLS_AT + RUN_MOST;  // ROWS: offset in q (64 bits), position, document, slope, token
    static constexpr uint32_t RANGE_AT = ROWS_AT + 6 * MB * 4, ODD_AT = RANGE_AT + 64, ITEM_AT = ODD_AT + RUN_MOST * 2, BAR_AT = ITEM_AT + 256, TREE_AT = BAR_AT + 256;
    static constexpr uint32_t SMEM = TREE_AT + 1024, SMEM_TREE = SMEM + TREE_MOST * 8 + MB * (TREE_MOST / 8);
    static_assert(SMEM_TREE <= 227 * 1024, "shared memory of an SM");
};
// barriers, 8 bytes each
enum { K_FULL = 0, V_FULL = 2, K_FREE = 4, V_FREE = 6, S_FULL = 8, P_FULL = 10, O_FULL = 12, TMEM_WORD = 13, FAIL_WORD = 14, META_FULL = 16, P_HALF = 20, Q_FULL = 22, V_CLEAN = 23 };

template <int N>
__device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }
// bits 31 and 15: whether the two bfloat16 are not finite (their exponents' bits are all set)
__device__ __forceinline__ uint32_t odd_pair(uint32_t w) { return (w & 0x7F807F80u) + 0x00800080u; }

// The rows as tensors of three dimensions: an element of a row, then row and KV head, the one of the smaller stride first.  Queries and outputs: element, head, token.
struct WideMaps {
    CUtensorMap k, v;
    CUtensorMap q, out;  // boxes of 32 query rows, where the head's group divides 32
    uint32_t k_head_first, v_head_first, q_boxes, out_boxes;
};
// What a CTA works on.
struct Item {
    CacheSeg sg;
    uint32_t head, item, row0, q_rows, n, ctx;
    CacheSight sight;
    uint64_t entry;
    uint32_t near_pos;                // where distances are taken from (see cache_distance)
    bool arrays, drafts_listed;  // positions or documents of the rows' own; drafted rows whose positions count
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

// Whether query row r sees row i of the segment, whose position is kp and whose document is kd.
__device__ __forceinline__ bool row_sees(const CacheArgs& a, const Item& w, const uint32_t* s_qp, const uint32_t* s_qd, const uint32_t* s_tok, const uint32_t* s_anc, uint32_t r, uint32_t i,
                                         uint32_t kp, uint32_t kd) {
    if (!w.sight.sees(s_qp[r], kp) || kd != s_qd[r]) return false;
    return !a.tree || i < w.ctx || (s_anc[s_tok[r] * (TREE_MOST / 32) + ((i - w.ctx) >> 5)] >> ((i - w.ctx) & 31) & 1u);
}
__device__ __forceinline__ uint32_t row_position(const CacheArgs& a, const Item& w, const uint32_t* s_depth, uint32_t i) {
    return a.row_pos ? a.row_pos[w.entry + i] : a.tree && i >= w.ctx ? w.sg.base + w.ctx + s_depth[i - w.ctx] : w.sg.base + i;
}

// Values that are not finite in tiles that not all see: the products took zeros in their place (a weight of zero would not keep them out of the sums).  Here they reach the sums of the
// query rows that see them: a bit for each query row, element and sign, then the results.  Only the rows that hold such values, and the seven beside each, are read again (256 query rows of 2 KV heads on
// 32768 rows with a row that nobody sees every 64: 44 us, 50 where those rows are NaN; 131072 rows 102 and 128, every other row 102 and 361).
template <int D>
__device__ __noinline__ void odd_values(const CacheArgs& a, unsigned char* sm, uint32_t cnt) {
    using S = Wide<D>;
    const Item& w = *reinterpret_cast<const Item*>(sm + S::ITEM_AT);
    const uint32_t* const s_qp = reinterpret_cast<const uint32_t*>(sm + S::ROWS_AT) + 2 * MB;
    const uint32_t *const s_qd = s_qp + MB, *const s_tok = s_qp + 3 * MB, *const s_depth = reinterpret_cast<const uint32_t*>(sm + S::TREE_AT) + TREE_MOST, *const s_anc = s_depth + TREE_MOST;
    const uint32_t *const s_list = reinterpret_cast<const uint32_t*>(sm + S::LIST_AT), *const s_odd = reinterpret_cast<const uint32_t*>(sm + S::ODD_AT);
    uint32_t* const s_sign = reinterpret_cast<uint32_t*>(sm + S::K_AT);  // [query row][+, -][128 elements]; the tiles are no longer needed
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, used = min((uint32_t)MB, w.q_rows - w.row0), c = lane * 4;
    for (uint32_t i = threadIdx.x; i < MB * 8; i += THREADS) s_sign[i] = 0;
    __syncthreads();
    const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.values) + w.sg.row_begin * a.vrs + w.head * a.vhs;
    uint32_t turn = 0;
    for (uint32_t l0 = 0; l0 < cnt; l0 += 32) {
        const uint32_t mine = l0 + lane < cnt ? s_odd[(l0 + lane) >> 1] >> (lane & 1) * 16 & 0xFFFFu : 0u;
        for (uint32_t tiles = __ballot_sync(0xFFFFFFFFu, mine != 0); tiles; tiles &= tiles - 1) {
            const uint32_t at = __ffs(tiles) - 1, first = (s_list[l0 + at] >> 2) * KT, rows = min((uint32_t)KT, w.n - first);
            for (uint32_t parts = __shfl_sync(0xFFFFFFFFu, mine, at); parts; parts &= parts - 1) {
                if (turn++ % WARPS != warp) continue;
                const uint32_t j0 = (__ffs(parts) - 1) * 8;
                uint2 x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = j0 + e < rows && c < a.d ? *reinterpret_cast<const uint2*>(v + (uint64_t)(first + j0 + e) * a.vrs + c) : make_uint2(0u, 0u);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t odd = odd_pair(x[e].x) | odd_pair(x[e].y);
                    if (!__any_sync(0xFFFFFFFFu, odd & 0x80008000u)) continue;
                    uint32_t plus = 0, minus = 0;  // of the lane's four elements; NaN: both
                    const uint32_t bits[4] = {x[e].x & 0xFFFFu, x[e].x >> 16, x[e].y & 0xFFFFu, x[e].y >> 16};
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const uint32_t size = bits[y] & 0x7FFFu;
                        if (size < 0x7F80u) continue;
                        if (size > 0x7F80u || !(bits[y] & 0x8000u)) plus |= 1u << y;
                        if (size > 0x7F80u || (bits[y] & 0x8000u)) minus |= 1u << y;
                    }
                    const uint32_t eight = 0xFFu << (lane & 24);
                    plus = __reduce_or_sync(eight, plus << (lane & 7) * 4);
                    minus = __reduce_or_sync(eight, minus << (lane & 7) * 4);
                    uint32_t word[8];
#pragma unroll
                    for (int y = 0; y < 4; ++y) word[y] = __shfl_sync(0xFFFFFFFFu, plus, y * 8), word[4 + y] = __shfl_sync(0xFFFFFFFFu, minus, y * 8);
                    const uint32_t i = first + j0 + e, kp = row_position(a, w, s_depth, i), kd = a.row_doc ? a.row_doc[w.entry + i] : 0u;
                    for (uint32_t r = lane; r < used; r += 32)
                        if (row_sees(a, w, s_qp, s_qd, s_tok, s_anc, r, i, kp, kd))
#pragma unroll
                            for (int y = 0; y < 8; ++y)
                                if (word[y] & ~s_sign[r * 8 + y]) atomicOr(s_sign + r * 8 + y, word[y]);
                }
            }
        }
    }
    __syncthreads();
    for (uint32_t r = warp; r < used; r += WARPS) {
        const uint32_t plus = s_sign[r * 8 + lane / 8] >> (lane & 7) * 4 & 15u, minus = s_sign[r * 8 + 4 + lane / 8] >> (lane & 7) * 4 & 15u;
        if (!(plus | minus) || c >= a.d) continue;
        const RowOut to = row_out(a, w, r);
        for (uint32_t y = 0; y < 4; ++y) {
            const float add = (plus >> y & 1u ? INFINITY : 0.0f) + (minus >> y & 1u ? -INFINITY : 0.0f);  // (both: NaN)
            if (add == 0.0f) continue;
            if (to.out) {
                __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(to.out) + c + y;
                *o = __float2bfloat16(__bfloat162float(*o) + add);
            } else {
                to.part[c + y] += add;
            }
        }
    }
}

// The item again on the CUDA cores, a warp a query row and a row of the cache at a time, where a wait ran out.
__device__ __noinline__ void by_rows(uint32_t bars, bool q_boxes, const CacheArgs& a, const Item& w, const uint32_t* s_qp, const uint32_t* s_qd, const float* s_slope, const uint32_t* s_tok,
                                     const uint32_t* s_depth, const uint32_t* s_anc, const uint32_t* s_list, uint32_t cnt) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // (where somebody gave up, copies may still be under way; a fill that was never begun lets the wait run out)
    bar_settle(bars + K_FULL * 8, cnt, 2);
    bar_settle(bars + V_FULL * 8, cnt, 2);
    bar_settle(bars + Q_FULL * 8, q_boxes ? 1 : 0, 1);
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
        for (uint32_t j = 0; j < cnt * KT; ++j) {
            const uint32_t i = (s_list[j / KT] >> 2) * KT + j % KT;
            if (i >= w.n) continue;
            const uint32_t kp = row_position(a, w, s_depth, i);
            if (!row_sees(a, w, s_qp, s_qd, s_tok, s_anc, r, i, kp, a.row_doc ? a.row_doc[w.entry + i] : 0u)) continue;
            float s = 0.0f;
            if (mine)
                for (int e = 0; e < 4; ++e) s = fmaf(x[e], __bfloat162float(k[(uint64_t)i * a.krs + c + e]), s);
            for (int b = 16; b; b >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, b);
            s = a.cap > 0.0f ? a.cap * LOG2E * cache_tanh(s * a.scale / a.cap) : s * a.scale * LOG2E;
            s = fmaf(-s_slope[r], cache_distance(s_qp[r], kp), s);
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

// A tile's scores that are more than products: capped, biased, masked.  Read from TMEM and written back, 32 columns at a time, in units of log 2 where a cap or a distance bends them; where
// all that a warp's rows see of 32 columns is all, they stay as they are.  (A function, in loops that are hardly
// unrolled, so that the loop over the tiles stays short: where the same stood in it, every tile's weights took 15 % longer.)  False where a wait ran out.
template <int D, bool CAP, bool SLOPED, bool APART = false>
__device__ __noinline__ bool bend_tile(const CacheArgs& a, unsigned char* sm, uint32_t ts, uint32_t r, uint32_t t, uint32_t li) {
    using S = Wide<D>;
    const Item& w = *reinterpret_cast<const Item*>(sm + S::ITEM_AT);
    const uint32_t* const s_qp = reinterpret_cast<const uint32_t*>(sm + S::ROWS_AT) + 2 * MB;
    const uint32_t bars = smem_addr(sm) + S::BAR_AT;
    const auto bar = [&](int which) { return bars + which * 8; };
    const uint32_t what = reinterpret_cast<const uint32_t*>(sm + S::LIST_AT)[li], first = (what >> 2) * KT, n = w.n, ctx = w.ctx;
    constexpr bool has_slope = SLOPED;
    const bool all = what >> t & 1, drafts = a.tree && first + KT > ctx;
    const bool by_pos = a.row_pos || (w.drafts_listed && drafts), listed = !all && (w.arrays || (w.drafts_listed && drafts));  // the fetching warp has left the rows' positions
    if ((has_slope || listed) && !__all_sync(0xFFFFFFFFu, bar_wait(bar(META_FULL + (li & 3)), li >> 2 & 1))) return false;
    const uint4* kp4 = reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(sm + S::META_AT) + (li & 3) * 3 * KT);
    const uint32_t qp = s_qp[r], qd = s_qp[MB + r];
    if constexpr (SLOPED && !APART)  // (in the same function: 250 us for 231 of 4096 tokens whose tiles are all bent)
        if (__any_sync(0xFFFFFFFFu, cache_distance(qp, w.near_pos) > (float)DISTANCE_NEAR)) return bend_tile<D, CAP, true, true>(a, sm, ts, r, t, li);
    const float slope = __uint_as_float(s_qp[2 * MB + r]), q_at = (float)((long long)qp - (long long)w.near_pos);
    const uint32_t* anc = reinterpret_cast<const uint32_t*>(sm + S::TREE_AT) + 2 * TREE_MOST + (a.tree ? s_qp[3 * MB + r] * (TREE_MOST / 32) : 0u);
    const CacheSight sight = w.sight;
    constexpr bool has_cap = CAP, bends = has_cap || has_slope;
    const float to_log2 = has_cap ? a.scale / a.cap : a.scale * LOG2E, cap2 = a.cap * LOG2E;
    // positions one after another: what is seen are one or two runs
    const long long at = (long long)w.sg.base + first;
    const long long low = (long long)qp - sight.window_last - at, high = (sight.causal ? (long long)qp : (long long)qp + sight.window_last) - at + 1;
    const int lo = (int)max(0ll, min(low, 128ll)), hi = (int)max(0ll, min(high, 128ll)), pre = (int)max(0ll, min((long long)sight.prefix - at, 128ll)), inside = (int)min(n - first, 128u);
#pragma unroll 1
    for (int j = 0; j < 4; ++j) {
        uint32_t seen = 0xFFFFFFFFu;  // bits of the rows that this query row sees
        if (!all) {
            seen = 0;
            if (by_pos) {
#pragma unroll 2
                for (int g = 0; g < 8; ++g) {
                    const uint4 p = kp4[j * 8 + g];
                    seen |= ((sight.sees(qp, p.x) ? 1u : 0u) | (sight.sees(qp, p.y) ? 2u : 0u) | (sight.sees(qp, p.z) ? 4u : 0u) | (sight.sees(qp, p.w) ? 8u : 0u)) << g * 4;
                }
            } else if (drafts) {  // (no window: what comes before the drafted rows is seen)
                seen = low_bits((int)ctx - (int)first - 32 * j);
            } else {
                seen = (low_bits(hi - 32 * j) & ~low_bits(lo - 32 * j)) | low_bits(pre - 32 * j);
            }
            if (a.row_doc) {
                uint32_t bits = 0;
#pragma unroll 4
                for (int g = 0; g < 8; ++g) {
                    const uint4 d = kp4[KT / 4 + j * 8 + g];
                    bits |= ((d.x == qd ? 1u : 0u) | (d.y == qd ? 2u : 0u) | (d.z == qd ? 4u : 0u) | (d.w == qd ? 8u : 0u)) << g * 4;
                }
                seen &= bits;
            }
            if (drafts) {  // of the drafted rows only itself and its ancestors
                const int from = (int)first + 32 * j - (int)ctx;  // the word's first row, counted among the drafted
                const uint32_t before = low_bits(-from);
                uint32_t line = 0;
                if (from > -32 && from < (int)TREE_MOST) {
                    const int word = from >> 5, off = from & 31;  // (word -1: the rows before)
                    const uint32_t l = word >= 0 ? anc[word] : 0u, h = word + 1 < (int)(TREE_MOST / 32) ? anc[word + 1] : 0u;
                    line = __funnelshift_r(l, h, off);
                }
                seen = w.drafts_listed ? seen & (before | line) : (seen & before) | (line & ~before);
            }
            seen &= low_bits(inside - 32 * j);
        }
        if (!bends && __all_sync(0xFFFFFFFFu, seen == 0xFFFFFFFFu)) continue;
        uint32_t u[32];
        float* s = reinterpret_cast<float*>(u);
        tmem_ld32(ts + 32 * j, u);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 32; ++c) asm volatile("" : "+r"(u[c]));
        if (has_cap) {
            float big = 0.0f;
#pragma unroll
            for (int c = 0; c < 32; ++c) big = fmaxf(big, fabsf(s[c]));
            if (__all_sync(0xFFFFFFFFu, big * to_log2 <= 1.0f || w.row0 + r >= w.q_rows)) {
                const uint64_t in = pair(to_log2, to_log2), out = pair(cap2, cap2);
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const uint64_t y = mul2(pair(s[c], s[c + 1]), in);
                    unpair(mul2(mul2(y, tanh_poly(mul2(y, y))), out), s[c], s[c + 1]);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 32; ++c) {  // tanh x = 1 - 2 / (exp(2 x) + 1)
                    const float e = exp2_fast(s[c] * to_log2 * (2.0f * LOG2E));
                    s[c] = fmaf(-2.0f * cap2, __fdividef(1.0f, e + 1.0f), cap2);
                }
            }
        } else if (has_slope) {
#pragma unroll
            for (int c = 0; c < 32; ++c) s[c] *= to_log2;
        }
        if constexpr (APART) {
#pragma unroll
            for (int c = 0; c < 32; ++c) s[c] = fmaf(-slope, cache_distance(qp, lds(smem_addr(kp4) + (j * 32 + c) * 4)), s[c]);
        } else if (has_slope) {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
                const float4 k = *reinterpret_cast<const float4*>(kp4 + KT / 2 + j * 8 + c / 4);
                s[c] = fmaf(-slope, fabsf(q_at - k.x), s[c]);
                s[c + 1] = fmaf(-slope, fabsf(q_at - k.y), s[c + 1]);
                s[c + 2] = fmaf(-slope, fabsf(q_at - k.z), s[c + 2]);
                s[c + 3] = fmaf(-slope, fabsf(q_at - k.w), s[c + 3]);
            }
        }
        if (!all)
#pragma unroll
            for (int c = 0; c < 32; ++c)
                if (!(seen >> c & 1u)) s[c] = -INFINITY;
        __syncwarp();
        tmem_st16(ts + 32 * j, u);
        tmem_st16(ts + 32 * j + 16, u + 16);
    }
    tmem_wait_st();
    __syncwarp();
    return true;
}

// CAP: scores are capped.  RICH: rows with positions or documents of their own, tokens with positions of their own, or trees; SLOPED: these or not, and a distance bias.  (Instances of
// their own: what a kernel does not need costs it registers and instruction cache in the loop over the tiles; with all in one, 8192 tokens of 32 heads took 937 us, alone 876.)
enum { PLAIN = 0, RICH = 1, SLOPED = 2 };
template <int D, bool CAP, int KIND>
__global__ void __launch_bounds__(THREADS, 1) cache_attend_wide_kernel(const __grid_constant__ CacheArgs a, const __grid_constant__ WideMaps maps, const __grid_constant__ CacheTable tab) {
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
    const uint32_t block = (w.item - w.sg.item_begin) / w.sg.n_chunks, chunk = (w.item - w.sg.item_begin) - block * w.sg.n_chunks, tiles = (w.n + KT - 1) / KT;
    {   // (the last blocks first: under a causal mask they see most)
        const uint32_t turned = w.sg.n_blocks - 1 - block;
        w.row0 = (w.sg.block_first + turned) * MB;
        w.item = w.sg.item_begin + turned * w.sg.n_chunks + chunk;  // (where the parts of its rows go)
    }
    w.sight = CacheSight{a.window_last, a.prefix ? a.prefix[w.sg.seg] : 0u, a.causal};
    const CacheSight sight = w.sight;
    w.entry = w.head * a.entry_hs + w.sg.row_begin;
    constexpr bool has_slope = KIND == SLOPED;
    const bool has_pos = KIND != PLAIN && a.row_pos, has_doc = KIND != PLAIN && a.row_doc, is_tree = KIND != PLAIN && a.tree;
    constexpr bool has_cap = CAP;
    const uint32_t used = min((uint32_t)MB, w.q_rows - w.row0);
    const bool two = used > 128;

    uint32_t* s_meta = reinterpret_cast<uint32_t*>(sm + S::META_AT);
    uint32_t* s_list = reinterpret_cast<uint32_t*>(sm + S::LIST_AT);
    unsigned char* s_cls = sm + S::CLS_AT;
    uint64_t* s_q = reinterpret_cast<uint64_t*>(sm + S::ROWS_AT);
    uint32_t* s_qp = reinterpret_cast<uint32_t*>(s_q + MB);
    uint32_t* s_qd = s_qp + MB;
    float* s_slope = reinterpret_cast<float*>(s_qd + MB);
    uint32_t* s_tok = reinterpret_cast<uint32_t*>(s_slope + MB);
    uint32_t* s_range = reinterpret_cast<uint32_t*>(sm + S::RANGE_AT);
    uint32_t* s_par = reinterpret_cast<uint32_t*>(sm + S::TREE_AT);
    uint32_t* s_depth = s_par + TREE_MOST;
    uint32_t* s_anc = s_depth + TREE_MOST;
    const uint32_t bars = sb + S::BAR_AT;
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(sm + S::BAR_AT + TMEM_WORD * 8);
    volatile uint32_t* s_fail = reinterpret_cast<volatile uint32_t*>(sm + S::BAR_AT + FAIL_WORD * 8);  // a wait ran out; a tile holds values that are not finite
    uint32_t* s_odd = reinterpret_cast<uint32_t*>(sm + S::ODD_AT);                                      // of each tile 16 bits, one for each eight rows in which there are such
    const auto bar = [&](int which) { return bars + which * 8; };
    const uint32_t tok0 = w.row0 / a.group;

    const bool arrays = has_pos || has_doc, drafts_listed = is_tree && (arrays || a.q_pos || sight.window_last != 0xFFFFFFFFu);  // drafted rows whose positions count
    const bool plain = KIND == PLAIN || (!arrays && !a.q_pos);  // all positions follow from the segment
    const uint32_t near_pos = a.q_pos ? a.q_pos[w.sg.query_begin + tok0] : w.sg.base + w.ctx + (is_tree ? 0u : tok0);
    w.near_pos = near_pos;
    w.arrays = arrays;
    w.drafts_listed = drafts_listed;
    if (tid == 0) *reinterpret_cast<Item*>(sm + S::ITEM_AT) = w;
    uint32_t cnt = 0;
    if (warp == FETCH_WARP) {
        for (uint32_t i = lane; i < RUN_MOST / 2; i += 32) s_odd[i] = 0;
        if (lane == 0) {
            for (int i = 0; i < 2; ++i) {
                bar_init(bar(K_FULL + i), 1);
                bar_init(bar(V_FULL + i), 1);
                bar_init(bar(K_FREE + i), 1);
                bar_init(bar(V_FREE + i), 3);
                bar_init(bar(V_CLEAN + i), 2);
                bar_init(bar(S_FULL + i), 1);
                bar_init(bar(P_HALF + i), 128);
                bar_init(bar(P_FULL + i), 128);
            }
            bar_init(bar(O_FULL), 1);
            bar_init(bar(Q_FULL), 1);
            for (int i = 0; i < 4; ++i) bar_init(bar(META_FULL + i), 1);
            s_fail[0] = s_fail[1] = 0;
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            if (maps.q_boxes) {  // 32 query rows a box
                const uint32_t boxes = two ? 8 : 4, step = 32 / a.group, t0 = w.sg.query_begin + tok0;
                bar_expect(bar(Q_FULL), boxes * S::TILE / 4);
                for (uint32_t i = 0; i < boxes; ++i)
#pragma unroll
                    for (int h = 0; h < S::HALVES; ++h)
                        tma_load(sb + (i >> 2) * S::TILE + h * HALF + (i & 3) * 4096, &maps.q, h * 64, w.head * a.group, t0 + i * step, bar(Q_FULL));
            }
        }
        __syncwarp();
    }
    if (plain) {
        // Which tiles are visited, and which of them either tile of query rows sees as a whole.  Of a split segment the item takes its share of them.  Every warp goes through
        // them, so that each knows how many there are; the fetching one writes the list.
        const uint32_t p0 = w.sg.base + w.ctx, last_tok = w.sg.n_queries - 1;
        // (of a tree's tokens: between the first one's and that of the last in a chain)
        const auto pos = [&](uint32_t row) { return is_tree ? p0 + (row == w.row0 || row == w.row0 + 128 ? 0u : last_tok) : p0 + min(row / a.group, last_tok); };
        const CacheRanges qa{pos(w.row0), pos(w.row0 + 127), 0u, 0u}, qb{pos(w.row0 + 128), pos(w.row0 + 255), 0u, 0u};
        const auto class_of = [&](uint32_t j) -> uint32_t {
            const uint32_t first = j * KT, last = first + KT - 1;
            if (j >= tiles) return 0u;
            const CacheRanges k{w.sg.base + first, w.sg.base + min(last, w.n - 1), 0u, 0u};
            const bool drafts = is_tree && last >= w.ctx;
            const int x = cache_tile_class(k, qa, sight, drafts, last < w.n), y = cache_tile_class(k, qb, sight, drafts, last < w.n);
            return (x || y ? 1u : 0u) | (x == 2 ? 2u : 0u) | (y == 2 ? 4u : 0u);
        };
        uint32_t skip = 0, most = RUN_MOST;
        if (w.sg.n_chunks > 1) {
            uint32_t visited = 0;
            for (uint32_t j0 = 0; j0 < tiles; j0 += 32) visited += __popc(__ballot_sync(0xFFFFFFFFu, class_of(j0 + lane) != 0));
            skip = (uint32_t)((uint64_t)visited * chunk / w.sg.n_chunks);
            most = (uint32_t)((uint64_t)visited * (chunk + 1) / w.sg.n_chunks) - skip;
        }
        uint32_t met = 0;
        for (uint32_t j0 = 0; j0 < tiles && met < skip + most; j0 += 32) {
            const uint32_t cls = class_of(j0 + lane), mask = __ballot_sync(0xFFFFFFFFu, cls != 0), at = met + __popc(mask & ((1u << lane) - 1u));
            if (warp == FETCH_WARP && cls && at >= skip && at < skip + most) s_list[at - skip] = (j0 + lane) << 2 | cls >> 1;
            met += __popc(mask);
        }
        cnt = met > skip ? min(met - skip, most) : 0u;
        __syncwarp();
    }
    const unsigned char* kb = static_cast<const unsigned char*>(a.keys) + (w.sg.row_begin * a.krs + w.head * a.khs) * 2;
    const unsigned char* vb = static_cast<const unsigned char*>(a.values) + (w.sg.row_begin * a.vrs + w.head * a.vhs) * 2;
    constexpr int PIECES = S::HALVES * 8;
    const auto fetch = [&](uint32_t dst, const CUtensorMap* map, bool head_first, const unsigned char* from, uint64_t stride, uint32_t first, uint32_t full) {
        if (first + KT <= w.n) {
            if (lane == 0) {
                const uint32_t row = (uint32_t)w.sg.row_begin + first;
                bar_expect(full, S::TILE);
#pragma unroll
                for (int h = 0; h < S::HALVES; ++h) tma_load(dst + h * HALF, map, h * 64, head_first ? w.head : row, head_first ? row : w.head, full);
            }
        } else {
            for (uint32_t i = lane; i < KT * PIECES; i += 32) {
                const uint32_t r = i / PIECES, c = i % PIECES, row = first + r;
                const bool there = row < w.n && c * 8 < a.d;
                copy16(dst + (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4), there ? from + row * stride * 2 + c * 16 : from, there);
            }
            copy_commit();
            copy_wait<0>();
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            __syncwarp();
            if (lane == 0) bar_arrive(full);
        }
    };
    if (warp == FETCH_WARP && plain && cnt) {  // the first keys, while the others get ready
        __syncwarp();
        fetch(sb + S::K_AT, &maps.k, maps.k_head_first, kb, a.krs, (s_list[0] >> 2) * KT, bar(K_FULL));
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(bar(TMEM_WORD)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (is_tree) {
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
    for (uint32_t r = tid; r < MB; r += THREADS) {  // (rows behind the last repeat it; their queries are zeros or, where boxes bring them, those of other tokens)
        const uint32_t row = min(w.row0 + r, w.q_rows - 1), tok = row / a.group, h = w.head * a.group + row - tok * a.group;
        s_q[r] = ((uint64_t)(w.sg.query_begin + tok) * a.qts + (uint64_t)h * a.qhs) * 2;
        s_qp[r] = a.q_pos ? a.q_pos[w.sg.query_begin + tok] : w.sg.base + w.ctx + (is_tree ? s_depth[tok] : tok);
        s_qd[r] = has_doc ? a.q_doc[w.sg.query_begin + tok] : 0u;
        s_slope[r] = has_slope ? a.slopes[h] * LOG2E : 0.0f;
        s_tok[r] = tok - tok0;
    }
    if (!maps.q_boxes) {
        __syncthreads();
        for (int i = tid; i < (two ? MB : 128) * S::HALVES * 8; i += THREADS) {
            const uint32_t r = i / (S::HALVES * 8), c = i % (S::HALVES * 8);
            const bool there = r < used && c * 8 < a.d;
            copy16(sb + (r >> 7) * S::TILE + (c >> 3) * HALF + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4), static_cast<const unsigned char*>(a.q) + (there ? s_q[r] + c * 16 : 0), there);
        }
        copy_commit();
        copy_wait<0>();
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // (the queries, read by the products)
    }
    if (!plain) {
        // the same, from the arrays: all warps look, a tile each at a time
        const uint32_t first_tile = min(tiles, chunk * w.sg.chunk_tiles), in_run = min(tiles - first_tile, w.sg.chunk_tiles);
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
        {   // which tiles are visited, and which of them either tile of query rows sees as a whole
            const CacheRanges qa{s_range[0], s_range[1], s_range[2], s_range[3]}, qb{s_range[4], s_range[5], s_range[6], s_range[7]};
            const auto classes = [&](const CacheRanges& k, uint32_t last) {
                const bool drafts = is_tree && last >= w.ctx, inside = last < w.n;
                const int x = cache_tile_class(k, qa, w.sight, drafts, inside), y = cache_tile_class(k, qb, w.sight, drafts, inside);
                return (x || y ? 1 : 0) | (x == 2 ? 2 : 0) | (y == 2 ? 4 : 0);
            };
            if (has_pos || has_doc) {
                constexpr int AT_ONCE = 3;  // tiles whose loads a warp has under way
                for (uint32_t j0 = warp; j0 < in_run; j0 += WARPS * AT_ONCE) {
                    CacheRanges k[AT_ONCE];
#pragma unroll
                    for (int x = 0; x < AT_ONCE; ++x) {
                        const uint32_t first = (first_tile + min(j0 + x * WARPS, in_run - 1)) * KT;
                        k[x] = CacheRanges{0xFFFFFFFFu, 0u, has_doc ? 0xFFFFFFFFu : 0u, 0u};
                    if (!has_pos) {  // (no token sees a row of them, whatever its document)
                        const CacheRanges by_place{w.sg.base + first, w.sg.base + min(first + KT - 1, w.n - 1), min(qa.dmin, qb.dmin), max(qa.dmax, qb.dmax)};
                        const CacheRanges both{min(qa.pmin, qb.pmin), max(qa.pmax, qb.pmax), by_place.dmin, by_place.dmax};
                        if (!cache_tile_class(by_place, both, sight, is_tree && first + KT > w.ctx, true)) continue;
                    }
#pragma unroll
                        for (int e = 0; e < KT / 32; ++e) {
                            const uint32_t i = min(first + lane + e * 32, w.n - 1);
                            const uint32_t p = has_pos ? a.row_pos[w.entry + i] : w.sg.base + i, d = has_doc ? a.row_doc[w.entry + i] : 0u;
                            k[x].pmin = min(k[x].pmin, p);
                            k[x].pmax = max(k[x].pmax, p);
                            k[x].dmin = min(k[x].dmin, d);
                            k[x].dmax = max(k[x].dmax, d);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < AT_ONCE; ++x) {
                        const uint32_t j = j0 + x * WARPS;
                        k[x].pmin = __reduce_min_sync(0xFFFFFFFFu, k[x].pmin);
                        k[x].pmax = __reduce_max_sync(0xFFFFFFFFu, k[x].pmax);
                        k[x].dmin = __reduce_min_sync(0xFFFFFFFFu, k[x].dmin);
                        k[x].dmax = __reduce_max_sync(0xFFFFFFFFu, k[x].dmax);
                        if (lane == 0 && j < in_run) s_cls[j] = k[x].pmin > k[x].pmax ? 0 : (unsigned char)classes(k[x], (first_tile + j) * KT + KT - 1);
                    }
                }
            } else {
                for (uint32_t j = tid; j < in_run; j += THREADS) {
                    const uint32_t first = (first_tile + j) * KT, last = first + KT - 1;
                    s_cls[j] = (unsigned char)classes(CacheRanges{w.sg.base + first, w.sg.base + min(last, w.n - 1), 0u, 0u}, last);
                }
            }
        }
        __syncthreads();
        for (uint32_t j0 = 0; j0 < in_run; j0 += 32) {  // (every warp counts, the first one writes)
            const int cls = j0 + lane < in_run ? s_cls[j0 + lane] : 0;
            const uint32_t mask = __ballot_sync(0xFFFFFFFFu, cls != 0);
            if (warp == 0 && cls) s_list[cnt + __popc(mask & ((1u << lane) - 1u))] = (first_tile + j0 + lane) << 2 | cls >> 1;
            cnt += __popc(mask);
        }
    }
    if (warp == FETCH_WARP && !cnt && maps.q_boxes) bar_wait(bar(Q_FULL), 0);  // (no product waits for the queries then, and rows of zeros leave through their place)
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *s_tmem;  // (read by all warps alike: with a value of its own for one of them, the compiler issued each product in a loop over the lanes)
    bool fail = false;

    if (warp < 8) {
        // ---- scores to weights: a query row a thread
        regs_more<REGS_ROWS>();
        const uint32_t t = warp >> 2, r = tid;
        if (t == 0 || two) {
            const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21), ts = lanes + t * 128, to = lanes + 256 + t * 128;
            const float to_log2 = has_cap ? a.scale / a.cap : a.scale * LOG2E, cap2 = a.cap * LOG2E;
            float m = -INFINITY, l = 0.0f;
            const bool there = r < used;  // (rows behind the last have no part in what a warp decides for all its rows: equal inputs give equal bits)
            for (uint32_t li = 0; li < cnt; ++li) {
                if (!__all_sync(0xFFFFFFFFu, bar_wait(bar(S_FULL + t), li & 1))) {
                    fail = true;
                    break;
                }
                tc_after();
                const bool all = s_list[li] >> t & 1;
                // Where a tile is seen as a whole and the warp's rows all have it on one side, the bias is near + step column, added on the way to the weights; its largest score is then only
                // bounded, by the largest product and the largest bias, which may be 2^64 too high and still leaves weights from 2^-62 of the row's largest on.
                // (8192 causal tokens, 32 heads: 900 us with all tiles bent, 587 so.)
                bool straight = false;
                float step = 0.0f, near = 0.0f;
                if constexpr (has_slope && !CAP) {
                    const long long at = (long long)w.sg.base + (s_list[li] >> 2) * KT;
                    const bool after = (long long)s_qp[r] >= at + KT - 1;
                    const float slope = s_slope[r];
                    step = after ? slope : -slope;
                    near = -slope * fabsf((float)((long long)s_qp[r] - at));
                    straight = __all_sync(0xFFFFFFFFu, all && !has_pos && !is_tree && (after || (long long)s_qp[r] <= at) && fabsf(slope) * (KT - 1) <= 64.0f);
                }
                const bool bent = !straight && (!all || has_slope);
                if (bent && !bend_tile<D, CAP, has_slope>(a, sm, ts, r, t, li)) {
                    fail = true;
                    break;
                }
                uint32_t u[128];
                float* s = reinterpret_cast<float*>(u);
                const auto load = [&]() {
#pragma unroll
                    for (int c = 0; c < 128; c += 32) tmem_ld32(ts + c, u + c);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 128; ++c) asm volatile("" : "+r"(u[c]));
                };
                load();
                float mul = bent && (CAP || has_slope) ? 1.0f : to_log2, top;
                bool fused = false, brief = false;  // the cap is applied on the way to the weights, by a polynomial of degree 6 or of degree 4
                if (CAP && !bent) {
                    float high[2] = {-INFINITY, -INFINITY}, low[2] = {INFINITY, INFINITY};
#pragma unroll
                    for (int c = 0; c < 128; c += 4)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            high[e] = fmaxf(high[e], fmaxf(s[c + 2 * e], s[c + 2 * e + 1]));
                            low[e] = fminf(low[e], fminf(s[c + 2 * e], s[c + 2 * e + 1]));
                        }
                    const float x = fmaxf(high[0], high[1]) * to_log2;
                    mul = 1.0f;
                    const float furthest = fmaxf(x, -fminf(low[0], low[1]) * to_log2);
                    fused = __all_sync(0xFFFFFFFFu, furthest <= 1.0f || !there);
                    brief = __all_sync(0xFFFFFFFFu, furthest <= TANH_BRIEF || !there);
                    if (fused) {  // (tanh grows: the largest score is that of the largest product)
                        top = cap2 * tanh_small(x);
                    } else {
                        if (!bend_tile<D, CAP, has_slope>(a, sm, ts, r, t, li)) {
                            fail = true;
                            break;
                        }
                        load();
                    }
                }
                if (!fused) {
                    float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < 128; c += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = fmaxf(x[e], fmaxf(s[c + 2 * e], s[c + 2 * e + 1]));
                    top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * mul;
                    if (straight) top += fmaxf(near, fmaf(step, KT - 1, near));
                }
                if (__any_sync(0xFFFFFFFFu, top > m + LAZY && there)) {
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
                const uint64_t mul_2 = pair(mul, mul), use_2 = pair(-use, -use);
                uint64_t sum_a = pair(0.0f, 0.0f), sum_b = sum_a;
                constexpr int BIASED = 3;
                const auto weights = [&](auto capped) {
                    const uint64_t in = pair(to_log2, to_log2), out = pair(cap2, cap2);
#pragma unroll
                    for (int c = 0; c < 128; c += 32) {
                        uint32_t p[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float x, y;
                            uint64_t z = pair(s[c + e], s[c + e + 1]);
                            if constexpr (decltype(capped)::value == 1 || decltype(capped)::value == 2) {
                                z = mul2(z, in);
                                z = fma2(mul2(z, decltype(capped)::value == 1 ? tanh_poly(mul2(z, z)) : tanh_poly_brief(mul2(z, z))), out, use_2);
                            } else if constexpr (decltype(capped)::value == BIASED) {
                                z = fma2(z, mul_2, pair(fmaf(step, (float)(c + e), near - use), fmaf(step, (float)(c + e + 1), near - use)));
                            } else {
                                z = fma2(z, mul_2, use_2);
                            }
                            unpair(z, x, y);
                            x = exp2_fast(x);
                            y = exp2_fast(y);
                            if (e & 2) sum_a = add2(sum_a, pair(x, y));
                            else sum_b = add2(sum_b, pair(x, y));
                            p[e / 2] = pack_bf16(x, y);
                        }
                        tmem_st16(ts + c / 2, p);
                        if (c == 32) {  // the products with the first half of the values may begin
                            tmem_wait_st();
                            tc_before();
                            bar_arrive(bar(P_HALF + t));
                        }
                    }
                };
                if constexpr (CAP) {
                    if (brief) weights(std::integral_constant<int, 2>());
                    else if (fused) weights(std::integral_constant<int, 1>());
                    else weights(std::integral_constant<int, 0>());
                } else if (has_slope && straight) {
                    weights(std::integral_constant<int, BIASED>());
                } else {
                    weights(std::integral_constant<int, 0>());
                }
                {
                    float x, y;
                    unpair(add2(sum_a, sum_b), x, y);
                    l += x + y;
                }
                tmem_wait_st();
                tc_before();
                bar_arrive(bar(P_FULL + t));
            }
            if (cnt && !fail) {
                fail = !__all_sync(0xFFFFFFFFu, bar_wait(bar(O_FULL), 0));
                tc_after();
            }
            // Rows leave through shared memory, where the queries were: a warp writes whole rows.
            const uint32_t tok = tok0 + s_tok[r], q_head = w.head * a.group + (there ? w.row0 + r - tok * a.group : 0u);
            const bool whole = w.sg.n_chunks == 1;
            const uint64_t part = ((uint64_t)w.item * a.n_kv + w.head) * MB + r;
            const uint64_t mine = whole ? (uint64_t)a.out + ((uint64_t)(w.sg.query_begin + tok) * a.ots + (uint64_t)q_head * a.ohs) * 2 : (uint64_t)(a.part_o + part * a.d);
            const float inv = !cnt || l == 0.0f ? 0.0f : whole ? 1.0f / l : 1.0f;
            constexpr int LINE = D * 2, LINE_PIECES = LINE / 16;  // bytes of a row at a time: all of its bfloat16 elements, or half of its float32 ones
            unsigned char* const stage = sm + t * S::TILE + (warp & 3) * 4096;  // 32 lines of 128 bytes in either half, as the boxes have them
            const auto piece = [&](int row, int c) { return reinterpret_cast<uint4*>(stage + (c >> 3) * HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4)); };
            const bool boxed = whole && maps.out_boxes && (uint32_t)(warp + 1) * 32 <= used;  // all 32 rows of the warp at once
            if (boxed) {
                __syncwarp();
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    uint32_t o[16];
                    tmem_ld16(to + c * 16, o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = inv != 0.0f ? __float_as_uint(__uint_as_float(o[e]) * inv) : 0u;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = pack_bf16(__uint_as_float(o[8 * h + 2 * e]), __uint_as_float(o[8 * h + 2 * e + 1]));
                        *piece(lane, c * 2 + h) = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) {
#pragma unroll
                    for (int h = 0; h < S::HALVES; ++h)
                        tma_store(&maps.out, sb + t * S::TILE + h * HALF + (warp & 3) * 4096, h * 64, w.head * a.group, w.sg.query_begin + tok0 + warp * (32 / a.group));
                    asm volatile("cp.async.bulk.commit_group;\ncp.async.bulk.wait_group.read 0;\n" ::: "memory");
                }
            }
            __syncwarp();
            for (int pass = 0; pass < (boxed ? 0 : whole ? 1 : 2); ++pass) {
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    if (!whole && c >= D / 32) break;
                    uint32_t o[16];
                    tmem_ld16(to + pass * (D / 2) + c * 16, o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = inv != 0.0f ? __float_as_uint(__uint_as_float(o[e]) * inv) : 0u;
                    if (whole) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t x[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] = pack_bf16(__uint_as_float(o[8 * h + 2 * e]), __uint_as_float(o[8 * h + 2 * e + 1]));
                            *piece(lane, c * 2 + h) = make_uint4(x[0], x[1], x[2], x[3]);
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < 4; ++h)
                            *piece(lane, c * 4 + h) = make_uint4(o[4 * h], o[4 * h + 1], o[4 * h + 2], o[4 * h + 3]);
                    }
                }
                __syncwarp();
#pragma unroll 4
                for (int i = lane; i < 32 * LINE_PIECES; i += 32) {
                    const int row = i / LINE_PIECES, c = i % LINE_PIECES;
                    const uint64_t dst = __shfl_sync(0xFFFFFFFFu, mine, row);
                    const uint4 x = *piece(row, c);
                    const uint32_t col = whole ? c * 8 : pass * (D / 2) + c * 4;
                    if ((warp * 32 + row) < (int)used && col < a.d) *reinterpret_cast<uint4*>(dst + col * (whole ? 2 : 4)) = x;
                }
                __syncwarp();
            }
            if (there) {
                if (whole) {
                    if (a.lse) a.lse[(uint64_t)(w.sg.query_begin + tok) * a.n_heads + q_head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
                } else {
                    a.part_ml[part * 2] = l == 0.0f ? -INFINITY : m;
                    a.part_ml[part * 2 + 1] = l;
                }
            }
        }
        regs_less<REGS_ALL>();
    } else {
        regs_less<REGS_REST>();
        if (warp == MMA_WARP) {
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
            const auto values = [&](uint32_t li, uint32_t t) {  // in two halves, as the weights come
                const uint32_t v = sb + S::V_AT + (li & 1) * S::TILE;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (!bar_wait(bar((h ? P_FULL : P_HALF) + t), li & 1)) return false;
                    tc_after();
#pragma unroll
                    for (int kk = h * 4; kk < h * 4 + 4; ++kk) mma_tmem(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, desc_across(v + kk * 2048), wide_idesc(D, true), li > 0 || kk > 0);
                }
                return true;
            };
            fail = (maps.q_boxes && !bar_wait(bar(Q_FULL), 0)) || !bar_wait(bar(K_FULL), 0);
            if (!fail) {
                scores(0, 0);
                if (two) scores(0, 1);
                tc_commit_to(bar(K_FREE));
            }
            for (uint32_t li = 0; li < cnt && !fail; ++li) {
                const bool more = li + 1 < cnt;
                // (the two warps have waited for the values; so for tiles that all see, too, which nobody looks over.  With a bias the loops come out quicker where the values are waited for
                // here too: 8192 causal tokens 609 us for 644, but a chunk under window and cap 225 for 217)
                if ((has_slope && !bar_wait(bar(V_FULL + (li & 1)), li >> 1 & 1)) || !bar_wait(bar(V_CLEAN + (li & 1)), li >> 1 & 1) || !values(li, 0)) {
                    fail = true;
                    break;
                }
                if (more) {
                    if (!bar_wait(bar(K_FULL + (li + 1 & 1)), (li + 1) >> 1 & 1)) {
                        fail = true;
                        break;
                    }
                    scores(li + 1, 0);
                }
                if (two && !values(li, 1)) {
                    fail = true;
                    break;
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
        } else if (warp == FETCH_WARP) {
        // ---- rows into shared memory
        for (uint32_t li = 0; li < cnt; ++li) {
            const uint32_t slot = li & 1, what = s_list[li], first = (what >> 2) * KT;
            if (li >= 2 && !__all_sync(0xFFFFFFFFu, bar_wait(bar(K_FREE + slot), (li >> 1) - 1 & 1))) {
                fail = true;
                break;
            }
            if (!plain || li > 0) fetch(sb + S::K_AT + slot * S::TILE, &maps.k, maps.k_head_first, kb, a.krs, first, bar(K_FULL + slot));
            // (the tile four before this one has been turned into weights: its positions are no longer read)
            const bool whole = (what & (two ? 3u : 1u)) == (two ? 3u : 1u);
            if (has_slope || (!whole && (arrays || (drafts_listed && first + KT > w.ctx)))) {
                for (uint32_t i = lane; i < KT; i += 32) {
                    const uint32_t row = min(first + i, w.n - 1);
                    uint32_t* at = s_meta + (li & 3) * 3 * KT + i;
                    const uint32_t p = has_pos ? a.row_pos[w.entry + row] : is_tree && row >= w.ctx ? w.sg.base + w.ctx + s_depth[row - w.ctx] : w.sg.base + row;
                    at[0] = p;
                    if (has_doc) at[KT] = a.row_doc[w.entry + row];
                    at[2 * KT] = __float_as_uint((float)((long long)p - (long long)near_pos));
                }
            }
            __syncwarp();
            if (lane == 0) bar_arrive(bar(META_FULL + (li & 3)));
            if (li >= 2 && !__all_sync(0xFFFFFFFFu, bar_wait(bar(V_FREE + slot), (li >> 1) - 1 & 1))) {
                fail = true;
                break;
            }
            fetch(sb + S::V_AT + slot * S::TILE, &maps.v, maps.v_head_first, vb, a.vrs, first, bar(V_FULL + slot));
        }
        } else {
        // ---- values of tiles that not all see: zeros take the place of those that are not finite, before the products (see odd_values)
        for (uint32_t li = 0; li < cnt; ++li) {
            if (!__all_sync(0xFFFFFFFFu, bar_wait(bar(V_FULL + (li & 1)), li >> 1 & 1))) {
                fail = true;
                break;
            }
            if ((s_list[li] & (two ? 3u : 1u)) != (two ? 3u : 1u)) {
                uint4* const tile = reinterpret_cast<uint4*>(sm + S::V_AT + (li & 1) * S::TILE);
                uint32_t odd = 0, parts = 0;
#pragma unroll 8
                for (uint32_t i = tid - 320; i < S::TILE / 16; i += 64) {
                    const uint4 x = tile[i];
                    odd |= odd_pair(x.x) | odd_pair(x.y) | odd_pair(x.z) | odd_pair(x.w);
                }
                if (__any_sync(0xFFFFFFFFu, odd & 0x80008000u)) {
                    const auto finite = [](uint32_t x) {
                        const uint32_t bad = odd_pair(x);
                        return x & ~((bad & 0x80000000u ? 0xFFFF0000u : 0u) | (bad & 0x00008000u ? 0xFFFFu : 0u));
                    };
                    for (uint32_t i = tid - 320; i < S::TILE / 16; i += 64) {  // (64 pieces are eight rows)
                        const uint4 x = tile[i];
                        if ((odd_pair(x.x) | odd_pair(x.y) | odd_pair(x.z) | odd_pair(x.w)) & 0x80008000u) parts |= 1u << (i / 64 & 15);
                        tile[i] = make_uint4(finite(x.x), finite(x.y), finite(x.z), finite(x.w));
                    }
                    parts = __reduce_or_sync(0xFFFFFFFFu, parts);
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    if (lane == 0) {
                        atomicOr(s_odd + (li >> 1), parts << (li & 1) * 16);
                        s_fail[1] = 1u;
                    }
                }
            }
            __syncwarp();
            if (lane == 0) {
                bar_arrive(bar(V_CLEAN + (li & 1)));
                bar_arrive(bar(V_FREE + (li & 1)));
            }
        }
        }
    }
    if (fail) s_fail[0] = 1u;
    tc_before();
    __syncthreads();  // (the rows' warps have given their registers back: none of the others takes them while one still has to get them)
    tc_after();
    if (warp >= 8) regs_more<REGS_ALL>();
    if (warp == MMA_WARP && s_fail[0] && cnt) bar_wait(bar(O_FULL), 0);  // (no product is under way when TMEM is given back, whoever gave up before)
    if (warp == MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
    if (s_fail[0] | s_fail[1]) {
        asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");  // (rows that left as boxes lie there before they are written again)
        __syncthreads();
        if (!s_fail[0]) odd_values<D>(a, sm, cnt);
        else by_rows(bars, maps.q_boxes != 0, a, *reinterpret_cast<const Item*>(sm + S::ITEM_AT), s_qp, s_qd, s_slope, s_tok, s_depth, s_anc, s_list, cnt);
    }
}

// Shares the segments' tiles out: each block of query rows visits some, in n_chunks items.  In units of a tile's time (1.8 us) an item costs about eight to begin and to end; what
// fits on the GPU at once takes as long as its longest item, more than that the mean load and half an item.  Where there are two blocks for every SM nothing is split.
void wide_share(const CacheArgs& a, CacheWork* w, uint32_t slots) {
    const bool known = !a.row_pos && !a.row_doc && !a.q_pos && !a.tree && !a.prefix && !a.rows;  // what a block visits follows from the table
    std::vector<uint32_t> most(w->segs.size());
    double total = 0.0, blocks = 0.0;
    uint32_t longest = 1;
    for (size_t i = 0; i < w->segs.size(); ++i) {
        const CacheSeg& s = w->segs[i];
        const uint32_t n = s.n_rows, tiles = std::max(1u, (uint32_t)(((uint64_t)n + KT - 1) / KT)), ctx = n - std::min(n, s.n_queries);
        const uint64_t count = ((uint64_t)s.n_queries * a.group + MB - 1) / MB;
        most[i] = known ? 1 : tiles;
        if (known && n)
            for (uint64_t b = 0; b < count; ++b) {
                const uint64_t p0 = ctx + b * MB / a.group, p1 = ctx + std::min<uint64_t>((b * MB + MB - 1) / a.group, s.n_queries - 1);
                const uint64_t lo = p0 > a.window_last ? p0 - a.window_last : 0, hi = std::min<uint64_t>(n - 1, a.causal ? p1 : p1 + a.window_last);
                const uint32_t visited = hi >= lo ? (uint32_t)(hi / KT - lo / KT + 1) : 1;
                most[i] = std::max(most[i], visited);
                total += (double)visited * a.n_kv;
            }
        else total += (double)count * tiles * a.n_kv;
        blocks += (double)count * a.n_kv;
        longest = std::max(longest, most[i]);
    }
    uint32_t best = std::min(longest, RUN_MOST);
    if (blocks < 2.0 * slots) {
        double best_time = 1e300;
        for (uint32_t run = best;; run = std::min(run - 1, run * 7 / 8)) {
            double items = 0.0;
            for (size_t i = 0; i < w->segs.size(); ++i) items += (double)(((uint64_t)w->segs[i].n_queries * a.group + MB - 1) / MB) * ((most[i] + run - 1) / run) * a.n_kv;
            const double time = items <= slots ? run + 8.0 : total / slots + 8.0 * items / slots + 0.5 * run;
            if (time + (run < longest ? 3.0 : 0.0) < best_time) best_time = time + (run < longest ? 3.0 : 0.0), best = run;
            if (run <= 2) break;
        }
    }
    for (size_t i = 0; i < w->segs.size(); ++i) {
        CacheSeg& s = w->segs[i];
        const uint32_t tiles = std::max(1u, (uint32_t)(((uint64_t)s.n_rows + KT - 1) / KT));
        s.n_chunks = (most[i] + best - 1) / best;
        s.chunk_tiles = (tiles + s.n_chunks - 1) / s.n_chunks;
    }
}
// The launches of a call: one, or where its parts would take more than CACHE_PARTS_MOST several, each of some blocks of query rows (262144 causal tokens of 32 heads on as many rows,
// 8.3 GB at once: 512 MB, and 596 ms for 630).
std::vector<CacheWork> wide_launches(const CacheArgs& a, const std::vector<CacheSeg>& segs) {
    bool split = false;
    for (const CacheSeg& s : segs) split |= s.n_chunks > 1;
    const uint64_t most = split ? std::max<uint64_t>(1, CACHE_PARTS_MOST / cache_part_bytes(1, a.n_kv, MB, a.d)) : ~0ull;
    std::vector<CacheWork> works(1);
    for (CacheSeg s : segs) {
        const uint64_t count = ((uint64_t)s.n_queries * a.group + MB - 1) / MB;
        for (uint64_t first = 0; first < count; first += s.n_blocks) {
            if (works.back().items && works.back().items + s.n_chunks > most) works.emplace_back();
            CacheWork& w = works.back();
            s.block_first = (uint32_t)first;
            s.n_blocks = (uint32_t)std::min(count - first, std::max<uint64_t>(1, (most - std::min(most, w.items)) / s.n_chunks));
            s.item_begin = (uint32_t)w.items;
            s.block_begin = (uint32_t)w.blocks;
            w.items += (uint64_t)s.n_blocks * s.n_chunks;
            if (s.n_chunks > 1) w.blocks += s.n_blocks;
            w.chunks = std::max(w.chunks, s.n_chunks);
            w.segs.push_back(s);
        }
    }
    return works;
}

template <int D, bool CAP, int KIND>
Status launch_wide(Ctx* c, CacheArgs a, CacheWork w, const WideMaps& maps) {
    using S = Wide<D>;
    wide_share(a, &w, (uint32_t)sm_count(c->device));
    const std::vector<CacheWork> works = wide_launches(a, w.segs);
    uint64_t parts = 0;
    for (const CacheWork& x : works) {
        if (x.items * a.n_kv > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "attention over a cache: too many blocks of query rows");
        if (x.blocks) parts = std::max(parts, x.items);
    }
    CacheMemory mem{c};
    SLHA_TRY(cache_part_memory(&a, parts, MB, &mem));
    constexpr auto kernel = cache_attend_wide_kernel<D, CAP, KIND>;
    SLHA_TRY((cache_smem<kernel>(c, S::SMEM_TREE)));
    static const int regs = []() {
        cudaFuncAttributes at;
        return cudaFuncGetAttributes(&at, cache_attend_wide_kernel<D, CAP, KIND>) == cudaSuccess ? at.numRegs : 0;
    }();
    if (regs != REGS_ALL) return Status(SLHA_ERR_DEVICE, "attention over a cache: the kernel was built with other registers than its warps share out");
    g_cache_kernels |= SLHA_B200_CACHE_ATTEND_WIDE;
    for (const CacheWork& x : works) {
        CacheTable tab;
        SLHA_TRY(cache_table(c, x.segs, &tab, &a.table));
        a.n_segs = (uint32_t)x.segs.size();
        SLHA_CUDA(launch_behind(kernel, dim3((uint32_t)(x.items * a.n_kv)), dim3(THREADS), a.tree ? S::SMEM_TREE : S::SMEM, c->stream, a, maps, tab));
        count_launch();
        if (x.blocks) SLHA_TRY(launch_cache_join(c, a, SLHA_B200_BF16, x, MB));
    }
    return mem.done();
}

template <int D>
Status launch_wide_d(Ctx* c, const CacheArgs& a, CacheWork w, const WideMaps& maps, int kind) {
    const bool cap = a.cap > 0.0f;
    if (kind == PLAIN) return cap ? launch_wide<D, true, PLAIN>(c, a, std::move(w), maps) : launch_wide<D, false, PLAIN>(c, a, std::move(w), maps);
    if (kind == RICH) return cap ? launch_wide<D, true, RICH>(c, a, std::move(w), maps) : launch_wide<D, false, RICH>(c, a, std::move(w), maps);
    return cap ? launch_wide<D, true, SLOPED>(c, a, std::move(w), maps) : launch_wide<D, false, SLOPED>(c, a, std::move(w), maps);
}

}  // namespace

Status launch_attend_wide(Ctx* c, CacheArgs a, CacheWork w, bool* taken) {
    uint64_t rows = 0;
    for (const CacheSeg& s : w.segs) rows = std::max(rows, s.row_begin + s.n_rows);
    WideMaps maps;
    *taken = wide_map(&maps.k, a.keys, a.krs, a.khs, std::max<uint64_t>(rows, 1), a.n_kv, a.d, &maps.k_head_first) &&
             wide_map(&maps.v, a.values, a.vrs, a.vhs, std::max<uint64_t>(rows, 1), a.n_kv, a.d, &maps.v_head_first);
    if (!*taken) return Status();
    maps.q_boxes = wide_row_map(&maps.q, a.q, a.qts, a.qhs, a);
    maps.out_boxes = wide_row_map(&maps.out, a.out, a.ots, a.ohs, a);
    const int kind = a.slopes ? SLOPED : a.row_pos || a.row_doc || a.q_pos || a.tree ? RICH : PLAIN;
    return a.d <= 64 ? launch_wide_d<64>(c, a, std::move(w), maps, kind) : launch_wide_d<128>(c, a, std::move(w), maps, kind);
}

}  // namespace slha
