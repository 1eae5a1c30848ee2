// Exact attention of query tokens over a cache of key and value rows (slha_b200_attend_cache, slha_b200_attend_tree).
//
// For query head g of KV head h, token t and the rows r that t sees:
//   s_r = scale <q, k_r>, capped to cap tanh(s_r / cap), minus slope_g |pos_t - pos_r|;   out = sum_r exp(s_r - lse) v_r,   lse = log sum_r exp(s_r)
// in one pass over the rows: a running maximum m and sum l a query row, out's sums scaled by exp(m_old - m_new) when the maximum grows.  Scores are held in
// units of log 2 (exp is one instruction there).
//
// One token's work is bound by the bytes of its rows: 131072 rows of 8 KV heads of 128 dimensions (537 MB), 91 to 101 us = 5.3 to 5.9 TB/s with scores capped, 84 without; 48 sequences of 6000
// on the average with positions and a distance bias 227 to 232 us (1.2 GB, 5.2 to 5.3 TB/s); 512 rows 6.5 us: a launch and the chain of one tile's loads, products, softmax and the join.  float32 rows are bound by the products (three of tf32 for one): 5 x 37 tokens of 12 heads of 96 dimensions over 1500 rows each 54 us.
//
// A CTA takes a block of 16, 32 or 64 query rows of one KV head (row = token x the head's group of query heads, so that the keys are read once for the group) and
// a run of the segment's rows in tiles of 64 (float32: 32).  Four warps: with 16 query rows each takes a quarter of a tile's keys, with 64 each takes
// its own 16 rows.  Tiles arrive by cp.async, one to three ahead (STAGES - 1, by what fits).
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "cache.cuh"
#include "cache_mma.cuh"

namespace slha {
thread_local uint32_t g_cache_kernels = 0;
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int ATT_THREADS = 128;
constexpr int ROUND = 256;  // tiles that are looked over at a time

template <typename T, int D, int WM>
struct Shape {
    static constexpr int MB = WM * 16, WN = 4 / WM;       // query rows; warps along the keys
    static constexpr int KT = sizeof(T) == 2 ? 64 : 32;   // keys of a tile
    static constexpr int KW = KT / WN, NT = KW / 8;       // a warp's
    static constexpr int STAGES = D == 64 ? 4 : WM == 4 || (D == 256 && WM == 2) ? 2 : 3;
    static constexpr uint32_t TILE = KT * D * sizeof(T), STAGE = 2 * TILE + 2 * KT * 4;
    static constexpr uint32_t Q_BYTES = MB * D * sizeof(T);
    // after the stages and Q: per query row position, document, slope, token within the block; per tile of a round its class; tree
    static constexpr uint32_t ROWS_AT = STAGES * STAGE + Q_BYTES, LIST_AT = ROWS_AT + 4 * MB * 4, CLS_AT = LIST_AT + ROUND * 2, RANGE_AT = CLS_AT + ROUND,
                              ML_AT = RANGE_AT + 32, TREE_AT = ML_AT + 64 * 2 * 4;
    static constexpr uint32_t SMEM = TREE_AT, SMEM_TREE = TREE_AT + TREE_MOST * 8 + MB * (TREE_MOST / 8);
    static constexpr int PITCH = D + 8;  // floats of a query row on the way out
    static_assert(64 * PITCH * 4 <= STAGES * STAGE && (64 * PITCH + MB * (D + 2)) * 4 <= STAGES * STAGE + Q_BYTES, "the sums leave through the stages and the queries behind them");
    static constexpr int CTAS = D == 256 ? 1 : 2;
    static_assert(SMEM_TREE <= 227 * 1024, "shared memory of an SM");
};

template <typename T, int D, int WM>
__global__ void __launch_bounds__(ATT_THREADS, Shape<T, D, WM>::CTAS) cache_attend_kernel(const __grid_constant__ CacheArgs a, const __grid_constant__ CacheTable tab) {
    using S = Shape<T, D, WM>;
    using L = Tile<T, D>;
    dep_wait();
    extern __shared__ __align__(1024) unsigned char sm[];
    const uint32_t sb = smem_addr(sm);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp % WM, wn = warp / WM, g = lane >> 2, t4 = lane & 3;
    namespace cg = cooperative_groups;
    const uint32_t cl = a.cluster ? a.cluster : 1, of_cluster = blockIdx.x % cl;
    const uint32_t head = blockIdx.x / cl % a.n_kv, item = blockIdx.x / cl / a.n_kv * cl + of_cluster;
    const CacheSeg* table = a.table ? a.table : tab.s;
    const uint32_t seg = cache_find(a.n_segs, item, [&](uint32_t i) { return table[i].item_begin; });
    const CacheSeg sg = table[seg];
    const uint32_t local = item - sg.item_begin, chunk = local % sg.n_chunks, block = local / sg.n_chunks;
    const uint32_t n = a.rows ? min(a.rows[sg.seg], sg.n_rows) : sg.n_rows;
    const uint32_t q_rows = sg.n_queries * a.group, row0 = block * S::MB;
    const uint32_t ctx = n - min(n, sg.n_queries);  // rows before the tokens' own
    const CacheSight sight{a.window_last, a.prefix ? a.prefix[sg.seg] : 0u, a.causal};
    const bool has_pos = a.row_pos, has_doc = a.row_doc, arrays = has_pos || has_doc;
    const uint64_t entry = head * a.entry_hs + sg.row_begin;

    uint32_t* s_qp = reinterpret_cast<uint32_t*>(sm + S::ROWS_AT);
    uint32_t* s_qd = s_qp + S::MB;
    float* s_slope = reinterpret_cast<float*>(s_qd + S::MB);
    uint32_t* s_tok = reinterpret_cast<uint32_t*>(s_slope + S::MB);
    uint16_t* s_list = reinterpret_cast<uint16_t*>(sm + S::LIST_AT);
    unsigned char* s_cls = sm + S::CLS_AT;
    uint32_t* s_range = reinterpret_cast<uint32_t*>(sm + S::RANGE_AT);
    uint32_t* s_par = reinterpret_cast<uint32_t*>(sm + S::TREE_AT);
    uint32_t* s_depth = s_par + TREE_MOST;
    uint32_t* s_anc = s_depth + TREE_MOST;
    const uint32_t tok0 = row0 / a.group;

    if (a.tree) {
        for (uint32_t j = tid; j < sg.n_queries; j += ATT_THREADS) {
            const uint32_t p = a.parents[sg.query_begin + j];
            s_par[j] = p < j ? p : 0xFFFFFFFFu;
        }
        for (uint32_t i = tid; i < S::MB * (TREE_MOST / 32); i += ATT_THREADS) s_anc[i] = 0;
        __syncthreads();
        for (uint32_t j = tid; j < sg.n_queries; j += ATT_THREADS) {  // (parents are smaller than their children: every walk ends)
            const uint32_t mine = j - tok0;
            uint32_t depth = 0, at = j;
            while (true) {
                if (mine < S::MB) s_anc[mine * (TREE_MOST / 32) + (at >> 5)] |= 1u << (at & 31);
                if (s_par[at] == 0xFFFFFFFFu) break;
                at = s_par[at];
                ++depth;
            }
            s_depth[j] = depth;
        }
        __syncthreads();
    }
    // the block's query rows (rows behind the last repeat it and are not written)
    const unsigned char* qbase = static_cast<const unsigned char*>(a.q);
    for (int i = tid; i < S::MB * L::PIECES; i += ATT_THREADS) {
        const int r = i / L::PIECES, c = i % L::PIECES;
        const uint32_t row = row0 + r;
        const bool there = row < q_rows && c * 16 < (int)(a.d * sizeof(T));
        const uint64_t at = there ? (sg.query_begin + row / a.group) * a.qts + (head * a.group + row % a.group) * a.qhs : 0;
        copy16(L::at(sb + S::STAGES * S::STAGE, r, c), qbase + at * sizeof(T) + (there ? c * 16 : 0), there);
    }
    copy_commit();
    for (int r = tid; r < S::MB; r += ATT_THREADS) {
        const uint32_t row = min(row0 + r, q_rows - 1), tok = row / a.group;
        s_qp[r] = a.q_pos ? a.q_pos[sg.query_begin + tok] : sg.base + ctx + (a.tree ? s_depth[tok] : tok);
        s_qd[r] = has_doc ? a.q_doc[sg.query_begin + tok] : 0u;
        s_slope[r] = a.slopes ? a.slopes[head * a.group + row % a.group] * LOG2E : 0.0f;
        s_tok[r] = tok - tok0;
    }
    __syncthreads();
    if (warp == 0) {
        CacheRanges q{0xFFFFFFFFu, 0u, 0xFFFFFFFFu, 0u};
        for (int r = lane; r < S::MB; r += 32) {
            q.pmin = min(q.pmin, s_qp[r]);
            q.pmax = max(q.pmax, s_qp[r]);
            q.dmin = min(q.dmin, s_qd[r]);
            q.dmax = max(q.dmax, s_qd[r]);
        }
        q.pmin = __reduce_min_sync(0xFFFFFFFFu, q.pmin);
        q.pmax = __reduce_max_sync(0xFFFFFFFFu, q.pmax);
        q.dmin = __reduce_min_sync(0xFFFFFFFFu, q.dmin);
        q.dmax = __reduce_max_sync(0xFFFFFFFFu, q.dmax);
        if (lane == 0) s_range[0] = q.pmin, s_range[1] = q.pmax, s_range[2] = q.dmin, s_range[3] = q.dmax;
    }
    copy_wait<0>();
    __syncthreads();
    const CacheRanges qr{s_range[0], s_range[1], s_range[2], s_range[3]};
    AFrag<T> qa[sizeof(T) == 2 && D <= 128 ? D / 16 : 1];
    constexpr bool Q_HELD = sizeof(T) == 2 && D <= 128;
    constexpr int KSTEPS = D / (sizeof(T) == 2 ? 16 : 8);
    const uint32_t sq = sb + S::STAGES * S::STAGE;
    if constexpr (Q_HELD)
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) qa[kk].template load<D>(sq, wm * 16, kk, lane);

    const auto tile_class = [&](const CacheRanges& k, uint32_t last) { return cache_tile_class(k, qr, sight, a.tree && last >= ctx, last < n); };

    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    const float to_log2 = a.cap > 0.0f ? a.scale / a.cap : a.scale * LOG2E, cap2 = a.cap * LOG2E;
    const bool has_cap = a.cap > 0.0f, has_slope = a.slopes;

    const uint32_t tiles = (n + S::KT - 1) / S::KT, tile_end = min(tiles, (chunk + 1) * sg.chunk_tiles);
    const unsigned char* kb = static_cast<const unsigned char*>(a.keys) + (sg.row_begin * a.krs + head * a.khs) * sizeof(T);
    const unsigned char* vb = static_cast<const unsigned char*>(a.values) + (sg.row_begin * a.vrs + head * a.vhs) * sizeof(T);
    for (uint32_t r0 = chunk * sg.chunk_tiles; r0 < tile_end; r0 += ROUND) {
        const uint32_t in_round = min((uint32_t)ROUND, tile_end - r0);
        // which of the round's tiles are visited
        if (arrays) {
            for (uint32_t j = warp; j < in_round; j += ATT_THREADS / 32) {
                const uint32_t first = (r0 + j) * S::KT, last = first + S::KT - 1;
                CacheRanges k{0xFFFFFFFFu, 0u, has_doc ? 0xFFFFFFFFu : 0u, 0u};
#pragma unroll
                for (int e = 0; e < S::KT / 32; ++e) {
                    const uint32_t i = min(first + lane + e * 32, n - 1);
                    const uint32_t p = has_pos ? a.row_pos[entry + i] : sg.base + i;
                    k.pmin = min(k.pmin, p);
                    k.pmax = max(k.pmax, p);
                    if (has_doc) {
                        const uint32_t d = a.row_doc[entry + i];
                        k.dmin = min(k.dmin, d);
                        k.dmax = max(k.dmax, d);
                    }
                }
                k.pmin = __reduce_min_sync(0xFFFFFFFFu, k.pmin);
                k.pmax = __reduce_max_sync(0xFFFFFFFFu, k.pmax);
                if (has_doc) {
                    k.dmin = __reduce_min_sync(0xFFFFFFFFu, k.dmin);
                    k.dmax = __reduce_max_sync(0xFFFFFFFFu, k.dmax);
                }
                if (lane == 0) s_cls[j] = (unsigned char)tile_class(k, last);
            }
        } else {
            for (uint32_t j = tid; j < in_round; j += ATT_THREADS) {
                const uint32_t first = (r0 + j) * S::KT, last = first + S::KT - 1;
                s_cls[j] = (unsigned char)tile_class(CacheRanges{sg.base + first, sg.base + min(last, n - 1), 0u, 0u}, last);
            }
        }
        __syncthreads();
        uint32_t cnt = 0;
        for (uint32_t j0 = 0; j0 < in_round; j0 += 32) {  // (every warp counts, the first one writes)
            const int cls = j0 + lane < in_round ? s_cls[j0 + lane] : 0;
            const uint32_t mask = __ballot_sync(0xFFFFFFFFu, cls != 0);
            if (warp == 0 && cls) s_list[cnt + __popc(mask & ((1u << lane) - 1u))] = (uint16_t)((j0 + lane) << 1 | (cls == 2));
            cnt += __popc(mask);
        }
        __syncthreads();

        const auto fetch = [&](uint32_t at) {
            if (at < cnt) {
                const uint32_t st = sb + (at % S::STAGES) * S::STAGE, first = (r0 + (s_list[at] >> 1)) * S::KT;
#pragma unroll
                for (int i = 0; i < S::KT * L::PIECES / ATT_THREADS; ++i) {
                    const int x = i * ATT_THREADS + tid, r = x / L::PIECES, c = x % L::PIECES;
                    const uint32_t row = first + r;
                    const bool there = row < n && c * 16 < (int)(a.d * sizeof(T));
                    copy16(L::at(st, r, c), there ? kb + row * (a.krs * sizeof(T)) + c * 16 : kb, there);
                    copy16(L::at(st + S::TILE, r, c), there ? vb + row * (a.vrs * sizeof(T)) + c * 16 : vb, there);
                }
                if (arrays && tid < 2 * S::KT) {
                    const uint32_t r = tid % S::KT, row = first + r;
                    const uint32_t* from = tid < S::KT ? a.row_pos : a.row_doc;
                    if (from) copy4(st + 2 * S::TILE + tid * 4, from + entry + min(row, n - 1), true);
                }
            }
            copy_commit();
        };
#pragma unroll
        for (int i = 0; i < S::STAGES - 1; ++i) fetch(i);
        for (uint32_t li = 0; li < cnt; ++li) {
            copy_wait<S::STAGES - 2>();
            __syncthreads();
            fetch(li + S::STAGES - 1);
            const uint32_t st = sb + (li % S::STAGES) * S::STAGE;
            const uint32_t what = s_list[li], first = (r0 + (what >> 1)) * S::KT;
            const bool all = what & 1;
            const int key0 = wn * S::KW;
            float s[S::NT][4];
#pragma unroll
            for (int i = 0; i < S::NT; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
            if constexpr (Q_HELD) {
#pragma unroll
                for (int kk = 0; kk < KSTEPS; ++kk) scores_step<T, D, S::NT>(s, qa[kk], st, key0, kk, lane);
            } else {
                scores_of<T, D, S::NT>(s, [&](int kk) -> const AFrag<T>& { qa[0].template load<D>(sq, wm * 16, kk, lane); return qa[0]; }, st, key0, lane);
            }
            // scores in units of log 2
#pragma unroll
            for (int i = 0; i < S::NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[i][e] *= to_log2;
                    if (has_cap) s[i][e] = cap2 * cache_tanh(s[i][e]);
                }
            if (!all || has_slope) {
                const uint32_t* kp_s = reinterpret_cast<const uint32_t*>(sm + (li % S::STAGES) * S::STAGE + 2 * S::TILE);
                const int ra = wm * 16 + g;
                const uint32_t qp[2] = {s_qp[ra], s_qp[ra + 8]}, qd[2] = {s_qd[ra], s_qd[ra + 8]};
                const float sl[2] = {s_slope[ra], s_slope[ra + 8]};
#pragma unroll
                for (int i = 0; i < S::NT; ++i)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t col = key0 + i * 8 + t4 * 2 + c, row = first + col;
                        const bool drafted = a.tree && row >= ctx && row < n;
                        const uint32_t kp = has_pos ? kp_s[col] : drafted ? sg.base + ctx + s_depth[row - ctx] : sg.base + row;
                        const uint32_t kd = has_doc ? kp_s[S::KT + col] : 0u;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float& x = s[i][h * 2 + c];
                            const uint32_t away = kp <= qp[h] ? qp[h] - kp : kp - qp[h];
                            if (has_slope) x = fmaf(-sl[h], (float)away, x);
                            if (!all) {
                                bool seen = row < n && sight.sees(qp[h], kp) && kd == qd[h];
                                if (drafted) seen = seen && (s_anc[s_tok[ra + h * 8] * (TREE_MOST / 32) + ((row - ctx) >> 5)] >> ((row - ctx) & 31) & 1u);
                                if (!seen) x = -INFINITY;
                            }
                        }
                    }
            }
            // running maximum and sum
            float grow[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = m[h];
#pragma unroll
                for (int i = 0; i < S::NT; ++i) mx = fmaxf(mx, fmaxf(s[i][h * 2], s[i][h * 2 + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
                const float use = mx == -INFINITY ? 0.0f : mx;
                grow[h] = exp2_fast(m[h] - use);
                m[h] = mx;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < S::NT; ++i) {
                    s[i][h * 2] = exp2_fast(s[i][h * 2] - use);
                    s[i][h * 2 + 1] = exp2_fast(s[i][h * 2 + 1] - use);
                    sum += s[i][h * 2] + s[i][h * 2 + 1];
                }
                l[h] = fmaf(l[h], grow[h], sum);
            }
            if (__any_sync(0xFFFFFFFFu, grow[0] != 1.0f || grow[1] != 1.0f)) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    o[i][0] *= grow[0];
                    o[i][1] *= grow[0];
                    o[i][2] *= grow[1];
                    o[i][3] *= grow[1];
                }
            }
            // Where some rows are not seen, they may hold anything: a weight of zero does not keep an infinity out of the sum.
            bool odd = false;
            if (!all) {
                for (int i = lane; i < S::KW * L::PIECES; i += 32) {
                    const uint4 x = *reinterpret_cast<const uint4*>(sm + (L::at(st + S::TILE, key0 + i / L::PIECES, i % L::PIECES) - sb));
                    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        odd |= (w[e] & 0x7F800000u) == 0x7F800000u;
                        if (sizeof(T) == 2) odd |= (w[e] & 0x00007F80u) == 0x00007F80u;
                    }
                }
                odd = __any_sync(0xFFFFFFFFu, odd);
            }
            if (!odd) {
                values_step<T, D, S::NT>(o, s, st + S::TILE, key0, lane);
            } else {  // key by key, only those with a weight
#pragma unroll
                for (int i = 0; i < S::NT; ++i)
                    for (int k8 = 0; k8 < 8; ++k8) {
                        const int from = (lane & ~3) | (k8 >> 1);
                        const float p0 = __shfl_sync(0xFFFFFFFFu, k8 & 1 ? s[i][1] : s[i][0], from);
                        const float p1 = __shfl_sync(0xFFFFFFFFu, k8 & 1 ? s[i][3] : s[i][2], from);
#pragma unroll
                        for (int d = 0; d < D / 8; ++d)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const uint32_t at = L::elem(st + S::TILE, key0 + i * 8 + k8, d * 8 + t4 * 2 + c) - sb;
                                float v;
                                if constexpr (sizeof(T) == 2) v = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(sm + at) << 16);
                                else v = *reinterpret_cast<const float*>(sm + at);
                                if (p0 != 0.0f) o[d][c] = fmaf(p0, v, o[d][c]);
                                if (p1 != 0.0f) o[d][2 + c] = fmaf(p1, v, o[d][2 + c]);
                            }
                    }
            }
        }
        copy_wait<0>();
        __syncthreads();  // (the next round's list and stages)
    }

    // the warps' maxima and sums meet, then their rows of sums
    float* s_m = reinterpret_cast<float*>(sm + S::ML_AT);  // [wn][query row]
    float* s_l = s_m + 64;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 1);
        l[h] += __shfl_xor_sync(0xFFFFFFFFu, l[h], 2);
        if (t4 == 0) s_m[wn * S::MB + wm * 16 + g + h * 8] = m[h], s_l[wn * S::MB + wm * 16 + g + h * 8] = l[h];
    }
    __syncthreads();
    float* s_o = reinterpret_cast<float*>(sm);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = wm * 16 + g + h * 8;
        float top = s_m[r];
#pragma unroll
        for (int w = 1; w < S::WN; ++w) top = fmaxf(top, s_m[w * S::MB + r]);
        const float f = m[h] == -INFINITY ? 0.0f : exp2_fast(m[h] - top);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<float2*>(s_o + (wn * S::MB + r) * S::PITCH + i * 8 + t4 * 2) =
                m[h] == -INFINITY ? make_float2(0.0f, 0.0f) : make_float2(o[i][h * 2] * f, o[i][h * 2 + 1] * f);
    }
    __syncthreads();
    const bool whole = sg.n_chunks == 1, shared = cl > 1;
    const uint32_t used = min((uint32_t)S::MB, q_rows - row0);
    // of a cluster: the CTA's own sums, maxima and sums of weights for the others to read
    float* const s_own = s_o + 64 * S::PITCH;
    float* const s_own_m = s_own + S::MB * D;
    float* const s_own_l = s_own_m + S::MB;
    for (uint32_t i = tid; i < used * (D / 4); i += ATT_THREADS) {
        const uint32_t r = i / (D / 4), c = i % (D / 4) * 4, row = row0 + r;
        if (c >= a.d) continue;
        float top = s_m[r];
#pragma unroll
        for (int w = 1; w < S::WN; ++w) top = fmaxf(top, s_m[w * S::MB + r]);
        float sum = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < S::WN; ++w) {
            const float mw = s_m[w * S::MB + r];
            sum += mw == -INFINITY ? 0.0f : s_l[w * S::MB + r] * exp2_fast(mw - top);
            const float4 y = *reinterpret_cast<const float4*>(s_o + (w * S::MB + r) * S::PITCH + c);
            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
        }
        if (shared) {
            *reinterpret_cast<float4*>(s_own + r * D + c) = x;
            if (c == 0) s_own_m[r] = top, s_own_l[r] = sum;
        } else if (whole) {
            const uint64_t tok = sg.query_begin + row / a.group;
            const uint32_t qh = head * a.group + row % a.group;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            unsigned char* dst = static_cast<unsigned char*>(a.out) + (tok * a.ots + qh * a.ohs + c) * sizeof(T);
            if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
            else *reinterpret_cast<float4*>(dst) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
            if (a.lse && c == 0) a.lse[tok * a.n_heads + qh] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * LN2;
        } else {
            const uint64_t at = ((uint64_t)item * a.n_kv + head) * S::MB + r;
            *reinterpret_cast<float4*>(a.part_o + at * a.d + c) = x;
            if (c == 0) a.part_ml[at * 2] = top, a.part_ml[at * 2 + 1] = sum;
        }
    }
    if (!shared) return;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (uint32_t i = of_cluster * ATT_THREADS + tid; i < used * (D / 4); i += cl * ATT_THREADS) {
        const uint32_t r = i / (D / 4), c = i % (D / 4) * 4, row = row0 + r;
        if (c >= a.d) continue;
        float top = -INFINITY, sum = 0.0f;
        for (uint32_t p = 0; p < cl; ++p) top = fmaxf(top, cluster.map_shared_rank(s_own_m, p)[r]);
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t p = 0; p < cl; ++p) {
            const float mp = cluster.map_shared_rank(s_own_m, p)[r], f = mp == -INFINITY ? 0.0f : exp2_fast(mp - top);
            const float4 y = *reinterpret_cast<const float4*>(cluster.map_shared_rank(s_own, p) + r * D + c);
            sum = fmaf(f, cluster.map_shared_rank(s_own_l, p)[r], sum);
            x.x = fmaf(f, y.x, x.x);
            x.y = fmaf(f, y.y, x.y);
            x.z = fmaf(f, y.z, x.z);
            x.w = fmaf(f, y.w, x.w);
        }
        const uint64_t tok = sg.query_begin + row / a.group;
        const uint32_t qh = head * a.group + row % a.group;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        unsigned char* dst = static_cast<unsigned char*>(a.out) + (tok * a.ots + qh * a.ohs + c) * sizeof(T);
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
        else *reinterpret_cast<float4*>(dst) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        if (a.lse && c == 0) a.lse[tok * a.n_heads + qh] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * LN2;
    }
    cluster.sync();  // (the others have read this CTA's sums)
}

// Joins the parts of query rows whose segment's rows were split.  WARPS warps a query row: each takes every WARPS-th part, their sums meet in shared memory in the warps' order.
constexpr int JOIN_THREADS = 128;
template <typename T, int WARPS>
__global__ void __launch_bounds__(JOIN_THREADS) cache_join_kernel(const __grid_constant__ CacheArgs a, const __grid_constant__ CacheTable tab, uint32_t mb, uint32_t blocks_of) {
    dep_wait();
    constexpr int ROWS = JOIN_THREADS / 32 / WARPS, FLIGHT = WARPS > 1 ? 8 : 3;
    __shared__ float4 s_acc[WARPS > 1 ? WARPS : 1][64];
    __shared__ float s_sum[WARPS];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = warp % WARPS;
    const uint32_t part = blockIdx.x % blocks_of, at = blockIdx.x / blocks_of, head = at % a.n_kv, qb = at / a.n_kv;
    const CacheSeg* table = a.table ? a.table : tab.s;
    const uint32_t seg = cache_find(a.n_segs, qb, [&](uint32_t i) { return table[i].block_begin; });
    const CacheSeg sg = table[seg];
    const uint32_t block = qb - sg.block_begin, r = part * ROWS + warp / WARPS, row = (sg.block_first + block) * mb + r;
    if (r >= mb || row >= sg.n_queries * a.group) return;  // (with more than one warp a row: all of them)
    const uint64_t first = ((uint64_t)(sg.item_begin + block * sg.n_chunks) * a.n_kv + head) * mb + r, step = (uint64_t)a.n_kv * mb;
    float top = -INFINITY;
    for (uint32_t c = lane; c < sg.n_chunks; c += 32) top = fmaxf(top, a.part_ml[(first + c * step) * 2]);
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
    float4 acc[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
    float sum = 0.0f;
    const uint32_t v_count = a.d > 128 ? 2 : 1;
    for (uint32_t c0 = mine; c0 < sg.n_chunks; c0 += WARPS * FLIGHT) {
        float2 ml[FLIGHT];
        float4 x[FLIGHT];
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i) {
            const uint32_t c = c0 + i * WARPS;
            const bool there = c < sg.n_chunks;
            ml[i] = there ? *reinterpret_cast<const float2*>(a.part_ml + (first + c * step) * 2) : make_float2(-INFINITY, 0.0f);
            x[i] = there && lane * 4 < a.d ? *reinterpret_cast<const float4*>(a.part_o + (first + c * step) * a.d + lane * 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i) {
            const float f = ml[i].x == -INFINITY ? 0.0f : exp2_fast(ml[i].x - top);
            sum = fmaf(f, ml[i].y, sum);
            acc[0].x = fmaf(f, x[i].x, acc[0].x);
            acc[0].y = fmaf(f, x[i].y, acc[0].y);
            acc[0].z = fmaf(f, x[i].z, acc[0].z);
            acc[0].w = fmaf(f, x[i].w, acc[0].w);
        }
        if (v_count == 2)
#pragma unroll
            for (int i = 0; i < FLIGHT; ++i) {
                const uint32_t c = c0 + i * WARPS;
                if (c >= sg.n_chunks || lane * 4 + 128 >= a.d) continue;
                const float4 y = *reinterpret_cast<const float4*>(a.part_o + (first + c * step) * a.d + lane * 4 + 128);
                const float f = ml[i].x == -INFINITY ? 0.0f : exp2_fast(ml[i].x - top);
                acc[1].x = fmaf(f, y.x, acc[1].x);
                acc[1].y = fmaf(f, y.y, acc[1].y);
                acc[1].z = fmaf(f, y.z, acc[1].z);
                acc[1].w = fmaf(f, y.w, acc[1].w);
            }
    }
    if constexpr (WARPS > 1) {
        s_acc[mine][lane] = acc[0];
        s_acc[mine][32 + lane] = acc[1];
        if (lane == 0) s_sum[mine] = sum;
        __syncthreads();
        if (mine) return;
        for (int w = 1; w < WARPS; ++w) {
            sum += s_sum[w];
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const float4 y = s_acc[w][v * 32 + lane];
                acc[v].x += y.x, acc[v].y += y.y, acc[v].z += y.z, acc[v].w += y.w;
            }
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint64_t tok = sg.query_begin + row / a.group;
    const uint32_t qh = head * a.group + row % a.group;
    unsigned char* dst = static_cast<unsigned char*>(a.out) + (tok * a.ots + qh * a.ohs) * sizeof(T);
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const uint32_t c = lane * 4 + v * 128;
        if (c >= a.d) continue;
        const float4 x = acc[v];
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dst + c * 2) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
        else *reinterpret_cast<float4*>(dst + c * 4) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    }
    if (a.lse && lane == 0) a.lse[tok * a.n_heads + qh] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * LN2;
}

}  // namespace
uint64_t cache_blocks_of(const CacheSeg& s, uint32_t group, uint32_t mb) { return ((uint64_t)s.n_queries * group + mb - 1) / mb; }
void cache_cut(CacheWork* w, uint32_t group, uint32_t mb, uint32_t kt, uint32_t most, uint32_t cluster) {
    w->items = w->blocks = 0;
    w->chunks = 1;
    for (CacheSeg& c : w->segs) {
        const uint32_t tiles = std::max(1u, (uint32_t)(((uint64_t)c.n_rows + kt - 1) / kt));
        const uint64_t blocks = cache_blocks_of(c, group, mb);
        c.n_chunks = cluster ? cluster : (tiles + most - 1) / most;
        c.chunk_tiles = (tiles + c.n_chunks - 1) / c.n_chunks;
        if (!cluster) c.n_chunks = (tiles + c.chunk_tiles - 1) / c.chunk_tiles;
        c.item_begin = (uint32_t)w->items;
        c.block_begin = (uint32_t)w->blocks;
        w->items += blocks * c.n_chunks;
        if (c.n_chunks > 1 && !cluster) w->blocks += blocks;
        w->chunks = std::max(w->chunks, c.n_chunks);
    }
}
// The longest run of tiles of an item.  In units of a tile's time: what fits on the GPU at once takes as long as its longest item, more than that the mean load
// and half an item at the end; an item costs about four tiles to begin, joining about three and a little for every part.
// *cluster: how many CTAs share a block of query rows and join their sums through each other's shared memory, where that takes less time than a second kernel (0: none do).
// One token over 512 rows: 6.5 us by a cluster, 8.0 by a second kernel; 8 x 4096 rows 26.2 and 28.7; 1 x 2048, where more than eight parts are worth it, 9.1 and 8.5.
static uint32_t longest_run(const CacheWork& w, uint32_t group, uint32_t mb, uint32_t kt, uint32_t n_kv, uint32_t d, uint32_t slots, uint32_t* cluster) {
    uint32_t most = 1;
    double total = 0.0;
    for (const CacheSeg& c : w.segs) {
        const uint32_t tiles = std::max(1u, (uint32_t)(((uint64_t)c.n_rows + kt - 1) / kt));
        most = std::max(most, tiles);
        total += (double)cache_blocks_of(c, group, mb) * tiles * n_kv;
    }
    uint32_t best = most;
    double best_time = 1e300;
    for (uint32_t run = most;; run = std::min(run - 1, run * 7 / 8)) {
        double items = 0.0;
        for (const CacheSeg& c : w.segs) {
            const uint32_t tiles = std::max(1u, (uint32_t)(((uint64_t)c.n_rows + kt - 1) / kt));
            items += (double)cache_blocks_of(c, group, mb) * ((tiles + run - 1) / run) * n_kv;
        }
        if (run < most && cache_part_bytes((uint64_t)items, 1, mb, d) > CACHE_PARTS_MOST) break;  // (items: of all KV heads)
        const double time = (items <= slots ? run : total / slots + 0.5 * run) + 4.0 * std::ceil(items / slots) +
                            (run < most ? 3.0 + 0.05 * ((most + run - 1) / run) : 0.0);
        if (time < best_time) best_time = time, best = run;
        if (run <= 2) break;
    }
    *cluster = 0;
    for (uint32_t cl = 2; cl <= 8; cl *= 2) {
        double items = 0.0;
        for (const CacheSeg& c : w.segs) items += (double)cache_blocks_of(c, group, mb) * cl * n_kv;
        const uint32_t run = (most + cl - 1) / cl;
        const double time = (items <= slots ? run : total / slots + 0.5 * run) + 4.0 * std::ceil(items / slots) + 0.5;
        if (time < best_time) best_time = time, *cluster = cl;
    }
    return best;
}

// Joins the parts of the segments that were split: only they take part, their blocks of query rows are numbered through.
Status launch_cache_join(Ctx* c, CacheArgs a, int dtype, const CacheWork& w, uint32_t mb) {
    std::vector<CacheSeg> split;
    uint32_t rows = 0;
    for (const CacheSeg& s : w.segs)
        if (s.n_chunks > 1) {
            split.push_back(s);
            rows = std::max(rows, std::min(mb, s.n_queries * a.group));
        }
    CacheTable tab;
    SLHA_TRY(cache_table(c, split, &tab, &a.table));
    a.n_segs = (uint32_t)split.size();
    // four warps a row where it has many parts (131072 rows in 35 parts, scores not capped: 90 us in all with one warp, 84 with four; 64 x 4096 rows in 2 parts 177 with one, 180 with four)
    const uint32_t warps = w.chunks > 8 ? 4 : 1, at_once = JOIN_THREADS / 32 / warps, per = (rows + at_once - 1) / at_once;
    if (w.blocks * a.n_kv * per > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "attention over a cache: too many blocks of query rows");
    const dim3 grid((uint32_t)(w.blocks * a.n_kv * per));
    const bool bf = dtype == SLHA_B200_BF16;
    SLHA_CUDA(launch_behind(warps == 4 ? (bf ? cache_join_kernel<__nv_bfloat16, 4> : cache_join_kernel<float, 4>) : (bf ? cache_join_kernel<__nv_bfloat16, 1> : cache_join_kernel<float, 1>),
                            grid, dim3(JOIN_THREADS), 0, c->stream, a, tab, mb, per));
    count_launch();
    return Status();
}
Status cache_part_memory(CacheArgs* a, uint64_t items, uint32_t mb, CacheMemory* mem) {
    if (!items) return Status();
    const size_t rows = (size_t)items * a->n_kv * mb;
    void* p;
    SLHA_TRY(mem->get(pad256(rows * a->d * 4) + rows * 8, &p));
    a->part_o = (float*)p;
    a->part_ml = (float*)((char*)p + pad256(rows * a->d * 4));
    return Status();
}

namespace {
template <typename T, int D, int WM>
Status launch_class(Ctx* c, CacheArgs a, CacheWork w) {
    using S = Shape<T, D, WM>;
    const uint32_t slots = (uint32_t)sm_count(c->device) * S::CTAS;
    const uint32_t run = longest_run(w, a.group, S::MB, S::KT, a.n_kv, a.d, slots, &a.cluster);
    cache_cut(&w, a.group, S::MB, S::KT, run, a.cluster);
    if (w.items * a.n_kv > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "attention over a cache: too many blocks of query rows");
    CacheTable tab;
    SLHA_TRY(cache_table(c, w.segs, &tab, &a.table));
    a.n_segs = (uint32_t)w.segs.size();
    CacheMemory mem{c};
    SLHA_TRY(cache_part_memory(&a, w.blocks ? w.items : 0, S::MB, &mem));
    const size_t smem = a.tree ? S::SMEM_TREE : S::SMEM;
    SLHA_TRY((cache_smem<cache_attend_kernel<T, D, WM>>(c, S::SMEM_TREE)));
    g_cache_kernels |= SLHA_B200_CACHE_ATTEND;
    SLHA_CUDA(launch_cluster(cache_attend_kernel<T, D, WM>, dim3((uint32_t)(w.items * a.n_kv)), dim3(ATT_THREADS), smem, c->stream, std::max(a.cluster, 1u), a, tab));
    count_launch();
    if (w.blocks) SLHA_TRY(launch_cache_join(c, a, sizeof(T) == 2 ? SLHA_B200_BF16 : SLHA_B200_F32, w, S::MB));
    return mem.done();
}
template <typename T, int D>
Status launch_dim(Ctx* c, const CacheArgs& a, int wm, CacheWork w) {
    if constexpr (sizeof(T) == 2)
        if (wm == 2) return launch_class<T, D, 2>(c, a, std::move(w));
    return wm == 1 ? launch_class<T, D, 1>(c, a, std::move(w)) : launch_class<T, D, 4>(c, a, std::move(w));
}

}  // namespace

Status cache_table(Ctx* c, const std::vector<CacheSeg>& segs, CacheTable* inl, const CacheSeg** dev) {
    *dev = nullptr;
    if (segs.size() <= CACHE_TABLE) {
        std::copy(segs.begin(), segs.end(), inl->s);
        return Status();
    }
    void* p;
    SLHA_TRY(ctx_upload(c, segs.data(), segs.size() * sizeof(CacheSeg), &p));
    *dev = static_cast<const CacheSeg*>(p);
    return Status();
}

Status launch_attend_cache(Ctx* c, CacheArgs a, int dtype, const std::vector<SlhaB200Segment>& segs) {
    // Segments of at most 16, of at most 32 and of more query rows a KV head: a launch each, so that a batch of decoded tokens beside a prompt keeps
    // the kernel that suits it.  8 KV heads of 128 dimensions, us in blocks of 16, 32, 64 query rows and with the kernel for many (whose tensor cores take 128 rows at a time):
    //   bfloat16, 16 x 8192 rows: 4 query rows 82, 100, 138, 116; 16: 84, 104, 144, 120; 20: 140, 106, 145, 120; 32: 141, 107, 147, 119; 36: -, 194, 148, 120; 256: -, 724, 615, 140
    //             1 x 4096 rows: 4 query rows 10.0, 10.8, 12.4, 14.1; 20: 12.8, 13.5, 16.7, 16.2; 36: -, 15.6, 17.6, 16.5; 256: -, 35, 32, 24
    //   float32, 4 x 2048 rows: 16 query rows 30, 78, 58; 32: 49, 81, 59; 64: 90, 93, 63 (blocks of 32 are never the quickest)
    CacheWork of[3];
    for (size_t i = 0; i < segs.size(); ++i) {
        const SlhaB200Segment& s = segs[i];
        if (s.n_queries == 0) continue;
        CacheSeg g{};
        g.row_begin = s.tile_begin;
        g.n_rows = s.n_tiles;
        g.query_begin = s.query_begin;
        g.n_queries = s.n_queries;
        g.base = s.index_base;
        g.seg = (uint32_t)i;
        const uint64_t rows = (uint64_t)s.n_queries * a.group;
        of[rows <= 16 || (rows <= 32 && dtype == SLHA_B200_F32) ? 0 : rows <= 32 ? 1 : 2].segs.push_back(g);
    }
    for (int k = 0; k < 3; ++k) {
        if (of[k].segs.empty()) continue;
        const int wm = 1 << k;
        if (k == 2 && dtype == SLHA_B200_BF16 && a.d <= 128 && a.scale > 0.0f) {
            bool taken;
            SLHA_TRY(launch_attend_wide(c, a, of[k], &taken));
            if (taken) continue;
        }
        if (dtype == SLHA_B200_BF16)
            SLHA_TRY(a.d <= 64 ? (launch_dim<__nv_bfloat16, 64>(c, a, wm, std::move(of[k])))
                     : a.d <= 128 ? (launch_dim<__nv_bfloat16, 128>(c, a, wm, std::move(of[k])))
                                  : (launch_dim<__nv_bfloat16, 256>(c, a, wm, std::move(of[k]))));
        else
            SLHA_TRY(a.d <= 64 ? (launch_dim<float, 64>(c, a, wm, std::move(of[k])))
                     : a.d <= 128 ? (launch_dim<float, 128>(c, a, wm, std::move(of[k])))
                                  : (launch_dim<float, 256>(c, a, wm, std::move(of[k]))));
    }
    return Status();
}

}  // namespace slha
