// The weight that each cached row received from a call's query tokens (slha_b200_observe_cache):
//   w_r = decay w_r + sum over tokens t and query heads g of exp(s_tgr - lse_tg),   s as in cache_attend.cu.
//
// With lse at hand a row's weight is a sum of its own column, so a CTA takes 128 keys (float32: 64) of one KV head, which stay in shared memory (and as operands in
// registers), and goes through the segment's query rows: every key is read once, no sum is shared between CTAs and their order is fixed.  Scores are summed four steps of the
// tensor cores at a time (see scores_of; 256 dimensions, 64 tokens on 16384 rows: 1.8e-7 off without, 8.2e-8 with, 25 us either way; 800 query rows of 128 on 32768 rows 339 us without, 354 with).
// With few query rows bound by the rows' bytes (8 KV heads of 128 dimensions, 8 x 8192 rows, 4 query rows: 40 us, 3.5 TB/s), with many by the products and exponentials (256 query
// rows over 32768 rows: 119 us).  bfloat16 rows of up to 128 dimensions have a kernel that takes 25 and 40 us for these (cache_observe_wide.cu).
#include <cuda_bf16.h>

#include <algorithm>

#include "cache.cuh"
#include "cache_mma.cuh"

namespace slha {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int OBS_THREADS = 128;

template <typename T, int D, int QB>
struct ObsShape {
    static constexpr int KT = sizeof(T) == 2 ? 128 : 64, KW = KT / 4, NT = KW / 8;
    static constexpr uint32_t K_BYTES = KT * D * sizeof(T), Q_BYTES = QB * D * sizeof(T);
    // keys | two blocks of queries | per key position, document, sum | per query row, twice: position, document, slope, lse
    static constexpr uint32_t META_AT = K_BYTES + 2 * Q_BYTES, ROW_AT = META_AT + 3 * KT * 4, SMEM = ROW_AT + 2 * 4 * QB * 4;
    static_assert(SMEM <= 227 * 1024, "shared memory of an SM");
    static constexpr bool HELD = sizeof(T) == 2 && D <= 128;  // a warp's keys as operands in registers
};

template <typename T, int D, int QB>
__global__ void __launch_bounds__(OBS_THREADS) cache_observe_kernel(const __grid_constant__ CacheArgs a, const __grid_constant__ CacheTable tab) {
    using S = ObsShape<T, D, QB>;
    using L = Tile<T, D>;
    dep_wait();
    extern __shared__ __align__(1024) unsigned char sm[];
    const uint32_t sb = smem_addr(sm);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const uint32_t head = blockIdx.x % a.n_kv, item = blockIdx.x / a.n_kv;
    const CacheSeg* table = a.table ? a.table : tab.s;
    const CacheSeg sg = table[cache_find(a.n_segs, item, [&](uint32_t i) { return table[i].item_begin; })];
    const uint32_t n = a.rows ? min(a.rows[sg.seg], sg.n_rows) : sg.n_rows;
    const uint32_t first = (item - sg.item_begin) * S::KT;
    if (first >= n) return;
    const uint32_t q_rows = sg.n_queries * a.group, ctx = n - min(n, sg.n_queries);
    const CacheSight sight{a.window_last, a.prefix ? a.prefix[sg.seg] : 0u, a.causal};
    const bool has_pos = a.row_pos, has_doc = a.row_doc, has_slope = a.slopes, has_cap = a.cap > 0.0f;
    const uint64_t entry = head * a.entry_hs + sg.row_begin;
    uint32_t* s_kp = reinterpret_cast<uint32_t*>(sm + S::META_AT);
    uint32_t* s_kd = s_kp + S::KT;
    float* s_sum = reinterpret_cast<float*>(s_kd + S::KT);
    uint32_t* s_rows = reinterpret_cast<uint32_t*>(sm + S::ROW_AT);

    const unsigned char* kb = static_cast<const unsigned char*>(a.keys) + (sg.row_begin * a.krs + head * a.khs) * sizeof(T);
#pragma unroll 8
    for (int i = 0; i < S::KT * L::PIECES / OBS_THREADS; ++i) {
        const int x = i * OBS_THREADS + tid, r = x / L::PIECES, c = x % L::PIECES;
        const bool there = first + r < n && c * 16 < (int)(a.d * sizeof(T));
        copy16(L::at(sb, r, c), there ? kb + (uint64_t)(first + r) * (a.krs * sizeof(T)) + c * 16 : kb, there);
    }
    const unsigned char* qbase = static_cast<const unsigned char*>(a.q);
    const auto fetch = [&](uint32_t b) {
        const uint32_t buf = b & 1, row0 = b * QB;
        if (row0 < q_rows) {
            for (int i = tid; i < QB * L::PIECES; i += OBS_THREADS) {
                const int r = i / L::PIECES, c = i % L::PIECES;
                const uint32_t row = row0 + r;
                const bool there = row < q_rows && c * 16 < (int)(a.d * sizeof(T));
                const uint64_t at = there ? (sg.query_begin + row / a.group) * a.qts + (head * a.group + row % a.group) * a.qhs : 0;
                copy16(L::at(sb + S::K_BYTES + buf * S::Q_BYTES, r, c), qbase + at * sizeof(T) + (there ? c * 16 : 0), there);
            }
            if (tid < QB) {
                const uint32_t row = min(row0 + tid, q_rows - 1), tok = row / a.group, qh = head * a.group + row % a.group;
                uint32_t* at = s_rows + buf * 4 * QB + tid;
                at[0] = a.q_pos ? a.q_pos[sg.query_begin + tok] : sg.base + ctx + tok;
                at[QB] = has_doc ? a.q_doc[sg.query_begin + tok] : 0u;
                at[2 * QB] = __float_as_uint(has_slope ? a.slopes[qh] : 0.0f);
                const float lse = a.lse_in[(uint64_t)(sg.query_begin + tok) * a.n_heads + qh];
                // a token that saw nothing, and rows behind the last: a weight of zero everywhere
                at[3 * QB] = __float_as_uint(lse == -INFINITY || row0 + tid >= q_rows ? INFINITY : lse);
            }
        }
        copy_commit();
    };
    fetch(0);
    float before = 0.0f;
    if (tid < S::KT) {
        const uint32_t row = min(first + tid, n - 1);
        s_kp[tid] = has_pos ? a.row_pos[entry + row] : sg.base + row;
        s_kd[tid] = has_doc ? a.row_doc[entry + row] : 0u;
        if (a.w_in) before = a.w_in[head * a.w_hs + sg.row_begin + row];
    }
    __syncthreads();
    uint32_t kpmin = 0xFFFFFFFFu, kpmax = 0u, kdmin = 0xFFFFFFFFu, kdmax = 0u;
    for (int i = lane; i < S::KT; i += 32) {
        kpmin = min(kpmin, s_kp[i]);
        kpmax = max(kpmax, s_kp[i]);
        kdmin = min(kdmin, s_kd[i]);
        kdmax = max(kdmax, s_kd[i]);
    }
    kpmin = __reduce_min_sync(0xFFFFFFFFu, kpmin);
    kpmax = __reduce_max_sync(0xFFFFFFFFu, kpmax);
    kdmin = __reduce_min_sync(0xFFFFFFFFu, kdmin);
    kdmax = __reduce_max_sync(0xFFFFFFFFu, kdmax);
    const bool whole = first + S::KT <= n;

    constexpr int KSTEPS = D / (sizeof(T) == 2 ? 16 : 8);
    uint32_t kf[S::HELD ? KSTEPS : 1][S::HELD ? S::NT * 2 : 1];
    float sum[S::NT][2];
#pragma unroll
    for (int i = 0; i < S::NT; ++i) sum[i][0] = sum[i][1] = 0.0f;
    const int key0 = warp * S::KW;
    for (uint32_t b = 0; b * QB < q_rows; ++b) {
        fetch(b + 1);
        copy_wait<1>();
        __syncthreads();
        const uint32_t sq = sb + S::K_BYTES + (b & 1) * S::Q_BYTES;
        const uint32_t* rows = s_rows + (b & 1) * 4 * QB;
        if constexpr (S::HELD)
            if (b == 0)
#pragma unroll
                for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
                    for (int i = 0; i < S::NT; i += 2) {
                        uint32_t x[4];
                        ldm4(x, L::at(sb, key0 + i * 8 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
                        kf[kk][2 * i] = x[0], kf[kk][2 * i + 1] = x[1], kf[kk][2 * i + 2] = x[2], kf[kk][2 * i + 3] = x[3];
                    }
        uint32_t qpmin = 0xFFFFFFFFu, qpmax = 0u, qdmin = 0xFFFFFFFFu, qdmax = 0u;
        for (int i = lane; i < QB; i += 32) {
            qpmin = min(qpmin, rows[i]);
            qpmax = max(qpmax, rows[i]);
            qdmin = min(qdmin, rows[QB + i]);
            qdmax = max(qdmax, rows[QB + i]);
        }
        qpmin = __reduce_min_sync(0xFFFFFFFFu, qpmin);
        qpmax = __reduce_max_sync(0xFFFFFFFFu, qpmax);
        qdmin = __reduce_min_sync(0xFFFFFFFFu, qdmin);
        qdmax = __reduce_max_sync(0xFFFFFFFFu, qdmax);
        const uint32_t near_ = kpmax < qpmin ? qpmin - kpmax : kpmin > qpmax ? kpmin - qpmax : 0u;
        const uint32_t far_ = max(qpmax > kpmin ? qpmax - kpmin : 0u, kpmax > qpmin ? kpmax - qpmin : 0u);
        const bool none = kdmin > qdmax || kdmax < qdmin || (kpmin >= sight.prefix && ((sight.causal && kpmin > qpmax) || near_ > sight.window_last));
        const bool all = whole && kdmin == kdmax && qdmin == qdmax && kdmin == qdmin &&
                         (kpmax < sight.prefix || ((!sight.causal || kpmax <= qpmin) && far_ <= sight.window_last));
        if (!none) {
#pragma unroll 1
            for (int r0 = 0; r0 < QB && b * QB + r0 < q_rows; r0 += 16) {
                float s[S::NT][4];
#pragma unroll
                for (int i = 0; i < S::NT; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
                AFrag<T> q;
                const auto load = [&](int kk) -> const AFrag<T>& {
                    q.template load<D>(sq, r0, kk, lane);
                    return q;
                };
                if constexpr (S::HELD) {
#pragma unroll
                    for (int k4 = 0; k4 < KSTEPS; k4 += 4) {
                        float part[S::NT][4] = {};
#pragma unroll
                        for (int kk = k4; kk < k4 + 4; ++kk) {
                            load(kk);
#pragma unroll
                            for (int i = 0; i < S::NT; ++i) mma_bf16(part[i], q.a, kf[kk][2 * i], kf[kk][2 * i + 1]);
                        }
#pragma unroll
                        for (int i = 0; i < S::NT; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[i][e] += part[i][e];
                    }
                } else {
                    scores_of<T, D, S::NT, 4>(s, load, sb, key0, lane);
                }
                const int ra = r0 + g;
                const float lse[2] = {__uint_as_float(rows[3 * QB + ra]), __uint_as_float(rows[3 * QB + ra + 8])};
                const uint32_t qp[2] = {rows[ra], rows[ra + 8]}, qd[2] = {rows[QB + ra], rows[QB + ra + 8]};
                const float sl[2] = {__uint_as_float(rows[2 * QB + ra]), __uint_as_float(rows[2 * QB + ra + 8])};
#pragma unroll
                for (int i = 0; i < S::NT; ++i)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int col = key0 + i * 8 + t4 * 2 + c;
                        const uint32_t kp = s_kp[col], kd = s_kd[col];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float x = s[i][h * 2 + c] * a.scale;
                            if (has_cap) x = a.cap * cache_tanh(x / a.cap);
                            if (has_slope) x = fmaf(-sl[h], (float)(kp <= qp[h] ? qp[h] - kp : kp - qp[h]), x);
                            if (!all && !(first + col < n && sight.sees(qp[h], kp) && kd == qd[h])) x = -INFINITY;
                            sum[i][c] += exp2_fast((x - lse[h]) * LOG2E);
                        }
                    }
            }
        }
        __syncthreads();
    }
    copy_wait<0>();
#pragma unroll
    for (int i = 0; i < S::NT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float x = sum[i][c];
            x += __shfl_xor_sync(0xFFFFFFFFu, x, 4);
            x += __shfl_xor_sync(0xFFFFFFFFu, x, 8);
            x += __shfl_xor_sync(0xFFFFFFFFu, x, 16);
            if (g == 0) s_sum[key0 + i * 8 + t4 * 2 + c] = x;
        }
    __syncthreads();
    if (tid < S::KT && first + tid < n) {
        const uint64_t at = head * a.w_hs + sg.row_begin + first + tid;
        a.w_out[at] = a.w_in && a.decay != 0.0f ? fmaf(a.decay, before, s_sum[tid]) : s_sum[tid];
    }
}

template <typename T, int D, int QB>
Status launch_observe_t(Ctx* c, CacheArgs a, std::vector<CacheSeg>& segs) {
    using S = ObsShape<T, D, QB>;
    uint64_t items = 0;
    for (CacheSeg& s : segs) {
        s.item_begin = (uint32_t)items;
        items += ((uint64_t)s.n_rows + S::KT - 1) / S::KT;
    }
    if (items * a.n_kv > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "slha_b200_observe_cache: too many rows");
    CacheTable tab;
    SLHA_TRY(cache_table(c, segs, &tab, &a.table));
    a.n_segs = (uint32_t)segs.size();
    SLHA_TRY((cache_smem<cache_observe_kernel<T, D, QB>>(c, S::SMEM)));
    g_cache_kernels |= SLHA_B200_CACHE_OBSERVE;
    SLHA_CUDA(launch_behind(cache_observe_kernel<T, D, QB>, dim3((uint32_t)(items * a.n_kv)), dim3(OBS_THREADS), S::SMEM, c->stream, a, tab));
    count_launch();
    return Status();
}
template <typename T>
Status launch_observe_d(Ctx* c, const CacheArgs& a, std::vector<CacheSeg>& segs, bool few) {
    if (a.d <= 64) return few ? launch_observe_t<T, 64, 16>(c, a, segs) : launch_observe_t<T, 64, 64>(c, a, segs);
    if (a.d <= 128) return few ? launch_observe_t<T, 128, 16>(c, a, segs) : launch_observe_t<T, 128, 64>(c, a, segs);
    return few ? launch_observe_t<T, 256, 16>(c, a, segs) : launch_observe_t<T, 256, 32>(c, a, segs);
}

}  // namespace

Status launch_observe_cache(Ctx* c, CacheArgs a, int dtype, const std::vector<SlhaB200Segment>& segs) {
    std::vector<CacheSeg> table;
    uint64_t most = 0;
    for (size_t i = 0; i < segs.size(); ++i) {
        const SlhaB200Segment& s = segs[i];
        if (s.n_tiles == 0) continue;
        CacheSeg g{};
        g.row_begin = s.tile_begin;
        g.n_rows = s.n_tiles;
        g.query_begin = s.query_begin;
        g.n_queries = s.n_queries;
        g.base = s.index_base;
        g.seg = (uint32_t)i;
        table.push_back(g);
        most = std::max(most, (uint64_t)s.n_queries * a.group);
    }
    if (table.empty()) return Status();
    if (dtype == SLHA_B200_BF16) {
        bool taken;
        SLHA_TRY(launch_observe_wide(c, a, table, most, &taken));
        if (taken) return Status();
    }
    return dtype == SLHA_B200_BF16 ? launch_observe_d<__nv_bfloat16>(c, a, table, most <= 16) : launch_observe_d<float>(c, a, table, most <= 16);
}

}  // namespace slha
