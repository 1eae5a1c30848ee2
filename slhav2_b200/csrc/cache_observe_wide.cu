// The weight that each cached row received, for bfloat16 rows of up to 128 dimensions and up to 512 query rows a KV head (the arithmetic is that of cache_observe.cu).
//
// Scores as S^T = K Q^T on tcgen05: a tile of 128 keys is the M side, so that a thread has a key's scores in its own TMEM lane and its weight is a sum over the thread's own
// columns: no sum crosses threads (with many query rows four threads share a key).  A CTA takes the queries of one KV head, which stay in shared memory, and a run of key tiles,
// each of which is read once (TMA, the tile behind which a segment ends by cp.async).  While one block of scores is summed, the next is multiplied.
// With few query rows bound by the rows' bytes (16 sequences of 5750 rows on the average after a decode step: 39 us, 5.0 TB/s), with many by one exponential a score and what surrounds it (256 query
// rows of 8 KV heads over 32768 rows: 41 us, 1.6e12 scores a second; the special-function units alone would take 15 us).
#include <cuda_bf16.h>

#include <algorithm>

#include "cache_tc.cuh"

namespace slha {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int KT = 128;

// FEW: up to 32 query rows, a thread a key, two CTAs an SM, blocks of scores in two places by turns.  MID: up to 256, four groups of 128 threads, each with a tile and a place of its
// own, so that no sum crosses threads and nobody waits for another group.  MANY: up to 512, four threads a key, two places by turns.
//
// MID wants four tiles at a time and a run of them behind those, and has one CTA an SM: FEW takes up to 32 query rows where an SM's share is 8 tiles or less, and up to 16 where runs for
// all SMs would be uneven; MANY takes more than 32 where that share is 4 or less.  Measured, 8 KV heads of 128 dimensions, us:
//   4 query rows, sequences: 64 x 1024 rows (runs of 8) FEW 31, MID 39, MANY 49; 1 x 8192 (4) 5.6, 6.0, 7.4; 8 x 8192 (28) 27, 25, 36; 16 of 2700 to 8192 35, 38
//   32 query rows: 64 x 1024 41, 47, 57; 32 x 4096 62, 54, 79; 8 x 8192 38, 27, 40
//   64 query rows: 1 x 4096 (2) MID 9.0, MANY 7.1; 1 x 16384 (7) 13.9, 14.9; 1 x 32768 (14) 16, 22; 256 query rows on 1 x 32768 41, 43
// and cache_observe.cu's kernel takes 40, 56 (4, 32 query rows on 8 x 8192), 39, 119 (64, 256 on 32768): it takes rows beyond 512 query rows, 128 dimensions, and float32.
enum { FEW = 0, MID = 1, MANY = 2 };
template <int D, int MODE>
struct Obs {
    static constexpr int HALVES = D / 64, ROWS = MODE == MANY ? 512 : MODE == MID ? 256 : 32, BLOCK = MODE == MANY ? 256 : MODE == MID ? 128 : 32;  // query rows in all, and of a product
    static constexpr int GROUPS = MODE == MID ? 4 : 1, PLACES = MODE == MID ? 4 : 2;
    static constexpr int SUMMERS = MODE == FEW ? 128 : 512, THREADS = SUMMERS + 64, MMA_WARP = SUMMERS / 32, FETCH_WARP = MMA_WARP + 1;
    static constexpr int STAGES = MODE == MANY ? 2 : MODE == MID ? 4 : (D == 64 ? 5 : 3);
    static constexpr uint32_t TILE = HALVES * HALF, Q_HALF = ROWS * 128, PLACE = MODE == FEW ? 64 : BLOCK, TMEM = PLACES * PLACE;  // columns of a place, and of all
    static constexpr uint32_t K_AT = HALVES * Q_HALF, ROW_AT = K_AT + STAGES * TILE;  // per query row: lse in units of log 2 (two parts), position, document, slope, distance
    static constexpr uint32_t SUM_AT = ROW_AT + 6 * ROWS * 4, BAR_AT = SUM_AT + (MODE == MANY ? 3 * KT * 4 : 0), SMEM = BAR_AT + 256 + 1024;
    static constexpr int CTAS = MODE == FEW ? 2 : 1;
    static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory of an SM");
};
enum { K_FULL = 0, K_FREE = 5, S_FULL = 10, S_FREE = 14, Q_FULL = 18, TMEM_WORD = 19, DONE = 20 };

// At the end of a block: no copy is under way, whoever gave up before.
__device__ __noinline__ void settle(uint32_t keys, uint32_t fills, uint32_t stages, uint32_t queries, uint32_t boxes) {
    bar_settle(keys, fills, stages);
    bar_settle(queries, boxes, 1);
}

struct ObsMaps {
    CUtensorMap k, q;
    uint32_t k_head_first, q_boxes;
};

template <int D, int MODE>
__global__ void __launch_bounds__(Obs<D, MODE>::THREADS, Obs<D, MODE>::CTAS)
    cache_observe_wide_kernel(const __grid_constant__ CacheArgs a, const __grid_constant__ ObsMaps maps, const __grid_constant__ CacheTable tab) {
    using S = Obs<D, MODE>;
    dep_wait();
    extern __shared__ unsigned char raw[];
    const uint32_t sb = (smem_addr(raw) + 1023u) & ~1023u;
    unsigned char* sm = raw + (sb - smem_addr(raw));
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
    const uint32_t head = blockIdx.x % a.n_kv, item = blockIdx.x / a.n_kv;
    const CacheSeg* table = a.table ? a.table : tab.s;
    const CacheSeg sg = table[cache_find(a.n_segs, item, [&](uint32_t i) { return table[i].item_begin; })];
    const uint32_t n = a.rows ? min(a.rows[sg.seg], sg.n_rows) : sg.n_rows;
    const uint32_t tiles = (n + KT - 1) / KT, first_tile = min(tiles, (item - sg.item_begin) * sg.chunk_tiles), end_tile = min(tiles, first_tile + sg.chunk_tiles);
    if (first_tile == end_tile) return;
    const uint32_t q_rows = sg.n_queries * a.group, ctx = n - min(n, sg.n_queries), blocks = (q_rows + S::BLOCK - 1) / S::BLOCK;
    const CacheSight sight{a.window_last, a.prefix ? a.prefix[sg.seg] : 0u, a.causal};
    const bool has_pos = a.row_pos, has_doc = a.row_doc, has_slope = a.slopes, has_cap = a.cap > 0.0f;
    const uint64_t entry = head * a.entry_hs + sg.row_begin;
    float* const s_hi = reinterpret_cast<float*>(sm + S::ROW_AT);
    float* const s_lo = s_hi + S::ROWS;
    uint32_t* const s_qp = reinterpret_cast<uint32_t*>(s_lo + S::ROWS);
    uint32_t* const s_qd = s_qp + S::ROWS;
    float* const s_slope = reinterpret_cast<float*>(s_qd + S::ROWS);
    float* const s_at = s_slope + S::ROWS;
    float* const s_sum = reinterpret_cast<float*>(sm + S::SUM_AT);
    const uint32_t bars = sb + S::BAR_AT;
    const auto bar = [&](int which) { return bars + which * 8; };
    // rows of a block of query rows, as columns: a multiple of 16
    // The tensor cores cut their sums off after each step of 16 elements, towards zero: eight steps of a score of 90 (8 once scaled) lose 1.3e-6 of its weight.  Where the columns
    // suffice a score is two sums, of 64 elements each, which halves that (8 x 8192 rows after a decode step: 1.1e-6 -> 4.1e-7).  With more query rows they are left as they are: the
    // losses of many scores partly make up for one another in a row's weight, and half the query rows a product cost more than that (256 query rows on 32768 rows: 3.3e-7 off and
    // 41.2 us, in halves 2.3e-7 and 45.9 us; the same in float32 products of the whole 1.7e-7 to 2.7e-7).
    constexpr uint32_t SECOND = S::PLACE / 2;
    const bool halved = D > 64 && MODE != MANY && q_rows <= SECOND;
    const auto columns = [&](uint32_t b) { return min((uint32_t)S::BLOCK, (q_rows - b * S::BLOCK + 31) / 32 * 32); };

    if (warp == S::FETCH_WARP) {
        if (lane == 0) {
            for (int i = 0; i < S::STAGES; ++i) bar_init(bar(K_FULL + i), 1), bar_init(bar(K_FREE + i), 1);
            for (int i = 0; i < S::PLACES; ++i) bar_init(bar(S_FULL + i), 1), bar_init(bar(S_FREE + i), S::SUMMERS / S::GROUPS);
            bar_init(bar(Q_FULL), 1);
            bar_init(bar(DONE), 1);
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
            if (maps.q_boxes && q_rows) {
                const uint32_t boxes = (q_rows + 31) / 32;
                bar_expect(bar(Q_FULL), boxes * 4096 * S::HALVES);
                for (uint32_t i = 0; i < boxes; ++i)
#pragma unroll
                    for (int h = 0; h < S::HALVES; ++h) tma_load(sb + h * S::Q_HALF + i * 4096, &maps.q, h * 64, head * a.group, sg.query_begin + i * (32 / a.group), bar(Q_FULL));
            }
        }
        __syncwarp();
    }
    if (warp == S::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(bar(TMEM_WORD)), "r"(S::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    const uint32_t near_pos = a.q_pos && sg.n_queries ? a.q_pos[sg.query_begin] : sg.base + ctx;  // distances are taken from here
    for (uint32_t r = tid; r < blocks * S::BLOCK; r += S::THREADS) {
        const uint32_t row = min(r, q_rows - 1), tok = row / a.group, qh = head * a.group + row - tok * a.group;
        const uint32_t p = a.q_pos ? a.q_pos[sg.query_begin + tok] : sg.base + ctx + tok;
        // a token that saw nothing, and columns behind the last row: no weight anywhere
        const float lse = a.lse_in[(uint64_t)(sg.query_begin + tok) * a.n_heads + qh], hi = lse * LOG2E;
        const bool none = r >= q_rows || lse == -INFINITY;
        s_hi[r] = none ? INFINITY : hi;
        s_lo[r] = none ? 0.0f : fmaf(lse, LOG2E, -hi);
        s_qp[r] = p;
        s_qd[r] = has_doc ? a.q_doc[sg.query_begin + tok] : 0u;
        s_slope[r] = has_slope ? a.slopes[qh] * LOG2E : 0.0f;
        s_at[r] = (float)((long long)p - (long long)near_pos);
        if (!maps.q_boxes)
            for (int c = 0; c < S::HALVES * 8; ++c) {
                const bool there = r < q_rows && c * 8 < (int)a.d;
                const uint64_t at = ((uint64_t)(sg.query_begin + tok) * a.qts + (uint64_t)qh * a.qhs + c * 8) * 2;
                copy16(sb + (c >> 3) * S::Q_HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4), static_cast<const unsigned char*>(a.q) + (there ? at : 0), there);
            }
    }
    copy_commit();
    copy_wait<0>();
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + S::BAR_AT + TMEM_WORD * 8);
    // positions and documents of all query rows
    CacheRanges qr{0xFFFFFFFFu, 0u, 0xFFFFFFFFu, 0u};
    for (uint32_t r = lane; r < blocks * S::BLOCK; r += 32) {
        qr.pmin = min(qr.pmin, s_qp[r]);
        qr.pmax = max(qr.pmax, s_qp[r]);
        qr.dmin = min(qr.dmin, s_qd[r]);
        qr.dmax = max(qr.dmax, s_qd[r]);
    }
    qr.pmin = __reduce_min_sync(0xFFFFFFFFu, qr.pmin);
    qr.pmax = __reduce_max_sync(0xFFFFFFFFu, qr.pmax);
    qr.dmin = __reduce_min_sync(0xFFFFFFFFu, qr.dmin);
    qr.dmax = __reduce_max_sync(0xFFFFFFFFu, qr.dmax);
    const bool apart = has_slope && qr.pmax - qr.pmin > DISTANCE_NEAR;  // (see cache_distance)
    // Tiles of which, by their place alone, no token sees a row are not read.
    const auto visited = [&](uint32_t j) {
        if (q_rows == 0) return false;
        const uint32_t first = j * KT, last = min(first + KT - 1, n - 1);
        return has_pos || cache_tile_class(CacheRanges{sg.base + first, sg.base + last, qr.dmin, qr.dmax}, qr, sight, false, true) != 0;
    };

    if (warp < S::SUMMERS / 32) {
        const uint32_t quarter = MODE == MANY ? warp >> 2 : 0, group = MODE == MID ? warp >> 2 : 0, k_row = (warp & 3) * 32 + lane;
        const float to_log2 = has_cap ? a.scale / a.cap : a.scale * LOG2E, cap2 = a.cap * LOG2E;
        const bool bent = has_cap || has_slope;
        bool alone = false;  // a wait ran out: this warp goes on with dot products of its own
        uint32_t use = 0;
        // what a key brings along, fetched while the tile before its own is summed
        uint32_t next_kp = 0, next_kd = 0;
        float next_w = 0.0f;
        const auto ahead = [&](uint32_t j) {
            const uint32_t row = j * KT + k_row, there = min(row, n - 1);
            next_kp = has_pos ? a.row_pos[entry + there] : sg.base + there;
            if (has_doc) next_kd = a.row_doc[entry + there];
            if (a.w_in && quarter == 0 && row < n) next_w = a.w_in[head * a.w_hs + sg.row_begin + row];
        };
        if (first_tile + group < end_tile) ahead(first_tile + group);
        for (uint32_t j = first_tile + group; j < end_tile; j += S::GROUPS) {
            const uint32_t row = j * KT + k_row, there = min(row, n - 1), kp = next_kp, kd = next_kd;
            const uint64_t at = head * a.w_hs + sg.row_begin + row;
            const float before = next_w, k_at = (float)((long long)kp - (long long)near_pos);
            if (j + S::GROUPS < end_tile) ahead(j + S::GROUPS);
            float sum = 0.0f;
            if (visited(j)) {
                // whether all query rows see the warp's keys
                const uint32_t far_ = max(qr.pmax > kp ? qr.pmax - kp : 0u, kp > qr.pmin ? kp - qr.pmin : 0u);
                const bool all = __all_sync(0xFFFFFFFFu, (!has_doc || (qr.dmin == qr.dmax && kd == qr.dmin)) && (kp < sight.prefix || ((!sight.causal || kp <= qr.pmin) && far_ <= sight.window_last)));
                for (uint32_t b = 0; b < blocks; ++b, ++use) {
                    const uint32_t cols = columns(b), buf = MODE == MID ? group : use & 1, r_from = b * S::BLOCK;
                    if (!alone) alone = !__all_sync(0xFFFFFFFFu, bar_wait(bar(S_FULL + buf), MODE == MID ? use & 1 : use >> 1 & 1));
                    tc_after();
                    for (uint32_t c0 = quarter * 16; c0 < cols && r_from + c0 < q_rows; c0 += MODE == MANY ? 64 : 16) {
                        uint32_t u[16];
                        float* s = reinterpret_cast<float*>(u);
                        __syncwarp();
                        if (!alone) {
                            const uint32_t from = tmem + ((uint32_t)(warp & 3) << 21) + buf * S::PLACE + c0;
                            tmem_ld16(from, u);
                            if (halved) {
                                uint32_t more[16];
                                tmem_ld16(from + SECOND, more);
#pragma unroll
                                for (int c = 0; c < 16; ++c) s[c] += __uint_as_float(more[c]);
                            }
                        } else {
#pragma unroll 1
                            for (int c = 0; c < 16; ++c) {
                                const uint32_t q = min(r_from + c0 + c, q_rows - 1), tok = q / a.group;
                                const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(a.q) + (uint64_t)(sg.query_begin + tok) * a.qts + (uint64_t)(head * a.group + q % a.group) * a.qhs;
                                const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(a.keys) + (sg.row_begin + there) * a.krs + head * a.khs;
                                float t = 0.0f;
                                for (uint32_t d = 0; d < a.d; ++d) t = fmaf(__bfloat162float(x[d]), __bfloat162float(k[d]), t);
#pragma unroll
                                for (int e = 0; e < 16; ++e)
                                    if (e == c) s[e] = t;
                            }
                        }
                        const uint32_t r0 = r_from + c0;
                        const bool edge = r0 + 16 > q_rows;  // (columns behind the last query row hold anything)
                        float part[2] = {0.0f, 0.0f};
#pragma unroll
                        for (int c = 0; c < 16; c += 4) {
                            if (edge && r0 + c >= q_rows) break;
                            const float4 hi = *reinterpret_cast<const float4*>(s_hi + r0 + c), lo = *reinterpret_cast<const float4*>(s_lo + r0 + c);
                            const float h4[4] = {hi.x, hi.y, hi.z, hi.w}, l4[4] = {lo.x, lo.y, lo.z, lo.w};
                            if (!bent && all && !edge) {
#pragma unroll
                                for (int e = 0; e < 4; ++e) part[e & 1] += exp2_fast(fmaf(s[c + e], to_log2, -h4[e]) - l4[e]);
                            } else {
                                const uint4 p4 = *reinterpret_cast<const uint4*>(s_qp + r0 + c), d4 = *reinterpret_cast<const uint4*>(s_qd + r0 + c);
                                const float4 sl = *reinterpret_cast<const float4*>(s_slope + r0 + c), qa = *reinterpret_cast<const float4*>(s_at + r0 + c);
                                const uint32_t qp[4] = {p4.x, p4.y, p4.z, p4.w}, qd[4] = {d4.x, d4.y, d4.z, d4.w};
                                const float slope[4] = {sl.x, sl.y, sl.z, sl.w}, q_at[4] = {qa.x, qa.y, qa.z, qa.w};
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    float x = (has_cap ? fmaf(cap2, cache_tanh(s[c + e] * to_log2), -h4[e]) : fmaf(s[c + e], to_log2, -h4[e])) - l4[e];
                                    x = exp2_fast(fmaf(-slope[e], apart ? cache_distance(qp[e], kp) : fabsf(q_at[e] - k_at), x));
                                    part[e & 1] += r0 + c + e < q_rows && (all || (sight.sees(qp[e], kp) && kd == qd[e])) ? x : 0.0f;
                                }
                            }
                        }
                        sum += part[0] + part[1];
                    }
                    tc_before();
                    bar_arrive(bar(S_FREE + buf));
                }
            }
            if constexpr (MODE == MANY) {  // a key's four sums meet
                if (quarter) s_sum[(quarter - 1) * KT + k_row] = sum;
                asm volatile("bar.sync 1, 512;\n" ::: "memory");
                if (!quarter) sum = (sum + s_sum[k_row]) + (s_sum[KT + k_row] + s_sum[2 * KT + k_row]);
                asm volatile("bar.sync 1, 512;\n" ::: "memory");
            }
            if (quarter == 0 && row < n) a.w_out[at] = a.w_in && a.decay != 0.0f ? fmaf(a.decay, before, sum) : sum;
        }
    } else if (warp == S::MMA_WARP) {
        uint32_t lead;
        asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(lead));
        if (lead && (q_rows == 0 || !maps.q_boxes || bar_wait(bar(Q_FULL), 0))) {
            uint32_t use = 0, step = 0;
            bool ok = true;
            const auto product = [&](uint32_t st, uint32_t b, uint32_t place) {
                const uint32_t k = sb + S::K_AT + st * S::TILE, q = sb + b * S::BLOCK * 128, idesc = wide_idesc(columns(b), false);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    mma_shared(tmem + place * S::PLACE + (halved && kk >= 4 ? SECOND : 0), desc_along(k + (kk >> 2) * HALF + (kk & 3) * 32), desc_along(q + (kk >> 2) * S::Q_HALF + (kk & 3) * 32), idesc,
                               kk > 0 && !(halved && kk == 4));
                tc_commit_to(bar(S_FULL + place));
            };
            if constexpr (MODE == MID) {
                uint32_t uses[4] = {0, 0, 0, 0};
                for (uint32_t j = first_tile; j < end_tile && ok; j += 4) {  // four tiles, a group's each; their first blocks, then their second ones
                    uint32_t stage[4];
                    for (uint32_t b = 0; b < blocks && ok; ++b)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            if (!ok || j + g >= end_tile || !visited(j + g)) continue;
                            if (b == 0) {
                                stage[g] = step % S::STAGES;
                                ok = bar_wait(bar(K_FULL + stage[g]), step / S::STAGES & 1);
                                ++step;
                            }
                            if (ok && uses[g]) ok = bar_wait(bar(S_FREE + g), (uses[g] - 1) & 1);
                            if (!ok) continue;
                            ++uses[g];
                            tc_after();
                            product(stage[g], b, g);
                            if (b + 1 == blocks) tc_commit_to(bar(K_FREE + stage[g]));
                        }
                }
            } else {
                for (uint32_t j = first_tile; j < end_tile && ok; ++j) {
                    if (!visited(j)) continue;
                    const uint32_t st = step % S::STAGES;
                    ok = bar_wait(bar(K_FULL + st), step / S::STAGES & 1);
                    for (uint32_t b = 0; b < blocks && ok; ++b, ++use) {
                        const uint32_t buf = use & 1;
                        if (use >= 2 && !bar_wait(bar(S_FREE + buf), (use >> 1) - 1 & 1)) {
                            ok = false;
                            break;
                        }
                        tc_after();
                        product(st, b, buf);
                    }
                    if (ok) tc_commit_to(bar(K_FREE + st));
                    ++step;
                }
            }
            tc_commit_to(bar(DONE));
            bar_wait(bar(DONE), 0);  // (no product is under way when TMEM is given back, whoever gave up before)
        }
        __syncwarp();
    } else {
        const unsigned char* kb = static_cast<const unsigned char*>(a.keys) + (sg.row_begin * a.krs + head * a.khs) * 2;
        constexpr int PIECES = S::HALVES * 8;
        uint32_t step = 0;
        for (uint32_t j = first_tile; j < end_tile; ++j) {
            if (!visited(j)) continue;
            const uint32_t st = step % S::STAGES, first = j * KT, dst = sb + S::K_AT + st * S::TILE, full = bar(K_FULL + st);
            if (step >= S::STAGES && !__all_sync(0xFFFFFFFFu, bar_wait(bar(K_FREE + st), step / S::STAGES - 1 & 1))) break;
            if (first + KT <= n) {
                if (lane == 0) {
                    const uint32_t row = (uint32_t)sg.row_begin + first;
                    bar_expect(full, S::TILE);
#pragma unroll
                    for (int h = 0; h < S::HALVES; ++h) tma_load(dst + h * HALF, &maps.k, h * 64, maps.k_head_first ? head : row, maps.k_head_first ? row : head, full);
                }
            } else {
                for (uint32_t i = lane; i < KT * PIECES; i += 32) {
                    const uint32_t r = i / PIECES, c = i % PIECES, row = first + r;
                    const bool there = row < n && c * 8 < a.d;
                    copy16(dst + (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4), there ? kb + (uint64_t)row * a.krs * 2 + c * 16 : kb, there);
                }
                copy_commit();
                copy_wait<0>();
                asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_arrive(full);
            }
            ++step;
        }
        settle(bar(K_FULL), step, S::STAGES, bar(Q_FULL), maps.q_boxes && q_rows ? 1 : 0);
        __syncwarp();
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == S::MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(S::TMEM) : "memory");
}

// How long runs of tiles may be: evenly shared by so many places, and so long that there is one for each place at most (`once`, unless the segments are too many or too short).
struct Runs {
    uint32_t even, fit;
    bool once;
    Runs(const std::vector<CacheSeg>& segs, uint32_t n_kv, uint64_t places) {
        uint64_t total = 0;
        uint32_t longest = 1;
        const auto tiles = [](const CacheSeg& s) { return (uint32_t)(((uint64_t)s.n_rows + KT - 1) / KT); };
        for (const CacheSeg& s : segs) {
            total += (uint64_t)tiles(s) * n_kv;
            longest = std::max(longest, tiles(s));
        }
        even = (uint32_t)std::min<uint64_t>(longest, (total + places - 1) / places);
        const auto fits = [&](uint32_t run) {
            uint64_t items = 0;
            for (const CacheSeg& s : segs) items += ((uint64_t)tiles(s) + run - 1) / run;
            return items * n_kv <= places;
        };
        fit = longest;
        once = fits(longest);
        for (uint32_t low = even; once && low < fit;) {  // (longer runs are never more)
            const uint32_t mid = low + (fit - low) / 2;
            if (fits(mid)) fit = mid;
            else low = mid + 1;
        }
    }
};

template <int D, int MODE>
Status launch_observe_wide_t(Ctx* c, CacheArgs a, std::vector<CacheSeg>& segs, const ObsMaps& maps) {
    using S = Obs<D, MODE>;
    // One run for each CTA that fits on the GPU at once, or of FEW, whose second CTA of an SM hides the first one's beginning and end, where such runs would be uneven (16 sequences of
    // 2700 to 8192 rows: 43 us, 39 in runs of two thirds) one and a half.
    const Runs r(segs, a.n_kv, (uint64_t)sm_count(c->device) * S::CTAS);
    const uint32_t run = MODE != FEW || r.fit <= std::max(4u, r.even + r.even / 10) ? r.fit : std::max(4u, r.even * 2 / 3);
    uint64_t items = 0;
    for (CacheSeg& s : segs) {
        const uint32_t tiles = (uint32_t)(((uint64_t)s.n_rows + KT - 1) / KT), parts = (tiles + run - 1) / run;
        s.chunk_tiles = (tiles + parts - 1) / parts;
        s.item_begin = (uint32_t)items;
        items += (tiles + s.chunk_tiles - 1) / s.chunk_tiles;
    }
    if (items * a.n_kv > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "slha_b200_observe_cache: too many rows");
    CacheTable tab;
    SLHA_TRY(cache_table(c, segs, &tab, &a.table));
    a.n_segs = (uint32_t)segs.size();
    constexpr auto kernel = cache_observe_wide_kernel<D, MODE>;
    SLHA_TRY((cache_smem<kernel>(c, S::SMEM)));
    g_cache_kernels |= MODE == FEW ? SLHA_B200_CACHE_OBSERVE_FEW : MODE == MID ? SLHA_B200_CACHE_OBSERVE_MID : SLHA_B200_CACHE_OBSERVE_MANY;
    SLHA_CUDA(launch_behind(kernel, dim3((uint32_t)(items * a.n_kv)), dim3(S::THREADS), S::SMEM, c->stream, a, maps, tab));
    count_launch();
    return Status();
}

}  // namespace

Status launch_observe_wide(Ctx* c, CacheArgs a, std::vector<CacheSeg> segs, uint64_t most_rows, bool* taken) {
    *taken = false;
    if (a.d > 128 || most_rows > 512) return Status();
    uint64_t rows = 1;
    for (const CacheSeg& s : segs) rows = std::max(rows, s.row_begin + s.n_rows);
    ObsMaps maps;
    if (!wide_map(&maps.k, a.keys, a.krs, a.khs, rows, a.n_kv, a.d, &maps.k_head_first)) return Status();
    maps.q_boxes = wide_row_map(&maps.q, a.q, a.qts, a.qhs, a);
    *taken = true;
    const Runs r(segs, a.n_kv, sm_count(c->device));
    const bool even = r.once && r.fit <= r.even + r.even / 5;
    const int mode = most_rows <= 32 && (r.even <= 8 || (most_rows <= 16 && !even)) ? FEW : most_rows <= 256 && (most_rows <= 32 || r.even > 4) ? MID : MANY;
    if (a.d <= 64)
        return mode == FEW ? launch_observe_wide_t<64, FEW>(c, a, segs, maps) : mode == MID ? launch_observe_wide_t<64, MID>(c, a, segs, maps) : launch_observe_wide_t<64, MANY>(c, a, segs, maps);
    return mode == FEW ? launch_observe_wide_t<128, FEW>(c, a, segs, maps) : mode == MID ? launch_observe_wide_t<128, MID>(c, a, segs, maps) : launch_observe_wide_t<128, MANY>(c, a, segs, maps);
}

}  // namespace slha
