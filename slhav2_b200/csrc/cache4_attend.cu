// Exact attention over a cache of rows in 4 bits (slha_b200_attend_cache4, slha_b200_attend_tree4).
//
// As cache_attend.cu, the scores transposed: S^T = K Q^T and O^T = V^T P^T, so that what the codes stand for is the tensor cores' A operand, made in registers, and 8 query rows are its
// narrow side.  An A operand holds pairs along the contraction.  Keys: pairs along a row, as the codes lie; a byte becomes two float16 numbers by one conversion, one product with the block's scale makes
// their values (exact).  Values: pairs of neighbouring rows; two rows' nibbles are put together into bytes before the conversion, their two scales into a pair.  Queries are
// float16 numbers, scaled by a power of two a row so that the largest has an exponent of 14 (bfloat16 ones exact down to 2^-31 of the largest; float32 ones as two numbers, 22 bits).
// Weights are float16 too: against a reference that is the largest score less 8 in units of log 2, and stays until a score is more than 15 above it, the largest is 2^8 to 2^15, and weights lose bits
// below 2^-22 of it, 2^-33 of it at most.
//
// A warp takes 32 rows of a tile of 128 and all of a block's 8, 16 or 32 query rows, with a maximum and sums of its own; it copies its own rows (cp.async, one to three tiles ahead), so that a block's
// warps meet only where its list of tiles ends.
//
// What bounds it: the conversions, the products with scales and mma.sync take turns on one pipe (2.1, 1.9 and 9.9 cycles of an SM's quarter each, measured, and additive), 810 cycles for the 32 rows of
// 128 dimensions of a warp beside 1080 in all: 131072 rows of 8 KV heads (151 MB) 39 us, of which the loads alone take 25 to 28 and the arithmetic alone 30; with a cap 44 us = 3.5 TB/s, 48
// sequences of up to 9001 rows with positions and slopes 101 us = 3.4 TB/s.  A short call is bound by its launch and the first pass through the kernel's instructions: 512 rows 6.6 us; 32 query rows
// a block have three times the instructions, and 9 us more, so that blocks of 8 or 16 are taken where that counts.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <functional>

#include "cache4.cuh"
#include "cache_mma.cuh"

namespace slha {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int ATT_THREADS = 128, WARPS = ATT_THREADS / 32;
constexpr int ROUND = 256;  // tiles that are looked over at a time
constexpr int KT = 128, KW = KT / WARPS, MT = KW / 16;  // rows of a tile, a warp's, and its groups of 16

template <typename T, int D, int NT>
struct Shape4 {
    static constexpr int MB = 8 * NT, PARTS = sizeof(T) == 2 ? 1 : 2;  // query rows; float16 numbers of a query's element
    static constexpr int CB = D / 2, SB = D / 16;                      // bytes of a row: codes, scales
    static constexpr uint32_t CODES = KT * CB, SCALES = KT * SB, STAGE = 2 * (CODES + SCALES) + 2 * KT * 4;
    static constexpr int STAGES = D == 64 ? 4 : D == 128 ? (NT == 1 ? 2 : 3) : 2;
    static constexpr int PITCH = D + 8;  // floats of a query row on the way out
    static constexpr uint32_t LEAVE = (WARPS * MB * PITCH + MB * (D + 2)) * 4;
    // behind the stages (the sums leave through them) the queries in the order of B operands; per query row position, document, slope, token within the block, factor; per tile of a round its class
    static constexpr uint32_t Q_AT = STAGES * STAGE > LEAVE ? STAGES * STAGE : (LEAVE + 127) / 128 * 128, Q_PART = D / 16 * NT * 256;
    static constexpr uint32_t ROWS_AT = Q_AT + PARTS * Q_PART, LIST_AT = ROWS_AT + 5 * MB * 4, CLS_AT = LIST_AT + ROUND * 2, RANGE_AT = CLS_AT + ROUND, ML_AT = RANGE_AT + 32,
                              TREE_AT = ML_AT + 2 * WARPS * MB * 4;
    static constexpr uint32_t SMEM = TREE_AT, SMEM_TREE = TREE_AT + TREE_MOST * 8 + MB * (TREE_MOST / 8);
    static constexpr int CTAS = D == 256 || NT == 4 ? 2 : NT == 1 ? 4 : 3;  // of an SM
    static_assert(CTAS * (SMEM_TREE + 1024) <= 228 * 1024, "shared memory of an SM");
};

// 16-byte pieces of a row in shared memory change places so that eight lanes' reads of keys (two rows) and of values (four rows) lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t piece_at(uint32_t row, uint32_t piece) {
    if constexpr (D == 64) return row * 32 + piece * 16;
    else if constexpr (D == 128) return row * 64 + ((piece ^ ((row >> 1) & 2)) << 4);
    else return row * 128 + ((piece ^ (((row & 1) ? 3 : 0) | (row & 4))) << 4);
}
// Row of a group of 8 that stands in place x of a tensor core tile.
__device__ __forceinline__ uint32_t row_of(uint32_t x) { return (x & 4) | (x & 1) << 1 | ((x >> 1 ^ x) & 1); }

// cp.async of N bytes, of which the first `there` are read and the others zeros
template <int N>
__device__ __forceinline__ void copy_some(uint32_t dst, const void* src, uint32_t there) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;\n" ::"r"(dst), "l"(src), "r"(there), "n"(N) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t x) { return make_float2(__half2float(__ushort_as_half((uint16_t)x)), __half2float(__ushort_as_half((uint16_t)(x >> 16)))); }
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t byte_pair(uint32_t w, int b) { return b == 0 ? e2m1_pair<0>(w) : b == 1 ? e2m1_pair<1>(w) : b == 2 ? e2m1_pair<2>(w) : e2m1_pair<3>(w); }

// (not in line: few scores come to it)
__device__ __noinline__ float tanh_far(float x) { return tanhf(x); }

template <typename T, int D, int NT>
__global__ void __launch_bounds__(ATT_THREADS, Shape4<T, D, NT>::CTAS) cache4_attend_kernel(const __grid_constant__ CacheArgs a, const __grid_constant__ Rows4 in4, const __grid_constant__ CacheTable tab) {
    using S = Shape4<T, D, NT>;
    dep_wait();
    extern __shared__ __align__(1024) unsigned char sm[];
    const uint32_t sb = smem_addr(sm);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
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
    float* s_factor = reinterpret_cast<float*>(s_tok + S::MB);
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
    __syncthreads();
    const CacheRanges qr{s_range[0], s_range[1], s_range[2], s_range[3]};
    // The block's query rows into shared memory, a warp each (rows behind the last: zeros; they are not written).
    const auto take_queries = [&]() {
        constexpr int CHUNKS = D / 128 > 0 ? D / 128 : 1, AT_ONCE = S::MB / WARPS < 4 ? S::MB / WARPS : 4;  // chunks of 4 elements a lane; rows whose loads are under way together
        const unsigned char* qbase = static_cast<const unsigned char*>(a.q);
#pragma unroll 1
        for (int r0 = warp * AT_ONCE; r0 < S::MB; r0 += WARPS * AT_ONCE) {
            float x[AT_ONCE][CHUNKS][4];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                const uint32_t row = row0 + r0 + j;
                const uint64_t at = row < q_rows ? (sg.query_begin + row / a.group) * a.qts + (head * a.group + row % a.group) * a.qhs : 0;
#pragma unroll
                for (int i = 0; i < CHUNKS; ++i) {
                    const uint32_t d = (lane + i * 32) * 4;
                    float(&y)[4] = x[j][i];
                    y[0] = y[1] = y[2] = y[3] = 0.0f;
                    if (row < q_rows && d < a.d) {
                        if constexpr (sizeof(T) == 2) {
                            const uint2 w = *reinterpret_cast<const uint2*>(qbase + (at + d) * 2);
                            y[0] = __uint_as_float(w.x << 16), y[1] = __uint_as_float(w.x & 0xFFFF0000u), y[2] = __uint_as_float(w.y << 16), y[3] = __uint_as_float(w.y & 0xFFFF0000u);
                        } else {
                            const float4 w = *reinterpret_cast<const float4*>(qbase + (at + d) * 4);
                            y[0] = w.x, y[1] = w.y, y[2] = w.z, y[3] = w.w;
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                const int r = r0 + j;
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) most = max(most, __float_as_uint(x[j][i][e]) & 0x7FFFFFFFu);
                most = __reduce_max_sync(0xFFFFFFFFu, most);
                // 2^k with k = 14 less the exponent of the largest; 1 where one is not finite
                const int k = most >= 0x7F800000u ? 0 : min(14 - (int)(max(most >> 23, 1u) - 127u), 126);
                const float up = __uint_as_float((uint32_t)(127 + k) << 23);
                if (lane == 0) s_factor[r] = __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
                for (int i = 0; i < CHUNKS; ++i) {
                    const uint32_t d = (lane + i * 32) * 4;
                    if (d >= D) continue;
                    const uint32_t to = S::Q_AT + ((d % (D / 4) / 4 * NT + r / 8) * 32 + r % 8 * 4 + d / (D / 4)) * 8;
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = x[j][i][e] * up;
                    const uint32_t h0 = pack_f16(v[0], v[1]), h1 = pack_f16(v[2], v[3]);
                    *reinterpret_cast<uint2*>(sm + to) = make_uint2(h0, h1);
                    if constexpr (S::PARTS == 2) {
                        const float2 f0 = unpack_f16(h0), f1 = unpack_f16(h1);
                        *reinterpret_cast<uint2*>(sm + to + S::Q_PART) = make_uint2(pack_f16(v[0] - f0.x, v[1] - f0.y), pack_f16(v[2] - f1.x, v[3] - f1.y));
                    }
                }
            }
        }
    };
    const auto tile_class = [&](const CacheRanges& k, uint32_t last) { return cache_tile_class(k, qr, sight, a.tree && last >= ctx, last < n); };

    // o[m]: elements 2 m and 2 m + 1 of the lane's D / 8 from g D / 8 on, of query rows 8 nt + 2 t4 and the next
    float o[D / 16][NT][4], m[NT][2], l[NT][2], factor[NT][2];
    const float to_log2 = a.cap > 0.0f ? a.scale / a.cap : a.scale * LOG2E, cap2 = a.cap * LOG2E;
    const bool has_cap = a.cap > 0.0f, has_slope = a.slopes;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) m[nt][c] = -INFINITY, l[nt][c] = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.0f;

    const uint32_t tiles = (n + KT - 1) / KT, tile_end = min(tiles, (chunk + 1) * sg.chunk_tiles);
    const unsigned char* codes[2] = {in4.codes[0] + sg.row_begin * in4.crs + head * in4.chs, in4.codes[1] + sg.row_begin * in4.crs + head * in4.chs};
    const unsigned char* scales[2] = {in4.scales[0] + sg.row_begin * in4.srs + head * in4.shs, in4.scales[1] + sg.row_begin * in4.srs + head * in4.shs};
    for (uint32_t r0 = chunk * sg.chunk_tiles; r0 < tile_end; r0 += ROUND) {
        const uint32_t in_round = min((uint32_t)ROUND, tile_end - r0);
        // which of the round's tiles are visited
        if (arrays) {
            for (uint32_t j = warp; j < in_round; j += WARPS) {
                const uint32_t first = (r0 + j) * KT, last = first + KT - 1;
                CacheRanges k{0xFFFFFFFFu, 0u, has_doc ? 0xFFFFFFFFu : 0u, 0u};
#pragma unroll
                for (int e = 0; e < KT / 32; ++e) {
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
                const uint32_t first = (r0 + j) * KT, last = first + KT - 1;
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

        // A warp's rows of tile `at` of the list into stage `slot`, by the warp that will read them.  A lane copies the same piece of rows PER apart, and one row's scales.
        const auto fetch = [&](uint32_t at, uint32_t slot) {
            if (at < cnt) {
                constexpr int PIECES = S::CB / 16, PER = 32 / PIECES;
                const uint32_t st = sb + slot * S::STAGE, first = (r0 + (s_list[at] >> 1)) * KT, mine = first + tid;
                const uint32_t r = warp * KW + lane / PIECES, c = lane % PIECES, there = c * 32 < a.d ? min(16u, a.d / 2 - c * 16) : 0u;
                const uint32_t to = st + piece_at<D>(r, c), to_scale = st + 2 * S::CODES + tid * S::SB;
                const auto place = [&](int i) { return to + i * PER * S::CB ^ (D == 256 && i & 1 ? 64u : 0u); };  // piece_at's, PER rows on
                const uint64_t at_code = there ? (first + r) * in4.crs + c * 16 : 0, step = there ? PER * in4.crs : 0;
                if (mine - lane + KW <= n) {
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const unsigned char* p = codes[v] + at_code;
#pragma unroll
                        for (int i = 0; i < KW / PER; ++i, p += step) copy_some<16>(place(i) + v * S::CODES, p, there);
                        copy_some<S::SB>(to_scale + v * S::SCALES, scales[v] + mine * in4.srs, a.d / 16);
                    }
                } else {  // (rows behind the last: zeros)
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
#pragma unroll
                        for (int i = 0; i < KW / PER; ++i) {
                            const bool row = first + r + i * PER < n;
                            copy_some<16>(place(i) + v * S::CODES, row ? codes[v] + at_code + i * step : codes[v], row ? there : 0u);
                        }
                        copy_some<S::SB>(to_scale + v * S::SCALES, mine < n ? scales[v] + mine * in4.srs : scales[v], mine < n ? a.d / 16 : 0u);
                    }
                }
                if (arrays) {
                    const uint64_t at_entry = entry + min(mine, n - 1);
                    const uint32_t to = st + 2 * (S::CODES + S::SCALES) + tid * 4;
                    if (has_pos) copy4(to, a.row_pos + at_entry, true);
                    if (has_doc) copy4(to + KT * 4, a.row_doc + at_entry, true);
                }
            }
            copy_commit();
        };
#pragma unroll
        for (int i = 0; i < S::STAGES - 1; ++i) fetch(i, i);
        if (r0 == chunk * sg.chunk_tiles) {  // (while the first rows are on their way)
            take_queries();
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) factor[nt][c] = to_log2 * s_factor[nt * 8 + t4 * 2 + c];
        }
        uint32_t slot = 0, slot_next = S::STAGES - 1;
        for (uint32_t li = 0; li < cnt; ++li) {
            copy_wait<S::STAGES - 2>();
            __syncwarp();
            fetch(li + S::STAGES - 1, slot_next);
            const unsigned char* st = sm + slot * S::STAGE;
            slot = slot + 1 == S::STAGES ? 0 : slot + 1;
            slot_next = slot_next + 1 == S::STAGES ? 0 : slot_next + 1;
            const uint32_t what = s_list[li], first = (r0 + (what >> 1)) * KT;
            const bool all = what & 1;
            const uint32_t key0 = warp * KW;

            // scores: c of s[mt][nt] is row key0 + 16 mt + row_of(g) (c & 2: + 8) and query row 8 nt + 2 t4 + (c & 1)
            float s[MT][NT][4];
            {
                uint32_t w[MT][2][D / 32], sc[MT][2][D / 64 > 1 ? D / 128 : 1];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t r = key0 + mt * 16 + h * 8 + row_of(g);
                        if constexpr (D == 64) {
                            const uint2 x = *reinterpret_cast<const uint2*>(st + piece_at<D>(r, t4 >> 1) + (t4 & 1) * 8);
                            w[mt][h][0] = x.x, w[mt][h][1] = x.y;
                            const uint32_t b = st[2 * S::CODES + r * S::SB + t4] & 0x7F;
                            sc[mt][h][0] = e4m3_pair(b | b << 8);
                        } else {
#pragma unroll
                            for (int i = 0; i < D / 128; ++i) {
                                const uint4 x = *reinterpret_cast<const uint4*>(st + piece_at<D>(r, t4 * (D / 128) + i));
                                w[mt][h][4 * i] = x.x, w[mt][h][4 * i + 1] = x.y, w[mt][h][4 * i + 2] = x.z, w[mt][h][4 * i + 3] = x.w;
                                sc[mt][h][i] = e4m3_pair(*reinterpret_cast<const uint16_t*>(st + 2 * S::CODES + r * S::SB + (t4 * (D / 128) + i) * 2) & 0x7F7F);
                            }
                        }
                    }
                // (float32: the products of four steps at a time are added here, to the nearest: the tensor cores cut their sums off towards zero)
                constexpr int AT_ONCE = S::PARTS == 2 ? 4 : D / 16;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.0f;
#pragma unroll
                for (int k0 = 0; k0 < D / 16; k0 += AT_ONCE) {
                    float part[MT][NT][4] = {};
#pragma unroll
                    for (int kk = k0; kk < k0 + AT_ONCE; ++kk) {
                        uint32_t x[MT][4];
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                // a lane's elements 4 kk .. 4 kk + 3, of block kk / 4 of its D / 64
                                const uint32_t two = sc[mt][h][kk / 8], scale = D == 64 ? two : __byte_perm(two, two, kk / 4 % 2 ? 0x3232 : 0x1010);
                                x[mt][h] = mul_f16x2(byte_pair(w[mt][h][kk / 2], kk % 2 * 2), scale);
                                x[mt][h + 2] = mul_f16x2(byte_pair(w[mt][h][kk / 2], kk % 2 * 2 + 1), scale);
                            }
#pragma unroll
                        for (int p = S::PARTS - 1; p >= 0; --p)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const uint2 b = *reinterpret_cast<const uint2*>(sm + S::Q_AT + p * S::Q_PART + ((kk * NT + nt) * 32 + lane) * 8);
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) mma_f16(S::PARTS == 2 ? part[mt][nt] : s[mt][nt], x[mt], b.x, b.y);
                            }
                    }
                    if constexpr (S::PARTS == 2) {
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[mt][nt][e] += part[mt][nt][e];
                    }
                }
            }
            // in units of log 2
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float& x = s[mt][nt][e];
                        x *= factor[nt][e & 1];
                        if (has_cap) x = cap2 * (fabsf(x) <= 1.0f ? tanh_small(x) : tanh_far(x));
                    }
            uint32_t seen = 0;  // where not all are: a bit for each of the lane's rows and query rows
            if (!all || has_slope) {
                const uint32_t* kp_s = reinterpret_cast<const uint32_t*>(st + 2 * (S::CODES + S::SCALES));
                const auto place = [&](int x) { return key0 + (x >> 1) * 16 + (x & 1) * 8 + row_of(g); };  // of the lane's x-th row in the tile
                const auto position = [&](uint32_t col) {
                    const uint32_t row = first + col;
                    return has_pos ? kp_s[col] : a.tree && row >= ctx && row < n ? sg.base + ctx + s_depth[row - ctx] : sg.base + row;
                };
                if (has_slope) {
#pragma unroll
                    for (int x = 0; x < 2 * MT; ++x) {
                        const uint32_t kp = position(place(x));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const int r = nt * 8 + t4 * 2 + c;
                                float& y = s[x >> 1][nt][(x & 1) * 2 + c];
                                y = fmaf(-s_slope[r], cache_distance(kp, s_qp[r]), y);
                            }
                    }
                }
                if (!all) {
                    // (which of them are seen is found out in a loop: unrolled, it pushed the rest of the loop over the tiles out of the instruction cache)
#pragma unroll 1
                    for (int x = 0; x < 2 * MT; ++x) {
                        const uint32_t col = place(x), row = first + col, kp = position(col), kd = has_doc ? kp_s[KT + col] : 0u;
                        const bool drafted = a.tree && row >= ctx && row < n;
#pragma unroll 1
                        for (int i = 0; i < 2 * NT; ++i) {
                            const int r = (i >> 1) * 8 + t4 * 2 + (i & 1);
                            bool sees = row < n && sight.sees(s_qp[r], kp) && kd == s_qd[r];
                            if (drafted) sees = sees && (s_anc[s_tok[r] * (TREE_MOST / 32) + ((row - ctx) >> 5)] >> ((row - ctx) & 31) & 1u);
                            seen |= (uint32_t)sees << (x * 2 * NT + i);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 2 * MT; ++x)
#pragma unroll
                        for (int i = 0; i < 2 * NT; ++i)
                            if (!(seen >> (x * 2 * NT + i) & 1)) s[x >> 1][i >> 1][(x & 1) * 2 + (i & 1)] = -INFINITY;
                }
            }
            // Weights against a reference: once a score is more than 15 above it, and for a row's first scores, it becomes the largest so far less 8.  (Looking for the largest over the
            // lanes each time cost a tenth of the instructions, and their latency.)
            bool above = false;
            float top[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    top[nt][c] = s[0][nt][c];
#pragma unroll
                    for (int x = 1; x < 2 * MT; ++x) top[nt][c] = fmaxf(top[nt][c], s[x >> 1][nt][(x & 1) * 2 + c]);
                    above |= top[nt][c] - m[nt][c] > 15.0f;  // (the difference: exact where it counts, infinite for a row's first scores; m + 15 is rounded from sizes of 2^24 on)
                }
            if (__any_sync(0xFFFFFFFFu, above)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float grow[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float mx = top[nt][c];
                        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
                        float ref = mx - 8.0f;
                        if (mx - ref > 12.0f) ref = mx;  // (sizes of 2^27 and more, where steps are 16)
                        if (!(mx - m[nt][c] > 15.0f)) ref = m[nt][c];
                        grow[c] = ref == -INFINITY ? 1.0f : exp2_fast(m[nt][c] - ref);
                        m[nt][c] = ref;
                        l[nt][c] *= grow[c];
                    }
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][nt][e] *= grow[e & 1];
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float use = m[nt][c] == -INFINITY ? 0.0f : m[nt][c];
#pragma unroll
                    for (int x = 0; x < 2 * MT; ++x) {
                        float& y = s[x >> 1][nt][(x & 1) * 2 + c];
                        y = exp2_fast(y - use);
                        l[nt][c] += y;
                    }
                }
            // values
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                uint32_t p[S::PARTS][NT][2];  // B operands: rows 2 t4, 2 t4 + 1 (and + 8) of the 16, query row g
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t x = pack_f16(s[mt][nt][h * 2], s[mt][nt][h * 2 + 1]);
                        p[0][nt][h] = transpose8(x);
                        if constexpr (S::PARTS == 2) {
                            const float2 f = unpack_f16(x);
                            p[1][nt][h] = transpose8(pack_f16(s[mt][nt][h * 2] - f.x, s[mt][nt][h * 2 + 1] - f.y));
                        }
                    }
                uint32_t w[2][2][D / 64], sc[2][D / 64 > 2 ? 2 : 1], twos[2][D / 64 > 2 ? 2 : 1];  // [+ 8][even or odd elements], of pairs of rows
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t raw[2][D / 64], b[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t r = key0 + mt * 16 + h * 8 + row_of(2 * t4 + j);
                        const unsigned char* v = st + S::CODES;
                        const unsigned char* vs = st + 2 * S::CODES + S::SCALES + r * S::SB;
                        if constexpr (D == 64) {
                            raw[j][0] = *reinterpret_cast<const uint32_t*>(v + piece_at<D>(r, g >> 2) + (g & 3) * 4);
                            b[j] = vs[g >> 1];
                        } else if constexpr (D == 128) {
                            const uint2 x = *reinterpret_cast<const uint2*>(v + piece_at<D>(r, g >> 1) + (g & 1) * 8);
                            raw[j][0] = x.x, raw[j][1] = x.y;
                            b[j] = vs[g];
                        } else {
                            const uint4 x = *reinterpret_cast<const uint4*>(v + piece_at<D>(r, g));
                            raw[j][0] = x.x, raw[j][1] = x.y, raw[j][2] = x.z, raw[j][3] = x.w;
                            b[j] = *reinterpret_cast<const uint16_t*>(vs + 2 * g);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < (D / 64 > 2 ? 2 : 1); ++i) {
                        twos[h][i] = __byte_perm(b[0], b[1], i ? 0x4451 : 0x4440) & 0x7F7F;
                        sc[h][i] = e4m3_pair(twos[h][i]);
                    }
#pragma unroll
                    for (int i = 0; i < D / 64; ++i) {
                        w[h][0][i] = (raw[0][i] & 0x0F0F0F0Fu) | (raw[1][i] << 4 & 0xF0F0F0F0u);
                        w[h][1][i] = (raw[0][i] >> 4 & 0x0F0F0F0Fu) | (raw[1][i] & 0xF0F0F0F0u);
                    }
                }
                // Where some rows are not seen, they may hold anything: a weight of zero does not keep a NaN out of the sum.  Its block's scale becomes zero, and the sums of the query rows
                // that see it become NaN, whatever is left of its weight.
                uint32_t nan[2][D / 64 > 2 ? 2 : 1];
                bool odd = false;
                if (!all) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < (D / 64 > 2 ? 2 : 1); ++i) {
                            nan[h][i] = ((twos[h][i] & 0xFF) == 0x7F ? 0x3C00u : 0u) | (twos[h][i] >> 8 == 0x7F ? 0x3C000000u : 0u);
                            odd |= nan[h][i] != 0;
                        }
                }
                if (!all && __any_sync(0xFFFFFFFFu, odd)) {
                    uint32_t one[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t two = seen >> ((2 * mt + h) * 2 * NT + 2 * nt);
                            one[nt][h] = transpose8((two & 1 ? 0x3C00u : 0u) | (two & 2 ? 0x3C000000u : 0u));
                        }
#pragma unroll
                    for (int i = 0; i < (D / 64 > 2 ? 2 : 1); ++i) {
                        const uint32_t x[4] = {nan[0][i], nan[0][i], nan[1][i], nan[1][i]};
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float count[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma_f16(count, x, one[nt][0], one[nt][1]);
#pragma unroll
                            for (int md = i * 8; md < (D / 64 > 2 ? i * 8 + 8 : D / 16); ++md)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (count[e] != 0.0f) o[md][nt][e] = NAN;
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (nan[h][i] & 0xFFFF) sc[h][i] &= 0xFFFF0000u;
                            if (nan[h][i] >> 16) sc[h][i] &= 0xFFFFu;
                        }
                    }
                }
#pragma unroll
                for (int md = 0; md < D / 16; ++md) {
                    uint32_t x[4];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 2; ++j) x[h * 2 + j] = mul_f16x2(byte_pair(w[h][j][md / 4], md % 4), sc[h][md / 8]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if constexpr (S::PARTS == 2) {  // (as for the scores)
                            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma_f16(part, x, p[1][nt][0], p[1][nt][1]);
                            mma_f16(part, x, p[0][nt][0], p[0][nt][1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[md][nt][e] += part[e];
                        } else {
                            mma_f16(o[md][nt], x, p[0][nt][0], p[0][nt][1]);
                        }
                    }
                }
            }
        }
        copy_wait<0>();
        __syncthreads();  // (the next round's list and stages)
    }

    // the warps' maxima and sums meet, then their rows of sums
    float* s_m = reinterpret_cast<float*>(sm + S::ML_AT);  // [warp][query row]
    float* s_l = s_m + WARPS * S::MB;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float& x = l[nt][c];
            x += __shfl_xor_sync(0xFFFFFFFFu, x, 4);
            x += __shfl_xor_sync(0xFFFFFFFFu, x, 8);
            x += __shfl_xor_sync(0xFFFFFFFFu, x, 16);
            if (g == 0) s_m[warp * S::MB + nt * 8 + t4 * 2 + c] = m[nt][c], s_l[warp * S::MB + nt * 8 + t4 * 2 + c] = x;
        }
    __syncthreads();
    float* s_o = reinterpret_cast<float*>(sm);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = nt * 8 + t4 * 2 + c;
            float top = s_m[r];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) top = fmaxf(top, s_m[w * S::MB + r]);
            const bool none = m[nt][c] == -INFINITY;
            const float f = none ? 0.0f : exp2_fast(m[nt][c] - top);
#pragma unroll
            for (int i = 0; i < D / 16; ++i)  // (pairs of elements of the lanes' parts in turn: side by side eight lanes' would lie in the same banks)
                *reinterpret_cast<float2*>(s_o + (warp * S::MB + r) * S::PITCH + (i * 8 + g) * 2) =
                    none ? make_float2(0.0f, 0.0f) : make_float2(o[i][nt][c] * f, o[i][nt][2 + c] * f);
        }
    __syncthreads();
    const bool whole = sg.n_chunks == 1, shared = cl > 1;
    const uint32_t used = min((uint32_t)S::MB, q_rows - row0);
    const float up = exp2f((float)in4.exponent[1]);
    const auto write = [&](uint32_t r, uint32_t c, const float4& x, float top, float sum) {
        const uint32_t row = row0 + r;
        const uint64_t tok = sg.query_begin + row / a.group;
        const uint32_t qh = head * a.group + row % a.group;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        unsigned char* dst = static_cast<unsigned char*>(a.out) + (tok * a.ots + qh * a.ohs + c) * sizeof(T);
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
        else *reinterpret_cast<float4*>(dst) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        if (a.lse && c == 0) a.lse[tok * a.n_heads + qh] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * LN2;
    };
    // of a cluster: the CTA's own sums, maxima and sums of weights for the others to read
    float* const s_own = s_o + WARPS * S::MB * S::PITCH;
    float* const s_own_m = s_own + S::MB * D;
    float* const s_own_l = s_own_m + S::MB;
    for (uint32_t i = tid; i < used * (D / 4); i += ATT_THREADS) {
        const uint32_t r = i / (D / 4), c = i % (D / 4) * 4;
        if (c >= a.d) continue;
        float top = s_m[r];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) top = fmaxf(top, s_m[w * S::MB + r]);
        float sum = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float mw = s_m[w * S::MB + r];
            sum += mw == -INFINITY ? s_l[w * S::MB + r] : s_l[w * S::MB + r] * exp2_fast(mw - top);  // (of scores that are all NaN: NaN, else zero)
            const float* from = s_o + (w * S::MB + r) * S::PITCH + (c % (D / 8) / 2 * 8 + c / (D / 8)) * 2;
            const float2 y = *reinterpret_cast<const float2*>(from), z = *reinterpret_cast<const float2*>(from + 16);
            x.x += y.x, x.y += y.y, x.z += z.x, x.w += z.y;
        }
        x.x *= up, x.y *= up, x.z *= up, x.w *= up;
        if (shared) {
            *reinterpret_cast<float4*>(s_own + r * D + c) = x;
            if (c == 0) s_own_m[r] = top, s_own_l[r] = sum;
        } else if (whole) {
            write(r, c, x, top, sum);
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
        const uint32_t r = i / (D / 4), c = i % (D / 4) * 4;
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
        write(r, c, x, top, sum);
    }
    cluster.sync();  // (the others have read this CTA's sums)
}

// Joins the parts of query rows whose segment's rows were split: WARPS warps a query row, each every WARPS-th part, eight at a time with their maxima and sums, so that nothing waits for what another
// load says; the warps' sums meet in shared memory, in the warps' order.  (131072 rows in 74 parts, one token: 44.0 us in all, 47.0 by two passes over the parts with four warps; 48 sequences in 2 to 6 parts 101.2 and 102.9.)
constexpr int JOIN_FLIGHT = 8;
template <typename T, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) cache4_join_kernel(const __grid_constant__ CacheArgs a, const __grid_constant__ CacheTable tab, uint32_t mb, uint32_t rows_of) {
    dep_wait();
    constexpr int ROWS = WARPS == 1 ? 4 : 1;  // of a block
    __shared__ float4 s_acc[WARPS > 1 ? WARPS : 1][64];
    __shared__ float2 s_ml[WARPS];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = WARPS == 1 ? 0 : warp;
    const uint32_t part = blockIdx.x % rows_of, at = blockIdx.x / rows_of, head = at % a.n_kv, qb = at / a.n_kv;
    const CacheSeg* table = a.table ? a.table : tab.s;
    const uint32_t seg = cache_find(a.n_segs, qb, [&](uint32_t i) { return table[i].block_begin; });
    const CacheSeg& sg = table[seg];
    const uint32_t block = qb - sg.block_begin, r = part * ROWS + (WARPS == 1 ? warp : 0), row = block * mb + r;
    if (r >= mb || row >= sg.n_queries * a.group) return;  // (with more than one warp a row: all of them)
    const uint64_t first = ((uint64_t)(sg.item_begin + block * sg.n_chunks) * a.n_kv + head) * mb + r, step = (uint64_t)a.n_kv * mb;
    float m = -INFINITY, sum = 0.0f;
    float4 acc[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
    const auto add = [](float4& x, float f, const float4& y) { x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w); };
    const auto times = [](float4& x, float f) { x.x *= f, x.y *= f, x.z *= f, x.w *= f; };
    for (uint32_t c0 = mine; c0 < sg.n_chunks; c0 += WARPS * JOIN_FLIGHT) {
        float2 ml[JOIN_FLIGHT];
        float4 x[JOIN_FLIGHT];
#pragma unroll
        for (int i = 0; i < JOIN_FLIGHT; ++i) {
            const uint32_t c = c0 + i * WARPS;
            const bool there = c < sg.n_chunks;
            ml[i] = there ? *reinterpret_cast<const float2*>(a.part_ml + (first + c * step) * 2) : make_float2(-INFINITY, 0.0f);
            x[i] = there && lane * 4 < a.d ? *reinterpret_cast<const float4*>(a.part_o + (first + c * step) * a.d + lane * 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < JOIN_FLIGHT; ++i) top = fmaxf(top, ml[i].x);
        const float keep = m == -INFINITY ? 0.0f : exp2_fast(m - top);
        if (m != -INFINITY) sum *= keep;  // (of scores that are all NaN: NaN, without a maximum)
        times(acc[0], keep);
        times(acc[1], keep);
        m = top;
#pragma unroll
        for (int i = 0; i < JOIN_FLIGHT; ++i) {
            const float f = ml[i].x == -INFINITY ? 0.0f : exp2_fast(ml[i].x - top);
            sum = fmaf(f, ml[i].y, sum);
            add(acc[0], f, x[i]);
        }
        if (a.d > 128)
#pragma unroll
            for (int i = 0; i < JOIN_FLIGHT; ++i) {
                const uint32_t c = c0 + i * WARPS;
                if (c >= sg.n_chunks || lane * 4 + 128 >= a.d) continue;
                add(acc[1], ml[i].x == -INFINITY ? 0.0f : exp2_fast(ml[i].x - top), *reinterpret_cast<const float4*>(a.part_o + (first + c * step) * a.d + lane * 4 + 128));
            }
    }
    if constexpr (WARPS > 1) {
        s_acc[mine][lane] = acc[0];
        s_acc[mine][32 + lane] = acc[1];
        if (lane == 0) s_ml[mine] = make_float2(m, sum);
        __syncthreads();
        if (mine) return;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_ml[w].x);
        sum = 0.0f;
        acc[0] = acc[1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float2 ml = s_ml[w];
            const float f = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - top);
            sum = fmaf(ml.x == -INFINITY ? 1.0f : f, ml.y, sum);
            add(acc[0], f, s_acc[w][lane]);
            if (a.d > 128) add(acc[1], f, s_acc[w][32 + lane]);
        }
        m = top;
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
    if (a.lse && lane == 0) a.lse[tok * a.n_heads + qh] = sum == 0.0f ? -INFINITY : (m + log2f(sum)) * LN2;
}

// How a call's segments are worked off: with blocks of 8 nt query rows, runs of at most `run` tiles an item, or each block by a cluster of `cluster` CTAs (0: none); and how long that takes, in us.
struct Plan4 {
    uint32_t run = 1, cluster = 0;
    double time = 1e300;
};
// By a model: a launch takes `fixed` (most of it the first pass through the kernel's instructions), a tile of 128 dimensions `tile` and `shared` more for each CTA that shares the SM, an item `item`
// of an SM's time to begin and end; a second kernel that joins parts 1.6 and a little for each part, a cluster 1.6.  What fits on the GPU at once takes as long as its longest item, more
// than that the mean load and 0.4 of an item.  The constants were fitted to 69 calls, each with every run and cluster and with all the blocks it can have: one to 64 sequences of 300 to
// 131072 rows, 4 to 512 query rows a KV head, 64 to 256 dimensions, both types.  What it picks takes 0.8 % longer than the best of each of those on the average, 8 % at most.  (One token over
// 4096 rows: 9.2 us in 128 items and a second kernel, 9.5 by 8 clusters of 8; 131072 rows 41.5 in 432 items, 43 in the 592 that it picks, for which it says 38, 49 in 824.  28 query rows over 1000 rows: 9.3 in blocks of 8, 10.8 of 16,
// 15.4 of 32; over 16 sequences of up to 8192 rows: 104, 77, 69.)
struct Cost4 {
    double tile, shared, item, fixed;
};
constexpr Cost4 COST_BF16[3] = {{0.51, 0.34, 0.95, 5.8}, {0.57, 0.49, 1.9, 6.8}, {0.84, 0.65, 4.5, 7.2}}, COST_F32[2] = {{0.62, 0.42, 1.24, 5.1}, {0.87, 0.6, 2.7, 5.6}};

Plan4 plan_of(const CacheWork& w, const CacheArgs& a, uint32_t mb, const Cost4& cost, uint32_t sms, uint32_t ctas) {
    // (64 segments and 60 runs to look at: 2 us of the host's time, 16 with divisions of whole numbers)
    std::vector<float> tiles, blocks;
    uint32_t most = 1;
    float total = 0.0f, all_blocks = 0.0f;
    for (const CacheSeg& c : w.segs) {
        const uint32_t n = std::max(1u, (uint32_t)(((uint64_t)c.n_rows + KT - 1) / KT));
        most = std::max(most, n);
        tiles.push_back((float)n);
        blocks.push_back((float)(cache_blocks_of(c, a.group, mb) * a.n_kv));
        total += tiles.back() * blocks.back();
        all_blocks += blocks.back();
    }
    const double slots = (double)sms * ctas, dims = a.d <= 64 ? 0.56 : a.d <= 128 ? 1.0 : 1.8;
    const auto time_of = [&](double items, uint32_t longest, uint32_t run) {
        const double load = std::min(std::max(std::ceil(items / sms), 1.0), (double)ctas), tile = (cost.tile + cost.shared * load) * dims;
        return (items <= slots ? longest : total / slots + 0.4 * run) * tile + cost.item * dims * load * std::max(items / slots, 1.0) + cost.fixed;
    };
    Plan4 best;
    std::vector<uint32_t> runs;
    for (uint32_t run = most; run >= 1; run = std::min(run - 1, run / 8 * 7 + run % 8 * 7 / 8)) runs.push_back(run);
    for (uint32_t of = 1; of <= 4 * ctas; ++of)  // runs that give each SM 1, 2, .. items
        for (uint32_t more = 0; more < 2; ++more) runs.push_back(std::min((uint32_t)std::min(total / sms / of, 4e9f) + more, most));
    std::sort(runs.begin(), runs.end(), std::greater<uint32_t>());
    runs.erase(std::unique(runs.begin(), runs.end()), runs.end());
    for (const uint32_t run : runs) {
        if (run < 1) continue;
        float items = 0.0f;
        const float up = (float)run - 0.5f, of_run = 1.0f / (float)run;  // (the half keeps a rounding from a whole number less)
        for (size_t i = 0; i < tiles.size(); ++i) items += blocks[i] * (float)(int)((tiles[i] + up) * of_run);
        if (run < most && cache_part_bytes((uint64_t)items, 1, mb, a.d) > CACHE_PARTS_MOST) continue;  // (items: of all KV heads)
        uint32_t longest = run;
        if (items <= slots) {  // (a segment's runs are evened out)
            float l = 1.0f;
            for (size_t i = 0; i < tiles.size(); ++i) {
                const float n = (float)(int)((tiles[i] + up) * of_run);
                l = std::max(l, (tiles[i] + n - 0.5f) / n);
            }
            longest = (uint32_t)l;
        }
        const uint32_t parts = (most - 1) / run + 1;
        const double time = time_of(items, longest, run) + (run < most ? 1.6 + 0.007 * parts : 0.0);
        if (time < best.time) best.time = time, best.run = run;
    }
    for (uint32_t cl = 2; cl <= 8; cl *= 2) {
        const uint32_t run = (most - 1) / cl + 1;
        const double time = time_of((double)all_blocks * cl, run, run) + 1.6 * std::max(all_blocks * cl / slots, 1.0);
        if (time < best.time) best.time = time, best.cluster = cl;
    }
    return best;
}

// The segments that were split, their blocks of query rows numbered through.
template <typename T>
Status launch_join4(Ctx* c, CacheArgs a, const CacheWork& w, uint32_t mb) {
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
    const int warps = w.chunks <= 8 ? 1 : w.chunks <= 32 ? 4 : 16;
    const uint32_t per = warps == 1 ? (rows + 3) / 4 : rows;
    if (w.blocks * a.n_kv * per > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "attention over a cache: too many blocks of query rows");
    const auto kernel = warps == 1 ? cache4_join_kernel<T, 1> : warps == 4 ? cache4_join_kernel<T, 4> : cache4_join_kernel<T, 16>;
    SLHA_CUDA(launch_behind(kernel, dim3((uint32_t)(w.blocks * a.n_kv * per)), dim3(warps == 16 ? 512 : 128), 0, c->stream, a, tab, mb, per));
    count_launch();
    return Status();
}

template <typename T, int D, int NT>
Status launch_class4(Ctx* c, CacheArgs a, const Rows4& r, CacheWork w, const Plan4& plan) {
    using S = Shape4<T, D, NT>;
    a.cluster = plan.cluster;
    cache_cut(&w, a.group, S::MB, KT, plan.run, plan.cluster);
    if (w.items * a.n_kv > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "attention over a cache: too many blocks of query rows");
    CacheTable tab;
    SLHA_TRY(cache_table(c, w.segs, &tab, &a.table));
    a.n_segs = (uint32_t)w.segs.size();
    CacheMemory mem{c};
    SLHA_TRY(cache_part_memory(&a, w.blocks ? w.items : 0, S::MB, &mem));
    const size_t smem = a.tree ? S::SMEM_TREE : S::SMEM;
    SLHA_TRY((cache_smem<cache4_attend_kernel<T, D, NT>>(c, S::SMEM_TREE)));
    g_cache_kernels |= SLHA_B200_CACHE_ATTEND4;
    SLHA_CUDA(launch_cluster(cache4_attend_kernel<T, D, NT>, dim3((uint32_t)(w.items * a.n_kv)), dim3(ATT_THREADS), smem, c->stream, std::max(a.cluster, 1u), a, r, tab));
    count_launch();
    if (w.blocks) SLHA_TRY(launch_join4<T>(c, a, w, S::MB));
    return mem.done();
}
template <typename T, int D>
Status launch_dim4(Ctx* c, const CacheArgs& a, const Rows4& r, int nt, CacheWork w, const Plan4& plan) {
    if constexpr (sizeof(T) == 2 && D <= 128)  // (32 query rows' sums fill the registers; for float32 blocks of 16 are never slower)
        if (nt == 4) return launch_class4<T, D, 4>(c, a, r, std::move(w), plan);
    return nt == 1 ? launch_class4<T, D, 1>(c, a, r, std::move(w), plan) : launch_class4<T, D, 2>(c, a, r, std::move(w), plan);
}

// Segments whose rows are laid out as rows of bfloat16 first, in order, as many at a time as CACHE4_ROWS_MOST holds (at least one).
Status attend_laid_out(Ctx* c, const CacheArgs& args, const Rows4& r, const std::vector<SlhaB200Segment>& segs) {
    constexpr uint64_t e = 2;
    const uint64_t row = 2 * args.n_kv * args.d * e;
    const uint32_t entries = (args.row_pos || args.row_doc) ? (args.entry_hs ? args.n_kv : 1) : 0;
    const uint64_t row_bytes = row + 4ull * entries * ((args.row_pos != nullptr) + (args.row_doc != nullptr));
    // a batch: segments first .. last, their rows one behind another
    struct Batch {
        size_t first, last;
        uint64_t rows;
    };
    std::vector<Batch> batches;
    uint64_t most = 0;
    for (size_t i = 0; i < segs.size(); ++i) {
        if (!segs[i].n_queries) continue;
        if (batches.empty() || (batches.back().rows + segs[i].n_tiles) * row_bytes > CACHE4_ROWS_MOST) batches.push_back({i, i, 0});
        batches.back().last = i;
        batches.back().rows += segs[i].n_tiles;
        most = std::max(most, batches.back().rows);
    }
    if (batches.empty()) return Status();
    CacheMemory mem{c};
    void* p;
    const uint64_t side = pad256(most * row / 2), entry = pad256(most * entries * 4ull);
    SLHA_TRY(mem.get(2 * side + 2 * entry + 256, &p));
    unsigned char* base = static_cast<unsigned char*>(p);
    for (const Batch& b : batches) {
        std::vector<SlhaB200Segment> of = segs, to = segs;
        uint64_t at = 0;
        for (size_t i = 0; i < segs.size(); ++i) {
            if (i < b.first || i > b.last || !segs[i].n_queries) {
                of[i].n_tiles = to[i].n_queries = 0;
                continue;
            }
            to[i].tile_begin = at;
            at += segs[i].n_tiles;
        }
        Rows4Args x{};
        x.in4 = r;
        x.in4.exponent[0] = 0;  // (in the scores' scale)
        const uint64_t hs = b.rows * args.d;  // [kv_head][row][d]
        for (int v = 0; v < 2; ++v) {
            x.rows.p[v] = base + v * side;
            x.rows.rs[v] = args.d * e;
            x.rows.hs[v] = hs * e;
        }
        x.counts = args.rows;
        x.pos = args.row_pos;
        x.doc = args.row_doc;
        x.to_pos = reinterpret_cast<uint32_t*>(base + 2 * side);
        x.to_doc = reinterpret_cast<uint32_t*>(base + 2 * side + entry);
        x.entry_hs = args.entry_hs;
        x.to_entry_hs = b.rows;
        x.entries = entries;
        x.n_kv = args.n_kv;
        x.d = args.d;
        // (where the order of rows is that of positions, and no prefix is seen from everywhere)
        x.seen_last = args.causal && !args.row_pos && !args.q_pos && !args.prefix && !args.tree ? args.window_last : 0xFFFFFFFFu;
        SLHA_TRY(launch_read_cache4(c, x, SLHA_B200_BF16, of, to));
        CacheArgs a = args;
        a.keys = x.rows.p[0];
        a.values = x.rows.p[1];
        a.krs = a.vrs = args.d;
        a.khs = a.vhs = hs;
        if (a.row_pos) a.row_pos = x.to_pos;
        if (a.row_doc) a.row_doc = x.to_doc;
        a.entry_hs = args.entry_hs ? b.rows : 0;
        SLHA_TRY(launch_attend_cache(c, a, SLHA_B200_BF16, to));
    }
    g_cache_kernels |= SLHA_B200_CACHE_LAID_OUT;
    return mem.done();
}

}  // namespace

Status launch_attend_cache4(Ctx* c, CacheArgs a, const Rows4& r, int dtype, const std::vector<SlhaB200Segment>& whole) {
    // Rows that the window of a segment's first token leaves behind are seen by none: where their number is known here, the segment begins behind them, so that the work is shared out by what is seen
    // (one token over 131072 rows, window 4096: 8.9 us, 20.0 where the table of all rows is shared out; 48 sequences of up to 9001, window 1000: 21.4 and 43.0).
    std::vector<SlhaB200Segment> segs = whole;
    if (a.causal && a.window_last != 0xFFFFFFFFu && !a.row_pos && !a.q_pos && !a.prefix && !a.tree && !a.rows)
        for (SlhaB200Segment& s : segs) {
            const uint32_t ctx = s.n_tiles - std::min(s.n_tiles, s.n_queries), behind = ctx - std::min(ctx, a.window_last);
            s.tile_begin += behind;
            s.n_tiles -= behind;
            s.index_base += behind;
        }
    // Segments of at most 8, 16, 64 and of more query rows a KV head: a launch each, so that decoded tokens beside a prompt keep the blocks that suit them.
    CacheWork of[4];
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
        of[rows <= 8 ? 0 : rows <= 16 ? 1 : rows <= 64 ? 2 : 3].segs.push_back(g);
    }
    const bool bf = dtype == SLHA_B200_BF16;
    const uint32_t sms = (uint32_t)sm_count(c->device);
    std::vector<SlhaB200Segment> rest;
    for (int k = 0; k < 4; ++k) {
        if (of[k].segs.empty()) continue;
        Plan4 plan;
        int nt = 1;
        for (int x = 0; x <= std::min(k, bf && a.d <= 128 ? 2 : 1); ++x) {
            const uint32_t ctas = a.d > 128 ? 2 : x == 0 ? 4 : x == 1 ? 3 : 2;  // (Shape4's)
            const Plan4 p = plan_of(of[k], a, 8u << x, bf ? COST_BF16[x] : COST_F32[x], sms, ctas);
            if (p.time < plan.time) plan = p, nt = 1 << x;
        }
        // What the kernel for many query rows takes: the rows laid out, and read again by it while it multiplies.  (16 sequences of 4096 rows, bfloat16, 128 dimensions, us: 64 query rows 120 against
        // 88 here, 96: 121 against 161; one of 8192 rows, 96: 29.3 and 29.2, 256: 36 and 53.)
        if (k >= 2 && bf && a.d <= 128 && a.scale > 0.0f) {
            double elements = 0.0, products = 0.0;
            for (const CacheSeg& g : of[k].segs) {
                const double rows = 2.0 * g.n_rows * a.n_kv * a.d;
                elements += rows;
                products += rows * g.n_queries * a.group;
            }
            if (16.0 + elements * 4.7e-7 + std::max(elements * 3.6e-7, products * 2e-9) < plan.time) {
                if (rest.empty()) {
                    rest = segs;
                    for (SlhaB200Segment& s : rest) s.n_queries = 0;
                }
                for (const CacheSeg& g : of[k].segs) rest[g.seg].n_queries = g.n_queries;
                continue;
            }
        }
        if (bf)
            SLHA_TRY(a.d <= 64 ? (launch_dim4<__nv_bfloat16, 64>(c, a, r, nt, std::move(of[k]), plan))
                     : a.d <= 128 ? (launch_dim4<__nv_bfloat16, 128>(c, a, r, nt, std::move(of[k]), plan))
                                  : (launch_dim4<__nv_bfloat16, 256>(c, a, r, nt, std::move(of[k]), plan)));
        else
            SLHA_TRY(a.d <= 64 ? (launch_dim4<float, 64>(c, a, r, nt, std::move(of[k]), plan))
                     : a.d <= 128 ? (launch_dim4<float, 128>(c, a, r, nt, std::move(of[k]), plan))
                                  : (launch_dim4<float, 256>(c, a, r, nt, std::move(of[k]), plan)));
    }
    return rest.empty() ? Status() : attend_laid_out(c, a, r, rest);
}

}  // namespace slha
