// Removal of the cached rows that received the least weight (slha_b200_evict_cache).
//
// Two kernels.  The first, a CTA for each KV head of a segment, finds which min(n, budget) of the n rows stay: the budget-th largest of the rows' keys by
// radix selection (11 bits, 11, 10), equal keys by the lower row, and writes for each place below the budget the row that comes to it.  The
// second moves rows.  A kept row below the budget stays where it is, so in place only rows from beyond the budget move, into places that no row is read from.
//
// Bound by latency where caches are short (1100 rows, 1024 stay: 13.5 us, two launches and three passes over a few words) and by bytes where rows move: 8 prompts of up to 32768 rows
// into caches of 4096, tiles with them, 93 us, of which the selection is 39 (its words are read once, into shared memory; its warps wait most at the barriers between the passes)
// and the moving 55 (6.2 TB/s).
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "cache.cuh"

namespace slha {
namespace {

constexpr int SEL_THREADS = 1024, SEL_WARPS = SEL_THREADS / 32, SEL_BINS = 2048;
constexpr uint32_t SEL_HELD = 49152;  // keys that fit in shared memory

// weights in the order of unsigned numbers: pinned rows above all, NaN below all, -0 like 0
__device__ __forceinline__ uint32_t weight_key(float w, bool pinned) {
    if (pinned) return 0xFFFFFFFFu;
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// the sum of `x` over the threads before this one
__device__ __forceinline__ uint32_t scan_threads(uint32_t x, uint32_t* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t s = x;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, s, o);
        if (lane >= o) s += y;
    }
    if (lane == 31) sh[warp] = s;
    __syncthreads();
    return s - x + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? sh[lane] : 0u);
}

// A cluster of C CTAs has a KV head of a segment: a run of its rows each, in it a run a warp, in 128s a run of four a lane.
template <int C>
__global__ void __cluster_dims__(C, 1, 1) __launch_bounds__(SEL_THREADS) cache_select_kernel(const __grid_constant__ EvictArgs a, const __grid_constant__ CacheTable tab) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    dep_wait();
    extern __shared__ __align__(16) uint32_t s_key[];
    __shared__ uint32_t s_hist[SEL_BINS], s_scan[SEL_WARPS], s_found[3], s_last, s_warp[SEL_WARPS], s_all[3];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t which = blockIdx.x / C, rank_of = C > 1 ? cluster.block_rank() : 0u, at = which / a.n_kv, head = which % a.n_kv;
    const CacheSeg sg = (a.table ? a.table : tab.s)[at];
    const uint32_t n = a.rows ? min(a.rows[sg.seg], sg.n_rows) : sg.n_rows;
    const uint32_t budget = a.budget, stay = min(n, budget);
    uint32_t* source = a.places + (uint64_t)which * a.room;
    uint32_t* hole = a.holes + (uint64_t)which * a.room;
    uint32_t* wanted = a.source ? a.source + ((uint64_t)sg.seg * a.n_kv + head) * budget : nullptr;
    if (tid == 0 && rank_of == 0) a.stay[which] = stay;
    if (n <= budget) {
        for (uint32_t i = rank_of * SEL_THREADS + tid; i < n; i += C * SEL_THREADS) {
            source[i] = i;
            if (wanted) wanted[i] = i;
        }
        return;
    }
    const uint64_t entry = head * a.entry_hs + sg.row_begin;
    const float* w = a.w + head * a.w_hs + sg.row_begin;
    // this CTA's rows and this warp's (of the CTA's, counted from its first)
    const uint32_t run = (n + C * SEL_WARPS * 128 - 1) / (C * SEL_WARPS * 128) * 128, base = min(n, rank_of * SEL_WARPS * run), own = min(n, base + SEL_WARPS * run) - base;
    const uint32_t from = min(own, warp * run), to = min(own, from + run);
    const auto position = [&](uint32_t i) { return a.pos ? a.pos[entry + base + i] : sg.base + base + i; };
    constexpr int FLIGHT = 8;  // loads that a thread has under way
    const bool held = own <= SEL_HELD, kept_pos = a.recent && a.pos && held;
    if (tid == 0) s_last = 0;
    for (int i = tid; i < SEL_BINS; i += SEL_THREADS) s_hist[i] = 0;
    __syncthreads();
    if (a.recent) {
        uint32_t last = a.pos ? 0u : sg.base + n - 1;
        if (a.pos)
            for (uint32_t i0 = tid; i0 < own; i0 += SEL_THREADS * FLIGHT) {
                uint32_t p[FLIGHT];
#pragma unroll
                for (int f = 0; f < FLIGHT; ++f) p[f] = i0 + f * SEL_THREADS < own ? a.pos[entry + base + i0 + f * SEL_THREADS] : 0u;
#pragma unroll
                for (int f = 0; f < FLIGHT; ++f) {
                    last = max(last, p[f]);
                    if (kept_pos && i0 + f * SEL_THREADS < own) s_key[i0 + f * SEL_THREADS] = p[f];  // (until the keys take their place)
                }
            }
        last = __reduce_max_sync(0xFFFFFFFFu, last);
        if (lane == 0) atomicMax(&s_last, last);
    }
    if (C > 1) cluster.sync();
    else __syncthreads();
    uint32_t newest = s_last;
    for (int r = 1; r < C; ++r) newest = max(newest, *cluster.map_shared_rank(&s_last, (rank_of + r) % C));
    const auto key_at = [&](uint32_t p, float x) { return weight_key(x, p < a.sink || (a.recent && newest - p < a.recent)); };
    // (a warp whose keys are all alike, as where nothing has been seen yet, adds once)
    const auto add = [&](uint32_t bin, bool in) {
        int alike;
        __match_all_sync(0xFFFFFFFFu, in ? bin : 0xFFFFFFFFu, &alike);
        if (alike ? in && lane == 0 : in) atomicAdd(&s_hist[bin], alike ? 32u : 1u);
    };
    if (held) {  // the keys take their places, and are counted by their first 11 bits
        for (uint32_t i00 = 0; i00 < own; i00 += SEL_THREADS * FLIGHT) {
            const uint32_t i0 = i00 + tid;
            float x[FLIGHT];
            uint32_t p[FLIGHT];
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f) {
                const uint32_t i = i0 + f * SEL_THREADS;
                x[f] = i < own ? w[base + i] : 0.0f;
                p[f] = i < own ? (kept_pos ? s_key[i] : position(i)) : 0u;
            }
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f) {
                const bool in = i0 + f * SEL_THREADS < own;
                const uint32_t k = key_at(p[f], x[f]);
                if (in) s_key[i0 + f * SEL_THREADS] = k;
                add(k >> 21, in);
            }
        }
    }
    // four rows' keys from row i on (of the CTA's); rows behind the warp's last: 0, which is below all that stay but perhaps their equal
    const auto four = [&](uint32_t i, uint32_t (&k)[4]) {
        if (held) {
            const uint4 x = *reinterpret_cast<const uint4*>(s_key + i);
            k[0] = x.x, k[1] = x.y, k[2] = x.z, k[3] = x.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e >= to) k[e] = 0u;
            else if (!held) k[e] = key_at(position(i + e), w[base + i + e]);
    };

    // the stay-th largest key, and how many of the keys equal to it stay
    uint32_t prefix = 0, left = stay;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t bins = pass == 2 ? 1024u : 2048u, settled = pass == 0 ? 0u : pass == 1 ? 0xFFE00000u : 0xFFFFFC00u;
        if (pass > 0) {
            for (int i = tid; i < SEL_BINS; i += SEL_THREADS) s_hist[i] = 0;
            __syncthreads();
        }
        for (uint32_t i0 = from; i0 < to && !(held && pass == 0); i0 += 128) {  // (a warp without rows begins at no multiple of 128)
            const uint32_t i = i0 + lane * 4;
            uint32_t k[4];
            four(i, k);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = i + e < to && !((k[e] ^ prefix) & settled);
                add((k[e] >> shift) & (bins - 1), in);
            }
        }
        if (C > 1) cluster.sync();
        else __syncthreads();
        // buckets from the top, two a thread
        uint32_t c[2] = {s_hist[SEL_BINS - 1 - tid * 2], s_hist[SEL_BINS - 2 - tid * 2]};
        for (int r = 1; r < C; ++r) {
            const uint32_t* other = cluster.map_shared_rank(s_hist, (rank_of + r) % C);
            c[0] += other[SEL_BINS - 1 - tid * 2];
            c[1] += other[SEL_BINS - 2 - tid * 2];
        }
        uint32_t before = scan_threads(c[0] + c[1], s_scan);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (before < left && before + c[j] >= left) s_found[0] = SEL_BINS - 1 - tid * 2 - j, s_found[1] = left - before, s_found[2] = c[j];
            before += c[j];
        }
        if (C > 1) cluster.sync();  // (also: the others have read this CTA's buckets)
        else __syncthreads();
        prefix |= s_found[0] << shift;
        left = s_found[1];
        if (left == s_found[2] && prefix) {  // all of the bucket stay: so do those above the number before it, and no others
            --prefix;
            left = 0;
            break;
        }
    }
    // In the rows' order: how many equal the last key that stays; then which stay, the free places below the budget and the rows from beyond that take them.
    const auto before_me = [&](uint32_t x, int slot) {  // the sum over the warps, of this CTA and those before it, before this one (x: a lane's)
        x = __reduce_add_sync(0xFFFFFFFFu, x);
        __syncthreads();
        if (lane == 0) s_warp[warp] = x;
        __syncthreads();
        if (tid < 32) {
            const uint32_t all = __reduce_add_sync(0xFFFFFFFFu, s_warp[lane]);
            if (lane == 0) s_all[slot] = all;
        }
        uint32_t sum = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? s_warp[lane] : 0u);
        if (C > 1) {
            cluster.sync();
            for (uint32_t r = 0; r < rank_of; ++r) sum += *cluster.map_shared_rank(&s_all[slot], r);
        }
        return sum;
    };
    uint32_t equal_mine = 0;
    for (uint32_t i = from + lane * 4; i < to; i += 128) {
        uint32_t k[4];
        four(i, k);
#pragma unroll
        for (int e = 0; e < 4; ++e) equal_mine += i + e < to && k[e] == prefix;
    }
    const uint32_t equal = before_me(equal_mine, 0);
    uint32_t rank = equal;
    const auto sum_before = [&](uint32_t x) {  // over the lanes before this one, x at most 4
        const uint32_t below = (1u << lane) - 1u;
        return __popc(__ballot_sync(0xFFFFFFFFu, x & 1u) & below) + 2 * __popc(__ballot_sync(0xFFFFFFFFu, x & 2u) & below) + 4 * __popc(__ballot_sync(0xFFFFFFFFu, x & 4u) & below);
    };
    const auto keeps = [&](uint32_t i) {  // a bit for each of four rows
        uint32_t k[4], keep = 0, eq = 0;
        four(i, k);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            keep |= (i + e < to && k[e] > prefix ? 1u : 0u) << e;
            eq |= (i + e < to && k[e] == prefix ? 1u : 0u) << e;
        }
        if (__any_sync(0xFFFFFFFFu, eq)) {
            uint32_t r = rank + sum_before(__popc(eq));
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (eq >> e & 1u) keep |= (r++ < left ? 1u : 0u) << e;
            rank += __reduce_add_sync(0xFFFFFFFFu, __popc(eq));
        }
        return keep;
    };
    const auto lies = [&](uint32_t i, uint32_t end) { return base + i >= end ? 0u : end - base - i < 4 ? (1u << (end - base - i)) - 1u : 15u; };  // which of four rows lie below `end`
    uint32_t free_mine = 0, late_mine = 0;
    for (uint32_t i0 = from; i0 < to; i0 += 128) {
        const uint32_t i = i0 + lane * 4, keep = keeps(i), front = lies(i, budget);
        free_mine += __popc(~keep & lies(i, base + to) & front);
        late_mine += __popc(keep & ~front);
    }
    uint32_t free_at = before_me(free_mine, 1), late_at = before_me(late_mine, 2);
    rank = equal;
    for (uint32_t i0 = from; i0 < to && base + i0 < budget; i0 += 128) {
        const uint32_t i = i0 + lane * 4, keep = keeps(i), front = lies(i, budget), open = ~keep & lies(i, base + to) & front;
        uint32_t place = free_at + sum_before(__popc(open));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t row = base + i + e;
            if (open >> e & 1u) hole[place++] = row;
            if (keep & front & (1u << e)) {
                source[row] = row;
                if (wanted) wanted[row] = row;
            }
        }
        free_at += __reduce_add_sync(0xFFFFFFFFu, __popc(open));
    }
    if (C > 1) cluster.sync();  // (all free places are known)
    else __syncthreads();
    if (__all_sync(0xFFFFFFFFu, late_mine == 0)) return;
    rank = equal;
    for (uint32_t i0 = from; i0 < to; i0 += 128) {
        const uint32_t i = i0 + lane * 4, comes = keeps(i) & ~lies(i, budget);
        if (!__any_sync(0xFFFFFFFFu, comes)) continue;
        uint32_t next = late_at + sum_before(__popc(comes));
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (comes >> e & 1u) {
                const uint32_t place = hole[next++];
                source[place] = base + i + e;
                if (wanted) wanted[place] = base + i + e;
            }
        late_at += __reduce_add_sync(0xFFFFFFFFu, __popc(comes));
    }
}

// A block moves what belongs to 64 places of one KV head: keys and values by LANES lanes a row in 16-byte pieces, then tiles, then the single words.
constexpr int MOVE_THREADS = 256, MOVE_PLACES = 64;
template <int LANES>
__global__ void __launch_bounds__(MOVE_THREADS) cache_move_kernel(const __grid_constant__ EvictArgs a, const __grid_constant__ CacheTable tab, uint32_t blocks) {
    dep_wait();
    __shared__ uint32_t s_src[MOVE_PLACES];
    const int tid = threadIdx.x;
    const uint32_t part = blockIdx.x % blocks, which = blockIdx.x / blocks, at = which / a.n_kv, head = which % a.n_kv;
    const CacheSeg sg = (a.table ? a.table : tab.s)[at];
    const uint32_t stay = a.stay[which], p0 = part * MOVE_PLACES;
    if (a.rows_out && part == 0 && head == 0 && tid == 0) a.rows_out[sg.seg] = stay;
    if (p0 >= stay) return;
    const uint32_t places = min((uint32_t)MOVE_PLACES, stay - p0);
    // 0xFFFFFFFF: stays where it is
    if (tid < MOVE_PLACES) {
        const uint32_t src = tid < places ? a.places[(uint64_t)which * a.room + p0 + tid] : 0xFFFFFFFFu;
        s_src[tid] = a.in_place && src == p0 + tid ? 0xFFFFFFFFu : src;
    }
    __syncthreads();
    const unsigned char* k = static_cast<const unsigned char*>(a.keys) + sg.row_begin * a.krs + head * a.khs;
    const unsigned char* v = static_cast<const unsigned char*>(a.values) + sg.row_begin * a.vrs + head * a.vhs;
    unsigned char* tk = static_cast<unsigned char*>(a.to_keys) + sg.to_begin * a.tkrs + head * a.tkhs;
    unsigned char* tv = static_cast<unsigned char*>(a.to_values) + sg.to_begin * a.tvrs + head * a.tvhs;
    // (all loads of tiles and of single words are under way before the first row is stored)
    uint4 tile[2];
    uint32_t word[3];
    const unsigned char* from_tile = a.tiles + (head * a.tile_hs + sg.row_begin) * TILE_BYTES + tid % 8 * 16;
    if (a.tiles)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const uint32_t src = s_src[tid / 8 + f * 32];
            if (src != 0xFFFFFFFFu) tile[f] = *reinterpret_cast<const uint4*>(from_tile + (uint64_t)src * TILE_BYTES);
        }
    const bool words = tid < MOVE_PLACES && s_src[tid < MOVE_PLACES ? tid : 0] != 0xFFFFFFFFu;
    if (words) {
        const uint64_t src = head * a.entry_hs + sg.row_begin + s_src[tid];
        if (a.to_pos) word[0] = a.pos[src];
        if (a.to_doc) word[1] = a.doc[src];
        if (a.to_w) word[2] = __float_as_uint(a.w[head * a.w_hs + sg.row_begin + s_src[tid]]);
    }
    constexpr int AT_ONCE = MOVE_THREADS / LANES, FLIGHT = MOVE_PLACES / AT_ONCE < 8 ? MOVE_PLACES / AT_ONCE : 8;
    const uint32_t lane = tid % LANES, group = tid / LANES, half = a.row_bytes / 16;
    for (uint32_t piece = lane; piece < 2 * half; piece += LANES) {
        const bool value = piece >= half;
        const uint64_t off = (uint64_t)(value ? piece - half : piece) * 16, rs = value ? a.vrs : a.krs, trs = value ? a.tvrs : a.tkrs;
        const unsigned char* from = (value ? v : k) + off;
        unsigned char* to = (value ? tv : tk) + off;
        for (uint32_t i0 = group; i0 < MOVE_PLACES; i0 += AT_ONCE * FLIGHT) {
            uint4 x[FLIGHT];
            uint32_t src[FLIGHT];
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f) {
                src[f] = s_src[i0 + f * AT_ONCE];
                if (src[f] != 0xFFFFFFFFu) x[f] = *reinterpret_cast<const uint4*>(from + src[f] * rs);
            }
#pragma unroll
            for (int f = 0; f < FLIGHT; ++f)
                if (src[f] != 0xFFFFFFFFu) *reinterpret_cast<uint4*>(to + (uint64_t)(p0 + i0 + f * AT_ONCE) * trs) = x[f];
        }
    }
    if (a.tiles) {
        unsigned char* to = a.to_tiles + (head * a.to_tile_hs + sg.to_begin) * TILE_BYTES + tid % 8 * 16;
#pragma unroll
        for (int f = 0; f < 2; ++f)
            if (s_src[tid / 8 + f * 32] != 0xFFFFFFFFu) *reinterpret_cast<uint4*>(to + (uint64_t)(p0 + tid / 8 + f * 32) * TILE_BYTES) = tile[f];
    }
    if (words) {
        const uint64_t to = head * a.to_entry_hs + sg.to_begin + p0 + tid;
        if (a.to_pos) a.to_pos[to] = word[0];
        if (a.to_doc) a.to_doc[to] = word[1];
        if (a.to_w) a.to_w[head * a.to_w_hs + sg.to_begin + p0 + tid] = __uint_as_float(word[2]);
    }
}

}  // namespace

Status launch_evict_cache(Ctx* c, EvictArgs a, const std::vector<SlhaB200Segment>& segs, const std::vector<SlhaB200Segment>& to) {
    std::vector<CacheSeg> table;
    uint32_t most = 0;
    for (size_t i = 0; i < segs.size(); ++i) {
        CacheSeg g{};
        g.row_begin = segs[i].tile_begin;
        g.n_rows = segs[i].n_tiles;
        g.base = segs[i].index_base;
        g.to_begin = a.in_place ? segs[i].tile_begin : to[i].tile_begin;
        g.seg = (uint32_t)i;
        table.push_back(g);
        most = std::max(most, g.n_rows);
    }
    // (places beyond the longest segment are never filled)
    const uint32_t room = a.room = std::min(a.budget, most);
    const uint64_t heads = (uint64_t)table.size() * a.n_kv, blocks = ((uint64_t)room + MOVE_PLACES - 1) / MOVE_PLACES;
    if (heads == 0) return Status();
    if (heads * std::max<uint64_t>(blocks, 8) > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "slha_b200_evict_cache: too many rows");
    CacheTable tab;
    SLHA_TRY(cache_table(c, table, &tab, &a.table));
    a.n_segs = (uint32_t)table.size();
    CacheMemory mem{c};
    void* p;
    SLHA_TRY(mem.get(heads * (2ull * room + 1) * 4, &p));
    a.places = static_cast<uint32_t*>(p);
    a.holes = a.places + heads * room;
    a.stay = a.holes + heads * room;
    // CTAs of a cluster: as many as find an SM each, of eight only where they find it beyond doubt (a cluster lies within a group of SMs: 16 heads in eights took two turns, 52 us
    // for 26 in fours).  8 heads, selection and 64 rows' places, in ones, twos, fours, eights: 8192 rows 18, 19, 19, 19 us; 16384 27, 24, 22, 22; 32768 44, 33, 26, 30;
    // 65536 106, 51, 34, 34; 131072 204, 112, 50, 42.
    uint32_t c_size = most >= 65536 ? 8 : most >= 16384 ? 4 : 1;
    while (c_size > 1 && heads * c_size > (uint64_t)sm_count(c->device) * (c_size == 8 ? 2 : 3) / 3) c_size /= 2;
    const size_t share = ((size_t)most + c_size * SEL_WARPS * 128 - 1) / (c_size * SEL_WARPS * 128) * SEL_WARPS * 128, smem = std::min<size_t>(share, SEL_HELD) * 4;
    g_cache_kernels |= SLHA_B200_CACHE_SELECT(c_size);
    const auto select = [&](auto kernel_of) -> Status {
        constexpr auto kernel = cache_select_kernel<decltype(kernel_of)::value>;
        SLHA_TRY((cache_smem<kernel>(c, SEL_HELD * 4)));
        SLHA_CUDA(launch_behind(kernel, dim3((uint32_t)(heads * c_size)), dim3(SEL_THREADS), smem, c->stream, a, tab));
        return Status();
    };
    SLHA_TRY(c_size == 8 ? select(std::integral_constant<int, 8>()) : c_size == 4 ? select(std::integral_constant<int, 4>()) : c_size == 2 ? select(std::integral_constant<int, 2>())
                                                                                                                              : select(std::integral_constant<int, 1>()));
    count_launch();
    const uint32_t pieces = 2 * a.row_bytes / 16;
    const dim3 grid((uint32_t)(heads * std::max<uint64_t>(blocks, 1)));
    SLHA_CUDA(pieces <= 8 ? launch_behind(cache_move_kernel<8>, grid, dim3(MOVE_THREADS), 0, c->stream, a, tab, (uint32_t)std::max<uint64_t>(blocks, 1))
              : pieces <= 16 ? launch_behind(cache_move_kernel<16>, grid, dim3(MOVE_THREADS), 0, c->stream, a, tab, (uint32_t)std::max<uint64_t>(blocks, 1))
                             : launch_behind(cache_move_kernel<32>, grid, dim3(MOVE_THREADS), 0, c->stream, a, tab, (uint32_t)std::max<uint64_t>(blocks, 1)));
    count_launch();
    return mem.done();
}

}  // namespace slha
