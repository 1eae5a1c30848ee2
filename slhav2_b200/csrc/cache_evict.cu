// Removal of the cached rows that received the least weight (slha_b200_evict_cache).
//
// Two kernels.  The first, a CTA for each KV head of a segment, finds which min(n, budget) of the n rows stay: the budget-th largest of the rows' keys by
// radix selection (8 bits a pass, from the top), equal keys by the lower row, and writes for each place below the budget the row that comes to it.  The
// second moves rows.  A kept row below the budget stays where it is, so in place only rows from beyond the budget move, into places that no row is read from.
#include <algorithm>

#include "cache.cuh"

namespace slha {
namespace {

constexpr int SEL_THREADS = 1024, SEL_WARPS = SEL_THREADS / 32, SEL_EACH = 4;
constexpr uint32_t SEL_HELD = 49152;  // keys that fit in shared memory

// weights in the order of unsigned numbers: pinned rows above all, NaN below all, -0 like 0
__device__ __forceinline__ uint32_t weight_key(float w, bool pinned) {
    if (pinned) return 0xFFFFFFFFu;
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// sums of `x` over the threads before this one, and over all
__device__ __forceinline__ uint32_t scan_threads(uint32_t x, uint32_t* sh, uint32_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t s = x;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, s, o);
        if (lane >= o) s += y;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = s;
    __syncthreads();
    if (warp == 0) {
        uint32_t v = sh[lane];
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, v, o);
            if (lane >= o) v += y;
        }
        sh[lane] = v;
    }
    __syncthreads();
    *total = sh[SEL_WARPS - 1];
    return s - x + (warp ? sh[warp - 1] : 0u);
}

__global__ void __launch_bounds__(SEL_THREADS) cache_select_kernel(const __grid_constant__ EvictArgs a, const __grid_constant__ CacheTable tab) {
    dep_wait();
    extern __shared__ uint32_t s_key[];
    __shared__ uint32_t s_hist[8][256], s_scan[SEL_WARPS], s_found[2], s_last;
    const int tid = threadIdx.x, lane = tid & 31;
    const uint32_t at = blockIdx.x / a.n_kv, head = blockIdx.x % a.n_kv;
    const CacheSeg sg = (a.table ? a.table : tab.s)[at];
    const uint32_t n = a.rows ? min(a.rows[sg.seg], sg.n_rows) : sg.n_rows;
    const uint32_t budget = a.budget, stay = min(n, budget);
    uint32_t* source = a.places + (uint64_t)blockIdx.x * a.room;
    uint32_t* hole = a.holes + (uint64_t)blockIdx.x * a.room;
    uint32_t* wanted = a.source ? a.source + ((uint64_t)sg.seg * a.n_kv + head) * budget : nullptr;
    if (tid == 0) a.stay[blockIdx.x] = stay;
    const uint64_t entry = head * a.entry_hs + sg.row_begin;
    const float* w = a.w + head * a.w_hs + sg.row_begin;
    if (n <= budget) {
        for (uint32_t i = tid; i < n; i += SEL_THREADS) {
            source[i] = i;
            if (wanted) wanted[i] = i;
        }
        return;
    }
    const auto position = [&](uint32_t i) { return a.pos ? a.pos[entry + i] : sg.base + i; };
    if (tid == 0) s_last = 0;
    __syncthreads();
    if (a.recent) {
        uint32_t last = 0;
        if (a.pos)
            for (uint32_t i = tid; i < n; i += SEL_THREADS) last = max(last, a.pos[entry + i]);
        else last = sg.base + n - 1;
        last = __reduce_max_sync(0xFFFFFFFFu, last);
        if (lane == 0) atomicMax(&s_last, last);
        __syncthreads();
    }
    const uint32_t newest = s_last;
    const auto make_key = [&](uint32_t i) {
        const uint32_t p = position(i);
        return weight_key(w[i], p < a.sink || (a.recent && newest - p < a.recent));
    };
    const bool held = n <= SEL_HELD;
    if (held) {
        for (uint32_t i = tid; i < n; i += SEL_THREADS) s_key[i] = make_key(i);
        __syncthreads();
    }
    const auto key_of = [&](uint32_t i) { return held ? s_key[i] : make_key(i); };

    // the stay-th largest key, and how many of the keys equal to it stay
    uint32_t prefix = 0, left = stay;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 8 * 256; i += SEL_THREADS) (&s_hist[0][0])[i] = 0;
        __syncthreads();
        for (uint32_t i0 = 0; i0 < n; i0 += SEL_THREADS) {
            const uint32_t i = i0 + tid;
            const uint32_t k = i < n ? key_of(i) : 0u;
            const bool in = i < n && (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)));
            // one addition for the lanes of a warp that share a bucket with the first of them; the others add alone
            const uint32_t bin = (k >> shift) & 255u, who = __ballot_sync(0xFFFFFFFFu, in);
            if (who) {
                const int lead = __ffs(who) - 1;
                const uint32_t lead_bin = __shfl_sync(0xFFFFFFFFu, bin, lead);
                const uint32_t same = __ballot_sync(0xFFFFFFFFu, in && bin == lead_bin);
                if (lane == lead) atomicAdd(&s_hist[(tid >> 5) & 7][bin], (uint32_t)__popc(same));
                else if (in && bin != lead_bin) atomicAdd(&s_hist[(tid >> 5) & 7][bin], 1u);
            }
        }
        __syncthreads();
        if (tid < 32) {  // buckets from the top: lane 0 the highest eight
            uint32_t c[8], sum = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t x = 0;
                for (int h = 0; h < 8; ++h) x += s_hist[h][255 - lane * 8 - j];
                c[j] = x;
                sum += x;
            }
            uint32_t before = sum;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, before, o);
                if (lane >= o) before += y;
            }
            before -= sum;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (before < left && before + c[j] >= left) s_found[0] = 255 - lane * 8 - j, s_found[1] = left - before;
                before += c[j];
            }
        }
        __syncthreads();
        prefix |= s_found[0] << shift;
        left = s_found[1];
        __syncthreads();
    }
    // rows in order: which stay, the free places below the budget, the rows from beyond that take them
    uint32_t equal = 0, holes = 0, late = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += SEL_THREADS * SEL_EACH) {
        uint32_t k[SEL_EACH], eq = 0, total;
#pragma unroll
        for (int j = 0; j < SEL_EACH; ++j) {
            const uint32_t i = i0 + tid * SEL_EACH + j;
            k[j] = i < n ? key_of(i) : 0u;
            eq += i < n && k[j] == prefix;
        }
        uint32_t rank = equal + scan_threads(eq, s_scan, &total);
        equal += total;
        bool keep[SEL_EACH];
        uint32_t h = 0, f = 0;
#pragma unroll
        for (int j = 0; j < SEL_EACH; ++j) {
            const uint32_t i = i0 + tid * SEL_EACH + j;
            keep[j] = i < n && (k[j] > prefix || (k[j] == prefix && rank < left));
            rank += i < n && k[j] == prefix;
            h += i < budget && !keep[j];
            f += i >= budget && keep[j];
        }
        // (free places in the low half, rows from beyond in the high one: at most 4096 of each here)
        const uint32_t both = scan_threads(h | f << 16, s_scan, &total);
        uint32_t free_at = holes + (both & 0xFFFFu), late_at = late + (both >> 16);
        holes += total & 0xFFFFu;
        late += total >> 16;
#pragma unroll
        for (int j = 0; j < SEL_EACH; ++j) {
            const uint32_t i = i0 + tid * SEL_EACH + j;
            if (i >= budget) continue;
            if (!keep[j]) {
                hole[free_at++] = i;
            } else {
                source[i] = i;
                if (wanted) wanted[i] = i;
            }
        }
        __syncthreads();  // (all places below the budget are known before the first row from beyond it asks for one)
#pragma unroll
        for (int j = 0; j < SEL_EACH; ++j) {
            const uint32_t i = i0 + tid * SEL_EACH + j;
            if (i < budget || !keep[j]) continue;
            const uint32_t place = hole[late_at++];
            source[place] = i;
            if (wanted) wanted[place] = i;
        }
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
        const unsigned char* from = a.tiles + (head * a.tile_hs + sg.row_begin) * TILE_BYTES;
        unsigned char* to = a.to_tiles + (head * a.to_tile_hs + sg.to_begin) * TILE_BYTES;
        uint4 x[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const uint32_t i = tid / 8 + f * 32;
            if (s_src[i] != 0xFFFFFFFFu) x[f] = *reinterpret_cast<const uint4*>(from + (uint64_t)s_src[i] * TILE_BYTES + tid % 8 * 16);
        }
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const uint32_t i = tid / 8 + f * 32;
            if (s_src[i] != 0xFFFFFFFFu) *reinterpret_cast<uint4*>(to + (uint64_t)(p0 + i) * TILE_BYTES + tid % 8 * 16) = x[f];
        }
    }
    if (tid < MOVE_PLACES && s_src[tid] != 0xFFFFFFFFu) {
        const uint64_t src = head * a.entry_hs + sg.row_begin + s_src[tid], to = head * a.to_entry_hs + sg.to_begin + p0 + tid;
        if (a.to_pos) a.to_pos[to] = a.pos[src];
        if (a.to_doc) a.to_doc[to] = a.doc[src];
        if (a.to_w) a.to_w[head * a.to_w_hs + sg.to_begin + p0 + tid] = a.w[head * a.w_hs + sg.row_begin + s_src[tid]];
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
    if (heads * std::max<uint64_t>(blocks, 1) > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "slha_b200_evict_cache: too many rows");
    CacheTable tab;
    SLHA_TRY(cache_table(c, table, &tab, &a.table));
    a.n_segs = (uint32_t)table.size();
    CacheMemory mem{c};
    void* p;
    SLHA_TRY(mem.get(heads * (2ull * room + 1) * 4, &p));
    a.places = static_cast<uint32_t*>(p);
    a.holes = a.places + heads * room;
    a.stay = a.holes + heads * room;
    const size_t smem = (size_t)std::min(most, SEL_HELD) * 4;
    SLHA_TRY((cache_smem<cache_select_kernel>(c, SEL_HELD * 4)));
    SLHA_CUDA(launch_behind(cache_select_kernel, dim3((uint32_t)heads), dim3(SEL_THREADS), smem, c->stream, a, tab));
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
