// Exact attention over a cache of rows in 4 bits (slha_b200_attend_cache4, slha_b200_attend_tree4).
#include <algorithm>

#include "cache4.cuh"

namespace slha {
namespace {

// Segments whose rows are laid out as rows of the queries' type first, in order, as many at a time as CACHE4_ROWS_MOST holds (at least one).
Status attend_laid_out(Ctx* c, const CacheArgs& args, const Rows4& r, int dtype, const std::vector<SlhaB200Segment>& segs) {
    const uint64_t e = dtype == SLHA_B200_BF16 ? 2 : 4, row = 2 * args.n_kv * args.d * e;
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
                of[i].n_tiles = of[i].n_queries = to[i].n_queries = 0;
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
        x.units = args.d / 8;
        SLHA_TRY(launch_read_cache4(c, x, dtype, of, to));
        CacheArgs a = args;
        a.keys = x.rows.p[0];
        a.values = x.rows.p[1];
        a.krs = a.vrs = args.d;
        a.khs = a.vhs = hs;
        if (a.row_pos) a.row_pos = x.to_pos;
        if (a.row_doc) a.row_doc = x.to_doc;
        a.entry_hs = args.entry_hs ? b.rows : 0;
        SLHA_TRY(launch_attend_cache(c, a, dtype, to));
    }
    g_cache_kernels |= SLHA_B200_CACHE_LAID_OUT;
    return mem.done();
}

}  // namespace

Status launch_attend_cache4(Ctx* c, CacheArgs a, const Rows4& r, int dtype, const std::vector<SlhaB200Segment>& segs) { return attend_laid_out(c, a, r, dtype, segs); }

}  // namespace slha
