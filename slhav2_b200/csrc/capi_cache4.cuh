// Part 2 of the C ABI, rows of 4 bits and what fills a cache: argument checks of slha_b200_rotate_heads, _write_cache4, _read_cache4, _attend_cache4 and _attend_tree4.
// Included at the end of capi.cu.
#pragma once

namespace {

uint64_t scale_bytes4(uint32_t head_dim) { return head_dim <= 64 ? 4 : head_dim <= 128 ? 8 : 16; }

Status cache4_check(const SlhaB200KvCache4* k, const char* fn) {
    const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
    if (!k->key_codes || !k->value_codes || !k->key_scales || !k->value_scales) return Status(SLHA_ERR_NULL, name("codes or scales are NULL"));
    if (k->dtype != SLHA_B200_F32 && k->dtype != SLHA_B200_BF16) return Status(SLHA_ERR_DIMENSION, name("dtype must be SLHA_B200_F32 or SLHA_B200_BF16"));
    if (k->head_dim == 0 || k->head_dim > CACHE_DIM_MOST || k->head_dim % BLOCK4) return Status(SLHA_ERR_DIMENSION, name("head_dim must be a multiple of 16 in 16..256"));
    if (k->n_kv_heads == 0 || k->n_kv_heads > 65535) return Status(SLHA_ERR_DIMENSION, name("n_kv_heads must be in 1..65535"));
    if (k->code_row_stride % 16 || k->code_head_stride % 16 || !cache_aligned(k->key_codes) || !cache_aligned(k->value_codes))
        return Status(SLHA_ERR_DIMENSION, name("codes must begin on a multiple of 16 bytes and their strides be multiples of 16 bytes"));
    const uint64_t s = scale_bytes4(k->head_dim);
    if (k->scale_row_stride % s || k->scale_head_stride % s || reinterpret_cast<uintptr_t>(k->key_scales) % s || reinterpret_cast<uintptr_t>(k->value_scales) % s)
        return Status(SLHA_ERR_DIMENSION, name("scales must begin on a multiple of ") + std::to_string(s) + " bytes and their strides be multiples of it");
    for (const int32_t e : {k->key_exponent, k->value_exponent})
        if (e < -64 || e > 64) return Status(SLHA_ERR_DIMENSION, name("key_exponent and value_exponent must be in -64..64"));
    return cache_words(fn, {k->positions, k->documents, k->rows});
}
Status cache4_memory(Ctx* c, const SlhaB200KvCache4* k, const char* fn) {
    SLHA_TRY(cache_device_memory(c, k->key_codes, fn, "key_codes"));
    SLHA_TRY(cache_device_memory(c, k->value_codes, fn, "value_codes"));
    SLHA_TRY(cache_device_memory(c, k->key_scales, fn, "key_scales"));
    SLHA_TRY(cache_device_memory(c, k->value_scales, fn, "value_scales"));
    if (k->positions) SLHA_TRY(cache_device_memory(c, k->positions, fn, "positions of rows"));
    if (k->documents) SLHA_TRY(cache_device_memory(c, k->documents, fn, "documents of rows"));
    return Status();
}
Rows4 cache4_rows(const SlhaB200KvCache4* k) {
    Rows4 r{};
    r.codes[0] = static_cast<const unsigned char*>(k->key_codes);
    r.codes[1] = static_cast<const unsigned char*>(k->value_codes);
    r.scales[0] = static_cast<const unsigned char*>(k->key_scales);
    r.scales[1] = static_cast<const unsigned char*>(k->value_scales);
    r.crs = k->code_row_stride;
    r.chs = k->code_head_stride;
    r.srs = k->scale_row_stride;
    r.shs = k->scale_head_stride;
    r.exponent[0] = k->key_exponent;
    r.exponent[1] = k->value_exponent;
    return r;
}
// Rows (or tokens) of float32 or bfloat16 beside a 4-bit cache: type, alignment and strides of what is there.
Status rows_check(const SlhaB200KvCache* k, uint32_t head_dim, uint32_t n_kv, bool both, const char* fn, const char* what) {
    const auto name = [&](const char* s) { return std::string(fn) + ": " + what + ": " + s; };
    if (both ? !k->keys || !k->values : !k->keys && !k->values) return Status(SLHA_ERR_NULL, name("keys or values are NULL"));
    if (k->dtype != SLHA_B200_F32 && k->dtype != SLHA_B200_BF16) return Status(SLHA_ERR_DIMENSION, name("dtype must be SLHA_B200_F32 or SLHA_B200_BF16"));
    if (k->head_dim != head_dim || k->n_kv_heads != n_kv) return Status(SLHA_ERR_DIMENSION, name("head_dim and n_kv_heads must be the same as beside it"));
    const size_t each = 16 / key_elem_bytes(k->dtype);
    if ((k->keys && (k->key_row_stride % each || k->key_head_stride % each || !cache_aligned(k->keys))) ||
        (k->values && (k->value_row_stride % each || k->value_head_stride % each || !cache_aligned(k->values))))
        return Status(SLHA_ERR_DIMENSION, name("keys and values must begin on a multiple of 16 bytes and their strides be multiples of 16 bytes"));
    return Status();
}
// What a call writes of a table's segments, a range of rows each: their tokens' rows, all of them (where `at` says), or their tokens as rows of queries.
struct Written {
    enum Of { TOKENS, ROWS, QUERIES } of;
    const std::vector<SlhaB200Segment>&segs, &at;
    const uint32_t* rows;       // counts on the host, or null
    bool known = true;          // false: counts in device memory, rows are among these
    uint64_t first = ~0ull, end = 0;
    bool single = true;         // one row each
    Written(Of of, const std::vector<SlhaB200Segment>& segs, const std::vector<SlhaB200Segment>& at, const uint32_t* counts) : of(of), segs(segs), at(at), rows(counts) {
        if (rows && is_device_ptr(rows)) {
            known = false;
            rows = nullptr;
        }
        for (size_t i = 0; i < segs.size(); ++i) {
            const auto [from, to] = range(i);
            if (from >= to) continue;
            first = std::min(first, from);
            end = std::max(end, to);
            single &= to - from == 1;
        }
    }
    std::pair<uint64_t, uint64_t> range(size_t i) const {  // first, behind the last
        const SlhaB200Segment& s = segs[i];
        if (of == QUERIES) return {s.query_begin, (uint64_t)s.query_begin + s.n_queries};
        const uint64_t n = rows ? std::min(rows[i], s.n_tiles) : s.n_tiles, begin = at[i].tile_begin;
        if (of == ROWS) return {begin, begin + n};
        return {begin + (known ? n - std::min<uint64_t>(n, s.n_queries) : s.n_queries ? 0 : n), begin + n};
    }
};
// Where rows go, every row that is written has a place of its own of `bytes` for each head; strides in bytes.  Where neither a row's heads lie before the next row nor a head's rows before the
// next head, places are compared: of rows `by` apart, the one h heads on.
Status rows_apart(unsigned __int128 row, unsigned __int128 head, uint32_t n_heads, uint64_t bytes, const Written& w, const char* fn, const char* what) {
    const auto apart = [&]() {
        if (row == 0 || (n_heads > 1 && head == 0)) return false;
        if (w.first >= w.end) return true;
        if (n_heads > 1 && head < bytes) return false;
        if (!w.known) return row >= bytes || w.single;
        if (row >= (n_heads > 1 ? head * (n_heads - 1) : 0) + bytes) return true;
        const uint64_t most = w.end - 1 - w.first;  // between two rows
        if (row >= bytes && head >= row * most + bytes) return true;
        std::vector<std::pair<uint64_t, uint64_t>> r;  // (they share no row)
        for (size_t i = 0; i < w.segs.size(); ++i)
            if (w.range(i).first < w.range(i).second) r.push_back(w.range(i));
        std::sort(r.begin(), r.end());
        const auto twice = [&](uint64_t by) {  // whether two rows lie `by` apart
            for (size_t i = 0, j = 0; i < r.size() && j < r.size();) {
                if (r[i].second <= r[j].first + by) ++i;
                else if (r[j].second + by <= r[i].first) ++j;
                else return true;
            }
            return false;
        };
        for (uint32_t h = 0; h < n_heads; ++h) {
            const unsigned __int128 on = head * h, least = h ? (on - bytes) / row + 1 : 1;  // (the first multiple of row beyond on - bytes; head >= bytes)
            if (least > most) break;
            for (unsigned __int128 by = least; by <= most && by * row < on + bytes; ++by)
                if (twice((uint64_t)by)) return false;
        }
        return true;
    };
    return apart() ? Status() : Status(SLHA_ERR_DIMENSION, std::string(fn) + ": " + what + " must have a place for each row and head (strides)");
}
Status rows_to_apart(const SlhaB200KvCache* to, const Written& w, const char* fn) {
    const unsigned __int128 e = key_elem_bytes(to->dtype);
    const uint64_t bytes = to->head_dim * (uint64_t)e;
    if (to->keys) SLHA_TRY(rows_apart(to->key_row_stride * e, to->key_head_stride * e, to->n_kv_heads, bytes, w, fn, "keys"));
    if (to->values) SLHA_TRY(rows_apart(to->value_row_stride * e, to->value_head_stride * e, to->n_kv_heads, bytes, w, fn, "values"));
    return Status();
}
RowsOf rows_of(const SlhaB200KvCache* k) {
    const uint64_t e = key_elem_bytes(k->dtype);
    RowsOf r{};
    r.p[0] = static_cast<const unsigned char*>(k->keys);
    r.p[1] = static_cast<const unsigned char*>(k->values);
    r.rs[0] = k->key_row_stride * e;
    r.hs[0] = k->key_head_stride * e;
    r.rs[1] = k->value_row_stride * e;
    r.hs[1] = k->value_head_stride * e;
    return r;
}
// Segments whose tokens there are, and (w: where they are written to their last rows) whose rows no other segment's tokens are written to.
Status token_segments(const std::vector<SlhaB200Segment>& segs, uint32_t n_tokens, const Written* w, const char* fn) {
    for (const SlhaB200Segment& s : segs)
        if ((uint64_t)s.query_begin + s.n_queries > n_tokens) return Status(SLHA_ERR_DIMENSION, std::string(fn) + ": a segment's tokens reach beyond n_tokens");
    if (!w || !w->known || segs.size() < 2) return Status();
    return cache_overlap(segs.size(), [&](size_t i) { return w->range(i); }) ? Status(SLHA_ERR_DIMENSION, std::string(fn) + ": two segments' tokens have the same rows") : Status();
}

int32_t attend_cache4_any(const char* fn, const SlhaB200KvCache4* cache, const SlhaB200Segment* segments, size_t n_segments, const SlhaB200CacheQueries* queries,
                          const uint32_t* parents, bool tree, void* out, uint64_t out_token_stride, uint64_t out_head_stride, float* lse_out) {
    return ffi([&]() -> Status {
        g_cache_kernels = 0;
        const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
        if (!cache || !queries || (n_segments && !segments)) return Status(SLHA_ERR_NULL, std::string(fn) + " received a NULL pointer");
        if (n_segments == 0 || queries->n_tokens == 0) return Status();
        if (!out || (tree && !parents)) return Status(SLHA_ERR_NULL, std::string(fn) + " received a NULL pointer");
        SLHA_TRY(cache4_check(cache, fn));
        // the same queries over rows of their own type, of which nothing but heads, positions and documents is looked at; the keys' exponent is part of the scale
        SlhaB200KvCache k{};
        k.dtype = cache->dtype;
        k.head_dim = cache->head_dim;
        k.n_kv_heads = cache->n_kv_heads;
        k.positions = cache->positions;
        k.documents = cache->documents;
        k.entry_head_stride = cache->entry_head_stride;
        k.rows = cache->rows;
        SlhaB200CacheQueries q = *queries;
        q.scale = std::ldexp(q.scale, cache->key_exponent);
        if (q.scale != 0.0f && !std::isnormal(q.scale)) return Status(SLHA_ERR_NONFINITE, name("scale * 2^key_exponent must be finite and a normal float32"));
        SLHA_TRY(cache_check_queries(&k, &q, fn));
        SLHA_TRY(cache_words(fn, {parents, lse_out}));
        const size_t each = 16 / key_elem_bytes(cache->dtype);
        if (out_token_stride % each || out_head_stride % each || !cache_aligned(out))
            return Status(SLHA_ERR_DIMENSION, name("out must begin on a multiple of 16 bytes and its strides be multiples of 16 bytes"));
        std::vector<SlhaB200Segment> segs;
        bool device_segs;
        cache_host_segments(segments, n_segments, &segs, &device_segs);
        const auto check_segments = [&]() -> Status {
            SLHA_TRY(cache_check_segments(&k, segs, &q, tree, fn));
            const auto tokens = [&](size_t i) { return std::pair<uint64_t, uint64_t>(segs[i].query_begin, (uint64_t)segs[i].query_begin + segs[i].n_queries); };
            return cache_overlap(segs.size(), tokens) ? Status(SLHA_ERR_DIMENSION, name("two segments have the same query tokens")) : Status();
        };
        if (!device_segs) SLHA_TRY(check_segments());
        CallScope cs;
        if (!cs.ok()) return cs.st;
        Ctx* c = cs.c;
        SLHA_TRY(cache_device_segments(c, segments, &segs, device_segs, fn));
        if (device_segs) SLHA_TRY(check_segments());
        SLHA_TRY(cache4_memory(c, cache, fn));
        SLHA_TRY(cache_device_memory(c, out, fn, "out"));
        if (lse_out) SLHA_TRY(cache_device_memory(c, lse_out, fn, "lse_out"));
        CacheArgs a;
        SLHA_TRY(cache_arguments(c, &k, n_segments, &q, fn, &a));
        if (tree) {
            SLHA_TRY(cache_stage(c, parents, q.n_tokens, &a.parents, fn, "parents"));
            a.tree = 1;
        }
        a.out = out;
        a.ots = out_token_stride;
        a.ohs = out_head_stride;
        a.lse = lse_out;
        SLHA_TRY(launch_attend_cache4(c, a, cache4_rows(cache), cache->dtype, segs));
        if (sync_by_default(c)) SLHA_CUDA(cudaStreamSynchronize(c->stream));
        return Status();
    });
}

}  // namespace

extern "C" {

int32_t slha_b200_attend_cache4(const SlhaB200KvCache4* cache, const SlhaB200Segment* segments, size_t n_segments, const SlhaB200CacheQueries* queries, void* out,
                                uint64_t out_token_stride, uint64_t out_head_stride, float* lse_out) {
    return attend_cache4_any("slha_b200_attend_cache4", cache, segments, n_segments, queries, nullptr, false, out, out_token_stride, out_head_stride, lse_out);
}
int32_t slha_b200_attend_tree4(const SlhaB200KvCache4* cache, const SlhaB200Segment* segments, size_t n_segments, const SlhaB200CacheQueries* queries,
                               const uint32_t* parents, void* out, uint64_t out_token_stride, uint64_t out_head_stride, float* lse_out) {
    return attend_cache4_any("slha_b200_attend_tree4", cache, segments, n_segments, queries, parents, true, out, out_token_stride, out_head_stride, lse_out);
}

int32_t slha_b200_write_cache4(const SlhaB200KvCache4* cache, const SlhaB200Segment* segments, size_t n_segments, const SlhaB200KvCache* from, uint32_t n_tokens) {
    return ffi([&]() -> Status {
        g_cache_kernels = 0;
        const char* fn = "slha_b200_write_cache4";
        if (!cache || !from || (n_segments && !segments)) return Status(SLHA_ERR_NULL, std::string(fn) + " received a NULL pointer");
        if (n_segments == 0 || n_tokens == 0) return Status();
        SLHA_TRY(cache4_check(cache, fn));
        SLHA_TRY(rows_check(from, cache->head_dim, cache->n_kv_heads, true, fn, "from"));
        std::vector<SlhaB200Segment> segs;
        bool device_segs;
        cache_host_segments(segments, n_segments, &segs, &device_segs);
        const auto check_segments = [&]() -> Status {
            const Written w(Written::TOKENS, segs, segs, cache->rows);
            SLHA_TRY(token_segments(segs, n_tokens, &w, fn));
            SLHA_TRY(rows_apart(cache->code_row_stride, cache->code_head_stride, cache->n_kv_heads, cache->head_dim / 2, w, fn, "codes"));
            return rows_apart(cache->scale_row_stride, cache->scale_head_stride, cache->n_kv_heads, cache->head_dim / BLOCK4, w, fn, "scales");
        };
        if (!device_segs) SLHA_TRY(check_segments());
        CallScope cs;
        if (!cs.ok()) return cs.st;
        Ctx* c = cs.c;
        SLHA_TRY(cache_device_segments(c, segments, &segs, device_segs, fn));
        if (device_segs) SLHA_TRY(check_segments());
        SLHA_TRY(cache4_memory(c, cache, fn));
        SLHA_TRY(cache_device_memory(c, from->keys, fn, "keys"));
        SLHA_TRY(cache_device_memory(c, from->values, fn, "values"));
        Rows4Args a{};
        a.in4 = cache4_rows(cache);
        a.rows = rows_of(from);
        SLHA_TRY(cache_stage(c, cache->rows, n_segments, &a.counts, fn, "rows"));
        a.n_kv = cache->n_kv_heads;
        a.d = cache->head_dim;
        SLHA_TRY(launch_write_cache4(c, a, from->dtype, segs));
        if (sync_by_default(c)) SLHA_CUDA(cudaStreamSynchronize(c->stream));
        return Status();
    });
}

int32_t slha_b200_read_cache4(const SlhaB200KvCache4* cache, const SlhaB200Segment* segments, size_t n_segments, const SlhaB200KvCache* to,
                              const SlhaB200Segment* to_segments) {
    return ffi([&]() -> Status {
        g_cache_kernels = 0;
        const char* fn = "slha_b200_read_cache4";
        const auto name = [&](const std::string& what) { return std::string(fn) + ": " + what; };
        if (!cache || !to || (n_segments && !segments)) return Status(SLHA_ERR_NULL, std::string(fn) + " received a NULL pointer");
        if (n_segments == 0) return Status();
        SLHA_TRY(cache4_check(cache, fn));
        SLHA_TRY(rows_check(to, cache->head_dim, cache->n_kv_heads, false, fn, "to"));
        std::vector<SlhaB200Segment> segs, to_segs;
        bool device_segs, device_to = false;
        cache_host_segments(segments, n_segments, &segs, &device_segs);
        if (to_segments) cache_host_segments(to_segments, n_segments, &to_segs, &device_to);
        const auto check_segments = [&]() -> Status {
            if (!to_segments) to_segs = segs;
            for (size_t i = 0; i < segs.size(); ++i)
                if (to_segs[i].n_tiles < segs[i].n_tiles) return Status(SLHA_ERR_CAPACITY, name("segment " + std::to_string(i) + " has no room for its rows where they go"));
            SLHA_TRY(cache_own_rows(segs, to_segs, cache->rows, 0xFFFFFFFFu, fn));
            const Written w(Written::ROWS, segs, to_segs, cache->rows);
            return rows_to_apart(to, w, fn);
        };
        if (!device_segs && !device_to) SLHA_TRY(check_segments());
        CallScope cs;
        if (!cs.ok()) return cs.st;
        Ctx* c = cs.c;
        SLHA_TRY(cache_device_segments(c, segments, &segs, device_segs, fn));
        if (to_segments) SLHA_TRY(cache_device_segments(c, to_segments, &to_segs, device_to, fn));
        if (device_segs || device_to) SLHA_TRY(check_segments());
        SLHA_TRY(cache4_memory(c, cache, fn));
        if (to->keys) SLHA_TRY(cache_device_memory(c, to->keys, fn, "keys"));
        if (to->values) SLHA_TRY(cache_device_memory(c, to->values, fn, "values"));
        Rows4Args a{};
        a.in4 = cache4_rows(cache);
        a.rows = rows_of(to);
        SLHA_TRY(cache_stage(c, cache->rows, n_segments, &a.counts, fn, "rows"));
        a.n_kv = cache->n_kv_heads;
        a.d = cache->head_dim;
        a.seen_last = 0xFFFFFFFFu;
        SLHA_TRY(launch_read_cache4(c, a, to->dtype, segs, to_segs));
        if (sync_by_default(c)) SLHA_CUDA(cudaStreamSynchronize(c->stream));
        return Status();
    });
}

int32_t slha_b200_rotate_heads(const SlhaB200HeadRows* heads, const SlhaB200Rotation* rotation, const SlhaB200Segment* segments, size_t n_segments, void* q_out,
                               uint64_t q_out_token_stride, uint64_t q_out_head_stride, const SlhaB200KvCache* to) {
    return ffi([&]() -> Status {
        g_cache_kernels = 0;
        const char* fn = "slha_b200_rotate_heads";
        const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
        if (!heads || (n_segments && !segments)) return Status(SLHA_ERR_NULL, std::string(fn) + " received a NULL pointer");
        if (!heads->q && !heads->k && !heads->v) return Status(SLHA_ERR_NULL, name("no heads are given"));
        if (heads->n_tokens == 0 || (segments && n_segments == 0)) return Status();
        if (heads->q && !q_out) return Status(SLHA_ERR_NULL, name("q_out is NULL"));
        if ((heads->k || heads->v) && !to) return Status(SLHA_ERR_NULL, name("there are keys or values, but no rows that they go to"));
        if ((heads->k && !to->keys) || (heads->v && !to->values)) return Status(SLHA_ERR_NULL, name("to: keys or values are NULL"));
        if (heads->dtype != SLHA_B200_F32 && heads->dtype != SLHA_B200_BF16) return Status(SLHA_ERR_DIMENSION, name("dtype must be SLHA_B200_F32 or SLHA_B200_BF16"));
        const uint32_t d = heads->head_dim, n_kv = heads->k || heads->v ? heads->n_kv_heads : 0;
        if (d == 0 || d > CACHE_DIM_MOST || d % 8) return Status(SLHA_ERR_DIMENSION, name("head_dim must be a multiple of 8 in 8..256"));
        if ((heads->q && (heads->n_heads == 0 || heads->n_heads > 0x3FFFFFFFu)) || ((heads->k || heads->v) && (n_kv == 0 || n_kv > 65535)))
            return Status(SLHA_ERR_DIMENSION, name("n_heads must be positive and n_kv_heads in 1..65535"));
        const uint64_t e = key_elem_bytes(heads->dtype), each = 16 / e;
        const auto lies = [&](const void* p, uint64_t ts, uint64_t hs) { return !p || (cache_aligned(p) && ts % each == 0 && hs % each == 0); };
        if (!lies(heads->q, heads->q_token_stride, heads->q_head_stride) || !lies(heads->k, heads->k_token_stride, heads->k_head_stride) ||
            !lies(heads->v, heads->v_token_stride, heads->v_head_stride) || (heads->q && !lies(q_out, q_out_token_stride, q_out_head_stride)))
            return Status(SLHA_ERR_DIMENSION, name("heads and q_out must begin on a multiple of 16 bytes and their strides be multiples of 16 bytes"));
        SlhaB200KvCache there{};  // what is written of `to`
        if (n_kv) {
            there = *to;
            if (!heads->k) there.keys = nullptr;
            if (!heads->v) there.values = nullptr;
            if (to->dtype != heads->dtype) return Status(SLHA_ERR_DIMENSION, name("heads and rows must have the same dtype"));
            SLHA_TRY(rows_check(&there, d, n_kv, false, fn, "to"));
            SLHA_TRY(cache_words(fn, {to->rows}));
        }
        if (heads->norm) {
            if (!std::isfinite(heads->eps) || heads->eps < 0.0f) return Status(SLHA_ERR_NONFINITE, name("eps must be finite and not negative"));
            for (const float* w : {heads->q_weight, heads->k_weight})  // (read word by word)
                if (!cache_aligned(w) && (reinterpret_cast<uintptr_t>(w) % 4 || !is_device_ptr(w)))
                    return Status(SLHA_ERR_DIMENSION, name("weights must begin on a multiple of 4 bytes in device memory, of 16 in host memory"));
        } else if (heads->q_weight || heads->k_weight) {
            return Status(SLHA_ERR_DIMENSION, name("weights are given, but no norm"));
        }
        if (rotation) {
            if (!rotation->frequencies || !rotation->positions) return Status(SLHA_ERR_NULL, name("frequencies or positions are NULL"));
            if (rotation->rotary_dim == 0 || rotation->rotary_dim > d || rotation->rotary_dim % 8)
                return Status(SLHA_ERR_DIMENSION, name("rotary_dim must be a multiple of 8 in 8..head_dim"));
            if (rotation->n_axes == 0 || rotation->n_axes > 256 || (rotation->n_axes > 1 && !rotation->axes))
                return Status(SLHA_ERR_DIMENSION, name("n_axes must be in 1..256, and axes given for more than one"));
            if (!std::isfinite(rotation->magnitude)) return Status(SLHA_ERR_NONFINITE, name("magnitude is not finite"));
            SLHA_TRY(cache_words(fn, {rotation->frequencies, rotation->positions}));
            if (rotation->axes && !is_device_ptr(rotation->axes))
                for (uint32_t p = 0; p < rotation->rotary_dim / 2; ++p)
                    if (rotation->axes[p] >= rotation->n_axes) return Status(SLHA_ERR_DIMENSION, name("an axis is not below n_axes"));
        }
        std::vector<SlhaB200Segment> segs;
        bool device_segs = false;
        const uint32_t* rows = n_kv && segments ? to->rows : nullptr;
        if (segments) cache_host_segments(segments, n_segments, &segs, &device_segs);
        else segs.push_back(SlhaB200Segment{0, heads->n_tokens, 0, heads->n_tokens, 0});
        const auto check_segments = [&]() -> Status {
            const Written w(Written::TOKENS, segs, segs, rows), turned(Written::QUERIES, segs, segs, nullptr);
            SLHA_TRY(token_segments(segs, heads->n_tokens, n_kv ? &w : nullptr, fn));
            if (n_kv) SLHA_TRY(rows_to_apart(&there, w, fn));
            if (heads->q) SLHA_TRY(rows_apart((unsigned __int128)q_out_token_stride * e, (unsigned __int128)q_out_head_stride * e, heads->n_heads, d * e, turned, fn, "q_out"));
            const auto tokens = [&](size_t i) { return std::pair<uint64_t, uint64_t>(segs[i].query_begin, (uint64_t)segs[i].query_begin + segs[i].n_queries); };
            return heads->q && cache_overlap(segs.size(), tokens) ? Status(SLHA_ERR_DIMENSION, name("two segments have the same tokens")) : Status();
        };
        if (!device_segs) SLHA_TRY(check_segments());
        CallScope cs;
        if (!cs.ok()) return cs.st;
        Ctx* c = cs.c;
        if (segments) {
            SLHA_TRY(cache_device_segments(c, segments, &segs, device_segs, fn));
            if (device_segs) SLHA_TRY(check_segments());
        }
        RotateArgs a{};
        const auto in = [&](const void* p, const unsigned char** at, const char* what) -> Status {
            if (p) SLHA_TRY(cache_device_memory(c, p, fn, what));
            *at = static_cast<const unsigned char*>(p);
            return Status();
        };
        SLHA_TRY(in(heads->q, &a.q, "q"));
        SLHA_TRY(in(heads->k, &a.k, "k"));
        SLHA_TRY(in(heads->v, &a.v, "v"));
        const unsigned char* at;
        if (heads->q) {
            SLHA_TRY(in(q_out, &at, "q_out"));
            a.q_out = const_cast<unsigned char*>(at);
        }
        if (heads->k) {
            SLHA_TRY(in(to->keys, &at, "keys"));
            a.k_out = const_cast<unsigned char*>(at);
            a.kors = to->key_row_stride * e;
            a.kohs = to->key_head_stride * e;
        }
        if (heads->v) {
            SLHA_TRY(in(to->values, &at, "values"));
            a.v_out = const_cast<unsigned char*>(at);
            a.vors = to->value_row_stride * e;
            a.vohs = to->value_head_stride * e;
        }
        a.qts = heads->q_token_stride * e;
        a.qhs = heads->q_head_stride * e;
        a.kts = heads->k_token_stride * e;
        a.khs = heads->k_head_stride * e;
        a.vts = heads->v_token_stride * e;
        a.vhs = heads->v_head_stride * e;
        a.qots = q_out_token_stride * e;
        a.qohs = q_out_head_stride * e;
        a.n_heads = heads->n_heads;
        a.n_kv = n_kv;
        a.d = d;
        a.n_tokens = heads->n_tokens;
        a.norm = heads->norm != 0;
        a.eps = heads->eps;
        if (rows) SLHA_TRY(cache_stage(c, rows, n_segments, &a.counts, fn, "rows"));
        if (heads->norm) {
            SLHA_TRY(cache_stage(c, heads->q_weight, d, &a.q_weight, fn, "q_weight"));
            SLHA_TRY(cache_stage(c, heads->k_weight, d, &a.k_weight, fn, "k_weight"));
        }
        if (rotation) {
            a.rotary = rotation->rotary_dim;
            a.n_axes = rotation->n_axes;
            a.interleaved = rotation->interleaved != 0;
            a.magnitude = rotation->magnitude;
            SLHA_TRY(cache_stage(c, rotation->frequencies, rotation->rotary_dim / 2, &a.freq, fn, "frequencies"));
            SLHA_TRY(cache_stage(c, rotation->axes, rotation->rotary_dim / 2, &a.axes, fn, "axes"));
            SLHA_TRY(cache_stage(c, rotation->positions, (size_t)rotation->n_axes * heads->n_tokens, &a.positions, fn, "positions"));
        }
        SLHA_TRY(launch_rotate_heads(c, a, heads->dtype, segs));
        if (sync_by_default(c)) SLHA_CUDA(cudaStreamSynchronize(c->stream));
        return Status();
    });
}

}  // extern "C"
