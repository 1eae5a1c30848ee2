// Part 2 of the C ABI, the cache of key and value rows: argument checks of slha_b200_attend_cache, _attend_tree, _observe_cache and _evict_cache.
// Included at the end of capi.cu.
#pragma once

namespace {

// Memory that kernels of the calling thread's device read or write in place.
Status cache_device_memory(Ctx* c, const void* p, const char* fn, const char* what, bool* host = nullptr) {
    cudaPointerAttributes at;
    const bool known = cudaPointerGetAttributes(&at, p) == cudaSuccess;
    if (!known) cudaGetLastError();
    if (host) {  // (asked for: memory of the host is no fault)
        *host = !known || (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged);
        if (*host) return Status();
    }
    if (!known || (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged))
        return Status(SLHA_ERR_DEVICE, std::string(fn) + ": " + what + " must be device memory");
    if (at.type == cudaMemoryTypeDevice && at.device != c->device)
        return Status(SLHA_ERR_DEVICE, std::string(fn) + ": " + what + " lies on another device than the calling thread's");
    return Status();
}
// Short arrays, host or device; host ones cannot be captured.  They are copied before the call returns, from page-locked memory too, which a copy on the stream would read later.
template <typename T>
Status cache_stage(Ctx* c, const T* p, size_t n, const T** dev, const char* fn, const char* what) {
    *dev = p;
    if (!p || !n) return Status();
    bool host;
    SLHA_TRY(cache_device_memory(c, p, fn, what, &host));
    if (!host) return Status();
    void* d;
    SLHA_TRY(ctx_upload(c, p, n * sizeof(T), &d));
    *dev = static_cast<const T*>(d);
    return Status();
}
// A table in device memory is read behind the caller's work on this stream; one in host memory is there before the device is asked for anything.
void cache_host_segments(const SlhaB200Segment* segments, size_t n, std::vector<SlhaB200Segment>* out, bool* on_device) {
    out->resize(n);
    *on_device = n && is_device_ptr(segments);
    if (n && !*on_device) std::memcpy(out->data(), segments, n * sizeof(SlhaB200Segment));
}
Status cache_device_segments(Ctx* c, const SlhaB200Segment* segments, std::vector<SlhaB200Segment>* out, bool on_device, const char* fn) {
    if (on_device) {
        SLHA_TRY(ctx_no_capture(c));
        SLHA_TRY(cache_device_memory(c, segments, fn, "segments"));
        SLHA_CUDA(cudaMemcpyAsync(out->data(), segments, out->size() * sizeof(SlhaB200Segment), cudaMemcpyDeviceToHost, c->stream));
        SLHA_CUDA(cudaStreamSynchronize(c->stream));
    }
    if (out->size() > CACHE_TABLE) SLHA_TRY(ctx_no_capture(c));
    return Status();
}
bool cache_aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
// Arrays of single words begin on a word: the GPU faults on others.
Status cache_words(const char* fn, std::initializer_list<const void*> arrays) {
    for (const void* p : arrays)
        if (reinterpret_cast<uintptr_t>(p) % 4) return Status(SLHA_ERR_DIMENSION, std::string(fn) + ": positions, documents, counts, slopes, lse and weights must begin on a multiple of 4 bytes");
    return Status();
}

Status cache_check(const SlhaB200KvCache* k, const char* fn, bool with_values) {
    const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
    if (!k->keys || (with_values && !k->values)) return Status(SLHA_ERR_NULL, name("keys or values are NULL"));
    if (k->dtype != SLHA_B200_F32 && k->dtype != SLHA_B200_BF16) return Status(SLHA_ERR_DIMENSION, name("dtype must be SLHA_B200_F32 or SLHA_B200_BF16"));
    const size_t each = 16 / key_elem_bytes(k->dtype);
    if (k->head_dim == 0 || k->head_dim > CACHE_DIM_MOST || k->head_dim % each)
        return Status(SLHA_ERR_DIMENSION, name("head_dim must be a multiple of 16 bytes in 1..256 elements"));
    if (k->n_kv_heads == 0 || k->n_kv_heads > 65535) return Status(SLHA_ERR_DIMENSION, name("n_kv_heads must be in 1..65535"));
    if (k->key_row_stride % each || k->key_head_stride % each || (with_values && (k->value_row_stride % each || k->value_head_stride % each)))
        return Status(SLHA_ERR_DIMENSION, name("row and head strides must be multiples of 16 bytes"));
    if (!cache_aligned(k->keys) || (with_values && !cache_aligned(k->values))) return Status(SLHA_ERR_DIMENSION, name("keys and values must begin on a multiple of 16 bytes"));
    return cache_words(fn, {k->positions, k->documents, k->rows});
}
Status cache_memory(Ctx* c, const SlhaB200KvCache* k, const char* fn, bool with_values) {
    const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
    SLHA_TRY(cache_device_memory(c, k->keys, fn, "keys"));
    if (with_values) SLHA_TRY(cache_device_memory(c, k->values, fn, "values"));
    if (k->positions) SLHA_TRY(cache_device_memory(c, k->positions, fn, "positions of rows"));
    if (k->documents) SLHA_TRY(cache_device_memory(c, k->documents, fn, "documents of rows"));
    return Status();
}
// Rows of a table whose last position, index_base + n_tiles - 1, no longer fits.
Status cache_positions_fit(const std::vector<SlhaB200Segment>& segs, const char* fn) {
    for (const SlhaB200Segment& s : segs)
        if ((uint64_t)s.index_base + s.n_tiles > 0x100000000ull || s.n_tiles > 0xFFFFFF00u)
            return Status(SLHA_ERR_DIMENSION, std::string(fn) + ": index_base + n_tiles exceeds 2^32");
    return Status();
}

// Whether two of n ranges (first, behind the last) share something.
template <typename F>
bool cache_overlap(size_t n, F range) {
    uint64_t end = 0;
    size_t i = 0;
    for (; i < n; ++i) {  // (most tables are in order)
        const auto [from, to] = range(i);
        if (from >= to) continue;
        if (from < end) break;
        end = to;
    }
    if (i == n) return false;
    std::vector<std::pair<uint64_t, uint64_t>> r;
    for (i = 0; i < n; ++i)
        if (range(i).first < range(i).second) r.push_back(range(i));
    std::sort(r.begin(), r.end());
    for (i = 1; i < r.size(); ++i)
        if (r[i].first < r[i - 1].second) return true;
    return false;
}
// Rows that a call writes, or whose weights it does, belong to one segment each.  (Row counts in device memory are not known here: the caller's to see to.)
Status cache_own_rows(const std::vector<SlhaB200Segment>& segs, const std::vector<SlhaB200Segment>& at, const uint32_t* rows, uint32_t most, const char* fn) {
    if (segs.size() < 2 || (rows && is_device_ptr(rows))) return Status();
    const auto range = [&](size_t i) {
        return std::pair<uint64_t, uint64_t>(at[i].tile_begin, at[i].tile_begin + std::min({segs[i].n_tiles, rows ? rows[i] : segs[i].n_tiles, most}));
    };
    return cache_overlap(segs.size(), range) ? Status(SLHA_ERR_DIMENSION, std::string(fn) + ": two segments have the same rows") : Status();
}

Status cache_check_queries(const SlhaB200KvCache* k, const SlhaB200CacheQueries* q, const char* fn) {
    const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
    const size_t each = 16 / key_elem_bytes(k->dtype);
    if (!q->q) return Status(SLHA_ERR_NULL, name("q is NULL"));
    if (q->n_heads == 0 || q->n_heads % k->n_kv_heads) return Status(SLHA_ERR_DIMENSION, name("n_heads must be a positive multiple of n_kv_heads"));
    if (q->token_stride % each || q->head_stride % each || !cache_aligned(q->q))
        return Status(SLHA_ERR_DIMENSION, name("q must begin on a multiple of 16 bytes and its strides be multiples of 16 bytes"));
    if (!std::isfinite(q->scale) || !std::isfinite(q->softcap) || q->softcap < 0.0f)
        return Status(SLHA_ERR_NONFINITE, name("scale must be finite, softcap finite and not negative"));
    if (q->softcap > 0.0f && !std::isfinite(q->scale / q->softcap)) return Status(SLHA_ERR_NONFINITE, name("scale / softcap must be finite"));
    // (in units of log 2; tanh(scale / softcap * product) of a larger cap would lose the small scores, and a factor below the smallest normal number its bits)
    if (!std::isfinite(q->scale * 1.4426950408889634f)) return Status(SLHA_ERR_NONFINITE, name("scale / log 2 must be finite"));
    if (q->softcap > 0x1p100f || (q->softcap > 0.0f && q->scale != 0.0f && !std::isnormal(q->scale / q->softcap)))
        return Status(SLHA_ERR_NONFINITE, name("softcap must be at most 2^100, and scale / softcap a normal float32"));
    if (k->positions && !q->positions) return Status(SLHA_ERR_NULL, name("the cache's rows have positions, the queries have none"));
    if ((k->documents != nullptr) != (q->documents != nullptr)) return Status(SLHA_ERR_NULL, name("documents must be given for rows and queries, or for neither"));
    return cache_words(fn, {q->slopes, q->prefix, q->positions, q->documents});
}
Status cache_check_segments(const SlhaB200KvCache* k, const std::vector<SlhaB200Segment>& segs, const SlhaB200CacheQueries* q, bool tree, const char* fn) {
    const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
    for (const SlhaB200Segment& s : segs) {
        if ((uint64_t)s.query_begin + s.n_queries > q->n_tokens) return Status(SLHA_ERR_DIMENSION, name("a segment's query tokens reach beyond n_tokens"));
        if ((uint64_t)s.n_queries * (q->n_heads / k->n_kv_heads) > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, name("too many query rows in a segment"));
        if (!q->positions && (uint64_t)s.index_base + s.n_queries > 0x100000000ull) return Status(SLHA_ERR_DIMENSION, name("index_base + n_queries exceeds 2^32"));
        if (tree && (s.n_queries > TREE_MOST || s.n_queries > s.n_tiles))
            return Status(SLHA_ERR_DIMENSION, name("a segment's drafted tokens are at most 256, and its last rows are theirs"));
    }
    return cache_positions_fit(segs, fn);
}
// What attention and observation share: cache and queries into the kernels' arguments.
Status cache_arguments(Ctx* c, const SlhaB200KvCache* k, size_t n_segs, const SlhaB200CacheQueries* q, const char* fn, CacheArgs* a) {
    const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
    SLHA_TRY(cache_device_memory(c, q->q, fn, "q"));
    *a = CacheArgs{};
    a->keys = k->keys;
    a->values = k->values;
    a->q = q->q;
    a->krs = k->key_row_stride;
    a->khs = k->key_head_stride;
    a->vrs = k->value_row_stride;
    a->vhs = k->value_head_stride;
    a->qts = q->token_stride;
    a->qhs = q->head_stride;
    a->row_pos = k->positions;
    a->row_doc = k->documents;
    a->entry_hs = k->entry_head_stride;
    SLHA_TRY(cache_stage(c, k->rows, n_segs, &a->rows, fn, "rows"));
    SLHA_TRY(cache_stage(c, q->positions, q->n_tokens, &a->q_pos, fn, "positions of queries"));
    SLHA_TRY(cache_stage(c, q->documents, q->n_tokens, &a->q_doc, fn, "documents of queries"));
    SLHA_TRY(cache_stage(c, q->prefix, n_segs, &a->prefix, fn, "prefix"));
    SLHA_TRY(cache_stage(c, q->slopes, q->n_heads, &a->slopes, fn, "slopes"));
    a->n_kv = k->n_kv_heads;
    a->n_heads = q->n_heads;
    a->group = q->n_heads / k->n_kv_heads;
    a->d = k->head_dim;
    a->n_tokens = q->n_tokens;
    a->scale = q->scale;
    a->cap = q->softcap;
    a->window_last = q->window ? q->window - 1 : 0xFFFFFFFFu;
    a->causal = q->causal != 0;
    return Status();
}

int32_t attend_cache_any(const char* fn, const SlhaB200KvCache* cache, const SlhaB200Segment* segments, size_t n_segments, const SlhaB200CacheQueries* queries,
                         const uint32_t* parents, bool tree, void* out, uint64_t out_token_stride, uint64_t out_head_stride, float* lse_out) {
    return ffi([&]() -> Status {
        g_cache_kernels = 0;
        const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
        if (!cache || !queries || (n_segments && !segments)) return Status(SLHA_ERR_NULL, std::string(fn) + " received a NULL pointer");
        if (n_segments == 0 || queries->n_tokens == 0) return Status();
        if (!out || (tree && !parents)) return Status(SLHA_ERR_NULL, std::string(fn) + " received a NULL pointer");
        SLHA_TRY(cache_check(cache, fn, true));
        SLHA_TRY(cache_check_queries(cache, queries, fn));
        SLHA_TRY(cache_words(fn, {parents, lse_out}));
        const size_t each = 16 / key_elem_bytes(cache->dtype);
        if (out_token_stride % each || out_head_stride % each || !cache_aligned(out))
            return Status(SLHA_ERR_DIMENSION, name("out must begin on a multiple of 16 bytes and its strides be multiples of 16 bytes"));
        std::vector<SlhaB200Segment> segs;
        bool device_segs;
        cache_host_segments(segments, n_segments, &segs, &device_segs);
        const auto check_segments = [&]() -> Status {
            SLHA_TRY(cache_check_segments(cache, segs, queries, tree, fn));
            const auto tokens = [&](size_t i) { return std::pair<uint64_t, uint64_t>(segs[i].query_begin, (uint64_t)segs[i].query_begin + segs[i].n_queries); };
            return cache_overlap(segs.size(), tokens) ? Status(SLHA_ERR_DIMENSION, name("two segments have the same query tokens")) : Status();
        };
        if (!device_segs) SLHA_TRY(check_segments());
        CallScope cs;
        if (!cs.ok()) return cs.st;
        Ctx* c = cs.c;
        SLHA_TRY(cache_device_segments(c, segments, &segs, device_segs, fn));
        if (device_segs) SLHA_TRY(check_segments());
        SLHA_TRY(cache_memory(c, cache, fn, true));
        SLHA_TRY(cache_device_memory(c, out, fn, "out"));
        if (lse_out) SLHA_TRY(cache_device_memory(c, lse_out, fn, "lse_out"));
        CacheArgs a;
        SLHA_TRY(cache_arguments(c, cache, n_segments, queries, fn, &a));
        if (tree) {
            SLHA_TRY(cache_stage(c, parents, queries->n_tokens, &a.parents, fn, "parents"));
            a.tree = 1;
        }
        a.out = out;
        a.ots = out_token_stride;
        a.ohs = out_head_stride;
        a.lse = lse_out;
        SLHA_TRY(launch_attend_cache(c, a, cache->dtype, segs));
        if (sync_by_default(c)) SLHA_CUDA(cudaStreamSynchronize(c->stream));
        return Status();
    });
}

}  // namespace

extern "C" {

int32_t slha_b200_debug_last_cache_kernels(uint32_t* out) {
    return ffi([&]() -> Status {
        if (!out) return Status(SLHA_ERR_NULL, "slha_b200_debug_last_cache_kernels received a NULL pointer");
        *out = g_cache_kernels;
        return Status();
    });
}

int32_t slha_b200_attend_cache(const SlhaB200KvCache* cache, const SlhaB200Segment* segments, size_t n_segments, const SlhaB200CacheQueries* queries, void* out,
                               uint64_t out_token_stride, uint64_t out_head_stride, float* lse_out) {
    return attend_cache_any("slha_b200_attend_cache", cache, segments, n_segments, queries, nullptr, false, out, out_token_stride, out_head_stride, lse_out);
}
int32_t slha_b200_attend_tree(const SlhaB200KvCache* cache, const SlhaB200Segment* segments, size_t n_segments, const SlhaB200CacheQueries* queries,
                              const uint32_t* parents, void* out, uint64_t out_token_stride, uint64_t out_head_stride, float* lse_out) {
    return attend_cache_any("slha_b200_attend_tree", cache, segments, n_segments, queries, parents, true, out, out_token_stride, out_head_stride, lse_out);
}

int32_t slha_b200_observe_cache(const SlhaB200KvCache* cache, const SlhaB200Segment* segments, size_t n_segments, const SlhaB200CacheQueries* queries,
                                const float* lse, const float* weights_in, float decay, float* weights_out, uint64_t weight_head_stride) {
    return ffi([&]() -> Status {
        g_cache_kernels = 0;
        const char* fn = "slha_b200_observe_cache";
        const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
        if (!cache || !queries || !lse || !weights_out || (n_segments && !segments)) return Status(SLHA_ERR_NULL, std::string(fn) + " received a NULL pointer");
        if (n_segments == 0) return Status();
        if (!std::isfinite(decay)) return Status(SLHA_ERR_NONFINITE, name("decay is not finite"));
        SLHA_TRY(cache_check(cache, fn, false));
        SLHA_TRY(cache_check_queries(cache, queries, fn));
        SLHA_TRY(cache_words(fn, {lse, weights_in, weights_out}));
        std::vector<SlhaB200Segment> segs;
        bool device_segs;
        cache_host_segments(segments, n_segments, &segs, &device_segs);
        const auto check_segments = [&]() -> Status {
            SLHA_TRY(cache_check_segments(cache, segs, queries, false, fn));
            return cache_own_rows(segs, segs, cache->rows, 0xFFFFFFFFu, fn);
        };
        if (!device_segs) SLHA_TRY(check_segments());
        CallScope cs;
        if (!cs.ok()) return cs.st;
        Ctx* c = cs.c;
        SLHA_TRY(cache_device_segments(c, segments, &segs, device_segs, fn));
        if (device_segs) SLHA_TRY(check_segments());
        SLHA_TRY(cache_memory(c, cache, fn, false));
        SLHA_TRY(cache_device_memory(c, lse, fn, "lse"));
        SLHA_TRY(cache_device_memory(c, weights_out, fn, "weights_out"));
        if (weights_in) SLHA_TRY(cache_device_memory(c, weights_in, fn, "weights_in"));
        CacheArgs a;
        SLHA_TRY(cache_arguments(c, cache, n_segments, queries, fn, &a));
        a.lse_in = lse;
        a.w_in = weights_in;
        a.w_out = weights_out;
        a.w_hs = weight_head_stride;
        a.decay = decay;
        SLHA_TRY(launch_observe_cache(c, a, cache->dtype, segs));
        if (sync_by_default(c)) SLHA_CUDA(cudaStreamSynchronize(c->stream));
        return Status();
    });
}

int32_t slha_b200_evict_cache(const SlhaB200KvCache* cache, const SlhaB200Segment* segments, size_t n_segments, const SlhaB200CacheEviction* ev) {
    return ffi([&]() -> Status {
        g_cache_kernels = 0;
        const char* fn = "slha_b200_evict_cache";
        const auto name = [&](const char* what) { return std::string(fn) + ": " + what; };
        if (!cache || !ev || (n_segments && !segments) || (ev && (!ev->weights || (ev->to && !ev->to_segments))))
            return Status(SLHA_ERR_NULL, std::string(fn) + " received a NULL pointer");
        if (n_segments == 0) return Status();
        if (ev->budget == 0) return Status(SLHA_ERR_DIMENSION, name("budget must be at least 1"));
        const SlhaB200KvCache* to = ev->to ? ev->to : cache;
        const bool in_place = !ev->to;
        if (to->dtype != cache->dtype || to->head_dim != cache->head_dim || to->n_kv_heads != cache->n_kv_heads)
            return Status(SLHA_ERR_DIMENSION, name("both caches must have the same dtype, head_dim and n_kv_heads"));
        if ((to->positions && !cache->positions) || (to->documents && !cache->documents))
            return Status(SLHA_ERR_NULL, name("positions or documents are to be moved, but the rows have none"));
        if ((to->positions || to->documents) && to->n_kv_heads > 1 && to->entry_head_stride == 0)
            return Status(SLHA_ERR_DIMENSION, name("each KV head keeps other rows: positions and documents must be its own where they go (entry_head_stride > 0)"));
        if (ev->tiles && !in_place && !ev->tiles_to) return Status(SLHA_ERR_NULL, name("tiles are given without tiles_to"));
        if (in_place && ev->weights_to && (ev->weights_to != ev->weights || ev->weights_to_head_stride != ev->weight_head_stride))
            return Status(SLHA_ERR_DIMENSION, name("in place, weights_to is the array of weights or NULL"));
        if (in_place && ev->tiles_to && (ev->tiles_to != ev->tiles || ev->tiles_to_head_stride != ev->tile_head_stride))
            return Status(SLHA_ERR_DIMENSION, name("in place, tiles_to is the array of tiles or NULL"));
        SciRustSlhaTile* tiles_to = in_place ? const_cast<SciRustSlhaTile*>(ev->tiles) : ev->tiles_to;
        if (ev->tiles && (!cache_aligned(ev->tiles) || !cache_aligned(tiles_to))) return Status(SLHA_ERR_DIMENSION, name("tiles must begin on a multiple of 16 bytes"));
        // (the heads keep the same rows where they share the weights, and the positions too or no row is kept for its position)
        const bool alike = cache->n_kv_heads == 1 || (ev->weight_head_stride == 0 && (!cache->positions || cache->entry_head_stride == 0 || (!ev->sink_window && !ev->recent_window)));
        if (!alike && ev->weights_to && (in_place ? ev->weight_head_stride : ev->weights_to_head_stride) == 0)
            return Status(SLHA_ERR_DIMENSION, name("each KV head keeps other rows: weights_to must be its own (weights_to_head_stride > 0)"));
        if (!alike && ev->tiles && (in_place ? ev->tile_head_stride : ev->tiles_to_head_stride) == 0)
            return Status(SLHA_ERR_DIMENSION, name("each KV head keeps other rows: tiles must be its own where they go (tiles_to_head_stride > 0)"));
        if (!alike && (to->key_head_stride == 0 || to->value_head_stride == 0))
            return Status(SLHA_ERR_DIMENSION, name("each KV head keeps other rows: rows must be its own where they go (head strides > 0)"));
        SLHA_TRY(cache_check(cache, fn, true));
        if (!in_place) SLHA_TRY(cache_check(to, fn, true));
        SLHA_TRY(cache_words(fn, {ev->weights, ev->weights_to, ev->source_out, ev->rows_out}));
        std::vector<SlhaB200Segment> segs, to_segs;
        bool device_segs, device_to = false;
        cache_host_segments(segments, n_segments, &segs, &device_segs);
        if (!in_place) cache_host_segments(ev->to_segments, n_segments, &to_segs, &device_to);
        const auto check_segments = [&]() -> Status {
            SLHA_TRY(cache_positions_fit(segs, fn));
            for (size_t i = 0; i < to_segs.size(); ++i)
                if (to_segs[i].n_tiles < std::min(segs[i].n_tiles, ev->budget))
                    return Status(SLHA_ERR_CAPACITY, name("segment ") + std::to_string(i) + " of the other cache has no room for the rows that stay");
            return cache_own_rows(segs, in_place ? segs : to_segs, cache->rows, in_place ? 0xFFFFFFFFu : ev->budget, fn);
        };
        if (!device_segs && !device_to) SLHA_TRY(check_segments());
        CallScope cs;
        if (!cs.ok()) return cs.st;
        Ctx* c = cs.c;
        SLHA_TRY(cache_device_segments(c, segments, &segs, device_segs, fn));
        if (!in_place) SLHA_TRY(cache_device_segments(c, ev->to_segments, &to_segs, device_to, fn));
        if (device_segs || device_to) SLHA_TRY(check_segments());
        SLHA_TRY(cache_memory(c, cache, fn, true));
        if (!in_place) SLHA_TRY(cache_memory(c, to, fn, true));
        SLHA_TRY(cache_device_memory(c, ev->weights, fn, "weights"));
        if (ev->weights_to) SLHA_TRY(cache_device_memory(c, ev->weights_to, fn, "weights_to"));
        if (ev->tiles) {
            SLHA_TRY(cache_device_memory(c, ev->tiles, fn, "tiles"));
            SLHA_TRY(cache_device_memory(c, tiles_to, fn, "tiles_to"));
        }
        if (ev->source_out) SLHA_TRY(cache_device_memory(c, ev->source_out, fn, "source_out"));
        if (ev->rows_out) SLHA_TRY(cache_device_memory(c, ev->rows_out, fn, "rows_out"));
        EvictArgs a{};
        const uint64_t e = key_elem_bytes(cache->dtype);
        a.keys = cache->keys;
        a.values = cache->values;
        a.to_keys = const_cast<void*>(to->keys);
        a.to_values = const_cast<void*>(to->values);
        a.krs = cache->key_row_stride * e;
        a.khs = cache->key_head_stride * e;
        a.vrs = cache->value_row_stride * e;
        a.vhs = cache->value_head_stride * e;
        a.tkrs = to->key_row_stride * e;
        a.tkhs = to->key_head_stride * e;
        a.tvrs = to->value_row_stride * e;
        a.tvhs = to->value_head_stride * e;
        a.pos = cache->positions;
        a.doc = cache->documents;
        a.to_pos = const_cast<uint32_t*>(to->positions);
        a.to_doc = const_cast<uint32_t*>(to->documents);
        a.entry_hs = cache->entry_head_stride;
        a.to_entry_hs = to->entry_head_stride;
        a.w = ev->weights;
        a.to_w = ev->weights_to;
        a.w_hs = ev->weight_head_stride;
        a.to_w_hs = ev->weights_to_head_stride;
        a.tiles = reinterpret_cast<const unsigned char*>(ev->tiles);
        a.to_tiles = reinterpret_cast<unsigned char*>(tiles_to);
        a.tile_hs = ev->tile_head_stride;
        a.to_tile_hs = in_place ? ev->tile_head_stride : ev->tiles_to_head_stride;
        SLHA_TRY(cache_stage(c, cache->rows, n_segments, &a.rows, fn, "rows"));
        a.rows_out = ev->rows_out;
        a.source = ev->source_out;
        a.n_kv = cache->n_kv_heads;
        a.row_bytes = (uint32_t)(cache->head_dim * e);
        a.budget = ev->budget;
        a.sink = ev->sink_window;
        a.recent = ev->recent_window;
        a.in_place = in_place;
        SLHA_TRY(launch_evict_cache(c, a, segs, to_segs));
        if (sync_by_default(c)) SLHA_CUDA(cudaStreamSynchronize(c->stream));
        return Status();
    });
}

}  // extern "C"
