// A cache of key and value rows in 4 bits, and the norms and rotation of heads on their way into a cache: what rotate.cu, cache4_rows.cu and cache4_attend.cu
// share and the launchers that the C ABI calls (capi_cache4.cuh).
//
// Blocks of 16 elements along a row of a head: a scale in e4m3 (4 significant bits), elements in e2m1 (2 significant bits), the value their product times a power of two.  A
// product has 6 significant bits and lies between 2^-10 and 2688: exact in float16 and in bfloat16, so that what the codes stand for goes to the tensor cores as it is.
#pragma once

#include "cache.cuh"

namespace slha {

constexpr uint32_t BLOCK4 = 16;  // elements of a scale
// Bytes of the rows that a launch lays out for attention by many tokens (a segment's own may be more).
constexpr uint64_t CACHE4_ROWS_MOST = 512ull << 20;

// Where 4-bit rows lie; strides in bytes.
struct Rows4 {
    const unsigned char *codes[2], *scales[2];  // keys, values
    uint64_t crs, chs, srs, shs;
    int32_t exponent[2];
};
// Rows of float32 or bfloat16; strides in bytes, null where there are none.
struct RowsOf {
    const unsigned char* p[2];
    uint64_t rs[2], hs[2];
};
struct Rows4Args {
    Rows4 in4;
    RowsOf rows;
    const uint32_t *counts, *pos, *doc;  // pos, doc: entries to be laid out with the rows, to_pos and to_doc
    uint32_t *to_pos, *to_doc;
    uint64_t entry_hs, to_entry_hs;
    const CacheSeg* table;
    uint32_t seen_last;  // reading: rows further than this before a segment's first token are left out; 0xFFFFFFFF: none are
    uint32_t n_segs, n_kv, d, entries;                                      // entries: heads whose entries are laid out
    uint32_t each, units, columns, passes, step, per_column, per_unit;  // rows of a work item and what a thread takes of them, see cache4_rows.cu
};
// One call's heads: strides in bytes.
struct RotateArgs {
    const unsigned char *q, *k, *v;
    unsigned char *q_out, *k_out, *v_out;
    uint64_t qts, qhs, kts, khs, vts, vhs, qots, qohs, kors, kohs, vors, vohs;
    const float *q_weight, *k_weight, *freq;
    const uint8_t* axes;
    const uint32_t *positions, *counts;
    const CacheSeg* table;
    float eps, magnitude, per_dim;  // per_dim: 1 / d
    uint32_t n_segs, n_heads, n_kv, d, rotary, n_axes, n_tokens, each;  // each: tokens of a work item
    int32_t norm, interleaved;
};

// Rows of a segment into 4 bits (write: the segment's tokens' rows) or back.  to_segs: where a segment's rows go.
Status launch_write_cache4(Ctx* c, Rows4Args a, int dtype, const std::vector<SlhaB200Segment>& segs);
Status launch_read_cache4(Ctx* c, Rows4Args a, int dtype, const std::vector<SlhaB200Segment>& segs, const std::vector<SlhaB200Segment>& to_segs);
Status launch_rotate_heads(Ctx* c, RotateArgs a, int dtype, const std::vector<SlhaB200Segment>& segs);
// a: queries, masks and outputs as for launch_attend_cache, its scale with the keys' exponent; keys, values and their strides are r's.
Status launch_attend_cache4(Ctx* c, CacheArgs a, const Rows4& r, int dtype, const std::vector<SlhaB200Segment>& segs);

#ifdef __CUDACC__
// The two elements of byte B of a word as float16.
template <int B>
__device__ __forceinline__ uint32_t e2m1_pair(uint32_t w) {
    uint32_t r;
    asm("{\n.reg .b8 b<4>;\nmov.b32 {b0, b1, b2, b3}, %1;\ncvt.rn.f16x2.e2m1x2 %0, b%2;\n}\n" : "=r"(r) : "r"(w), "n"(B));
    return r;
}
// Two scales as float16.
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"((uint16_t)two));
    return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
#endif

}  // namespace slha
