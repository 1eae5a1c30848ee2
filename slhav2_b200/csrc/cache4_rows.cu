// Rows of keys and values into 4 bits and back (slha_b200_write_cache4, slha_b200_read_cache4, and the rows that attention by many tokens has laid out).
//
// Of a block of 16 elements x of a row of a head, with e the cache's exponent:  s = e4m3(max |x| / (6 2^e)),  code = e2m1(x / (s 2^e)),  value = code s 2^e.
// A quotient is rounded once more where it becomes 3 bits: where its own rounding could land it on the border of two codes that x does not lie on, the last bit says
// that something was cut off (rounding to odd), so that every code and scale is what the formula gives in exact arithmetic.
//
// Bound by bytes, 2 or 4 in for 9/16 out an element: a thread takes 8 elements (16 bytes of bfloat16, 4 of codes), four such units of a work item are under way at a time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "cache4.cuh"

namespace slha {
namespace {

constexpr int ROW_THREADS = 256, FLIGHT = 4;

// Unit u of a work item, counted through its rows, heads and units of 8 elements, in steps of the block's threads.
struct UnitWalk {
    uint32_t r, h, x, dr, dh, dx, kv, units;
    __device__ __forceinline__ UnitWalk(uint32_t first, uint32_t step, uint32_t kv_, uint32_t units_) : kv(kv_), units(units_) {
        const uint32_t h_all = first / units, dh_all = step / units;
        x = first - h_all * units;
        r = h_all / kv;
        h = h_all - r * kv;
        dx = step - dh_all * units;
        dr = dh_all / kv;
        dh = dh_all - dr * kv;
    }
    __device__ __forceinline__ void next() {
        x += dx;
        h += dh;
        r += dr;
        if (x >= units) x -= units, ++h;
        if (h >= kv) h -= kv, ++r;
    }
};
// x / y (y > 0) to the nearest, for r the nearest to 1 / y: Markstein's two steps, exact remainders by fused multiply-add.
__device__ __forceinline__ float quotient(float x, float y, float r) {
    const float q = x * r;
    return fmaf(fmaf(-q, y, x), r, q);
}
// The last bit of a quotient q >= 0 of x and y says whether it is exact: to the nearest -> cut off towards zero, its last bit set where anything was.
__device__ __forceinline__ float to_odd(float q, float x, float y) {
    const float rest = fmaf(-q, y, x);
    uint32_t b = __float_as_uint(q);
    if (rest < 0.0f) --b;
    if (rest != 0.0f) b |= 1;
    return __uint_as_float(b);
}
// Bit patterns of 8 elements of T as float32.
template <typename T>
struct Eight {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const unsigned char* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void values(float (&f)[8]) const {
        if constexpr (sizeof(T) == 2) {
            const uint32_t x[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(x[i] << 16), f[2 * i + 1] = __uint_as_float(x[i] & 0xFFFF0000u);
        } else {
            const uint32_t x[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(x[i]);
        }
    }
};
__device__ __forceinline__ uint32_t e2m1_pack(float lo, float hi) {
    uint32_t r;
    asm("{\n.reg .b8 b;\ncvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\ncvt.u32.u8 %0, b;\n}\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t e4m3_of(float x) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(0.0f), "f"(x));
    return r & 0xFF;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) { return __half2float(__ushort_as_half((uint16_t)(e4m3_pair(byte) & 0xFFFF))); }

// 8 elements, half a block (the other half is the neighbouring lane's): their codes and the block's scale.
template <typename T>
__device__ __forceinline__ uint32_t quantise(const Eight<T>& in, float down, uint32_t* scale) {
    float x[8];
    in.values(x);
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
    if (most > 0x7F800000u) {  // a NaN
        *scale = 0x7F;
        return 0;
    }
    constexpr float SIXTH = 1.0f / 6.0f, LARGEST = 3.0e38f;
    const float size = fminf(__uint_as_float(most) * down, LARGEST);
    *scale = e4m3_of(to_odd(quotient(size, 6.0f, SIXTH), size, 6.0f));
    const float s = e4m3_value(*scale), r = s > 0.0f ? __frcp_rn(s) : 0.0f;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float q[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float y = fminf(fabsf(x[i + j] * down), LARGEST);
            q[j] = quotient(y, s, r);
            // (a bfloat16's quotient by the 4 bits of a scale lies on a border, of at most 3 bits, or 2^-8 of it away)
            if constexpr (sizeof(T) == 4) q[j] = to_odd(q[j], y, s);
            q[j] = copysignf(q[j], x[i + j]);
        }
        codes |= e2m1_pack(q[0], q[1]) << (4 * i);
    }
    return codes;
}

template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) write_cache4_kernel(const __grid_constant__ Rows4Args a, const __grid_constant__ CacheTable tab) {
    dep_wait();
    const CacheSeg* table = a.table ? a.table : tab.s;
    const uint32_t seg = cache_find(a.n_segs, blockIdx.x, [&](uint32_t i) { return table[i].item_begin; });
    const CacheSeg& sg = table[seg];
    const uint32_t n = a.counts ? min(a.counts[sg.seg], sg.n_rows) : sg.n_rows, ctx = n - min(n, sg.n_queries);
    const uint32_t t0 = (blockIdx.x - sg.item_begin) * a.each;  // (below n_queries)
    const uint32_t tokens = min(min(a.each, sg.n_queries - t0), n - ctx - min(n - ctx, t0));
    const int v = blockIdx.y;
    const unsigned char* from = a.rows.p[v] + (uint64_t)(sg.query_begin + t0) * a.rows.rs[v];
    unsigned char* codes = const_cast<unsigned char*>(a.in4.codes[v]) + (sg.row_begin + ctx + t0) * a.in4.crs;
    unsigned char* scales = const_cast<unsigned char*>(a.in4.scales[v]) + (sg.row_begin + ctx + t0) * a.in4.srs;
    const float down = exp2f((float)-a.in4.exponent[v]);
    UnitWalk u(threadIdx.x, ROW_THREADS, a.n_kv, a.units);
    // (the two halves of a block are neighbours: the number of units is even, and so are a warp's first and the step)
    while (__any_sync(0xFFFFFFFFu, u.r < tokens)) {
        UnitWalk w = u;
        Eight<T> in[FLIGHT];
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i, w.next()) {
            if (w.r < tokens) in[i].load(from + w.r * a.rows.rs[v] + w.h * a.rows.hs[v] + w.x * (8 * sizeof(T)));
            else in[i].clear();
        }
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i, u.next()) {
            uint32_t scale;
            const uint32_t code = quantise<T>(in[i], down, &scale);
            if (u.r >= tokens) continue;
            *reinterpret_cast<uint32_t*>(codes + u.r * a.in4.crs + u.h * a.in4.chs + u.x * 4) = code;
            if (!(u.x & 1)) scales[u.r * a.in4.srs + u.h * a.in4.shs + u.x / 2] = (unsigned char)scale;
        }
    }
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) read_cache4_kernel(const __grid_constant__ Rows4Args a, const __grid_constant__ CacheTable tab) {
    dep_wait();
    const CacheSeg* table = a.table ? a.table : tab.s;
    const uint32_t seg = cache_find(a.n_segs, blockIdx.x, [&](uint32_t i) { return table[i].item_begin; });
    const CacheSeg& sg = table[seg];
    const uint32_t n = a.counts ? min(a.counts[sg.seg], sg.n_rows) : sg.n_rows;
    const uint32_t r0 = (blockIdx.x - sg.item_begin) * a.each, rows = min(a.each, n - min(n, r0));
    const int v = blockIdx.y;
    if (v == 0)
        for (uint32_t e = 0; e < a.entries; ++e)
            for (uint32_t r = threadIdx.x; r < rows; r += ROW_THREADS) {
                const uint64_t at = e * a.entry_hs + sg.row_begin + r0 + r, to = e * a.to_entry_hs + sg.to_begin + r0 + r;
                if (a.pos) a.to_pos[to] = a.pos[at];
                if (a.doc) a.to_doc[to] = a.doc[at];
            }
    if (!a.rows.p[v]) return;
    const unsigned char* codes = a.in4.codes[v] + (sg.row_begin + r0) * a.in4.crs;
    const unsigned char* scales = a.in4.scales[v] + (sg.row_begin + r0) * a.in4.srs;
    unsigned char* to = const_cast<unsigned char*>(a.rows.p[v]) + (sg.to_begin + r0) * a.rows.rs[v];
    const float up = exp2f((float)a.in4.exponent[v]);
    UnitWalk u(threadIdx.x, ROW_THREADS, a.n_kv, a.units);
    while (u.r < rows) {
        UnitWalk w = u;
        uint32_t code[FLIGHT], scale[FLIGHT];
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i, w.next()) {
            const bool there = w.r < rows;
            code[i] = there ? *reinterpret_cast<const uint32_t*>(codes + w.r * a.in4.crs + w.h * a.in4.chs + w.x * 4) : 0;
            scale[i] = there ? scales[w.r * a.in4.srs + w.h * a.in4.shs + w.x / 2] : 0;
        }
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i, u.next()) {
            if (u.r >= rows) break;
            const uint32_t s = e4m3_pair((scale[i] & 0x7F) * 0x0101u);
            const uint32_t h[4] = {mul_f16x2(e2m1_pair<0>(code[i]), s), mul_f16x2(e2m1_pair<1>(code[i]), s), mul_f16x2(e2m1_pair<2>(code[i]), s), mul_f16x2(e2m1_pair<3>(code[i]), s)};
            float f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[2 * j] = __half2float(__ushort_as_half((uint16_t)h[j])) * up;
                f[2 * j + 1] = __half2float(__ushort_as_half((uint16_t)(h[j] >> 16))) * up;
            }
            uint4* dst = reinterpret_cast<uint4*>(to + u.r * a.rows.rs[v] + u.h * a.rows.hs[v] + u.x * (8 * sizeof(T)));
            if constexpr (sizeof(T) == 2) {
                *dst = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
            } else {
                dst[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
                dst[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
            }
        }
    }
}

// Rows of a work item: about FLIGHT units a thread, more where that would be more work items than a grid takes.
Status cut_rows(Ctx* c, Rows4Args* a, std::vector<CacheSeg>* segs, bool write, CacheTable* tab, uint32_t* items) {
    const uint32_t per_row = a->n_kv * a->units;
    uint64_t each = std::max(1u, ROW_THREADS * FLIGHT / per_row), count;
    for (;; each *= 2) {
        count = 0;
        for (CacheSeg& s : *segs) {
            s.item_begin = (uint32_t)count;
            count += ((write ? s.n_queries : s.n_rows) + each - 1) / each;
        }
        if (count <= 0x7FFFFFFFull) break;
    }
    a->each = (uint32_t)std::min<uint64_t>(each, 0xFFFFFFFFu);
    a->n_segs = (uint32_t)segs->size();
    *items = (uint32_t)count;
    return cache_table(c, *segs, tab, &a->table);
}

}  // namespace

Status launch_write_cache4(Ctx* c, Rows4Args a, int dtype, const std::vector<SlhaB200Segment>& segs) {
    std::vector<CacheSeg> of;
    for (size_t i = 0; i < segs.size(); ++i) {
        if (!segs[i].n_queries) continue;
        CacheSeg g{};
        g.row_begin = segs[i].tile_begin;
        g.n_rows = segs[i].n_tiles;
        g.query_begin = segs[i].query_begin;
        g.n_queries = segs[i].n_queries;
        g.seg = (uint32_t)i;
        of.push_back(g);
    }
    if (of.empty()) return Status();
    CacheTable tab;
    uint32_t items;
    SLHA_TRY(cut_rows(c, &a, &of, true, &tab, &items));
    SLHA_CUDA(launch_behind(dtype == SLHA_B200_BF16 ? write_cache4_kernel<__nv_bfloat16> : write_cache4_kernel<float>, dim3(items, 2), dim3(ROW_THREADS), 0, c->stream, a, tab));
    count_launch();
    return Status();
}

Status launch_read_cache4(Ctx* c, Rows4Args a, int dtype, const std::vector<SlhaB200Segment>& segs, const std::vector<SlhaB200Segment>& to_segs) {
    std::vector<CacheSeg> of;
    for (size_t i = 0; i < segs.size(); ++i) {
        if (!segs[i].n_tiles) continue;
        CacheSeg g{};
        g.row_begin = segs[i].tile_begin;
        g.n_rows = segs[i].n_tiles;
        g.seg = (uint32_t)i;
        g.to_begin = to_segs[i].tile_begin;
        of.push_back(g);
    }
    if (of.empty()) return Status();
    CacheTable tab;
    uint32_t items;
    SLHA_TRY(cut_rows(c, &a, &of, false, &tab, &items));
    SLHA_CUDA(launch_behind(dtype == SLHA_B200_BF16 ? read_cache4_kernel<__nv_bfloat16> : read_cache4_kernel<float>, dim3(items, 2), dim3(ROW_THREADS), 0, c->stream, a, tab));
    count_launch();
    return Status();
}

}  // namespace slha
