// Rows of keys and values into 4 bits and back (slha_b200_write_cache4, slha_b200_read_cache4, and the rows that attention by many tokens has laid out).
//
// Of a block of 16 elements x of a row of a head, with e the cache's exponent:  s = e4m3(max |x| / (6 2^e)),  code = e2m1(x / (s 2^e)),  value = code s 2^e.
// A quotient is rounded once more where it becomes 3 bits, so its own rounding must not land it on the border of two codes, or beside one that x lies on.  bfloat16: x / s, of 8 bits and of 4, is a
// border or 2^-8 of it away; times 1 / s as the sum of two float32 it comes out on the border exactly.  float32: the quotient's last bit says whether something was cut off (rounding to
// odd).  So every code and scale is what the formula gives in exact arithmetic.
//
// Bytes bound it, 2 or 4 in for 9/16 out an element, once few instructions do: a thread takes one column of the rows' elements, 8 of them reading (4 bytes of codes, 16 of bfloat16) and a whole block
// of 16 writing, so that its addresses grow by a constant.  32768 tokens of 8 heads of 128 dimensions: written 31.7 us = 5.4 TB/s (bfloat16; float32 58, 5.3 TB/s), read back 30.3 = 5.7 TB/s
// (float32 63, 4.9 TB/s; 9001 rows of 7 prompts, 80 dimensions, float32 35 = 3.8 TB/s: rows of 80 dimensions leave 16 of 256 threads idle).  48 tokens are one launch each way, 3 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "cache4.cuh"

namespace slha {
namespace {

// Units under way at a time: reading, of 8 elements, and writing, of 16 (32768 tokens of 8 heads of 128 dimensions written, us, with 1, 2 and 3 blocks under way: bfloat16 31.7, 38.0, 33.5; float32
// 58.8, 80.5, 74.4: what the registers take in warps costs more than the loads gain).
constexpr int ROW_THREADS = 256, FLIGHT = 4, WRITE_FLIGHT = 1;

// A thread's part of a work item: a column of the rows' kv x units units (the `pass`-th of its columns; threads beyond them have none), and every step-th row from `row` on.  What is divided by is
// known to the host: below 256, x / y is x * ceil(2^16 / y) / 2^16.
struct Column {
    uint32_t row, head, unit;
    bool there;
    __device__ __forceinline__ Column(const Rows4Args& a, uint32_t pass) {
        row = a.passes == 1 ? threadIdx.x * a.per_column >> 16 : 0;
        const uint32_t column = pass * ROW_THREADS + threadIdx.x - row * a.columns;
        there = row < a.step && column < a.columns;
        head = !there ? 0 : a.passes == 1 ? column * a.per_unit >> 16 : column / a.units;
        unit = there ? column - head * a.units : 0;
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
// A block of 16 elements of T as they lie.
template <typename T>
struct Block16 {
    uint4 w[sizeof(T)];
    __device__ __forceinline__ void load(const unsigned char* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    // elements 4 i .. 4 i + 3
    __device__ __forceinline__ void four(int i, float (&f)[4]) const {
        if constexpr (sizeof(T) == 2) {
            const uint32_t x = i & 1 ? w[i / 2].z : w[i / 2].x, y = i & 1 ? w[i / 2].w : w[i / 2].y;
            f[0] = __uint_as_float(x << 16), f[1] = __uint_as_float(x & 0xFFFF0000u), f[2] = __uint_as_float(y << 16), f[3] = __uint_as_float(y & 0xFFFF0000u);
        } else {
            f[0] = __uint_as_float(w[i].x), f[1] = __uint_as_float(w[i].y), f[2] = __uint_as_float(w[i].z), f[3] = __uint_as_float(w[i].w);
        }
    }
    // the largest size, as the bits of a float32; a NaN where there is one
    __device__ __forceinline__ uint32_t largest() const {
        if constexpr (sizeof(T) == 2) {
            const auto both = [](uint32_t x, uint32_t y) {
                uint32_t m;
                asm("max.NaN.bf16x2 %0, %1, %2;\n" : "=r"(m) : "r"(x), "r"(y));
                return m;
            };
            constexpr uint32_t M = 0x7FFF7FFFu;
            const uint32_t m = both(both(both(w[0].x & M, w[0].y & M), both(w[0].z & M, w[0].w & M)), both(both(w[1].x & M, w[1].y & M), both(w[1].z & M, w[1].w & M)));
            return max(m << 16, m & 0xFFFF0000u);
        } else {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = max(m, max(max(w[i].x & 0x7FFFFFFFu, w[i].y & 0x7FFFFFFFu), max(w[i].z & 0x7FFFFFFFu, w[i].w & 0x7FFFFFFFu)));
            return m;
        }
    }
};
__device__ __forceinline__ uint32_t e4m3_of(float x) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(0.0f), "f"(x));
    return r & 0xFF;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) { return __half2float(__ushort_as_half((uint16_t)(e4m3_pair(byte) & 0xFFFF))); }

// 1 / s to the nearest, for the scales' significands of 4 bits: two steps from an approximation.
__device__ __forceinline__ float inverse(float s) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(s));
    r = fmaf(fmaf(-s, r, 1.0f), r, r);
    return fmaf(fmaf(-s, r, 1.0f), r, r);
}
// A block's codes and scale.  down = 2^-e, up = 2^e.
template <typename T>
__device__ __forceinline__ uint2 quantise(const Block16<T>& in, float down, float up, uint32_t* scale) {
    const uint32_t most = in.largest();
    constexpr float SIXTH = 1.0f / 6.0f, BEYOND = 8192.0f;  // (what is larger takes the largest scale and code)
    const float size = sizeof(T) == 2 ? __uint_as_float(most) * down : fminf(__uint_as_float(most) * down, BEYOND), limit = BEYOND * up;
    // (a bfloat16's sixth needs no more: checked for every significand of a tie, the product with 1 / 6 comes out on it)
    *scale = e4m3_of(sizeof(T) == 2 ? size * SIXTH : to_odd(quotient(size, 6.0f, SIXTH), size, 6.0f));
    // (the scale's exponent apart: 1 / s within what an approximation takes)
    const float held = e4m3_value(*scale), s = held * up;
    float r = held > 0.0f ? inverse(held) : 0.0f, rest = 0.0f;
    if constexpr (sizeof(T) == 2) {
        // 1 / s = r + rest, r the float32 below it: both parts of x / s have x's sign, so that what overflows comes out as the infinity that it should
        rest = fmaf(-held, r, 1.0f);
        if (rest < 0.0f) {
            r = __uint_as_float(__float_as_uint(r) - 1);
            rest = fmaf(-held, r, 1.0f);
        }
        rest *= r * down;
    }
    r *= down;
    uint32_t codes[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float q[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float x[4];
            in.four(2 * i + h, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(T) == 2) {
                    q[4 * h + e] = fmaf(x[e], r, x[e] * rest);
                } else {
                    const float y = fminf(fabsf(x[e]), limit);
                    q[4 * h + e] = copysignf(to_odd(quotient(y, s, r), y, s), x[e]);
                }
            }
        }
        asm("{\n.reg .b8 a, b, c, d;\ncvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\ncvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
            "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\nmov.b32 %0, {a, b, c, d};\n}\n"
            : "=r"(codes[i]) : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
    }
    if (most <= 0x7F800000u) return make_uint2(codes[0], codes[1]);
    *scale = 0x7F;  // a NaN
    return make_uint2(0, 0);
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
    const float down = exp2f((float)-a.in4.exponent[v]), up = exp2f((float)a.in4.exponent[v]);
    const uint32_t step = a.step;  // (in a register: read from the parameters each time the loop was unrolled another way, a fifth slower)
    for (uint32_t pass = 0; pass < a.passes; ++pass) {
        const Column u(a, pass);
        if (!u.there) continue;
        const unsigned char* from = a.rows.p[v] + (sg.query_begin + t0 + u.row) * a.rows.rs[v] + u.head * a.rows.hs[v] + u.unit * (16 * sizeof(T));
        const uint64_t at = sg.row_begin + ctx + t0 + u.row, from_step = step * a.rows.rs[v], code_step = step * a.in4.crs, scale_step = step * a.in4.srs;
        unsigned char* codes = const_cast<unsigned char*>(a.in4.codes[v]) + at * a.in4.crs + u.head * a.in4.chs + u.unit * 8;
        unsigned char* scales = const_cast<unsigned char*>(a.in4.scales[v]) + at * a.in4.srs + u.head * a.in4.shs + u.unit;
        for (uint32_t r = u.row; r < tokens; r += WRITE_FLIGHT * step) {
            Block16<T> in[WRITE_FLIGHT];
#pragma unroll
            for (int i = 0; i < WRITE_FLIGHT; ++i, from += from_step)
                if (r + i * step < tokens) in[i].load(from);
#pragma unroll
            for (int i = 0; i < WRITE_FLIGHT; ++i, codes += code_step, scales += scale_step) {
                if (r + i * step >= tokens) break;
                uint32_t scale;
                *reinterpret_cast<uint2*>(codes) = quantise<T>(in[i], down, up, &scale);
                *scales = (unsigned char)scale;
            }
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
    // (rows to be attended to: those before what the window of the segment's first token leaves are seen by none)
    const uint32_t ctx = n - min(n, sg.n_queries);
    if (a.seen_last != 0xFFFFFFFFu && ctx > a.seen_last && r0 + rows <= ctx - a.seen_last) return;
    const int v = blockIdx.y;
    if (v == 0)
        for (uint32_t e = 0; e < a.entries; ++e)
            for (uint32_t r = threadIdx.x; r < rows; r += ROW_THREADS) {
                const uint64_t at = e * a.entry_hs + sg.row_begin + r0 + r, to = e * a.to_entry_hs + sg.to_begin + r0 + r;
                if (a.pos) a.to_pos[to] = a.pos[at];
                if (a.doc) a.to_doc[to] = a.doc[at];
            }
    if (!a.rows.p[v]) return;
    const float up = exp2f((float)a.in4.exponent[v]);
    const uint32_t step = a.step;
    for (uint32_t pass = 0; pass < a.passes; ++pass) {
        const Column u(a, pass);
        if (!u.there) continue;
        const uint64_t at = sg.row_begin + r0 + u.row, to_step = step * a.rows.rs[v], code_step = step * a.in4.crs, scale_step = step * a.in4.srs;
        const unsigned char* codes = a.in4.codes[v] + at * a.in4.crs + u.head * a.in4.chs + u.unit * 4;
        const unsigned char* scales = a.in4.scales[v] + at * a.in4.srs + u.head * a.in4.shs + u.unit / 2;
        unsigned char* to = const_cast<unsigned char*>(a.rows.p[v]) + (sg.to_begin + r0 + u.row) * a.rows.rs[v] + u.head * a.rows.hs[v] + u.unit * (8 * sizeof(T));
        for (uint32_t r = u.row; r < rows; r += FLIGHT * step) {
            uint32_t code[FLIGHT], scale[FLIGHT];
#pragma unroll
            for (int i = 0; i < FLIGHT; ++i, codes += code_step, scales += scale_step) {
                const bool there = r + i * step < rows;
                code[i] = there ? *reinterpret_cast<const uint32_t*>(codes) : 0;
                scale[i] = there ? *scales : 0;
            }
#pragma unroll
            for (int i = 0; i < FLIGHT; ++i, to += to_step) {
                if (r + i * step >= rows) break;
                const float s = e4m3_value(scale[i] & 0x7F) * up;
                const uint32_t h[4] = {e2m1_pair<0>(code[i]), e2m1_pair<1>(code[i]), e2m1_pair<2>(code[i]), e2m1_pair<3>(code[i])};
                float f[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
                    f[2 * j] = x.x * s;
                    f[2 * j + 1] = x.y * s;
                }
                if constexpr (sizeof(T) == 2) {
                    *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
                } else {
                    // Neighbours exchange halves, so that each of the two stores fills whole sectors of 32 bytes (32768 tokens read, us: 62.7, 78.6 without).  (Units come in pairs, the even one to an even lane, of one row and head.)
                    const bool odd = u.unit & 1;
                    const uint32_t both = 3u << (threadIdx.x & 30);
                    float4 own = odd ? make_float4(f[4], f[5], f[6], f[7]) : make_float4(f[0], f[1], f[2], f[3]), other = odd ? make_float4(f[0], f[1], f[2], f[3]) : make_float4(f[4], f[5], f[6], f[7]);
                    other.x = __shfl_xor_sync(both, other.x, 1);
                    other.y = __shfl_xor_sync(both, other.y, 1);
                    other.z = __shfl_xor_sync(both, other.z, 1);
                    other.w = __shfl_xor_sync(both, other.w, 1);
                    float4* pair = reinterpret_cast<float4*>(to) - (odd ? 1 : 0);  // (of the four halves the even lane writes the first and third, the odd one the others)
                    pair[0] = odd ? other : own;
                    pair[2] = odd ? own : other;
                }
            }
        }
    }
}

// Rows of a work item: what is under way at a time, up to eight times as many where that leaves 8 work items an SM (16 of writing), more where there would be more than a grid takes.
Status cut_rows(Ctx* c, Rows4Args* a, std::vector<CacheSeg>* segs, bool write, CacheTable* tab, uint32_t* items) {
    uint64_t rows = 0, count;
    for (const CacheSeg& s : *segs) rows += write ? s.n_queries : s.n_rows;
    a->units = a->d / (write ? 16 : 8);
    a->columns = a->n_kv * a->units;
    a->passes = (a->columns + ROW_THREADS - 1) / ROW_THREADS;
    a->step = std::max(1u, ROW_THREADS / a->columns);
    a->per_column = (65536 + a->columns - 1) / a->columns;
    a->per_unit = (65536 + a->units - 1) / a->units;
    const uint64_t least = (uint64_t)a->step * (write ? WRITE_FLIGHT : FLIGHT);
    uint64_t each = least * std::min<uint64_t>(std::max<uint64_t>(rows / (least * (write ? 16 : 8) * sm_count(c->device)), 1), 8);
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
        g.n_queries = segs[i].n_queries;
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
