// Tensor-core steps of the cache kernels for rows of bfloat16 and of float32, 16 query rows a warp (mma.sync).
//
// bfloat16: one m16n8k16 product, exact terms, float32 sums.  float32: each factor as the sum of two tf32 numbers (11 bits and the next 11), three m16n8k8
// products; the lowest one, 2^-22 of the term, is left out.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace slha {
namespace {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes, or zeros where `there` does not hold (the address is then not read)
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 4u : 0u) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t lds(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x as the nearest number of 11 bits (ties away from zero) and the exact rest, of which the products take the first 11 bits.  (In integers: cvt.rna.tf32 takes three
// instructions, two of them with the rest's made this kernel's largest part.)  An infinity's rest is NaN.
__device__ __forceinline__ void tf32_split(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_f32(float (&d)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], float b0, float b1) {
    uint32_t bh0, bl0, bh1, bl1;
    tf32_split(b0, bh0, bl0);
    tf32_split(b1, bh1, bl1);
    mma_tf32(d, al, bh0, bh1);
    mma_tf32(d, ah, bl0, bl1);
    mma_tf32(d, ah, bh0, bh1);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Tiles of rows in shared memory: rows of D elements, their 16-byte pieces exchanged by the row's low three bits, so that eight rows' pieces of one column
// lie in eight different groups of banks.
template <typename T, int D>
struct Tile {
    static constexpr int ROW = D * (int)sizeof(T), PIECES = ROW / 16, EACH = 16 / (int)sizeof(T);
    static __device__ __forceinline__ uint32_t at(uint32_t base, int row, int piece) { return base + row * ROW + ((piece ^ (row & 7)) << 4); }
    static __device__ __forceinline__ uint32_t elem(uint32_t base, int row, int col) { return at(base, row, col / EACH) + (col % EACH) * (uint32_t)sizeof(T); }
};

// A operand: 16 query rows x one k step (16 bfloat16, 8 float32), from shared memory
template <typename T>
struct AFrag;
template <>
struct AFrag<__nv_bfloat16> {
    uint32_t a[4];
    template <int D>
    __device__ __forceinline__ void load(uint32_t base, int row0, int kk, int lane) {
        ldm4(a, Tile<__nv_bfloat16, D>::at(base, row0 + (lane & 7) + ((lane >> 3) & 1) * 8, kk * 2 + (lane >> 4)));
    }
};
template <>
struct AFrag<float> {
    uint32_t h[4], l[4];
    template <int D>
    __device__ __forceinline__ void load(uint32_t base, int row0, int kk, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < 4; ++i) tf32_split(__uint_as_float(lds(Tile<float, D>::elem(base, row0 + g + (i & 1) * 8, kk * 8 + t + (i >> 1) * 4))), h[i], l[i]);
    }
};
// s[n][.] += Q K^T of a k step for 8 N keys from key0 on
template <typename T, int D, int N>
__device__ __forceinline__ void scores_step(float (&s)[N][4], const AFrag<T>& a, uint32_t kbase, int key0, int kk, int lane) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int n = 0; n < N; n += 2) {
            uint32_t b[4];
            ldm4(b, Tile<T, D>::at(kbase, key0 + n * 8 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1)));
            mma_bf16(s[n], a.a, b[0], b[1]);
            mma_bf16(s[n + 1], a.a, b[2], b[3]);
        }
    } else {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float b0 = __uint_as_float(lds(Tile<T, D>::elem(kbase, key0 + n * 8 + g, kk * 8 + t)));
            const float b1 = __uint_as_float(lds(Tile<T, D>::elem(kbase, key0 + n * 8 + g, kk * 8 + t + 4)));
            mma_f32(s[n], a.h, a.l, b0, b1);
        }
    }
}
// All k steps of s[n][.] = Q K^T; load(kk) brings the A operand of one.  The tensor cores cut each product's sum off towards zero: sums of which more than bfloat16 counts are taken four
// steps at a time (AT_ONCE; 0: all) and added here, to the nearest (float32, 7 x 18 drafted tokens over 390 rows, 128 dimensions: outputs 2.2e-6 off without, 6.5e-7 with; 5 % of the time).
template <typename T, int D, int N, int AT_ONCE = sizeof(T) == 2 ? 0 : 4, typename Load>
__device__ __forceinline__ void scores_of(float (&s)[N][4], Load load, uint32_t kbase, int key0, int lane) {
    if constexpr (!AT_ONCE) {
#pragma unroll 4
        for (int kk = 0; kk < D / 16; ++kk) scores_step<T, D, N>(s, load(kk), kbase, key0, kk, lane);
    } else {
#pragma unroll 1
        for (int k4 = 0; k4 < D / (sizeof(T) == 2 ? 16 : 8); k4 += AT_ONCE) {
            float part[N][4] = {};
#pragma unroll
            for (int kk = 0; kk < AT_ONCE; ++kk) scores_step<T, D, N>(part, load(k4 + kk), kbase, key0, k4 + kk, lane);
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] += part[n][e];
        }
    }
}
// o[.] += P V for the 8 N keys from key0 on; p as scores_step leaves its sums (a thread's columns 2t and 2t + 1: for float32 they stand for the k indices t and
// t + 4, the rows of V accordingly)
template <typename T, int D, int N>
__device__ __forceinline__ void values_step(float (&o)[D / 8][4], const float (&p)[N][4], uint32_t vbase, int key0, int lane) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int n = 0; n < N; n += 2) {
            const uint32_t a[4] = {pack_bf16(p[n][0], p[n][1]), pack_bf16(p[n][2], p[n][3]), pack_bf16(p[n + 1][0], p[n + 1][1]), pack_bf16(p[n + 1][2], p[n + 1][3])};
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                uint32_t b[4];
                ldm4t(b, Tile<T, D>::at(vbase, key0 + n * 8 + (lane & 7) + ((lane >> 3) & 1) * 8, d * 2 + (lane >> 4)));
                mma_bf16(o[2 * d], a, b[0], b[1]);
                mma_bf16(o[2 * d + 1], a, b[2], b[3]);
            }
        }
    } else {
        const int g = lane >> 2, t = lane & 3;
        uint32_t h[N][4], l[N][4];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            tf32_split(p[n][0], h[n][0], l[n][0]);
            tf32_split(p[n][2], h[n][1], l[n][1]);
            tf32_split(p[n][1], h[n][2], l[n][2]);
            tf32_split(p[n][3], h[n][3], l[n][3]);
        }
#pragma unroll
        for (int d = 0; d < D / 8; ++d) {
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // (as for the scores)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const float b0 = __uint_as_float(lds(Tile<T, D>::elem(vbase, key0 + n * 8 + 2 * t, d * 8 + g)));
                const float b1 = __uint_as_float(lds(Tile<T, D>::elem(vbase, key0 + n * 8 + 2 * t + 1, d * 8 + g)));
                mma_f32(part, h[n], l[n], b0, b1);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d][e] += part[e];
        }
    }
}

}  // namespace
}  // namespace slha
