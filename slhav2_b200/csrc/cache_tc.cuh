// What the cache kernels on tcgen05 share: barriers, TMA, operands in shared memory, TMEM, and the maps of rows that TMA reads.
#pragma once

#include <cuda.h>

#include "cache.cuh"
#include "cache_mma.cuh"

namespace slha {
namespace {

constexpr uint32_t HALF = 128 * 128;  // bytes of 128 rows x 64 elements
constexpr uint32_t SPINS = 1u << 22;  // polls of a wait before it gives up (a fraction of a second)

__device__ __forceinline__ void bar_init(uint32_t addr, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(addr), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t addr) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(addr) : "memory"); }
__device__ __forceinline__ bool bar_wait(uint32_t addr, uint32_t parity) {
    for (uint32_t i = 0; i < SPINS; ++i) {
        uint32_t ok;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(addr), "r"(parity) : "memory");
        if (ok) return true;
        if (i > 64) __nanosleep(32);
    }
    return false;
}
// Waits for the last fills of a ring of `stages` barriers of which `fills` were begun, so that no copy is under way when a block ends, whoever gave up before.
__device__ __forceinline__ void bar_settle(uint32_t bars, uint32_t fills, uint32_t stages) {
    for (uint32_t i = fills > stages ? fills - stages : 0; i < fills; ++i) bar_wait(bars + i % stages * 8, i / stages & 1);
}
__device__ __forceinline__ void bar_expect(uint32_t addr, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(addr), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t y, uint32_t z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst), "l"(map), "r"(x), "r"(y),
                 "r"(z), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, uint32_t x, uint32_t y, uint32_t z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];\n" ::"l"(map), "r"(x), "r"(y), "r"(z), "r"(src) : "memory");
}
__device__ __forceinline__ void tc_commit_to(uint32_t addr) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
// Shared-memory operands, 128-byte swizzle.  Contraction along the 128-byte lines (Q, K): groups of eight lines 1024 bytes apart.  Contraction across the lines (V): eight lines
// 1024 bytes apart likewise, the next 64 elements of a line one HALF further.
__device__ __forceinline__ uint64_t desc_along(uint32_t s) {
    return (uint64_t)((s & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t desc_across(uint32_t s) {
    return (uint64_t)((s & 0x3FFFFu) >> 4) | (uint64_t)(HALF >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D float32, A and B bfloat16, M = 128, N columns; across: B's contraction runs across its lines
__host__ __device__ constexpr uint32_t wide_idesc(uint32_t n, bool across) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (across ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
// two float32 at a time
__device__ __forceinline__ uint64_t pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;\n" : "=f"(x), "=f"(y) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// tanh_small's polynomial at v = x^2
__device__ __forceinline__ uint64_t tanh_poly(uint64_t v) {
    uint64_t p = fma2(v, pair(TANH_6, TANH_6), pair(TANH_5, TANH_5));
    p = fma2(v, p, pair(TANH_4, TANH_4));
    p = fma2(v, p, pair(TANH_3, TANH_3));
    p = fma2(v, p, pair(TANH_2, TANH_2));
    p = fma2(v, p, pair(TANH_1, TANH_1));
    return fma2(v, p, pair(TANH_0, TANH_0));
}
// the same to |x| = 0.6 with two terms fewer (7e-8 relative)
constexpr float TANH_BRIEF = 0.6f;
__device__ __forceinline__ uint64_t tanh_poly_brief(uint64_t v) {
    uint64_t p = fma2(v, pair(1.5475427487757746e-2f, 1.5475427487757746e-2f), pair(-5.210148011562652e-2f, -5.210148011562652e-2f));
    p = fma2(v, p, pair(1.3310173657966862e-1f, 1.3310173657966862e-1f));
    p = fma2(v, p, pair(-3.3332309974403695e-1f, -3.3332309974403695e-1f));
    return fma2(v, p, pair(9.999999268689624e-1f, 9.999999268689624e-1f));
}
// the low x bits of a word
__device__ __forceinline__ uint32_t low_bits(int x) { return x <= 0 ? 0u : x >= 32 ? 0xFFFFFFFFu : (1u << x) - 1u; }
#define R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define W8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])
// Columns of this thread's TMEM lane; to be waited for (tmem_wait) and held before they are used.
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t* x) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : R8(x, 0), R8(x, 8), R8(x, 16), R8(x, 24) : "r"(t) : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t t, uint32_t* x) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\ntcgen05.wait::ld.sync.aligned;\n"
                 : "=&r"(x[0]), "=&r"(x[1]), "=&r"(x[2]), "=&r"(x[3]), "=&r"(x[4]), "=&r"(x[5]), "=&r"(x[6]), "=&r"(x[7]), "=&r"(x[8]), "=&r"(x[9]), "=&r"(x[10]), "=&r"(x[11]),
                   "=&r"(x[12]), "=&r"(x[13]), "=&r"(x[14]), "=&r"(x[15]) : "r"(t) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t* x) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(t), W8(x, 0), W8(x, 8) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

using WideEncode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
WideEncode wide_encode() {
    static const WideEncode encode = []() -> WideEncode {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        return reinterpret_cast<WideEncode>(p);
    }();
    return encode;
}
// A map of rows x KV heads x elements in boxes of 128 rows of one KV head x 64 elements; false where the driver does not take the layout.
bool wide_map(CUtensorMap* map, const void* base, uint64_t row_stride, uint64_t head_stride, uint64_t rows, uint32_t heads, uint32_t d, uint32_t* head_first) {
    const WideEncode encode = wide_encode();
    if (!encode || rows > 0x7FFFFFFFull) return false;
    if (heads == 1) head_stride = row_stride * rows;  // (never stepped by)
    *head_first = head_stride < row_stride;
    const cuuint64_t dims[3] = {d, *head_first ? heads : rows, *head_first ? rows : heads};
    const cuuint64_t strides[2] = {(*head_first ? head_stride : row_stride) * 2, (*head_first ? row_stride : head_stride) * 2};
    const cuuint32_t box[3] = {64, *head_first ? 1u : 128u, *head_first ? 128u : 1u}, each[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Queries or outputs in boxes of 32 rows of a KV head (32 / group tokens of its group); false where the layout or the group does not allow it.
bool wide_row_map(CUtensorMap* map, const void* base, uint64_t token_stride, uint64_t head_stride, const CacheArgs& a) {
    if (32 % a.group || (a.n_heads > 1 && head_stride >= token_stride) || a.n_tokens > 0x7FFFFFFFu) return false;
    const WideEncode encode = wide_encode();
    if (!encode) return false;
    if (a.n_heads == 1) head_stride = token_stride;  // (never stepped by)
    const cuuint64_t dims[3] = {a.d, a.n_heads, a.n_tokens}, strides[2] = {head_stride * 2, token_stride * 2};
    const cuuint32_t box[3] = {64, a.group, 32 / a.group}, each[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace slha
