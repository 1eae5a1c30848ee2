// Norms of query and key heads and their rotation by position, on the way into a cache of rows (slha_b200_rotate_heads).
//
//   y = x (mean x^2 + eps)^(-1/2) w;   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),  t = position[axis[p]] frequency[p] for pair p
// The angle is taken in turns and in float64, t / 2 pi less the nearest integer: positions of 2^32 keep 2^-23 of a turn.  Its cosine and sine are float32, one pair of them a token for all
// heads.
//
// Bytes bound it, every head read and written once, once few instructions do: 8, 16 or 32 lanes take a head, 8 elements each: four pairs (two 8- or 16-byte loads, half a rotation apart) or, of
// interleaved pairs and what is not turned, 8 elements side by side.  A group of lanes takes a head of a block's tokens, two of them at a time, so that its addresses grow by a constant and its
// weights stay in registers; then its next head.  No element is read by another lane than the one that writes it, so that heads may be turned in place.
//
// Squares are summed in float32; a head for which that is too narrow is scaled by a power of two first (44.8 us instead of 43.4 for the look at each sum, in the case below).
//
// 8192 tokens of 32 + 8 + 8 heads of 128 dimensions, three axes: bfloat16 44.8 us = 4.5 TB/s (without norms 40.2), float32 69.4 us = 5.8 TB/s.  146 instructions for 8 elements take
// 63 % of the issue slots; the largest wait is for loads (4.5 of 11 warps an issue), of which a group of lanes has two tokens' under way.  One token 2.2 us, its call 6.5 with the host's time.
#include <cuda_bf16.h>

#include <algorithm>

#include "cache4.cuh"

namespace slha {
namespace {

constexpr int ROT_THREADS = 256, ROT_FLIGHT = 2, ROT_TOKENS = 16;  // tokens under way at a time, and most of a block
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
constexpr double PER_TURN = 0.15915494309189533577;  // 1 / (2 pi)

template <typename T>
struct HeadUnit {  // 8 elements as they lie: two times 4
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void load(const unsigned char* a, const unsigned char* b, bool apart) {
        if constexpr (sizeof(T) == 2) {
            if (apart) {
                const uint2 x = *reinterpret_cast<const uint2*>(a), y = *reinterpret_cast<const uint2*>(b);
                w[0] = x.x, w[1] = x.y, w[2] = y.x, w[3] = y.y;
            } else {
                const uint4 x = *reinterpret_cast<const uint4*>(a);
                w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
            }
        } else {
            const uint4 x = *reinterpret_cast<const uint4*>(a), y = *reinterpret_cast<const uint4*>(b);
            w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w, w[4] = y.x, w[5] = y.y, w[6] = y.z, w[7] = y.w;
        }
    }
    __device__ __forceinline__ void store(unsigned char* a, unsigned char* b, bool apart) const {
        if constexpr (sizeof(T) == 2) {
            if (apart) {
                *reinterpret_cast<uint2*>(a) = make_uint2(w[0], w[1]);
                *reinterpret_cast<uint2*>(b) = make_uint2(w[2], w[3]);
            } else {
                *reinterpret_cast<uint4*>(a) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else {
            *reinterpret_cast<uint4*>(a) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(b) = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 2) f[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
            else f[i] = __uint_as_float(w[i]);
        }
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(w[i]) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(f[i]);
        }
    }
};

template <int LANES>
__device__ __forceinline__ float mean_square(const float (&f)[8], bool there, float per_dim, float eps, uint32_t lanes) {
    float sum = 0.0f;
    if (there) {
        uint64_t two = 0;
#pragma unroll
        for (int e = 0; e < 8; e += 2) two = fma2(pair(f[e], f[e + 1]), pair(f[e], f[e + 1]), two);
        float odd;
        unpair(two, sum, odd);
        sum += odd;
    }
#pragma unroll
    for (int m = LANES / 2; m; m >>= 1) sum += __shfl_xor_sync(lanes, sum, m);
    return sum * per_dim + eps;
}
// Whether a sum of squares has overflown, or squares that count have lost bits: their mean is below 2^-96, or no number.
__device__ __forceinline__ bool beyond(float mean) { return __float_as_uint(mean) - (31u << 23) >= (224u << 23); }
// What such a head is multiplied with, a power of two, so that its largest element (eps' root where that is larger) is 1 to 4: y stays the same, and elements that lose bits are below 2^-120 of
// the largest.  1 where there is an infinity, a NaN or nothing but zeros.
template <int LANES>
__device__ __noinline__ float head_down(float most, float eps, uint32_t lanes) {
#pragma unroll
    for (int m = LANES / 2; m; m >>= 1) most = fmaxf(most, __shfl_xor_sync(lanes, most, m));
    most = fmaxf(most, sqrtf(eps));
    if (__float_as_uint(most) >= 0x7F800000u || most == 0.0f) return 1.0f;
    const int k = min((int)(max(__float_as_uint(most) >> 23, 1u) - 127u), 126);
    return __uint_as_float((uint32_t)(127 - k) << 23);
}

template <typename T, int LANES>
__global__ void __launch_bounds__(ROT_THREADS) rotate_heads_kernel(const __grid_constant__ RotateArgs a, const __grid_constant__ CacheTable tab) {
    dep_wait();
    __shared__ __align__(16) float s_turn[ROT_TOKENS][2][CACHE_DIM_MOST / 2];  // cosines, sines
    const CacheSeg* table = a.table ? a.table : tab.s;
    const uint32_t seg = cache_find(a.n_segs, blockIdx.x, [&](uint32_t i) { return table[i].item_begin; });
    const CacheSeg& sg = table[seg];
    const uint32_t t0 = (blockIdx.x - sg.item_begin) * a.each, tokens = min(a.each, sg.n_queries - t0), tok0 = sg.query_begin + t0;
    const uint32_t n = a.counts ? min(a.counts[sg.seg], sg.n_rows) : sg.n_rows, ctx = n - min(n, sg.n_queries);
    const uint32_t placed = min(tokens, n - ctx - min(n - ctx, t0));  // the tokens that have a row
    const uint64_t row0 = sg.row_begin + ctx + t0;
    const uint32_t nq = a.q ? a.n_heads : 0, nk = a.k ? a.n_kv : 0, nv = a.v ? a.n_kv : 0, all = nq + nk + nv;

    const uint32_t x = threadIdx.x % LANES, group = threadIdx.x / LANES, groups = blockDim.x / LANES;
    const bool mine = x < a.d / 8, turned = x < a.rotary / 8, apart = turned && !a.interleaved;
    const uint32_t first = apart ? 4 * x : 8 * x, second = apart ? a.rotary / 2 + 4 * x : 8 * x + 4;

    for (uint32_t i = threadIdx.x; i < tokens * (a.rotary / 2); i += blockDim.x) {
        const uint32_t t = i / (a.rotary / 2), p = i % (a.rotary / 2), axis = a.axes ? min((uint32_t)a.axes[p], a.n_axes - 1) : 0;
        const double turns = (double)a.positions[(uint64_t)axis * a.n_tokens + tok0 + t] * (double)a.freq[p] * PER_TURN;
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        s_turn[t][0][p] = c * a.magnitude;
        s_turn[t][1][p] = s * a.magnitude;
    }
    __syncthreads();
    // (a warp's groups go through the loops together: sums are taken over a group's lanes)
    for (uint32_t i = blockIdx.y * groups + group; __any_sync(0xFFFFFFFFu, i < all); i += gridDim.y * groups) {
        const bool q = i < nq, k = !q && i < nq + nk, value = !q && !k;
        const uint32_t h = q ? i : k ? i - nq : i - nq - nk, last = i >= all || !mine ? 0 : q ? tokens : placed;  // last: tokens whose head is written
        const uint64_t step = q ? a.qts : k ? a.kts : a.vts, to_step = q ? a.qots : k ? a.kors : a.vors;
        const unsigned char* from = (q ? a.q + h * a.qhs : k ? a.k + h * a.khs : a.v + h * a.vhs) + tok0 * step;
        unsigned char* to = (q ? a.q_out + h * a.qohs : k ? a.k_out + h * a.kohs : a.v_out + h * a.vohs) + (q ? tok0 : row0) * to_step;
        const float* weight = q ? a.q_weight : k ? a.k_weight : nullptr;
        uint64_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t at = e < 2 ? first + 2 * e : second + 2 * e - 4;
            w[e] = weight && last ? pair(weight[at], weight[at + 1]) : pair(1.0f, 1.0f);
        }
        for (uint32_t t = 0; t < tokens; t += ROT_FLIGHT) {
            HeadUnit<T> in[ROT_FLIGHT];
#pragma unroll
            for (int j = 0; j < ROT_FLIGHT; ++j, from += step)
                if (t + j < last) in[j].load(from + first * sizeof(T), from + second * sizeof(T), apart);
#pragma unroll
            for (int j = 0; j < ROT_FLIGHT; ++j, to += to_step) {
                if (t + j >= tokens) break;
                const bool there = t + j < last;
                if (!value || a.norm) {  // (values go through the sums over the lanes: their neighbours' heads may be keys)
                    float f[8], factor = 1.0f;
                    if (there) in[j].get(f);
                    if (a.norm) {
                        float mean = mean_square<LANES>(f, there, a.per_dim, a.eps, 0xFFFFFFFFu);
                        if (beyond(mean)) {  // (elements of 2^60 and more; an eps of zero and elements below 2^-48.  All lanes of a head or none)
                            const uint32_t lanes = LANES == 32 ? 0xFFFFFFFFu : ((1u << LANES % 32) - 1) << (threadIdx.x & 31 & ~(LANES - 1));
                            float most = 0.0f;
#pragma unroll
                            for (int e = 0; e < 8; ++e) most = there ? fmaxf(most, fabsf(f[e])) : 0.0f;
                            const float down = head_down<LANES>(most, a.eps, lanes);
#pragma unroll
                            for (int e = 0; e < 8; ++e) f[e] *= down;
                            mean = mean_square<LANES>(f, there, a.per_dim, a.eps * down * down, lanes);
                        }
                        factor = rsqrtf(mean);
                    }
                    if (there && !value) {
                        uint64_t y[4];  // two elements at a time: apart, of two pairs; side by side, a pair's
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            y[e] = pair(f[2 * e], f[2 * e + 1]);
                            if (a.norm) y[e] = mul2(mul2(y[e], pair(factor, factor)), w[e]);
                        }
                        if (turned) {
                            const float4 c = *reinterpret_cast<const float4*>(&s_turn[t + j][0][4 * x]), s = *reinterpret_cast<const float4*>(&s_turn[t + j][1][4 * x]);
                            if (apart) {
                                const uint64_t cs[2] = {pair(c.x, c.y), pair(c.z, c.w)}, sn[2] = {pair(s.x, s.y), pair(s.z, s.w)}, back[2] = {pair(-s.x, -s.y), pair(-s.z, -s.w)};
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const uint64_t u = y[e], v = y[2 + e];
                                    y[e] = fma2(u, cs[e], mul2(v, back[e]));
                                    y[2 + e] = fma2(u, sn[e], mul2(v, cs[e]));
                                }
                            } else {
                                const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    float u, v;
                                    unpair(y[e], u, v);
                                    y[e] = fma2(pair(u, u), pair(cs[e], sn[e]), mul2(pair(v, v), pair(-sn[e], cs[e])));
                                }
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) unpair(y[e], f[2 * e], f[2 * e + 1]);
                        in[j].set(f);
                    }
                }
                if (there) in[j].store(to + first * sizeof(T), to + second * sizeof(T), apart);  // (values as they are, NaN too)
            }
        }
    }
}

template <typename T>
Status launch_lanes(Ctx* c, const RotateArgs& a, const CacheTable& tab, uint32_t items) {
    const uint32_t lanes = a.d <= 64 ? 8 : a.d <= 128 ? 16 : 32, heads = (a.q ? a.n_heads : 0) + ((a.k != nullptr) + (a.v != nullptr)) * a.n_kv;
    const uint32_t threads = std::min<uint64_t>(ROT_THREADS, ((uint64_t)heads * lanes + 31) / 32 * 32);
    const auto kernel = lanes == 8 ? rotate_heads_kernel<T, 8> : lanes == 16 ? rotate_heads_kernel<T, 16> : rotate_heads_kernel<T, 32>;
    // few tokens: their heads go to as many blocks as they fill (one token of 48 heads: 3.4 us in three blocks, 4.4 in one)
    const uint32_t at_once = threads / lanes, blocks = items < 2u * sm_count(c->device) ? std::min((heads + at_once - 1) / at_once, 64u) : 1;
    SLHA_CUDA(launch_behind(kernel, dim3(items, blocks), dim3(threads), 0, c->stream, a, tab));
    count_launch();
    return Status();
}

}  // namespace

Status launch_rotate_heads(Ctx* c, RotateArgs a, int dtype, const std::vector<SlhaB200Segment>& segs) {
    uint64_t tokens = 0, items = 0;
    for (const SlhaB200Segment& s : segs) tokens += s.n_queries;
    if (!tokens) return Status();
    // tokens of a block: up to 16, so that the blocks come in whole rounds of what an SM holds of them (8192 tokens, bfloat16: two rounds of 7 each took 2.4 us more than one of 14)
    const uint64_t round = (dtype == SLHA_B200_BF16 ? 4ull : 3ull) * sm_count(c->device), rounds = (tokens + round * ROT_TOKENS - 1) / (round * ROT_TOKENS);
    a.each = (uint32_t)((tokens + round * rounds - 1) / (round * rounds));
    a.per_dim = 1.0f / (float)a.d;
    std::vector<CacheSeg> of;
    for (size_t i = 0; i < segs.size(); ++i) {
        if (!segs[i].n_queries) continue;
        CacheSeg g{};
        g.row_begin = segs[i].tile_begin;
        g.n_rows = segs[i].n_tiles;
        g.query_begin = segs[i].query_begin;
        g.n_queries = segs[i].n_queries;
        g.item_begin = (uint32_t)items;
        g.seg = (uint32_t)i;
        items += ((uint64_t)g.n_queries + a.each - 1) / a.each;
        of.push_back(g);
    }
    if (items > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "slha_b200_rotate_heads: too many tokens");
    CacheTable tab;
    SLHA_TRY(cache_table(c, of, &tab, &a.table));
    a.n_segs = (uint32_t)of.size();
    return dtype == SLHA_B200_BF16 ? launch_lanes<__nv_bfloat16>(c, a, tab, (uint32_t)items) : launch_lanes<float>(c, a, tab, (uint32_t)items);
}

}  // namespace slha
