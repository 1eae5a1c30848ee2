// Norms of query and key heads and their rotation by position, on the way into a cache of rows (slha_b200_rotate_heads).
//
//   y = x (mean x^2 + eps)^(-1/2) w;   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),  t = position[axis[p]] frequency[p] for pair p
// The angle is taken in turns and in float64, t / 2 pi less the nearest integer: positions of 2^32 keep 2^-23 of a turn.  Its cosine and sine are float32, one pair of them a token for all
// heads.
//
// Bound by bytes, every head read and written once.  A block takes a token; 8, 16 or 32 lanes take a head, 8 elements each: four pairs (two 8- or 16-byte loads, half a rotation apart) or,
// of interleaved pairs and what is not turned, 8 elements side by side.  No element is read by another lane than the one that writes it, so that heads may be turned in place.
#include <cuda_bf16.h>

#include <algorithm>

#include "cache4.cuh"

namespace slha {
namespace {

constexpr int ROT_THREADS = 256, ROT_FLIGHT = 3;  // heads under way at a time for each group of lanes
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

template <typename T, int LANES>
__global__ void __launch_bounds__(ROT_THREADS) rotate_heads_kernel(const __grid_constant__ RotateArgs a, const __grid_constant__ CacheTable tab) {
    dep_wait();
    __shared__ float s_cos[CACHE_DIM_MOST / 2], s_sin[CACHE_DIM_MOST / 2];
    const CacheSeg* table = a.table ? a.table : tab.s;
    const uint32_t seg = cache_find(a.n_segs, blockIdx.x, [&](uint32_t i) { return table[i].item_begin; });
    const CacheSeg& sg = table[seg];
    const uint32_t t = blockIdx.x - sg.item_begin, tok = sg.query_begin + t;
    const uint32_t n = a.counts ? min(a.counts[sg.seg], sg.n_rows) : sg.n_rows, ctx = n - min(n, sg.n_queries);
    const bool placed = ctx + t < n;  // the token has a row
    const uint64_t row = sg.row_begin + ctx + t;
    const uint32_t nq = a.q ? a.n_heads : 0, nk = a.k && placed ? a.n_kv : 0, nv = a.v && placed ? a.n_kv : 0, all = nq + nk + nv;

    const uint32_t x = threadIdx.x % LANES, group = threadIdx.x / LANES, groups = blockDim.x / LANES;
    const bool mine = x < a.d / 8;
    const bool turned = x < a.rotary / 8, apart = turned && !a.interleaved;
    const uint32_t first = apart ? 4 * x : 8 * x, second = apart ? a.rotary / 2 + 4 * x : 8 * x + 4;
    const auto from = [&](uint32_t i) {
        return i < nq ? a.q + tok * a.qts + i * a.qhs : i < nq + nk ? a.k + tok * a.kts + (i - nq) * a.khs : a.v + tok * a.vts + (i - nq - nk) * a.vhs;
    };
    const auto to = [&](uint32_t i) {
        return i < nq ? a.q_out + tok * a.qots + i * a.qohs : i < nq + nk ? a.k_out + row * a.kors + (i - nq) * a.kohs : a.v_out + row * a.vors + (i - nq - nk) * a.vohs;
    };
    HeadUnit<T> in[ROT_FLIGHT];
    const auto fetch = [&](uint32_t i0) {
#pragma unroll
        for (int j = 0; j < ROT_FLIGHT; ++j) {
            const uint32_t i = i0 + j * groups;
            if (i < all && mine) {
                const unsigned char* p = from(i);
                in[j].load(p + first * sizeof(T), p + second * sizeof(T), apart);
            }
        }
    };
    fetch(group);
    for (uint32_t p = threadIdx.x; p < a.rotary / 2; p += blockDim.x) {
        const uint32_t axis = a.axes ? min((uint32_t)a.axes[p], a.n_axes - 1) : 0;
        const double turns = (double)a.positions[(uint64_t)axis * a.n_tokens + tok] * (double)a.freq[p] * PER_TURN;
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        s_cos[p] = c * a.magnitude;
        s_sin[p] = s * a.magnitude;
    }
    __syncthreads();
    float cs[4], sn[4];
    if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) cs[i] = s_cos[4 * x + i], sn[i] = s_sin[4 * x + i];
    }
    // (a warp's groups go through the loop together: sums are taken over a group's lanes)
    for (uint32_t i0 = group; __any_sync(0xFFFFFFFFu, i0 < all); i0 += ROT_FLIGHT * groups) {
        if (i0 != group) fetch(i0);
#pragma unroll
        for (int j = 0; j < ROT_FLIGHT; ++j) {
            const uint32_t i = i0 + j * groups;
            const bool there = i < all && mine;
            float f[8];
            if (a.norm) {
                float sum = 0.0f;
                if (there) {
                    in[j].get(f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum = fmaf(f[e], f[e], sum);
                }
#pragma unroll
                for (int m = LANES / 2; m; m >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, m);
                if (!there) continue;
                if (i < nq + nk) {
                    const float factor = rsqrtf(sum / (float)a.d + a.eps);
                    const float* weight = i < nq ? a.q_weight : a.k_weight;
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= factor;
                    if (weight) {
                        const float4 u = *reinterpret_cast<const float4*>(weight + first), v = *reinterpret_cast<const float4*>(weight + second);
                        f[0] *= u.x, f[1] *= u.y, f[2] *= u.z, f[3] *= u.w, f[4] *= v.x, f[5] *= v.y, f[6] *= v.z, f[7] *= v.w;
                    }
                }
            } else {
                if (!there) continue;
                in[j].get(f);
            }
            const auto turn = [&](float& u, float& v, int e) {
                const float one = fmaf(u, cs[e], -v * sn[e]);
                v = fmaf(u, sn[e], v * cs[e]);
                u = one;
            };
            if (turned && i < nq + nk) {
                if (apart) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) turn(f[e], f[4 + e], e);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) turn(f[2 * e], f[2 * e + 1], e);
                }
            }
            if (i < nq + nk) in[j].set(f);  // (values as they are, NaN too)
            unsigned char* p = to(i);
            in[j].store(p + first * sizeof(T), p + second * sizeof(T), apart);
        }
    }
}

template <typename T>
Status launch_lanes(Ctx* c, const RotateArgs& a, const CacheTable& tab, uint32_t tokens) {
    const uint32_t lanes = a.d <= 64 ? 8 : a.d <= 128 ? 16 : 32, heads = (a.q ? a.n_heads : 0) + ((a.k != nullptr) + (a.v != nullptr)) * a.n_kv;
    const uint32_t threads = std::min<uint64_t>(ROT_THREADS, ((uint64_t)heads * lanes + 31) / 32 * 32);
    const auto kernel = lanes == 8 ? rotate_heads_kernel<T, 8> : lanes == 16 ? rotate_heads_kernel<T, 16> : rotate_heads_kernel<T, 32>;
    SLHA_CUDA(launch_behind(kernel, dim3(tokens), dim3(threads), 0, c->stream, a, tab));
    count_launch();
    return Status();
}

}  // namespace

Status launch_rotate_heads(Ctx* c, RotateArgs a, int dtype, const std::vector<SlhaB200Segment>& segs) {
    std::vector<CacheSeg> of;
    uint64_t tokens = 0;
    for (size_t i = 0; i < segs.size(); ++i) {
        if (!segs[i].n_queries) continue;
        CacheSeg g{};
        g.row_begin = segs[i].tile_begin;
        g.n_rows = segs[i].n_tiles;
        g.query_begin = segs[i].query_begin;
        g.n_queries = segs[i].n_queries;
        g.item_begin = (uint32_t)tokens;
        g.seg = (uint32_t)i;
        tokens += g.n_queries;
        of.push_back(g);
    }
    if (of.empty()) return Status();
    if (tokens > 0x7FFFFFFFull) return Status(SLHA_ERR_CAPACITY, "slha_b200_rotate_heads: too many tokens");
    CacheTable tab;
    SLHA_TRY(cache_table(c, of, &tab, &a.table));
    a.n_segs = (uint32_t)of.size();
    return dtype == SLHA_B200_BF16 ? launch_lanes<__nv_bfloat16>(c, a, tab, (uint32_t)tokens) : launch_lanes<float>(c, a, tab, (uint32_t)tokens);
}

}  // namespace slha
