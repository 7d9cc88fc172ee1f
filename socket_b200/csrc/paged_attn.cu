// Softmax attention of one new token per sequence over a paged cache.
#include "paged.cuh"

namespace sk {
namespace {

// One block per (sequence, key/value head), its query heads one after the other: a warp takes every eighth key, its lanes the head's
// elements; running maximum and sums per warp, joined at the end.  With mass the scores are taken a second time once maximum and
// sum are known.
constexpr int PT_WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(PT_WARPS * 32)
paged_attn_kernel(const __grid_constant__ sk_paged_cache c, const T* q, int64_t q_bs, int64_t q_hs, T* out, int64_t o_bs, int64_t o_hs, int H,
                  int extra, float scale) {
    constexpr int E = 8;                                       // elements of a head per lane: 256 / 32
    __shared__ float ms[PT_WARPS], ls[PT_WARPS], os[PT_WARPS][256];
    const int g = blockIdx.x % c.G, b = blockIdx.x / c.G, rep = H / c.G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, shift = 31 - __clz(c.page);
    bool over;
    const int n = paged_length(c, b, extra, &over);
    if (over && threadIdx.x == 0 && c.status != nullptr) atomicOr(c.status, SK_DEV_POS_OUT_OF_RANGE);
    for (int h = g * rep; h < (g + 1) * rep; ++h) {
        float x[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = lane + 32 * e;
            x[e] = d < c.D ? to_f32(q[b * q_bs + h * q_hs + d]) : 0.f;
            o[e] = 0.f;
        }
        auto score = [&](int j, int page) {
            const T* k = (const T*)c.k + page * c.k_ps + g * c.k_hs + (j & (c.page - 1)) * c.k_rs;
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (lane + 32 * e < c.D) s = fmaf(x[e], to_f32(k[lane + 32 * e]), s);
            return warp_sum(s) * scale;
        };
        for (int j = warp; j < n; j += PT_WARPS) {
            const int page = c.table[b * c.table_ld + (j >> shift)];
            if (!paged_page_ok(c, page)) {
                if (lane == 0 && c.status != nullptr) atomicOr(c.status, SK_DEV_INDEX_OUT_OF_RANGE);
                continue;
            }
            const float s = score(j, page), mn = fmaxf(m, s);
            const float mc = mn == -INFINITY ? 0.f : mn, f = expf(m - mc), w = expf(s - mc);      // a NaN score is a NaN weight
            const T* v = (const T*)c.v + page * c.v_ps + g * c.v_hs + (j & (c.page - 1)) * c.v_rs;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (lane + 32 * e < c.D) o[e] = fmaf(w, to_f32(v[lane + 32 * e]), o[e] * f);
            l = l * f + w;
            m = mn;
        }
        if (lane == 0) {
            ms[warp] = m;
            ls[warp] = l;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) os[warp][lane + 32 * e] = o[e];
        __syncthreads();
        m = -INFINITY;
        for (int w = 0; w < PT_WARPS; ++w) m = fmaxf(m, ms[w]);
        const float mc = m == -INFINITY ? 0.f : m;
        l = 0.f;
        for (int w = 0; w < PT_WARPS; ++w) l += ls[w] * expf(ms[w] - mc);
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        for (int d = threadIdx.x; d < c.D; d += PT_WARPS * 32) {
            float s = 0.f;
            for (int w = 0; w < PT_WARPS; ++w) s += os[w][d] * expf(ms[w] - mc);
            out[b * o_bs + h * o_hs + d] = from_f32<T>(s * inv);
        }
        if (c.mass != nullptr)
            for (int j = warp; j < n; j += PT_WARPS) {
                const int page = c.table[b * c.table_ld + (j >> shift)];
                if (!paged_page_ok(c, page)) continue;
                const float w = expf(score(j, page) - mc) * inv;
                if (lane == 0) c.mass[b * c.mass_bs + g * c.mass_hs + j] += w;
            }
        __syncthreads();
    }
}

}  // namespace

size_t paged_attn_workspace(const sk_paged_cache& c, int H) { return 0; }

int launch_paged_attn(const sk_paged_cache& c, const void* q, int64_t q_bs, int64_t q_hs, void* out, int64_t o_bs, int64_t o_hs, int H,
                      int extra, float scale, void* workspace, cudaStream_t st) {
    auto go = [&](auto t) {
        using T = decltype(t);
        paged_attn_kernel<T><<<c.B * c.G, PT_WARPS * 32, 0, st>>>(c, (const T*)q, q_bs, q_hs, (T*)out, o_bs, o_hs, H, extra, scale);
    };
    if (c.dtype == SK_F32) go(float{});
    else if (c.dtype == SK_BF16) go(__nv_bfloat16{});
    else go(__half{});
    return check_launch("paged_attn_kernel");
}

}  // namespace sk
