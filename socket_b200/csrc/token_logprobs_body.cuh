// How likely tokens were: log probabilities, entropy and the likeliest alternatives of rows of logits.
//
//   Z = sum exp(x - m),  log p_t = x_t - m - log Z,  H = log Z - sum exp(x - m) (x - m) / Z
//
// Bound by reading the logits, once: every thread keeps a reference m of its own among its logits, raised only for one LP_SLACK above it, with
// the two sums over its other ones; they are brought to one reference at the end.  Alternatives are (logit, index) pairs as one number, so that equal logits have an
// order and no two are the same.  A block walks its row in tiles and knows a bound that at least `top` pairs reach.  Threads whose maximum
// of a tile (it comes with the sums) reaches the bound append what does to a list in shared memory; from time to time the block meets, and
// cuts a list grown long to its `top` largest, whose last one is the new bound.  The first bound is the least of what `top` maxima of
// the first tile's threads reach, an equal share from each warp.  Where more is appended than the list holds - rising rows - the block
// takes the tiles since it last met again, one by one, and first raises the bound to what `top` of a tile's maxima reach.
// Few rows are split over clusters, whose first block joins the sums and lists.
#pragma once
#include "token_rows_body.cuh"
#include "warp_mma.cuh"

namespace sk {
namespace {

// Threads of a block.  Many rows: small ones, seven an SM, whose barriers few warps wait at (2048 rows of 128256 bf16, 8 alternatives: 121 us, 4.3 TB/s,
// with six an SM 128; without alternatives 92).  In clusters rows are few, and larger blocks leave fewer tiles in a row (8 rows of 128256: 13 us, with
// 128 threads 18).
template <int CL> constexpr int LP_WORK = CL == 1 ? 28 : 24;    // warps of an SM
constexpr int LP_CLUSTERED = 256;
template <int CL> constexpr int LP_THREADS = CL == 1 ? 128 : LP_CLUSTERED;
constexpr int LP_VECTORS = 4, LP_TOP = 64;
constexpr int LP_STAGES = 3;                                   // tiles in shared memory: 96 KB on their way to an SM at a time
constexpr int LP_FEW = 8, LP_LONG = 4;                         // top + LP_FEW threads may append from one tile; a list longer than top + LP_LONG is cut
constexpr int LP_RANKED = 384;                                 // the longest list that is cut by counting, pair by pair
constexpr float LP_SLACK = 5.f, LP_LOG2E = 1.4426950408889634f;

typedef unsigned long long LpPair;                             // order of the logit (NaN largest) << 32 | ~index
__device__ __forceinline__ uint32_t lp_key(float x) { return x != x ? 0xFFFFFFFFu : order_key(x); }
__device__ __forceinline__ LpPair lp_pair(float x, int i) { return (LpPair)lp_key(x) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float lp_value(LpPair p) {
    const uint32_t k = (uint32_t)(p >> 32);
    return k == 0xFFFFFFFFu ? NAN : __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// A 16-byte vector of logits: its elements two by two, and its largest one, NaN if there is one
__device__ __forceinline__ float lp_max(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
template <typename T> struct LpVector;
template <> struct LpVector<float> {
    static constexpr int V = 4, WORD = 1;                      // elements, and elements of a word
    static __device__ __forceinline__ float of(uint32_t w, int) { return __uint_as_float(w); }
    uint32_t w[4];
    __device__ __forceinline__ float2 two(int i) const { return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])); }
    __device__ __forceinline__ float largest() const {
        const float2 a = two(0), b = two(1);
        return lp_max(lp_max(a.x, a.y), lp_max(b.x, b.y));
    }
};
template <> struct LpVector<__nv_bfloat16> {
    static constexpr int V = 8, WORD = 2;
    static __device__ __forceinline__ float of(uint32_t w, int i) { return __uint_as_float(i ? w & 0xFFFF0000u : w << 16); }
    uint32_t w[4];
    __device__ __forceinline__ float2 two(int i) const { return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u)); }
    __device__ __forceinline__ float largest() const {
        const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(w);
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
        return lp_max(to_f32(m.x), to_f32(m.y));
    }
};
template <> struct LpVector<__half> {
    static constexpr int V = 8, WORD = 2;
    static __device__ __forceinline__ float of(uint32_t w, int i) { return __half2float(__ushort_as_half((unsigned short)(i ? w >> 16 : w))); }
    uint32_t w[4];
    __device__ __forceinline__ float2 two(int i) const { return __half22float2(reinterpret_cast<const __half2*>(w)[i]); }
    __device__ __forceinline__ float largest() const {
        const __half2* p = reinterpret_cast<const __half2*>(w);
        const __half2 m = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
        return lp_max(to_f32(m.x), to_f32(m.y));
    }
};

// A vector at a row's end, by the element; -inf outside
template <typename T> __device__ __noinline__ LpVector<T> lp_edge(const T* x, int at, int vocab) {
    alignas(16) T e[LpVector<T>::V];
    LpVector<T> v;
    for (int k = 0; k < LpVector<T>::V; ++k) e[k] = at + k >= 0 && at + k < vocab ? x[at + k] : from_f32<T>(-INFINITY);
    for (int k = 0; k < 4; ++k) v.w[k] = reinterpret_cast<const uint32_t*>(e)[k];
    return v;
}

// Two fp32 numbers in one instruction
typedef unsigned long long Lp2;
__device__ __forceinline__ Lp2 lp_two(float x, float y) {
    Lp2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void lp_split(Lp2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a)); }
__device__ __forceinline__ Lp2 lp_add(Lp2 a, Lp2 b) {
    Lp2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Lp2 lp_mul(Lp2 a, Lp2 b) {
    Lp2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Lp2 lp_fma(Lp2 a, Lp2 b, Lp2 c) {
    Lp2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// A reference m, one of the logits; over all the others the sum z of exp(x - m), and of that times x - m.  The logit m itself, whose weight is 1,
// is left out: where it has nearly all of the probability, 1 + z would keep next to nothing of z, which is what its log probability is made of
struct LpSums {
    float m, z, zd;
};
// to a larger reference, which is not among the sums
__device__ __forceinline__ void lp_raise(LpSums& s, float m) {
    if (s.m != -INFINITY) {
        const float d = s.m - m, f = exp2_fast(d * LP_LOG2E), all = s.z + 1.f;
        s.zd = f * fmaf(fmaxf(d, -200.f), all, s.zd);          // below -200 the factor is zero
        s.z = f * all;
    }
    s.m = m;
}
__device__ __forceinline__ void lp_join(LpSums& a, LpSums b) {
    if (b.m > a.m) {
        const LpSums x = a;
        a = b;
        b = x;
    }
    if (b.m == -INFINITY) {                                    // no logit above -inf: zeros or NaN
        a.z += b.z;
        a.zd += b.zd;
        return;
    }
    const float d = b.m - a.m, f = exp2_fast(d * LP_LOG2E), all = b.z + 1.f;
    a.zd += f * fmaf(fmaxf(d, -200.f), all, b.zd);
    a.z = fmaf(f, all, a.z);
}

template <int THREADS> struct LpShared {
    uint4 tiles[LP_STAGES][LP_VECTORS][THREADS];            // a thread's vectors are its own
    LpPair best[LP_TOP];
    LpPair got[THREADS == 128 ? 1 : 8][LP_TOP];                                     // in a cluster's first block: what each has found
    LpSums sums[8], parts[THREADS / 32];
    uint32_t least[THREADS / 32];
    int n, count;
    LpPair list[];                                             // of lp_room pairs
};
// a list that is not long, and all that the threads of a tile append
constexpr int lp_room(int top, int of_thread) { return (top + LP_FEW) * of_thread + top + LP_LONG; }

// list[0, n) -> best: its `top` largest, in order (all of them if there are fewer); returns how many.  The whole block calls it, with the list complete
template <int THREADS> __device__ __forceinline__ int lp_cut(LpShared<THREADS>& s, int n, int top) {
    const int t = threadIdx.x;
    if (n > LP_RANKED) {                                       // the top-th pair by halving, then what reaches it
        LpPair lo = 0, hi = ~0ull, mid = hi;                   // at least `top` reach lo; fewer reach hi, once that is tested
        for (;;) {
            __syncthreads();
            if (t == 0) s.count = 0;
            __syncthreads();
            int c = 0;
            for (int i = t; i < n; i += THREADS) c += s.list[i] >= mid;
            c = __reduce_add_sync(FULL, c);
            if ((t & 31) == 0) atomicAdd(&s.count, c);
            __syncthreads();
            c = s.count;
            if (c >= top) lo = mid;
            else hi = mid;
            if (c == top || hi - lo <= 1) break;
            mid = lo + (hi - lo) / 2;
        }
        __syncthreads();
        if (t == 0) s.count = 0;
        __syncthreads();
        for (int i = t; i < n; i += THREADS) {
            const LpPair p = s.list[i];
            if (p >= lo) s.best[atomicAdd(&s.count, 1)] = p;   // `top` of them: no two pairs are equal
        }
        __syncthreads();
        n = top;
        if (t < n) s.list[t] = s.best[t];
        __syncthreads();
    }
    for (int i = t; i < n; i += THREADS) {
        const LpPair p = s.list[i];
        int above = 0;
        for (int x = 0; x < n; ++x) above += s.list[x] > p;
        if (above < top) s.best[above] = p;
    }
    __syncthreads();
    return min(n, top);
}

template <typename T, int CL>
__global__ void __launch_bounds__(LP_THREADS<CL>, LP_WORK<CL> * 32 / LP_THREADS<CL>)
token_logprobs_kernel(const T* logits, int64_t ld, int vocab, const int64_t* token, int top, float* logprob, float* entropy, float* top_logprob,
                      int64_t* top_token, int32_t* status) {
    pdl_begin();
    constexpr int THREADS = LP_THREADS<CL>;
    constexpr int V = 16 / sizeof(T), U = LP_VECTORS, TILE = THREADS * U;      // vectors of a tile
    extern __shared__ __align__(16) char lp_raw[];
    LpShared<THREADS>& s = *reinterpret_cast<LpShared<THREADS>*>(lp_raw);
    if (CL > 1) cluster_arrive();
    const int t = threadIdx.x, lane = t & 31, rank = CL > 1 ? blockIdx.x % CL : 0;
    const int64_t r = blockIdx.x / CL;
    const T* x = logits + r * ld;
    float x_token = NAN;
    if (rank == 0 && t == 0 && token != nullptr) {
        const int64_t i = token[r];
        if (i >= 0 && i < vocab) x_token = to_f32(x[i]);
        else if (status != nullptr) atomicOr(status, SK_DEV_INDEX_OUT_OF_RANGE);
    }
    // the row in 16-byte vectors from the boundary in front of it; this block's share of them
    const int skew = (int)((uintptr_t)x % 16 / sizeof(T)), vectors = (vocab + skew + V - 1) / V, share = (vectors + CL - 1) / CL;
    const int begin = rank * share, end = min(begin + share, vectors);
    if (t == 0) s.n = 0;

    typedef LpVector<T> Vec;
    auto load = [&](int i0, Vec (&v)[U]) {
        const int at = (i0 + t) * V - skew;
        const T* p = x + at;
        auto take = [&](int u) {
            const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p + u * THREADS * V));
            v[u].w[0] = a.x;
            v[u].w[1] = a.y;
            v[u].w[2] = a.z;
            v[u].w[3] = a.w;
        };
        if (i0 * V >= skew && i0 + TILE <= end && (i0 + TILE) * V - skew <= vocab) {      // a tile inside the row
#pragma unroll
            for (int u = 0; u < U; ++u) take(u);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int a = at + u * THREADS * V;
                if (i0 + u * THREADS + t >= end) v[u] = lp_edge(x, vocab, vocab);
                else if (a >= 0 && a + V <= vocab) take(u);
                else v[u] = lp_edge(x, a, vocab);
            }
        }
    };
    auto ask = [&](int i0, int stage) {                        // a tile into shared memory; one commit group each, an empty one behind the row
        if (i0 < end) {
            const int at = (i0 + t) * V - skew;
            if (i0 * V >= skew && i0 + TILE <= end && (i0 + TILE) * V - skew <= vocab) {
#pragma unroll
                for (int u = 0; u < U; ++u) cp16(saddr(&s.tiles[stage][u][t]), x + at + u * THREADS * V, true);
            } else {
#pragma unroll 1
                for (int u = 0; u < U; ++u) {
                    const int a = at + u * THREADS * V;
                    if (i0 + u * THREADS + t < end && a >= 0 && a + V <= vocab) {
                        cp16(saddr(&s.tiles[stage][u][t]), x + a, true);
                    } else {
                        const Vec v = lp_edge(x, i0 + u * THREADS + t < end ? a : vocab, vocab);
                        s.tiles[stage][u][t] = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // What of a tile reaches `bound` goes to the list, vector by vector of the threads that have some: a lane per element, word(u, k, from)
    // the k-th word of the u-th vector of lane `from`
    const int room = lp_room(top, U * V);
    auto append = [&](int i0, bool mine, LpPair bound, auto&& word) {
        for (unsigned who = __ballot_sync(FULL, mine); who != 0u; who &= who - 1) {
            const int from = __ffs(who) - 1, u = lane / Vec::WORD / 4 % U, k = lane / Vec::WORD % 4;
            const uint32_t w = word(u, k, from);
            const int i = i0 + u * THREADS + (t & ~31) + from, at = i * V - skew + k * Vec::WORD + lane % Vec::WORD;
            const LpPair p = lp_pair(Vec::of(w, lane % Vec::WORD), at);
            const bool in = lane < U * V && i < end && at >= 0 && at < vocab && p >= bound;
            const unsigned all = __ballot_sync(FULL, in);
            int place = 0;
            if (lane == 0 && all != 0u) place = atomicAdd(&s.n, __popc(all));
            place = __shfl_sync(FULL, place, 0) + __popc(all & ((1u << lane) - 1));
            if (in && place < room) s.list[place] = p;
        }
    };
    // a thread's pairs of a tile are at most (its largest logit, its first index); a thread outside the row has key 0
    auto key_of = [&](int i0, float most) { return i0 + t < end ? lp_key(most) : 0u; };
    auto reaches = [&](int i0, uint32_t key, LpPair bound) {
        return key != 0u && ((LpPair)key << 32 | (uint32_t)~max((i0 + t) * V - skew, 0)) >= bound;
    };
    // to the list's `top` largest, if it is long; the bound that follows
    auto meet = [&](int n, LpPair bound) {
        if (n <= top + LP_LONG) return bound;
        n = lp_cut(s, n, top);
        if (t < n) s.list[t] = s.best[t];
        if (t == 0) s.n = n;
        if (n == top && s.best[top - 1] > bound) bound = s.best[top - 1];
        __syncthreads();
        return bound;
    };
    // One tile with the whole block: raises the bound where more threads would append than the list has room for
    auto careful = [&](int i0, LpPair bound) {
        Vec v[U];
        load(i0, v);
        float most = v[0].largest();
#pragma unroll
        for (int u = 1; u < U; ++u) most = lp_max(most, v[u].largest());
        const uint32_t key = key_of(i0, most);
        const int some = __syncthreads_count(reaches(i0, key, bound));
        if (some > top + LP_FEW) {
            uint32_t lo = (uint32_t)(bound >> 32);
            int64_t hi = 1ll << 32;                            // at least `top` reach lo, fewer reach hi
            int n = some;
            while (hi - lo > 1) {
                const uint32_t mid = lo + (uint32_t)((hi - lo) / 2);
                const int c = __syncthreads_count(key >= mid);
                if (c >= top) {
                    lo = mid;
                    n = c;
                    if (c <= top + LP_FEW) break;
                } else {
                    hi = mid;
                }
            }
            LpPair b = (LpPair)lo << 32;
            if (n > top + LP_FEW || lo == (uint32_t)(bound >> 32)) {           // many equal maxima: by the index of each thread's first one
                const int above = __syncthreads_count(key > lo);
                int at = INT32_MAX;
                if (key == lo && lo != 0u) {
#pragma unroll
                    for (int u = U - 1; u >= 0; --u)
#pragma unroll
                        for (int k = V / 2 - 1; k >= 0; --k) {
                            const int i = i0 + u * THREADS + t, a = i * V - skew + k * 2;
                            const float2 e = v[u].two(k);
                            if (i < end && a + 1 >= 0 && a + 1 < vocab && lp_key(e.y) == lo) at = a + 1;
                            if (i < end && a >= 0 && a < vocab && lp_key(e.x) == lo) at = a;
                        }
                }
                int il = -1, ih = INT32_MAX - 1;               // fewer than `top` with an index up to il, enough up to ih
                if (above + __syncthreads_count(at <= ih) >= top) {
                    while (ih - il > 1) {
                        const int mid = il + (ih - il) / 2;
                        if (above + __syncthreads_count(at <= mid) >= top) ih = mid;
                        else il = mid;
                    }
                    b |= (uint32_t)~ih;
                }
            }
            if (b > bound) bound = b;
        }
        append(i0, reaches(i0, key, bound), bound, [&](int u, int k, int from) {
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 4 * U; ++j) {
                const uint32_t y = __shfl_sync(FULL, v[j / 4].w[j % 4], from);
                if (u * 4 + k == j) w = y;
            }
            return w;
        });
        __syncthreads();
        return meet(min(s.n, room), bound);
    };

    LpSums sum = {-INFINITY, 0.f, 0.f};
    LpPair bound = 0;                                          // at least `top` pairs of this block reach it, once it is not 0
    int met = begin, n_met = 0;                                // tiles in front of `met` are in the list, of n_met pairs then
    for (int k = 0; k < LP_STAGES - 1; ++k) ask(begin + k * TILE, k);
    int stage = 0;
    for (int i0 = begin, tile = 1; i0 < end; i0 += TILE, ++tile) {
        asm volatile("cp.async.wait_group %0;" ::"n"(LP_STAGES - 2) : "memory");
        __syncwarp();                                          // lanes read one another's words, in this stage and the one to be filled
        ask(i0 + (LP_STAGES - 1) * TILE, (stage + LP_STAGES - 1) % LP_STAGES);
        Vec cur[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint4 a = s.tiles[stage][u][t];
            cur[u].w[0] = a.x;
            cur[u].w[1] = a.y;
            cur[u].w[2] = a.z;
            cur[u].w[3] = a.w;
        }
        float most = cur[0].largest();
#pragma unroll
        for (int u = 1; u < U; ++u) most = lp_max(most, cur[u].largest());
        const bool raise = most > sum.m + LP_SLACK || (sum.m == -INFINITY && most > -INFINITY);
        if (raise) lp_raise(sum, most);
        const float m = sum.m == -INFINITY ? 0.f : sum.m;
        const Lp2 minus = lp_two(-m, -m), log2e = lp_two(LP_LOG2E, LP_LOG2E);
        Lp2 z[U], zd = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            z[u] = 0;
#pragma unroll
            for (int k = 0; k < V / 2; ++k) {
                const float2 e = cur[u].two(k);
                const Lp2 d = lp_add(lp_two(e.x, e.y), minus);
                float y[2];
                lp_split(lp_mul(d, log2e), y[0], y[1]);
                const Lp2 w = lp_two(exp2_fast(y[0]), exp2_fast(y[1]));
                z[u] = lp_add(z[u], w);
                zd = lp_fma(w, d, zd);
            }
        }
        if (raise) {                                           // the vector of the new reference again, without it
            bool out = false;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (!out && cur[u].largest() == most) {
                    float a = 0.f;
#pragma unroll
                    for (int k = 0; k < V / 2; ++k) {
                        const float2 e = cur[u].two(k);
                        const bool x_out = !out && e.x == most, y_out = !out && !x_out && e.y == most;
                        a += x_out ? 0.f : exp2_fast((e.x - m) * LP_LOG2E);
                        a += y_out ? 0.f : exp2_fast((e.y - m) * LP_LOG2E);
                        out |= x_out || y_out;
                    }
                    z[u] = lp_two(a, 0.f);
                }
        }
        float two[2];
        static_assert(U == 4, "the sum of the vectors' sums");
        lp_split(lp_add(lp_add(z[0], z[1]), lp_add(z[2], z[3])), two[0], two[1]);
        sum.z += two[0] + two[1];
        lp_split(zd, two[0], two[1]);
        if (two[0] + two[1] != two[0] + two[1]) {              // a logit of -inf: it adds 0, not 0 * -inf
            two[0] = two[1] = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < V / 2; ++k) {
                    const float2 e = cur[u].two(k);
                    two[0] = fmaf(exp2_fast((e.x - m) * LP_LOG2E), fmaxf(e.x - m, -200.f), two[0]);
                    two[1] = fmaf(exp2_fast((e.y - m) * LP_LOG2E), fmaxf(e.y - m, -200.f), two[1]);
                }
        }
        sum.zd += two[0] + two[1];
        if (top > 0) {
            if (tile == 1) {                                   // an equal share of `top` maxima from each warp inside the row
                const int warps = min((end - i0) / 32, THREADS / 32), each = warps > 0 ? (top + warps - 1) / warps : 33;
                uint32_t left = key_of(i0, most), least = 0;
                if (each <= 32 && t >> 5 < warps)
                    for (int i = 0; i < each; ++i) {
                        least = __reduce_max_sync(FULL, left);
                        const unsigned who = __ballot_sync(FULL, left == least);
                        if (lane == __ffs(who) - 1) left = 0;
                    }
                if (lane == 0) s.least[t >> 5] = least;
                __syncthreads();
                least = each <= 32 ? 0xFFFFFFFFu : 0u;
                for (int w = 0; w < warps; ++w) least = min(least, s.least[w]);
                bound = (LpPair)least << 32;
            }
            append(i0, !(most < lp_value(bound)) && reaches(i0, key_of(i0, most), bound), bound,
                   [&](int u, int k, int from) { return reinterpret_cast<const uint32_t*>(&s.tiles[stage][u][(t & ~31) + from])[k]; });
            if ((tile & (tile - 1)) == 0 || tile % 8 == 0 || i0 + TILE >= end) {
                __syncthreads();
                const int n = s.n;
                if (n <= top + LP_LONG) {
                    n_met = n;
                    __syncthreads();                           // everyone knows n before it grows
                } else if (n <= room) {
                    bound = meet(n, bound);
                    n_met = top;
                } else {                                       // too many: those tiles again, with care
                    __syncthreads();
                    if (t == 0) s.n = n_met;
                    __syncthreads();
                    for (int i = met; i <= i0; i += TILE) bound = careful(i, bound);
                    __syncthreads();
                    n_met = s.n;
                    __syncthreads();
                }
                met = i0 + TILE;
            }
        }
        stage = stage + 1 == LP_STAGES ? 0 : stage + 1;
    }
    // ---- the block's sums and list
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1)
        lp_join(sum, LpSums{__shfl_xor_sync(FULL, sum.m, o), __shfl_xor_sync(FULL, sum.z, o), __shfl_xor_sync(FULL, sum.zd, o)});
    if (lane == 0) s.parts[t >> 5] = sum;
    __syncthreads();
    const int found = top > 0 ? lp_cut(s, s.n, top) : 0;
    sum = s.parts[lane % (THREADS / 32)];
#pragma unroll
    for (int o = THREADS / 64; o >= 1; o >>= 1)
        lp_join(sum, LpSums{__shfl_xor_sync(FULL, sum.m, o), __shfl_xor_sync(FULL, sum.z, o), __shfl_xor_sync(FULL, sum.zd, o)});
    if (CL > 1) {
        cluster_wait();                                        // every block of the cluster has begun
        if (t < top) {                                         // 0 is no pair
            const LpPair p = t < found ? s.best[t] : 0;
            store_first_cta(reinterpret_cast<const uint32_t*>(&s.got[rank][t]), (uint32_t)p);
            store_first_cta(reinterpret_cast<const uint32_t*>(&s.got[rank][t]) + 1, (uint32_t)(p >> 32));
        }
        if (t == 0) {
            store_first_cta(&s.sums[rank].m, sum.m);
            store_first_cta(&s.sums[rank].z, sum.z);
            store_first_cta(&s.sums[rank].zd, sum.zd);
        }
        cluster_arrive();
        cluster_wait();
        if (rank > 0) return;
        sum = s.sums[lane % CL];
#pragma unroll
        for (int o = CL / 2; o >= 1; o >>= 1)
            lp_join(sum, LpSums{__shfl_xor_sync(FULL, sum.m, o), __shfl_xor_sync(FULL, sum.z, o), __shfl_xor_sync(FULL, sum.zd, o)});
        // the rank of a pair among all blocks': how many of each block's sorted list are larger
        if (top > 0) {
            for (int i = t; i < CL * top; i += THREADS) {
                const LpPair p = s.got[i / top][i % top];
                int above = 0;
                for (int c = 0; c < CL; ++c) {
                    int lo = 0, hi = top;                      // the first of the list that is not larger
                    while (lo < hi) {
                        const int mid = (lo + hi) / 2;
                        if (s.got[c][mid] > p) lo = mid + 1;
                        else hi = mid;
                    }
                    above += lo;
                }
                if (p != 0 && above < top) s.best[above] = p;
            }
            __syncthreads();
        }
    }
    // ---- the row's results, of one lane's sums: of two equal references either may have become the other's
    sum.m = __shfl_sync(FULL, sum.m, 0);
    sum.z = __shfl_sync(FULL, sum.z, 0);
    sum.zd = __shfl_sync(FULL, sum.zd, 0);
    const float lz = fabsf(sum.m) == INFINITY ? NAN : log1pf(sum.z);      // no logit above -inf, or one of +inf: no distribution
    if (t == 0) {
        if (entropy != nullptr) entropy[r] = lz - sum.zd / (1.f + sum.z);
        if (token != nullptr) logprob[r] = x_token - sum.m - lz;
    }
    if (t < top) {
        const LpPair p = s.best[t];
        top_logprob[r * top + t] = lp_value(p) - sum.m - lz;
        top_token[r * top + t] = (int)~(uint32_t)p;
    }
}

template <typename T, int CL>
int logprobs_launch(const void* logits, int64_t ld, int64_t rows, int vocab, const int64_t* token, int top, float* logprob, float* entropy,
                    float* top_logprob, int64_t* top_token, int32_t* status, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * CL));
    cfg.blockDim = dim3(LP_THREADS<CL>);
    constexpr int OF_THREAD = LP_VECTORS * 16 / (int)sizeof(T);
    cfg.dynamicSmemBytes = sizeof(LpShared<LP_THREADS<CL>>) + lp_room(top, OF_THREAD) * sizeof(LpPair);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CL;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CL > 1 ? 2 : 1;
    static SmemLimit limit;
    const cudaError_t e = limit.raise((const void*)token_logprobs_kernel<T, CL>, sizeof(LpShared<LP_THREADS<CL>>) + lp_room(LP_TOP, OF_THREAD) * sizeof(LpPair));
    if (e != cudaSuccess) return check_chained(e, "token_logprobs_kernel");
    return check_chained(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, CL>, (const T*)logits, ld, vocab, token, top, logprob, entropy,
                                            top_logprob, top_token, status), "token_logprobs_kernel");
}

}  // namespace

int token_logprobs(const void* logits, int dtype, int64_t ld, int64_t rows, int vocab, const int64_t* token, int top, float* logprob,
                   float* entropy, float* top_logprob, int64_t* top_token, int32_t* status, cudaStream_t st) {
    SK_REQUIRE(valid_dtype(dtype) && rows >= 0 && vocab > 0, "token_logprobs: bad sizes or dtype");
    SK_REQUIRE(top >= 0 && top <= LP_TOP && top <= vocab, "token_logprobs: %d alternatives of %d", top, vocab);
    if (rows == 0) return SK_OK;
    SK_REQUIRE(logits && (ld >= vocab || rows == 1) && (!token || logprob) && (top == 0 || (top_logprob && top_token)),
               "token_logprobs: null pointer or overlapping rows");
    if (!aligned(logits, esize(dtype))) return fail(SK_ERR_MISALIGNED, "token_logprobs: logits off an element's boundary");
    if (rows > 0x7fffffff / 8 || vocab > 0x7fffffff - 65536) return fail(SK_ERR_UNSUPPORTED, "token_logprobs: %lld rows of %d", (long long)rows, vocab);
    auto go = [&](auto t) {
        using T = decltype(t);
        auto with = [&](auto cl) {
            return logprobs_launch<T, decltype(cl)::value>(logits, ld, rows, vocab, token, top, logprob, entropy, top_logprob, top_token, status, st);
        };
        // blocks of a row: as long as they find a place at once on the SMs and have a tile to walk
        const int64_t places = (int64_t)sm_count() * (LP_WORK<8> * 32 / LP_CLUSTERED);
        if (rows * 8 <= places && vocab >= 8 * 2048) return with(std::integral_constant<int, 8>{});
        if (rows * 4 <= places && vocab >= 4 * 2048) return with(std::integral_constant<int, 4>{});
        if (rows * 2 <= places && vocab >= 2 * 2048) return with(std::integral_constant<int, 2>{});
        return with(std::integral_constant<int, 1>{});
    };
    if (dtype == SK_F32) return go(float{});
    return dtype == SK_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}

}  // namespace sk
