// Eviction from a paged cache by collected attention weight.
#include "paged.cuh"

namespace sk {
namespace {

constexpr int EV_THREADS = 1024;
struct EvMove {
    int from;
    float mass;
    int pos;
    int pad;
};

// What a slot is ranked by: slots kept for sure above all, NaN above numbers
__device__ __forceinline__ uint32_t ev_key(float mass, bool sure) {
    return sure ? 0xFFFFFFFFu : mass != mass ? 0xFFFFFFFEu : order_key(mass);
}

// Exclusive prefix sum over the block of one flag per thread, `total` over all
__device__ __forceinline__ int ev_scan(bool f, int* part, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned all = __ballot_sync(FULL, f);
    __syncthreads();
    if (lane == 0) part[warp] = __popc(all);
    __syncthreads();
    int before = 0, sum = 0;
    for (int w = 0; w < EV_THREADS / 32; ++w) {
        if (w < warp) before += part[w];
        sum += part[w];
    }
    total = sum;
    return before + __popc(all & ((1u << lane) - 1));
}

// One block per (sequence, key/value head).  The budget-th largest key by four digits of eight bits, then one walk over the slots in
// order: which stay, which go, which move where.
__global__ void __launch_bounds__(EV_THREADS)
paged_evict_kernel(const __grid_constant__ sk_paged_cache c, int budget, int recent, int sink, float* mass_out, int64_t mo_bs, int64_t mo_hs,
                   int32_t* pos_out, int64_t po_bs, int64_t po_hs, EvMove* moves) {
    __shared__ uint32_t hist[256];
    __shared__ int part[32], newest_s, need_s;
    __shared__ uint32_t prefix_s;
    const int g = blockIdx.x % c.G, b = blockIdx.x / c.G, t = threadIdx.x, cap = c.width * c.page, es = c.dtype == SK_F32 ? 4 : 2;
    const float* mass = c.mass + b * c.mass_bs + g * c.mass_hs;
    const int32_t* pos = c.positions + b * c.pos_bs + g * c.pos_hs;
    float* mo = mass_out + b * mo_bs + g * mo_hs;
    int32_t* po = pos_out + b * po_bs + g * po_hs;
    bool over;
    const int n = paged_length(c, b, 0, &over), kept = min(n, budget);
    if (over && t == 0 && c.status != nullptr) atomicOr(c.status, SK_DEV_POS_OUT_OF_RANGE);
    if (n <= budget) {
        for (int j = t; j < cap; j += EV_THREADS) {
            mo[j] = j < n ? mass[j] : 0.f;
            po[j] = j < n ? pos[j] : -1;
        }
        return;
    }
    if (t == 0) newest_s = INT32_MIN;
    __syncthreads();
    int newest = INT32_MIN;
    for (int j = t; j < n; j += EV_THREADS) newest = max(newest, pos[j]);
    atomicMax(&newest_s, newest);
    __syncthreads();
    const int64_t late = (int64_t)newest_s - recent;
    auto key = [&](int j) { return ev_key(mass[j], pos[j] < sink || pos[j] > late); };
    uint32_t prefix = 0;
    int need = budget;                                         // of the keys that share the prefix
    for (int digit = 24; digit >= 0; digit -= 8) {
        if (t < 256) hist[t] = 0;
        __syncthreads();
        for (int j = t; j < n; j += EV_THREADS) {
            const uint32_t k = key(j);
            if (digit == 24 || k >> (digit + 8) == prefix) atomicAdd(&hist[k >> digit & 255], 1u);
        }
        __syncthreads();
        if (t == 0) {
            int left = need, d = 255;
            while ((int)hist[d] < left) left -= hist[d--];
            need_s = left;
            prefix_s = prefix << 8 | d;
        }
        __syncthreads();
        need = need_s;
        prefix = prefix_s;
        __syncthreads();
    }
    // every key above the prefix and the first `need` that equal it are kept
    EvMove* mv = moves + (int64_t)blockIdx.x * budget;
    auto walk = [&](auto&& at) {                               // at(slot, live, kept, its place among the kept equal ones known)
        int equal = 0;
        for (int j0 = 0; j0 < n; j0 += EV_THREADS) {
            const int j = j0 + t;
            const uint32_t k = j < n ? key(j) : 0;
            int sum;
            const int place = ev_scan(j < n && k == prefix, part, sum);
            at(j, j < n, j < n && (k > prefix || (k == prefix && equal + place < need)));
            equal += sum;
        }
    };
    int moved = 0;
    walk([&](int j, bool live, bool keep) {
        int sum;
        const bool mover = live && keep && j >= budget;
        const int i = ev_scan(mover, part, sum);
        if (mover) mv[moved + i] = EvMove{j, mass[j], pos[j], 0};
        moved += sum;
    });
    __syncthreads();
    const int shift = 31 - __clz(c.page), pieces = c.D * es / 16;
    int freed = 0;
    walk([&](int j, bool live, bool keep) {
        int sum;
        const bool hole = live && !keep && j < budget;
        const int i = freed + ev_scan(hole, part, sum);
        freed += sum;
        const float m = live ? mass[j] : 0.f;
        const int p = live ? pos[j] : 0;
        __syncthreads();
        if (hole) {
            const EvMove e = mv[i];
            mo[j] = e.mass;
            po[j] = e.pos;
            const int from = c.table[b * c.table_ld + (e.from >> shift)], to = c.table[b * c.table_ld + (j >> shift)];
            if (paged_page_ok(c, from) && paged_page_ok(c, to)) {
                const int rf = e.from & (c.page - 1), rt = j & (c.page - 1);
                const uint4* ks = (const uint4*)((const char*)c.k + (from * c.k_ps + g * c.k_hs + rf * c.k_rs) * es);
                const uint4* vs = (const uint4*)((const char*)c.v + (from * c.v_ps + g * c.v_hs + rf * c.v_rs) * es);
                uint4* kd = (uint4*)((char*)c.k + (to * c.k_ps + g * c.k_hs + rt * c.k_rs) * es);
                uint4* vd = (uint4*)((char*)c.v + (to * c.v_ps + g * c.v_hs + rt * c.v_rs) * es);
                for (int x = 0; x < pieces; ++x) {
                    kd[x] = ks[x];
                    vd[x] = vs[x];
                }
            } else if (c.status != nullptr) {
                atomicOr(c.status, SK_DEV_INDEX_OUT_OF_RANGE);
            }
        } else if (live && j < budget) {
            mo[j] = m;
            po[j] = p;
        }
    });
    __syncthreads();
    for (int j = kept + t; j < cap; j += EV_THREADS) {
        mo[j] = 0.f;
        po[j] = -1;
    }
}

__global__ void paged_evict_lengths_kernel(const __grid_constant__ sk_paged_cache c, int budget, int32_t* lengths_out) {
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b < c.B) lengths_out[b] = min(paged_length(c, b, 0), budget);
}

}  // namespace

size_t paged_evict_workspace(const sk_paged_cache& c, int budget) { return (size_t)c.B * c.G * budget * sizeof(EvMove); }

int launch_paged_evict(const sk_paged_cache& c, int budget, int recent, int sink, float* mass_out, int64_t mo_bs, int64_t mo_hs,
                       int32_t* pos_out, int64_t po_bs, int64_t po_hs, int32_t* lengths_out, void* workspace, cudaStream_t st) {
    paged_evict_kernel<<<c.B * c.G, EV_THREADS, 0, st>>>(c, budget, recent, sink, mass_out, mo_bs, mo_hs, pos_out, po_bs, po_hs, (EvMove*)workspace);
    if (int rc = check_launch("paged_evict_kernel")) return rc;
    paged_evict_lengths_kernel<<<(c.B + 255) / 256, 256, 0, st>>>(c, budget, lengths_out);
    return check_launch("paged_evict_lengths_kernel");
}

}  // namespace sk
