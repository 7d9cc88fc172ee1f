// Eviction from a paged cache by collected attention weight.
//
// A cluster per (sequence, key/value head): slots are ranked by a 32-bit key that grows with their mass; the key of the
// last slot to be kept is found by four histograms of eight bits, summed over the cluster, and equal keys go by slot.  Then every slot
// is kept or not, and the i-th freed slot below the budget and the i-th kept one behind it are written side by side.  A
// list entry is a row of K, a row of V, a mass and a position to move; sources lie behind the budget and targets below it, so the
// cluster's blocks move entries in any order once the list is complete.  Of keys and values only what moves is read, 241 of 4352 rows; positions once and
// masses twice (the second time from L2), where a block's slots find room on chip.
//
// Measured, 8 heads of 128: 32 sequences from 4352 to 4096 slots 26.7 us (about 14 in passes of three barriers each, then 63 MB of rows), one from
// 32768 to 4096 25.7 us (13 until its moves begin: passes end in barriers of the cluster).  Always four passes: 28.2 and 28; list and table read when
// a move needs them instead of a turn ahead: 26.8 and 26.8; every warp finding the digit for itself, a barrier less a pass: 27.3 and 26.9.  With the moves in
// a kernel of their own 3 more, and a launch; with three histograms of 2048 bins 29 and 52, words of other blocks cost that much.
#include "paged.cuh"

#include <atomic>
#include <type_traits>

namespace sk {
namespace {

constexpr int EV_THREADS = 512, EV_WARPS = EV_THREADS / 32, EV_CLUSTER = 16;
// Two blocks an SM, which leaves registers for two moves a thread under way.  One block with four (4 sequences of 8 heads, 32768 to 4096 slots):
// 79 us, as their 256 blocks then come in two turns; two blocks with two moves 43
constexpr int EV_PER_SM = 2, EV_MOVES = 2;
constexpr int EV_SLOTS = 24576;                                // of a block, whose keys and positions find room in shared memory
constexpr int EV_SLOTS_OF_TWO = 13824;                         // where two blocks share an SM
struct alignas(16) EvMove {
    int from, to;
    float mass;
    int pos;
};
struct EvShared {
    uint32_t hist[2][256], total[256];
    int newest, equals, holes, movers;                         // of this block; read by the cluster
    int digit, need, equal;
    int part[3][EV_WARPS];
};

// What a slot is ranked by: slots kept for sure above all, NaN above numbers
__device__ __forceinline__ uint32_t ev_key(float mass) { return mass != mass ? 0xFFFFFFFEu : min(order_key(mass), 0xFFFFFFFEu); }

// A word of every block's shared memory, at the place `local` has in this one's, all asked for before the first is used; the caller has
// passed a cluster barrier behind their writes
template <int CL> __device__ __forceinline__ void ev_remote(const void* local, uint32_t (&v)[CL]) {
    uint32_t at[CL];
#pragma unroll
    for (int r = 0; r < CL; ++r) asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at[r]) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(r));
    if constexpr (CL == 8) {
        asm volatile(
            "ld.shared::cluster.u32 %0, [%8];\n\tld.shared::cluster.u32 %1, [%9];\n\tld.shared::cluster.u32 %2, [%10];\n\t"
            "ld.shared::cluster.u32 %3, [%11];\n\tld.shared::cluster.u32 %4, [%12];\n\tld.shared::cluster.u32 %5, [%13];\n\t"
            "ld.shared::cluster.u32 %6, [%14];\n\tld.shared::cluster.u32 %7, [%15];"
            : "=&r"(v[0]), "=&r"(v[1]), "=&r"(v[2]), "=&r"(v[3]), "=&r"(v[4]), "=&r"(v[5]), "=&r"(v[6]), "=&r"(v[7])
            : "r"(at[0]), "r"(at[1]), "r"(at[2]), "r"(at[3]), "r"(at[4]), "r"(at[5]), "r"(at[6]), "r"(at[7]) : "memory");
    } else {
#pragma unroll
        for (int r = 0; r < CL; ++r) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v[r]) : "r"(at[r]) : "memory");
    }
}
template <int CL> __device__ __forceinline__ void ev_sync() {
    if (CL == 1) __syncthreads();
    else {
        cluster_arrive();
        cluster_wait();
    }
}

template <int CL>
__global__ void __launch_bounds__(EV_THREADS, EV_PER_SM)
paged_evict_kernel(const __grid_constant__ sk_paged_cache c, int budget, int recent, int sink, float* mass_out, int64_t mo_bs, int64_t mo_hs,
                   int32_t* pos_out, int64_t po_bs, int64_t po_hs, int32_t* lengths_out, EvMove* moves, int most_moves, int room) {
    pdl_begin();
    extern __shared__ uint32_t ev_raw[];                       // keys, then positions of this block's slots
    __shared__ EvShared s;
    const int rank = CL > 1 ? blockIdx.x % CL : 0, row = blockIdx.x / CL, g = row % c.G, b = row / c.G, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int cap = c.width * c.page;
    const float* mass = c.mass + b * c.mass_bs + g * c.mass_hs;
    const int32_t* pos = c.positions + b * c.pos_bs + g * c.pos_hs;
    float* mo = mass_out + b * mo_bs + g * mo_hs;
    int32_t* po = pos_out + b * po_bs + g * po_hs;
    bool over;
    const int n = paged_length(c, b, 0, &over), kept = min(n, budget);
    if (rank == 0 && t == 0) {
        if (over && c.status != nullptr) atomicOr(c.status, SK_DEV_POS_OUT_OF_RANGE);
        if (lengths_out != nullptr && g == 0) lengths_out[b] = kept;
    }
    for (int j = n + rank * EV_THREADS + t; j < cap; j += CL * EV_THREADS) {
        mo[j] = 0.f;
        po[j] = -1;
    }
    if (n <= budget) {                                         // the whole cluster: nothing goes
        for (int j = rank * EV_THREADS + t; j < n; j += CL * EV_THREADS) {
            const float m = mass[j];
            const int p = pos[j];
            mo[j] = m;
            po[j] = p;
        }
        return;
    }
    const int share = (n + CL - 1) / CL, j0 = min(rank * share, n), j1 = min(j0 + share, n), count = j1 - j0;
    if (t == 0) s.newest = INT32_MIN;
    for (int i = t; i < 256; i += EV_THREADS) s.hist[0][i] = 0;
    __syncthreads();
    EvMove* list = moves + (int64_t)row * most_moves;
    int moves_n = 0;
    auto select = [&](auto on_chip) {
        constexpr bool HELD = decltype(on_chip)::value;        // keys and positions in shared memory; else they are read again
        uint32_t* keys = ev_raw;
        int32_t* places = reinterpret_cast<int32_t*>(ev_raw + room);
        int newest = INT32_MIN;
#pragma unroll 8
        for (int i = t; i < count; i += EV_THREADS) {
            const int p = pos[j0 + i];
            newest = max(newest, p);
            if (HELD) {
                keys[i] = ev_key(mass[j0 + i]);
                places[i] = p;
            }
        }
        newest = __reduce_max_sync(FULL, newest);
        if (lane == 0) atomicMax(&s.newest, newest);
        ev_sync<CL>();
        newest = s.newest;
        if constexpr (CL > 1) {
            uint32_t v[CL];
            ev_remote<CL>(&s.newest, v);
#pragma unroll
            for (int r = 0; r < CL; ++r) newest = max(newest, (int)v[r]);
        }
        const int late = (int)max((int64_t)newest - recent, (int64_t)INT32_MIN);
        auto sure = [&](int p) { return p < sink || p > late; };
        auto key = [&](int i) {                                // of slot j0 + i, after the first pass
            return HELD ? keys[i] : sure(pos[j0 + i]) ? 0xFFFFFFFFu : ev_key(mass[j0 + i]);
        };

        // ---- the smallest key that is kept, and how many of that key
        uint32_t prefix = 0;
        int need = budget;
        for (int i0 = 0; i0 < count; i0 += EV_THREADS) {       // masses share few exponents: equal bins are added up in the warp
            const int i = i0 + t;
            uint32_t k = 0;
            if (i < count) {
                k = HELD ? (sure(places[i]) ? 0xFFFFFFFFu : keys[i]) : key(i);
                if (HELD) keys[i] = k;
            }
            warp_hist_add(s.hist[0], k >> 24, i < count);
        }
#pragma unroll 1
        for (int pass = 0; pass < 4; ++pass) {
            uint32_t* hist = s.hist[pass & 1];
            if (pass > 0) {
                const int shift = 24 - 8 * pass;
#pragma unroll 4
                for (int i = t; i < count; i += EV_THREADS) {
                    const uint32_t k = key(i);
                    if (k >> shift >> 8 == prefix) atomicAdd(&hist[k >> shift & 255], 1u);
                }
            }
            ev_sync<CL>();
            if (t < 256) {
                uint32_t sum = hist[t];
                if constexpr (CL > 1) {
                    uint32_t v[CL];
                    ev_remote<CL>(hist + t, v);
                    sum = 0;
#pragma unroll
                    for (int r = 0; r < CL; ++r) sum += v[r];
                }
                s.total[t] = sum;
                s.hist[(pass + 1) & 1][t] = 0;                 // read by the others before the barrier
            }
            __syncthreads();
            if (warp == 0) {                                   // lane: eight bins, the largest first
                int mine = 0;
#pragma unroll
                for (int x = 0; x < 8; ++x) mine += s.total[255 - lane * 8 - x];
                int sum = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(FULL, sum, o);
                    if (lane >= o) sum += x;
                }
                int above = sum - mine;
                if (above < need && sum >= need) {
                    int d = 255 - lane * 8;
                    while (above + (int)s.total[d] < need) above += s.total[d--];
                    s.digit = d;
                    s.need = need - above;
                    s.equal = s.total[d];
                }
            }
            __syncthreads();
            prefix = prefix << 8 | s.digit;
            need = s.need;
            if (s.equal == need) {                             // all that are left are kept, in every block of the cluster
                prefix <<= 24 - 8 * pass;
                break;
            }
        }
        const bool ties = s.equal > need;                      // only some of the equal keys are kept: the first ones

        // ---- in slot order, a run of slots per warp: freed slots, kept slots behind the budget
        const int run = (count + EV_WARPS * 32 - 1) / (EV_WARPS * 32) * 32, i0 = min(warp * run, count), i1 = min(i0 + run, count);
        auto before = [&](int which, int& all) {               // sum over the warps in front; `all`: over the block
            const int x = lane < EV_WARPS ? s.part[which][lane] : 0;
            all = __reduce_add_sync(FULL, x);
            return __reduce_add_sync(FULL, lane < warp ? x : 0);
        };
        int equal_at = 0, all;
        if (ties) {
            int equal = 0;
            for (int i = i0 + lane; i - lane < i1; i += 32) equal += __popc(__ballot_sync(FULL, i < i1 && key(i) == prefix));
            if (lane == 0) s.part[0][warp] = equal;
            __syncthreads();
            equal_at = before(0, all);
            if constexpr (CL > 1) {
                if (t == 0) s.equals = all;
                ev_sync<CL>();
                uint32_t v[CL];
                ev_remote<CL>(&s.equals, v);
#pragma unroll
                for (int r = 0; r < CL; ++r) equal_at += r < rank ? (int)v[r] : 0;
            }
        }
        // one step of the walk over a warp's run: is slot i kept
        auto keeps = [&](int i, int& seen) {
            const uint32_t k = i < i1 ? key(i) : 0u;
            if (!ties) return i < i1 && k >= prefix;
            const unsigned same = __ballot_sync(FULL, i < i1 && k == prefix);
            const bool keep = i < i1 && (k > prefix || (k == prefix && seen + __popc(same & ((1u << lane) - 1)) < need));
            seen += __popc(same);
            return keep;
        };
        const int low = budget - j0;                           // slots of this block below the budget
        int holes = 0, movers = 0, seen = equal_at;
        for (int i = i0 + lane; i - lane < i1; i += 32) {
            const bool keep = keeps(i, seen);
            holes += i < i1 && !keep && i < low;
            movers += keep && i >= low;
        }
        holes = __reduce_add_sync(FULL, holes);
        movers = __reduce_add_sync(FULL, movers);
        if (lane == 0) {
            s.part[1][warp] = holes;
            s.part[2][warp] = movers;
        }
        __syncthreads();
        int all_holes, all_movers, hole_at = before(1, all_holes), mover_at = before(2, all_movers);
        if constexpr (CL > 1) {
            if (t == 0) {
                s.holes = all_holes;
                s.movers = all_movers;
            }
            ev_sync<CL>();
            uint32_t h[CL], m[CL];
            ev_remote<CL>(&s.holes, h);
            ev_remote<CL>(&s.movers, m);
            all_movers = 0;
#pragma unroll
            for (int r = 0; r < CL; ++r) {
                hole_at += r < rank ? (int)h[r] : 0;
                mover_at += r < rank ? (int)m[r] : 0;
                all_movers += (int)m[r];
            }
        }
        moves_n = all_movers;
        seen = equal_at;
        constexpr int STEPS = 4;                               // whose masses are asked for at a time
        for (int first = i0; first < i1; first += 32 * STEPS) {
            float m[STEPS];
            int p[STEPS];
#pragma unroll
            for (int u = 0; u < STEPS; ++u) {
                const int i = first + u * 32 + lane;
                m[u] = i < i1 ? mass[j0 + i] : 0.f;
                p[u] = i < i1 ? (HELD ? places[i] : pos[j0 + i]) : 0;
            }
#pragma unroll
            for (int u = 0; u < STEPS; ++u) {
                const int i = first + u * 32 + lane, j = j0 + i;
                const bool keep = keeps(i, seen), hole = i < i1 && !keep && i < low, mover = keep && i >= low;
                const unsigned h = __ballot_sync(FULL, hole), v = __ballot_sync(FULL, mover);
                if (hole) list[hole_at + __popc(h & ((1u << lane) - 1))].to = j;
                if (mover) {
                    EvMove* e = list + mover_at + __popc(v & ((1u << lane) - 1));
                    e->from = j;
                    e->mass = m[u];
                    e->pos = p[u];
                }
                if (i < i1 && !hole) {                         // a hole's are written with the move
                    mo[j] = i < low ? m[u] : 0.f;
                    po[j] = i < low ? p[u] : -1;
                }
                hole_at += __popc(h);
                mover_at += __popc(v);
            }
        }
    };
    if (share <= room) select(std::true_type{});
    else select(std::false_type{});
    ev_sync<CL>();                                             // the list is complete, and the others' counts are read

    // ---- moves: a thread per 16-byte piece of some of them
    const int es = c.dtype == SK_F32 ? 4 : 2, pieces = c.D * es / 16, per = 1 << (32 - __clz(pieces - 1)), p = t & (per - 1);
    const int step = EV_THREADS / per, shift = 31 - __clz(c.page);
    int4 next[EV_MOVES];
    int next_from[EV_MOVES], next_to[EV_MOVES];
    auto fetch = [&](int i0) {                                 // of the list and the table, a turn ahead
#pragma unroll
        for (int x = 0; x < EV_MOVES; ++x)
            if (i0 + x * step < moves_n) next[x] = __ldcg(reinterpret_cast<const int4*>(list + i0 + x * step));
#pragma unroll
        for (int x = 0; x < EV_MOVES; ++x)
            if (i0 + x * step < moves_n) {
                next_from[x] = __ldcg(c.table + b * c.table_ld + (next[x].x >> shift));
                next_to[x] = __ldcg(c.table + b * c.table_ld + (next[x].y >> shift));
            }
    };
    const int first = rank * EV_MOVES * step + t / per;
    fetch(first);
    for (int i0 = first; i0 < moves_n; i0 += CL * EV_MOVES * step) {
        int4 e[EV_MOVES];
        int from[EV_MOVES], to[EV_MOVES];
#pragma unroll
        for (int x = 0; x < EV_MOVES; ++x) {
            e[x] = next[x];
            from[x] = next_from[x];
            to[x] = next_to[x];
        }
        uint4 k[EV_MOVES], v[EV_MOVES];
        bool ok[EV_MOVES];
#pragma unroll
        for (int x = 0; x < EV_MOVES; ++x) {
            ok[x] = i0 + x * step < moves_n && paged_page_ok(c, from[x]) && paged_page_ok(c, to[x]);
            if (ok[x] && p < pieces) {
                const int r = e[x].x & (c.page - 1);
                k[x] = __ldcs(reinterpret_cast<const uint4*>((const char*)c.k + (from[x] * c.k_ps + g * c.k_hs + r * c.k_rs) * es) + p);
                v[x] = __ldcs(reinterpret_cast<const uint4*>((const char*)c.v + (from[x] * c.v_ps + g * c.v_hs + r * c.v_rs) * es) + p);
            }
        }
        fetch(i0 + CL * EV_MOVES * step);
#pragma unroll
        for (int x = 0; x < EV_MOVES; ++x) {
            if (i0 + x * step >= moves_n) continue;
            if (ok[x] && p < pieces) {
                const int r = e[x].y & (c.page - 1);
                reinterpret_cast<uint4*>((char*)c.k + (to[x] * c.k_ps + g * c.k_hs + r * c.k_rs) * es)[p] = k[x];
                reinterpret_cast<uint4*>((char*)c.v + (to[x] * c.v_ps + g * c.v_hs + r * c.v_rs) * es)[p] = v[x];
            }
            if (p == 0) {
                mo[e[x].y] = __int_as_float(e[x].z);
                po[e[x].y] = e[x].w;
                if (!ok[x] && c.status != nullptr) atomicOr(c.status, SK_DEV_INDEX_OUT_OF_RANGE);
            }
        }
    }
}

// New lengths in place of the old ones, which blocks of the kernel before read
__global__ void __launch_bounds__(256)
paged_evict_lengths_kernel(const __grid_constant__ sk_paged_cache c, int budget, int32_t* lengths_out) {
    pdl_begin();
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b < c.B) lengths_out[b] = min(paged_length(c, b, 0), budget);
}

// Do clusters of 16 blocks, more than every GPU takes, find a place on this device with all the shared memory that a block may have: asked of
// the driver once per device
bool ev_sixteen() {
    constexpr int MAX_DEV = 64;
    static std::atomic<int> known[MAX_DEV];                    // 0: not asked yet, 1: no, 2: yes
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEV) {
        cudaGetLastError();
        return false;
    }
    if (const int k = known[dev].load(std::memory_order_relaxed)) return k == 2;
    auto kern = paged_evict_kernel<EV_CLUSTER>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(EV_CLUSTER);
    cfg.blockDim = dim3(EV_THREADS);
    cfg.dynamicSmemBytes = (size_t)EV_SLOTS * 8;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = EV_CLUSTER;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_SLOTS * 8) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
        cudaGetLastError();                                    // no such clusters then, and no error of the next launch
        n = 0;
    }
    known[dev].store(n > 0 ? 2 : 1, std::memory_order_relaxed);
    return n > 0;
}

struct EvPlan {
    int cluster, room, most_moves;
    size_t total;                                              // bytes of the lists
};
EvPlan ev_plan(const sk_paged_cache& c, int budget) {
    EvPlan p;
    const int64_t rows = (int64_t)c.B * c.G, cap = (int64_t)c.width * c.page;
    // Blocks of a row: twice as many while they find a place at once, two an SM, and then have four slots a thread; more where a block's slots have no
    // room on chip.  Sixteen come later, with eight slots a thread (one row of 65536 slots 26 us by 16 and 34 by 8, eight of 32768 29 and 26), and for
    // more rows than half fill the GPU only where eight would not share SMs (16 rows of 131072 slots 192 and 281, of 70000 117 and 104).  Where the
    // device has no place for sixteen, eight do it too: slots without room on chip are read again
    p.cluster = 1;
    while (p.cluster < EV_CLUSTER) {
        const bool find_places = rows * 2 * p.cluster <= 2 * sm_count(), sixteen = p.cluster == 8;
        const bool pays = !sixteen ? cap >= (int64_t)8 * EV_THREADS * p.cluster
                                   : cap >= (int64_t)16 * EV_THREADS * 8 && (rows * 16 <= sm_count() || cap > (int64_t)EV_SLOTS_OF_TWO * 8);
        if (!(find_places && pays) && (cap + p.cluster - 1) / p.cluster <= EV_SLOTS) break;
        if (sixteen && !ev_sixteen()) break;
        p.cluster *= 2;
    }
    const int64_t share = (cap + p.cluster - 1) / p.cluster;
    p.room = (int)(share < EV_SLOTS ? share : EV_SLOTS);
    const int64_t behind = cap > budget ? cap - budget : 0;
    p.most_moves = (int)(behind < budget ? behind : budget);
    p.total = (size_t)rows * p.most_moves * sizeof(EvMove);
    return p;
}

template <int CL>
int evict_launch(const sk_paged_cache& c, int budget, int recent, int sink, float* mass_out, int64_t mo_bs, int64_t mo_hs, int32_t* pos_out,
                 int64_t po_bs, int64_t po_hs, int32_t* lengths_out, EvMove* moves, const EvPlan& p, cudaStream_t st) {
    static SmemLimit limit;
    cudaError_t e = limit.raise((const void*)paged_evict_kernel<CL>, (size_t)EV_SLOTS * 8);
    if (e != cudaSuccess) return check_chained(e, "paged_evict_kernel");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(c.B * c.G * CL));
    cfg.blockDim = dim3(EV_THREADS);
    cfg.dynamicSmemBytes = (size_t)p.room * 8;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CL;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CL > 1 ? 2 : 1;
    return check_chained(cudaLaunchKernelEx(&cfg, paged_evict_kernel<CL>, c, budget, recent, sink, mass_out, mo_bs, mo_hs, pos_out, po_bs, po_hs, lengths_out,
                                            moves, p.most_moves, p.room), "paged_evict_kernel");
}

}  // namespace

size_t paged_evict_workspace(const sk_paged_cache& c, int budget) { return ev_plan(c, budget).total; }

int launch_paged_evict(const sk_paged_cache& c, int budget, int recent, int sink, float* mass_out, int64_t mo_bs, int64_t mo_hs,
                       int32_t* pos_out, int64_t po_bs, int64_t po_hs, int32_t* lengths_out, void* workspace, cudaStream_t st) {
    const EvPlan p = ev_plan(c, budget);
    if ((int64_t)c.B * c.G * EV_CLUSTER > INT32_MAX) return fail(SK_ERR_UNSUPPORTED, "sk_paged_evict: %d sequences with %d heads", c.B, c.G);
    const bool apart = lengths_out + c.B <= c.lengths || c.lengths + c.B <= lengths_out;
    auto go = p.cluster == 16 ? evict_launch<16> : p.cluster == 8 ? evict_launch<8> : p.cluster == 4 ? evict_launch<4> : p.cluster == 2 ? evict_launch<2> : evict_launch<1>;
    if (int rc = go(c, budget, recent, sink, mass_out, mo_bs, mo_hs, pos_out, po_bs, po_hs, apart ? lengths_out : nullptr, (EvMove*)workspace, p, st))
        return rc;
    if (apart) return SK_OK;
    return check_chained(launch_after(paged_evict_lengths_kernel, dim3((unsigned)((c.B + 255) / 256)), dim3(256), 0, st, c, budget, lengths_out),
                         "paged_evict_lengths_kernel");
}

}  // namespace sk
