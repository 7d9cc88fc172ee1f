// Softmax attention of one new token per sequence over a paged cache, split over the keys and joined.
//
//   out_h = sum_j w_hj v_j,  w_hj = exp(s_hj - m_h) / l_h,  s_hj = scale q_h . k_j,  m_h = max_j s_hj,  l_h = sum_j exp(s_hj - m_h)
//
// in one pass over the keys with a running maximum, and mass_j += sum over the head's queries of w_hj.  Bound by the bytes of
// keys and values: 2 D elements a key, each read once for all query heads of its key/value head.
//
// Work: all keys of all (sequence, key/value head) pairs stand in one row of chunks of WARPS x 16 keys, and every block takes an
// equal run of it, so that ragged batches load the SMs evenly.  A warp works by itself on its 16 keys of a chunk - 16 keys never
// leave a page - with three stages of asynchronous copies of its own and no block barrier.  Only where a run crosses into the next
// pair, or ends, the block's warps join; a pair inside one run is then finished, others leave a partial result for a second kernel.
// The second kernel also adds the weights to mass, from scores that the first one leaves behind (they need the final maximum and sum).
//
// Measured, 32 / 8 heads of 128: 32768 keys 29 us (134 MB; first kernel 26 at 5.1 TB/s, the start and end of a block's run 5 of them), 4 x 131072 with
// mass 375 us (350 at 6.3 TB/s and 25), 64 sequences of 1 to 8003 with mass 57.7 us (49 and 8; fp16 59.0).  Eight warps a block and one block an SM: two blocks of
// four cost the ragged batch 2 us and the long one 4.  A pair's end counted as one chunk: as two 3 us more, with work measured in tiles 1 to 50.
//
// 16-bit types: S^T = K Q^T and O^T = V^T P^T by m16n8k16 products, keys and then value columns in the 16 rows and up to 8 query heads in
// the 8 columns, which wastes half of what heads in the rows would.  Weights go in as two halves (value and rounding rest), so that what is
// added up has 16 bits of each weight.  In fp16 both halves end at 2^-24: its reference stands below the maximum, so that weights reach 2^15, and those
// under 2^-9 go in by themselves, multiplied by 2^24.  fp32: fused multiply-adds, a lane per key for scores, a lane per four columns for values.
#include "paged.cuh"
#include "warp_mma.cuh"

namespace sk {
namespace {

constexpr float PT_LOG2E = 1.4426950408889634f;
constexpr int PT_KEYS = 16;                                    // keys of a warp's tile
// A running maximum is only raised for a score this far (in powers of two) above it: weights then reach 2^8, which neither a half nor
// the sums mind, and the six exchanges and the rescaling that a rise takes are left out of nearly every tile.
constexpr float PT_SLACK = 8.f;
// fp16: raised to PT16_BELOW under the maximum, for a score PT16_SLACK above that.  Weights then reach 2^15 of a largest half of 65504, and only those
// 20 powers of two under a maximum are small.  64 sequences of 1 to 8003 with mass, as called, 59.4 us, 58.0 with small weights lost; 4 x 131072 keys 348,
// of which all but one are small 373, and 397 where they take two turns (344, all lost)
constexpr float PT16_BELOW = 11.f, PT16_SLACK = 4.f, PT16_SMALL = 0x1p-9f, PT16_UP = 0x1p24f;

template <typename T, int DP_, int NT_> struct PtShape {
    static constexpr int DP = DP_, NT = NT_;                   // head size padded, groups of heads
    static constexpr bool F32 = sizeof(T) == 4;
    static constexpr int HG = (F32 ? 4 : 8) * NT;              // query heads of a block
    static constexpr int ROW = DP * (int)sizeof(T), HALF = PT_KEYS * ROW, TILE = 2 * HALF;
    static constexpr int WARPS = TILE <= 8192 ? 8 : 65536 / TILE, STAGES = !F32 && NT == 2 ? 2 : 3;
    static constexpr int CHUNK = WARPS * PT_KEYS, THREADS = WARPS * 32;
    static constexpr int OS = DP + 4;                          // row of the joined sums: columns of four query pairs in four bank groups
    static constexpr size_t SMEM = (size_t)WARPS * STAGES * TILE + (size_t)WARPS * HG * OS * 4 + (F32 ? (size_t)HG * DP * 4 + (size_t)WARPS * PT_KEYS * HG * 4 : 0);
    static constexpr int PER_SM = SMEM <= 113 * 1024 ? 2 : 1;
    static_assert(SMEM <= 226 * 1024, "shared memory of a block");
};

// What the second kernel has to know of a block's run: where it begins, how long it is, the chunks of every run; and the pair that begins
// in it and ends in a later run, `tail_last` (-1: none)
struct alignas(16) PtRun {
    int64_t per, first;                                        // chunks of a run, and before this one
    int b, g, grp, chunk, chunks, n, left, tail_last, tail_b, tail_g, tail_grp, tail_inside;
};

struct PtArgs {
    const void* q;
    void* out;
    PtRun* runs;
    float *parts, *stats, *scores;                             // partial results; final maximum and 1 / sum per head; scores for mass
    int64_t q_bs, q_hs, o_bs, o_hs;
    int H, extra, groups, rs;                                  // groups of HG heads per key/value head; scores of a key
    float scale;                                               // times log2(e)
};

// Sum over the block, `red` of one value per warp; every thread gets it
__device__ __forceinline__ int64_t pt_block_sum(int64_t v, int64_t* red) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v += red[w];
    __syncthreads();
    return v;
}

__device__ __forceinline__ uint32_t pt_turn(uint32_t x) {      // an 8 x 8 matrix of 16-bit elements, transposed
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
template <typename T> __device__ __forceinline__ uint32_t pt_pack(float x, float y);
template <> __device__ __forceinline__ uint32_t pt_pack<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pt_pack<__half>(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ float pt_low(uint32_t x);
template <> __device__ __forceinline__ float pt_low<__nv_bfloat16>(uint32_t x) { return __uint_as_float(x << 16); }
template <> __device__ __forceinline__ float pt_low<__half>(uint32_t x) { return __half2float(__ushort_as_half((unsigned short)x)); }
template <typename T> __device__ __forceinline__ float pt_high(uint32_t x);
template <> __device__ __forceinline__ float pt_high<__nv_bfloat16>(uint32_t x) { return __uint_as_float(x & 0xFFFF0000u); }
template <> __device__ __forceinline__ float pt_high<__half>(uint32_t x) { return __half2float(__ushort_as_half((unsigned short)(x >> 16))); }

// exp2(a - b) with exp2(-inf - -inf) = 0
__device__ __forceinline__ float pt_factor(float a, float b) { return exp2_fast(a - (b == -INFINITY ? 0.f : b)); }
__device__ __forceinline__ float pt_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// 64-bit division is some hundred instructions in a row, and chunks are rarely that many
__device__ __forceinline__ int64_t pt_div(int64_t a, int64_t b) { return (uint64_t)(a | b) >> 32 == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b; }

// A place in the row of chunks: chunk `chunk` of `chunks` of group grp of key/value head g of sequence b, which has n keys.  Behind the
// chunks of every group stand PT_PAD empty ones: what it costs a block to finish it and begin the next.
constexpr int PT_PAD = 1;
struct PtPlace {
    int b, g, grp, chunk, chunks, n;
};
// to the next chunk, with what is left of the run; past the end of the run nothing is read
template <int CHUNK> __device__ __forceinline__ void pt_step(const sk_paged_cache& c, const PtArgs& a, PtPlace& p, int& left) {
    --left;
    if (++p.chunk < p.chunks) return;
    left -= PT_PAD;
    p.chunk = 0;
    if (left <= 0 || ++p.grp < a.groups) return;
    p.grp = 0;
    if (++p.g < c.G) return;
    p.g = 0;
    do {
        p.n = ++p.b < c.B ? paged_length(c, p.b, a.extra) : 1;
    } while (p.n == 0);
    p.chunks = (p.n + CHUNK - 1) / CHUNK;
}

template <typename S, typename T>
__global__ void __launch_bounds__(S::THREADS, S::PER_SM)
paged_attn_kernel(const __grid_constant__ sk_paged_cache c, const __grid_constant__ PtArgs a) {
    pdl_begin();
    constexpr int DP = S::DP, HG = S::HG, WARPS = S::WARPS, STAGES = S::STAGES, CHUNK = S::CHUNK, VE = 16 / (int)sizeof(T), OS = S::OS;
    constexpr int PIECES = S::ROW / 16;                        // 16-byte pieces of a row
    extern __shared__ __align__(1024) char pt_smem[];
    __shared__ int64_t red[WARPS];
    __shared__ float ms[WARPS][HG], ls[WARPS][HG];
    __shared__ PtPlace start_s;
    char* tiles = pt_smem + (threadIdx.x >> 5) * STAGES * S::TILE;                                  // [stage][keys | values][16][ROW]
    float* os = reinterpret_cast<float*>(pt_smem + WARPS * STAGES * S::TILE);                       // [WARPS][HG][OS]
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, shift = 31 - __clz(c.page);
    const int units = c.G * a.groups, rep = a.H / c.G;
    auto slots_of = [](int n) { return n == 0 ? 0 : (n + CHUNK - 1) / CHUNK + PT_PAD; };

    // ---- this block's run of chunks
    int64_t total, before = 0;
    PtPlace cur;
    const bool few = c.B <= 32;                                // a lane per sequence, every warp by itself
    int n_lane = 0;
    if (few) {
        bool over = false;
        n_lane = lane < c.B ? paged_length(c, lane, a.extra, &over) : 0;
        if (over && blockIdx.x == 0 && warp == 0 && c.status != nullptr) atomicOr(c.status, SK_DEV_POS_OUT_OF_RANGE);
        before = slots_of(n_lane);                             // up to this lane's sequence, with it
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(FULL, before, o);
            if (lane >= o) before += x;
        }
        total = __shfl_sync(FULL, before, 31) * units;
    } else {
        total = 0;
        for (int b = t; b < c.B; b += S::THREADS) {
            bool over;
            total += slots_of(paged_length(c, b, a.extra, &over));
            if (over && blockIdx.x == 0 && c.status != nullptr) atomicOr(c.status, SK_DEV_POS_OUT_OF_RANGE);
        }
        total = pt_block_sum(total, red) * units;
    }
    for (int b = blockIdx.x; b < c.B; b += gridDim.x)          // no key, no run: zeros
        if (paged_length(c, b, a.extra) == 0)
            for (int i = t; i < a.H * c.D; i += S::THREADS) ((T*)a.out)[b * a.o_bs + i / c.D * a.o_hs + i % c.D] = from_f32<T>(0.f);
    const int64_t per = pt_div(total + gridDim.x - 1, gridDim.x), first = per * blockIdx.x;
    int left = (int)max(min(per, total - first), (int64_t)0);
    PtRun* run = a.runs == nullptr ? nullptr : a.runs + blockIdx.x;
    if (run != nullptr && t == 0) {
        run->left = 0;
        run->tail_last = -1;
    }
    if (left == 0) return;
    auto place = [&](int b, int n, int64_t lo) {               // of chunk `first` in sequence b, whose chunks begin at lo
        const int m = slots_of(n), unit = (int)pt_div(first - lo, m);
        return PtPlace{b, unit / a.groups, unit % a.groups, (int)(first - lo - (int64_t)unit * m), m - PT_PAD, n};
    };
    if (few) {
        const int b = __ffs(__ballot_sync(FULL, before * units > first)) - 1, n = __shfl_sync(FULL, n_lane, b);
        cur = place(b, n, (__shfl_sync(FULL, before, b) - slots_of(n)) * units);
    } else {
        for (int b0 = 0; b0 < c.B; b0 += S::THREADS) {         // the sequence that holds chunk `first`
            const int b = b0 + t, n = b < c.B ? paged_length(c, b, a.extra) : 0, m = slots_of(n);
            int64_t sum = m;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t x = __shfl_up_sync(FULL, sum, o);
                if (lane >= o) sum += x;
            }
            if (lane == 31) red[warp] = sum;
            __syncthreads();
            int64_t all = 0;
            for (int w = 0; w < WARPS; ++w) {
                if (w < warp) sum += red[w];
                all += red[w];
            }
            const int64_t lo = (before + sum - m) * units, hi = (before + sum) * units;
            if (lo <= first && first < hi) start_s = place(b, n, lo);
            before += all;
            __syncthreads();
            if (before * units > first) break;
        }
        cur = start_s;
    }
    int64_t flat = first;                                      // chunk in the row of all chunks
    if (cur.chunk >= cur.chunks) {                             // the run begins behind a pair
        const int skip = cur.chunks + PT_PAD - cur.chunk;
        cur.chunk = cur.chunks - 1;
        left += 1 + PT_PAD - skip;
        flat += skip;
        pt_step<CHUNK>(c, a, cur, left);
        if (left <= 0) return;
    }
    PtPlace ld = cur;
    if (run != nullptr && t == 0) *run = PtRun{per, flat, cur.b, cur.g, cur.grp, cur.chunk, cur.chunks, cur.n, left, -1, 0, 0, 0, 0};

    // ---- copies: this warp's tile of the chunk at `ld`, one commit group each; `live` has a bit per stage that holds keys
    constexpr int COPIES = PT_KEYS * PIECES / 32;              // of keys, and of values, per lane
    const int k_row = (int)c.k_rs * (int)sizeof(T), v_row = (int)c.v_rs * (int)sizeof(T);          // bytes; checked to fit
    const char *k_head = (const char*)c.k + ld.g * c.k_hs * (int)sizeof(T), *v_head = (const char*)c.v + ld.g * c.v_hs * (int)sizeof(T);
    const uint32_t ld_to = lane / PIECES * S::ROW + ((lane % PIECES ^ (lane / PIECES & 7)) << 4);
    int ld_left = left, ld_stage = 0, ld_page = 0;
    uint32_t live = 0;
    auto ask_page = [&]() {
        const int j = ld.chunk * CHUNK + warp * PT_KEYS;
        if (ld_left > 0 && j < ld.n) ld_page = __ldcg(c.table + ld.b * c.table_ld + (j >> shift));
    };
    auto issue = [&]() {
        live &= ~(1u << ld_stage);
        if (ld_left > 0) {
            const int j = ld.chunk * CHUNK + warp * PT_KEYS, rows = ld.n - j;
            if (rows > 0) {
                if (paged_page_ok(c, ld_page)) {
                    const char* k = k_head + ld_page * (c.k_ps * (int)sizeof(T)) + (int64_t)(j & (c.page - 1)) * k_row;
                    const char* v = v_head + ld_page * (c.v_ps * (int)sizeof(T)) + (int64_t)(j & (c.page - 1)) * v_row;
                    const uint32_t dst = saddr(tiles + ld_stage * S::TILE);
                    if (rows >= PT_KEYS && c.D == DP) {
                        const char* kl = k + (int64_t)(lane / PIECES) * k_row + lane % PIECES * 16;
                        const char* vl = v + (int64_t)(lane / PIECES) * v_row + lane % PIECES * 16;
#pragma unroll
                        for (int i = 0; i < COPIES; ++i) {
                            const int r = i * 32 / PIECES;     // of lane 0; lanes add at most bits that r has clear
                            const uint32_t at = (dst + ld_to) ^ ((r & 7) << 4);
                            cp16(at + r * S::ROW + i * 32 % PIECES * 16, kl + (int64_t)r * k_row + i * 32 % PIECES * 16, true);
                            cp16(at + r * S::ROW + i * 32 % PIECES * 16 + S::HALF, vl + (int64_t)r * v_row + i * 32 % PIECES * 16, true);
                        }
                    } else {
#pragma unroll 2
                        for (int i = 0; i < COPIES; ++i) {
                            const int x = i * 32 + lane, r = x / PIECES, p = x % PIECES;
                            const bool in = r < rows && p * VE < c.D;      // others are zeros
                            const uint32_t at = dst + r * S::ROW + ((p ^ (r & 7)) << 4);
                            cp16(at, in ? k + (int64_t)r * k_row + p * 16 : k, in);
                            cp16(at + S::HALF, in ? v + (int64_t)r * v_row + p * 16 : v, in);
                        }
                    }
                    live |= 1u << ld_stage;
                } else if (lane == 0 && c.status != nullptr) {
                    atomicOr(c.status, SK_DEV_INDEX_OUT_OF_RANGE);
                }
            }
            const int g = ld.g;
            pt_step<CHUNK>(c, a, ld, ld_left);
            if (ld.g != g) {
                k_head = (const char*)c.k + ld.g * c.k_hs * (int)sizeof(T);
                v_head = (const char*)c.v + ld.g * c.v_hs * (int)sizeof(T);
            }
            ask_page();
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ld_stage = ld_stage + 1 == STAGES ? 0 : ld_stage + 1;
    };
    ask_page();
    for (int s = 0; s < STAGES - 1; ++s) issue();

    // ---- queries of a pair, running maxima and sums
    constexpr int KK = DP / 16, NT = S::NT;
    constexpr bool NARROW = std::is_same_v<T, __half>;         // a type whose smallest weights need care
    constexpr int CPL = S::F32 ? (DP / 4 + 31) / 32 : 1;       // fp32: 16-byte pieces of a value row per lane
    uint32_t qf[S::F32 ? 1 : NT][S::F32 ? 1 : KK][2];
    float acc[S::F32 ? HG : KK][S::F32 ? CPL : NT][4];         // 16 bit: rows of value columns x heads; fp32: heads x columns
    constexpr int MC = S::F32 ? HG : 2 * NT;                   // heads whose maximum a lane keeps
    float m[MC], l[MC];
    float* qs = os + WARPS * HG * OS;                          // fp32: [HG][DP] queries, [WARPS][16][HG] weights
    float* ps = qs + HG * DP + warp * PT_KEYS * HG;
    auto queries = [&](const PtPlace& p) {
        const int h0 = p.g * rep + p.grp * HG, heads = min(HG, (p.g + 1) * rep - h0);
        const T* q = (const T*)a.q + p.b * a.q_bs + h0 * a.q_hs;
        if constexpr (S::F32) {
            for (int i = t; i < HG * DP; i += S::THREADS) qs[i] = i / DP < heads && i % DP < c.D ? q[i / DP * a.q_hs + i % DP] : 0.f;
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int h = nt * 8 + (lane >> 2), d = kk * 16 + i * 8 + (lane & 3) * 2;
                        qf[nt][kk][i] = h < heads && d < c.D ? *reinterpret_cast<const uint32_t*>(q + h * a.q_hs + d) : 0u;
                    }
        }
    };
    auto begin = [&]() {
#pragma unroll
        for (int i = 0; i < MC; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < (int)(sizeof(acc) / 4); ++i) (&acc[0][0][0])[i] = 0.f;
    };
    queries(cur);
    if (S::F32) __syncthreads();
    begin();
    int stage = 0, seg_chunk = cur.chunk;
    bool seg_first = flat == first;                            // what the run begins with, inside a pair or with it

    while (true) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();                                          // the tile is there, and the stage before is read
        issue();
        const int j = cur.chunk * CHUNK + warp * PT_KEYS, rows = cur.n - j;
        float* sc_out = a.scores == nullptr ? nullptr : a.scores + (flat * CHUNK + warp * PT_KEYS) * a.rs;
        if (rows > 0 && (live >> stage & 1)) {
            const char* kt = tiles + stage * S::TILE;
            const char* vt = kt + S::HALF;
            if constexpr (!S::F32) {
                // 16-byte piece p of row r lies at piece p ^ (r & 7): of two pieces a step, the step's bits are flipped in the address
                const uint32_t row = saddr(kt) + (lane & 15) * S::ROW + (((lane >> 4) ^ (lane & 7)) << 4);
                float sc[2][NT][4];
#pragma unroll
                for (int i = 0; i < 8 * NT; ++i) (&sc[0][0][0])[i] = 0.f;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    uint32_t k4[4];
                    ldsm4(row ^ (kk << 5), k4);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(sc[kk & 1][nt], k4[0], k4[1], k4[2], k4[3], qf[nt][kk][0], qf[nt][kk][1], (const T*)nullptr);
                }
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nt][e] = (sc[0][nt][e] + sc[1][nt][e]) * a.scale;
                if (rows < PT_KEYS) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if ((lane >> 2) + (e >> 1) * 8 >= rows) s[nt][e] = -INFINITY;
                }
                bool above = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (sc_out != nullptr && nt * 8 + (lane & 3) * 2 < a.rs) {
                        float* o = sc_out + (lane >> 2) * a.rs + nt * 8 + (lane & 3) * 2;
                        if ((lane >> 2) < rows) __stcg(reinterpret_cast<float2*>(o), make_float2(s[nt][0], s[nt][1]));
                        if ((lane >> 2) + 8 < rows) __stcg(reinterpret_cast<float2*>(o + 8 * a.rs), make_float2(s[nt][2], s[nt][3]));
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) above |= fmaxf(s[nt][i], s[nt][i + 2]) - m[nt * 2 + i] > (NARROW ? PT16_BELOW + PT16_SLACK : PT_SLACK);
                }
                if (__any_sync(FULL, above)) {                 // maxima follow, and what was summed up with them
#pragma unroll
                    for (int x = 0; x < MC; ++x) {
                        float mx = fmaxf(s[x / 2][x & 1], s[x / 2][(x & 1) + 2]);
                        mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 16));
                        if (NARROW) mx = __fsub_ru(mx, PT16_BELOW);            // of huge scores too no more than this below
                        const float mn = fmaxf(m[x], mx), f = pt_factor(m[x], mn);
                        m[x] = mn;
                        l[x] *= f;
#pragma unroll
                        for (int mt = 0; mt < KK; ++mt) {
                            acc[mt][x / 2][x & 1] *= f;
                            acc[mt][x / 2][(x & 1) + 2] *= f;
                        }
                    }
                }
                uint32_t ph[NT][2], pl[NT][2];
                auto halves = [&](const float (&w)[NT][4]) {   // keys x heads of a lane's row to those of its column
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t h = pt_pack<T>(w[nt][2 * i], w[nt][2 * i + 1]);
                            ph[nt][i] = pt_turn(h);
                            pl[nt][i] = pt_turn(pt_pack<T>(w[nt][2 * i] - pt_low<T>(h), w[nt][2 * i + 1] - pt_high<T>(h)));
                        }
                };
                float least = PT16_SMALL;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float mc = m[nt * 2 + i] == -INFINITY ? 0.f : m[nt * 2 + i];
                        s[nt][i] = exp2_fast(s[nt][i] - mc);
                        s[nt][i + 2] = exp2_fast(s[nt][i + 2] - mc);
                        l[nt * 2 + i] += s[nt][i] + s[nt][i + 2];
                        if (NARROW) least = fminf(least, fminf(s[nt][i], s[nt][i + 2]));
                    }
                }
                const uint32_t vrow = saddr(vt) + ((lane & 7) + (lane >> 4) * 8) * S::ROW + (((lane >> 3 & 1) ^ (lane & 7)) << 4);
                if constexpr (NARROW) {
                    if (__any_sync(FULL, least < PT16_SMALL)) {                // 24 powers of two at a time
                        float rest[NT][4];
#pragma unroll
                        for (int i = 0; i < 4 * NT; ++i) {
                            float& w = (&s[0][0])[i];
                            (&rest[0][0])[i] = w < PT16_SMALL ? w : 0.f;
                            w = w < PT16_SMALL ? 0.f : w;
                        }
                        float down = 1.f;
                        bool small;
                        do {
                            float w[NT][4];
                            down /= PT16_UP;
                            small = false;
#pragma unroll
                            for (int i = 0; i < 4 * NT; ++i) {
                                float& r = (&rest[0][0])[i];
                                r *= PT16_UP;
                                (&w[0][0])[i] = r < PT16_SMALL ? 0.f : r;
                                r = r < PT16_SMALL ? r : 0.f;
                                small |= r > 0.f;
                            }
                            halves(w);
#pragma unroll
                            for (int mt = 0; mt < KK; ++mt) {
                                uint32_t v4[4];
                                ldsm4t(vrow ^ (mt << 5), v4);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma16816(sum, v4[0], v4[1], v4[2], v4[3], ph[nt][0], ph[nt][1], (const T*)nullptr);
                                    mma16816(sum, v4[0], v4[1], v4[2], v4[3], pl[nt][0], pl[nt][1], (const T*)nullptr);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) acc[mt][nt][e] = fmaf(sum[e], down, acc[mt][nt][e]);
                                }
                            }
                        } while (__any_sync(FULL, small));
                    }
                }
                halves(s);
#pragma unroll
                for (int mt = 0; mt < KK; ++mt) {
                    uint32_t v4[4];
                    ldsm4t(vrow ^ (mt << 5), v4);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16816(acc[mt][nt], v4[0], v4[1], v4[2], v4[3], ph[nt][0], ph[nt][1], (const T*)nullptr);
                        mma16816(acc[mt][nt], v4[0], v4[1], v4[2], v4[3], pl[nt][0], pl[nt][1], (const T*)nullptr);
                    }
                }
            } else {
                // scores: lane = key, each half of the warp one half of the head
                const int key = lane & 15, half = lane >> 4;
                float s[HG];
#pragma unroll
                for (int h = 0; h < HG; ++h) s[h] = 0.f;
                const float4* kr = reinterpret_cast<const float4*>(kt + key * S::ROW);
#pragma unroll 4
                for (int i = 0; i < PIECES / 2; ++i) {
                    const int p = half * (PIECES / 2) + i;
                    const float4 k4 = kr[p ^ (key & 7)];
#pragma unroll
                    for (int h = 0; h < HG; ++h) {
                        const float4 q4 = *reinterpret_cast<const float4*>(qs + h * DP + p * 4);
                        s[h] = fmaf(k4.w, q4.w, fmaf(k4.z, q4.z, fmaf(k4.y, q4.y, fmaf(k4.x, q4.x, s[h]))));
                    }
                }
                bool above = false;
#pragma unroll
                for (int h = 0; h < HG; ++h) {
                    s[h] = (s[h] + __shfl_xor_sync(FULL, s[h], 16)) * a.scale;
                    if (key >= rows) s[h] = -INFINITY;
                    if (sc_out != nullptr && h < a.rs && key < rows && half == 0) __stcg(sc_out + key * a.rs + h, s[h]);
                    above |= s[h] > m[h] + PT_SLACK;
                }
                if (__any_sync(FULL, above)) {
#pragma unroll
                    for (int h = 0; h < HG; ++h) {
                        float mx = s[h];
#pragma unroll
                        for (int o = 8; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, o));
                        const float mn = fmaxf(m[h], mx), f = pt_factor(m[h], mn);
                        m[h] = mn;
                        l[h] *= f;
#pragma unroll
                        for (int i = 0; i < CPL; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[h][i][e] *= f;
                    }
                }
#pragma unroll
                for (int h = 0; h < HG; ++h) {
                    const float w = pt_factor(s[h], m[h]);
                    l[h] += w;                                 // both halves of the warp keep the same sums
                    if (half == 0) ps[key * HG + h] = w;
                }
                __syncwarp();
                constexpr int SPLIT = PIECES < 32 ? 32 / PIECES : 1;         // heads of 64: half a warp takes every second key
#pragma unroll 4
                for (int x = lane / (32 / SPLIT); x < PT_KEYS; x += SPLIT) {
                    float w[HG];
#pragma unroll
                    for (int h = 0; h < HG; h += 4) load_vec<float, 4>(ps + x * HG + h, reinterpret_cast<float(&)[4]>(w[h]));
#pragma unroll
                    for (int i = 0; i < CPL; ++i) {
                        const float4 v4 = reinterpret_cast<const float4*>(vt + x * S::ROW)[(lane % PIECES + i * 32) ^ (x & 7)];
#pragma unroll
                        for (int h = 0; h < HG; ++h) {
                            acc[h][i][0] = fmaf(w[h], v4.x, acc[h][i][0]);
                            acc[h][i][1] = fmaf(w[h], v4.y, acc[h][i][1]);
                            acc[h][i][2] = fmaf(w[h], v4.z, acc[h][i][2]);
                            acc[h][i][3] = fmaf(w[h], v4.w, acc[h][i][3]);
                        }
                    }
                }
                __syncwarp();                                  // the weights are read
            }
        } else if (sc_out != nullptr && rows > 0) {            // a page outside the pool: no weight
            for (int i = lane; i < min(rows, PT_KEYS) * a.rs; i += 32) __stcg(sc_out + i, -INFINITY);
        }
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        if (cur.chunk + 1 < cur.chunks && left > 1) {
            --left;
            ++flat;
            ++cur.chunk;
            continue;
        }
        // ---- the block's warps join what they have of this pair; the next one's queries are on their way meanwhile
        PtPlace next = cur;
        pt_step<CHUNK>(c, a, next, left);
        if (!S::F32 && left > 0) queries(next);
        const int tiles_here = (min(cur.n, (cur.chunk + 1) * CHUNK) - seg_chunk * CHUNK + PT_KEYS - 1) / PT_KEYS, busy = min(tiles_here, WARPS);
#pragma unroll
        for (int i = 0; i < MC; ++i) {
            if constexpr (S::F32) {
#pragma unroll
                for (int o = 8; o >= 1; o >>= 1) l[i] += __shfl_xor_sync(FULL, l[i], o);
                if (lane == 0) {
                    ms[warp][i] = m[i];
                    ls[warp][i] = l[i];
                }
            } else {
                l[i] += __shfl_xor_sync(FULL, l[i], 4);
                l[i] += __shfl_xor_sync(FULL, l[i], 8);
                l[i] += __shfl_xor_sync(FULL, l[i], 16);
                if (lane < 4) {
                    ms[warp][i / 2 * 8 + lane * 2 + (i & 1)] = m[i];
                    ls[warp][i / 2 * 8 + lane * 2 + (i & 1)] = l[i];
                }
            }
        }
        float* mine = os + warp * HG * OS;
        if constexpr (S::F32) {
#pragma unroll
            for (int h = 0; h < HG; ++h)
#pragma unroll
                for (int i = 0; i < CPL; ++i) {
                    float4 v = make_float4(acc[h][i][0], acc[h][i][1], acc[h][i][2], acc[h][i][3]);
                    if constexpr (PIECES < 32) {
                        v.x += __shfl_xor_sync(FULL, v.x, 16);
                        v.y += __shfl_xor_sync(FULL, v.y, 16);
                        v.z += __shfl_xor_sync(FULL, v.z, 16);
                        v.w += __shfl_xor_sync(FULL, v.w, 16);
                    }
                    if (PIECES >= 32 || lane < PIECES) *reinterpret_cast<float4*>(mine + h * OS + (lane % PIECES + i * 32) * 4) = v;
                }
        } else {
#pragma unroll
            for (int mt = 0; mt < KK; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (warp < busy && nt * 8 + (lane & 3) * 2 < rep) mine[(nt * 8 + (lane & 3) * 2 + (e & 1)) * OS + mt * 16 + (lane >> 2) + (e >> 1) * 8] = acc[mt][nt][e];
        }
        __syncthreads();
        const int h0 = cur.g * rep + cur.grp * HG, heads = min(HG, (cur.g + 1) * rep - h0);
        const bool whole = seg_chunk == 0 && cur.chunk + 1 == cur.chunks;
        float* part = whole ? nullptr : a.parts + ((int64_t)blockIdx.x * 2 + (seg_first ? 0 : 1)) * HG * (DP + 2);
        for (int i = t; i < heads * (DP / 4); i += S::THREADS) {
            const int h = i / (DP / 4), d = i % (DP / 4) * 4;
            float mm = -INFINITY, ll = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, ms[w][h]);
            float o[4] = {0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < busy; ++w) {                   // the others had no key of it
                const float f = pt_factor(ms[w][h], mm);
                const float4 x = *reinterpret_cast<const float4*>(os + (w * HG + h) * OS + d);
                ll = fmaf(ls[w][h], f, ll);
                o[0] = fmaf(x.x, f, o[0]);
                o[1] = fmaf(x.y, f, o[1]);
                o[2] = fmaf(x.z, f, o[2]);
                o[3] = fmaf(x.w, f, o[3]);
            }
            if (whole) {
                const float inv = pt_inverse(ll);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] *= inv;
                if (d < c.D) store_vec<T, 4>((T*)a.out + cur.b * a.o_bs + (h0 + h) * a.o_hs + d, o);
                if (d == 0 && a.stats != nullptr) *reinterpret_cast<float2*>(a.stats + ((int64_t)cur.b * a.H + h0 + h) * 2) = make_float2(mm, inv);
            } else {
                *reinterpret_cast<float4*>(part + h * DP + d) = make_float4(o[0], o[1], o[2], o[3]);
                if (d == 0) *reinterpret_cast<float2*>(part + HG * DP + h * 2) = make_float2(mm, ll);
            }
        }
        if (left <= 0) break;
        __syncthreads();                                       // sums are read
        flat += 1 + PT_PAD;
        cur = next;
        if (S::F32) {
            queries(cur);
            __syncthreads();
        }
        begin();
        seg_chunk = 0;
        seg_first = false;
    }
    if (run != nullptr && t == 0 && seg_chunk == 0 && cur.chunk + 1 < cur.chunks) {
        run->tail_b = cur.b;
        run->tail_g = cur.g;
        run->tail_grp = cur.grp;
        run->tail_inside = !seg_first;
        run->tail_last = (int)pt_div(flat - cur.chunk + cur.chunks - 1, per);
    }
}

// The partial result that block x left of a pair: its run's first one, or, of a pair that begins inside the run, its last one
template <typename S> __device__ __forceinline__ const float* pt_part(const PtArgs& a, int x, bool begins_inside) {
    return a.parts + ((int64_t)x * 2 + (begins_inside ? 1 : 0)) * S::HG * (S::DP + 2);
}

// A pair that ends in another run than it begins in belongs to the run it begins in; a run has one such pair at most.  With mass, the
// warps of the first `shares` blocks of a run (blockIdx.x) add the weights of a share of the run's keys each; the other blocks join the
// pair's partial results, one head each, a warp every eighth of them.
constexpr int PJ_WARPS = 8, PJ_SHARES = 4;
template <typename S, typename T>
__global__ void __launch_bounds__(PJ_WARPS * 32)
paged_join_kernel(const __grid_constant__ sk_paged_cache c, const __grid_constant__ PtArgs a, int shares) {
    pdl_begin();
    constexpr int DP = S::DP, HG = S::HG, E = DP / 32, CHUNK = S::CHUNK;
    __shared__ float ms[PJ_WARPS], ls[PJ_WARPS], os[PJ_WARPS][DP], stats[PJ_WARPS][2][HG];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31, rep = a.H / c.G, x0 = blockIdx.x;
    PtRun run;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(PtRun) / 16); ++i) reinterpret_cast<int4*>(&run)[i] = __ldcg(reinterpret_cast<const int4*>(a.runs + x0) + i);
    if ((int)blockIdx.y >= shares) {
        const int last = run.tail_last, h = blockIdx.y - shares, b = run.tail_b, g = run.tail_g, hh = run.tail_grp * HG + h;
        if (last < 0 || hh >= rep) return;
        float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = 0.f;
        constexpr int AHEAD = 3;                               // partial results asked for at a time: up to 24 of a pair in one trip
        for (int x = x0 + warp; x <= last; x += AHEAD * PJ_WARPS) {
            float2 ml[AHEAD];
            float v[AHEAD][E];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                ml[i] = make_float2(-INFINITY, 0.f);
                if (x + i * PJ_WARPS > last) continue;
                const float* part = pt_part<S>(a, x + i * PJ_WARPS, i == 0 && x == x0 && run.tail_inside);
                ml[i] = __ldcg(reinterpret_cast<const float2*>(part + HG * DP + h * 2));
#pragma unroll
                for (int e = 0; e < E; ++e) v[i][e] = __ldcg(part + h * DP + e * 32 + lane);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (x + i * PJ_WARPS > last) continue;
                const float mn = fmaxf(m, ml[i].x), f = pt_factor(m, mn), fx = pt_factor(ml[i].x, mn);
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = fmaf(v[i][e], fx, o[e] * f);
                l = fmaf(ml[i].y, fx, l * f);
                m = mn;
            }
        }
        if (lane == 0) {
            ms[warp] = m;
            ls[warp] = l;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) os[warp][e * 32 + lane] = o[e];
        __syncthreads();
        if (t < c.D) {
            m = -INFINITY;
            l = 0.f;
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < PJ_WARPS; ++w) m = fmaxf(m, ms[w]);
#pragma unroll
            for (int w = 0; w < PJ_WARPS; ++w) {
                const float f = pt_factor(ms[w], m);
                l = fmaf(ls[w], f, l);
                sum = fmaf(os[w][t], f, sum);
            }
            ((T*)a.out)[b * a.o_bs + (g * rep + hh) * a.o_hs + t] = from_f32<T>(sum * pt_inverse(l));
        }
        return;
    }
    // ---- mass: all groups of a key/value head add to the same keys.  Their chunks stand one behind the other, and who walks the first
    // group's adds for all of them
    const int share = blockIdx.y * PJ_WARPS + warp, of = PJ_SHARES * PJ_WARPS;
    const int from = (int)((int64_t)run.left * share / of), to = (int)((int64_t)run.left * (share + 1) / of);
    float (*stat)[HG] = stats[warp];
    const int64_t per = run.per;
    PtPlace p = {run.b, run.g, run.grp, run.chunk, run.chunks, run.n};
    int64_t flat = run.first;
    for (int done = 0; done < to;) {
        const int some = min(p.chunks - p.chunk, to - done);   // of this pair
        const int lo = max(from - done, 0);
        if (lo < some && p.grp == 0) {
            const int g = p.g, j0 = (p.chunk + lo) * CHUNK, j1 = min((p.chunk + some) * CHUNK, p.n);
            float* mass = c.mass + p.b * c.mass_bs + g * c.mass_hs;
            for (int grp = 0; grp < a.groups; ++grp) {
                const int heads = min(HG, rep - grp * HG);
                const int64_t begin = flat - p.chunk + (int64_t)grp * (p.chunks + PT_PAD);
                const int y0 = (int)pt_div(begin, per), y1 = (int)pt_div(begin + p.chunks - 1, per);
                const float* sc = a.scores + begin * CHUNK * a.rs;
                // four heads a key: the first keys' scores and masses are asked for before the heads' maxima are, of four keys at a time (64 ragged
                // sequences 59.0 us, key by key as with other numbers of heads 63.7; 4 x 131072 keys 375 and 407)
                float4 x[4];
                float w[4];
                auto ask = [&](int j) {
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (j + u * 32 < j1) {
                            x[u] = __ldcs(reinterpret_cast<const float4*>(sc) + j + u * 32);
                            w[u] = mass[j + u * 32];
                        }
                };
                if (a.rs == 4) ask(j0 + lane);
                __syncwarp();
                if (y0 == y1) {                                // final maximum and 1 / sum: there already
                    if (lane < heads) {
                        const float2 st = __ldcg(reinterpret_cast<const float2*>(a.stats + ((int64_t)p.b * a.H + g * rep + grp * HG + lane) * 2));
                        stat[0][lane] = st.x == -INFINITY ? 0.f : st.x;
                        stat[1][lane] = st.y;
                    }
                } else {                                       // as many lanes for every head
                    const int of_head = heads <= 4 ? 8 : heads <= 8 ? 4 : 2, h = lane / of_head;
                    float m = -INFINITY, l = 0.f;
                    if (h < heads)
                        for (int y = y0 + lane % of_head; y <= y1; y += of_head) {
                            const float2 ml = __ldcg(reinterpret_cast<const float2*>(pt_part<S>(a, y, begin > y * per) + HG * DP + h * 2));
                            const float mn = fmaxf(m, ml.x);
                            l = l * pt_factor(m, mn) + ml.y * pt_factor(ml.x, mn);
                            m = mn;
                        }
                    for (int o = of_head / 2; o >= 1; o >>= 1) {
                        const float m2 = __shfl_xor_sync(FULL, m, o), l2 = __shfl_xor_sync(FULL, l, o), mn = fmaxf(m, m2);
                        l = l * pt_factor(m, mn) + l2 * pt_factor(m2, mn);
                        m = mn;
                    }
                    if (h < heads && lane % of_head == 0) {
                        stat[0][h] = m == -INFINITY ? 0.f : m;
                        stat[1][h] = pt_inverse(l);
                    }
                }
                __syncwarp();
                if (a.rs == 4) {
                    const float4 m4 = make_float4(stat[0][0], stat[0][1], stat[0][2], stat[0][3]);
                    const float4 l4 = make_float4(stat[1][0], stat[1][1], stat[1][2], stat[1][3]);
                    for (int j = j0 + lane; j < j1; j += 128) {
                        if (j >= j0 + 128) ask(j);
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            if (j + u * 32 < j1) {
                                float s = exp2_fast(x[u].x - m4.x) * l4.x;
                                s = fmaf(exp2_fast(x[u].y - m4.y), l4.y, s);
                                s = fmaf(exp2_fast(x[u].z - m4.z), l4.z, s);
                                if (heads > 3) s = fmaf(exp2_fast(x[u].w - m4.w), l4.w, s);
                                mass[j + u * 32] = w[u] + s;
                            }
                    }
                } else {
                    const int vec = a.rs % 4 == 0 ? 4 : 2;
#pragma unroll 2
                    for (int j = j0 + lane; j < j1; j += 32) {
                        const float* row = sc + (int64_t)j * a.rs;
                        const float old = mass[j];
                        float s = 0.f;
                        for (int h = 0; h < heads; h += vec) {
                            float4 v;
                            if (vec == 4) {
                                v = __ldcs(reinterpret_cast<const float4*>(row + h));
                            } else {
                                const float2 two = __ldcs(reinterpret_cast<const float2*>(row + h));
                                v = make_float4(two.x, two.y, 0.f, 0.f);
                            }
                            s = fmaf(exp2_fast(v.x - stat[0][h]), stat[1][h], s);
                            if (h + 1 < heads) s = fmaf(exp2_fast(v.y - stat[0][h + 1]), stat[1][h + 1], s);
                            if (vec == 4 && h + 2 < heads) s = fmaf(exp2_fast(v.z - stat[0][h + 2]), stat[1][h + 2], s);
                            if (vec == 4 && h + 3 < heads) s = fmaf(exp2_fast(v.w - stat[0][h + 3]), stat[1][h + 3], s);
                        }
                        mass[j] = old + s;
                    }
                }
            }
        }
        int skip = to - done - some + 1;                       // what is left from the pair's last chunk on
        const int before = skip;
        p.chunk += some - 1;
        pt_step<CHUNK>(c, a, p, skip);
        done += some - 1 + before - skip;
        flat += some - 1 + before - skip;
    }
}

struct PtPlan {
    int groups, rs, chunk, blocks;
    bool join;
    size_t parts, stats, scores, total;                        // bytes in front of them, and of all
};
template <typename S> PtPlan pt_plan(const sk_paged_cache& c, int H) {
    PtPlan p;
    const int rep = H / c.G;
    p.groups = (rep + S::HG - 1) / S::HG;
    p.rs = rep < S::HG ? (rep + 1) / 2 * 2 : S::HG;
    const int64_t cap = (int64_t)c.width * c.page, chunks = ((cap + S::CHUNK - 1) / S::CHUNK + PT_PAD) * c.B * c.G * p.groups;
    const int64_t most = (int64_t)sm_count() * S::PER_SM;
    p.blocks = (int)(chunks < most ? (chunks < 1 ? 1 : chunks) : most);
    p.join = cap > S::CHUNK || c.mass != nullptr;
    p.parts = p.join ? up256((size_t)p.blocks * sizeof(PtRun)) : 0;
    p.stats = p.parts + (cap > S::CHUNK ? up256((size_t)p.blocks * 2 * S::HG * (S::DP + 2) * 4) : 0);
    p.scores = p.stats + (c.mass != nullptr ? up256((size_t)c.B * H * 8) : 0);
    p.total = p.scores + (c.mass != nullptr ? up256((size_t)chunks * S::CHUNK * p.rs * 4) : 0);
    return p;
}

// f(shape, element) of the kernel for this cache: heads padded to 64, 128 or 256; up to 8 (fp32: 4) query heads a block where a
// key/value head has no more, else up to 16 (8): a key is read once for all of them.
template <typename F> auto pt_with(const sk_paged_cache& c, int H, F&& f) {
    auto sized = [&](auto t, auto nt) {
        using T = decltype(t);
        constexpr int NT = decltype(nt)::value;
        if (c.D <= 64) return f(PtShape<T, 64, NT>{}, t);
        if (c.D <= 128) return f(PtShape<T, 128, NT>{}, t);
        return f(PtShape<T, 256, NT>{}, t);
    };
    auto typed = [&](auto t) {
        if (H / c.G <= (sizeof(t) == 4 ? 4 : 8)) return sized(t, std::integral_constant<int, 1>{});
        return sized(t, std::integral_constant<int, 2>{});
    };
    if (c.dtype == SK_F32) return typed(float{});
    if (c.dtype == SK_BF16) return typed(__nv_bfloat16{});
    return typed(__half{});
}

}  // namespace

size_t paged_attn_workspace(const sk_paged_cache& c, int H) {
    return pt_with(c, H, [&](auto s, auto) { return pt_plan<decltype(s)>(c, H).total; });
}

int launch_paged_attn(const sk_paged_cache& c, const void* q, int64_t q_bs, int64_t q_hs, void* out, int64_t o_bs, int64_t o_hs, int H,
                      int extra, float scale, void* workspace, cudaStream_t st) {
    return pt_with(c, H, [&](auto shape, auto t) -> int {
        using S = decltype(shape);
        using T = decltype(t);
        const PtPlan p = pt_plan<S>(c, H);
        PtArgs a;
        a.q = q;
        a.out = out;
        a.runs = p.join ? (PtRun*)workspace : nullptr;
        a.parts = (float*)((char*)workspace + p.parts);
        a.stats = c.mass != nullptr ? (float*)((char*)workspace + p.stats) : nullptr;
        a.scores = c.mass != nullptr ? (float*)((char*)workspace + p.scores) : nullptr;
        a.q_bs = q_bs;
        a.q_hs = q_hs;
        a.o_bs = o_bs;
        a.o_hs = o_hs;
        a.H = H;
        a.extra = extra;
        a.groups = p.groups;
        a.rs = p.rs;
        a.scale = scale * PT_LOG2E;
        static SmemLimit limit;
        cudaError_t e = limit.raise((const void*)paged_attn_kernel<S, T>, S::SMEM);
        if (e == cudaSuccess) e = launch_after(paged_attn_kernel<S, T>, dim3(p.blocks), dim3(S::THREADS), S::SMEM, st, c, a);
        if (int rc = check_chained(e, "paged_attn_kernel")) return rc;
        if (!p.join) return SK_OK;
        const int shares = c.mass != nullptr ? PJ_SHARES : 0, heads = H / c.G < S::HG ? H / c.G : S::HG;
        return check_chained(launch_after(paged_join_kernel<S, T>, dim3(p.blocks, shares + heads), dim3(PJ_WARPS * 32), 0, st, c, a, shares), "paged_join_kernel");
    });
}

}  // namespace sk
