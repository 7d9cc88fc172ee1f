// Entry points of the paged cache, and the append that fills its pages.
#include "paged.cuh"

#include <algorithm>

namespace sk {
namespace {

// A thread per 16-byte piece of four new rows (sequence, token, head) of its own: the pieces of both tensors are asked for before the
// table is, and written behind it.  Nothing but copies, bound by memory: a padded batch of 8 prompts of up to 4096 tokens, 176 MB, in 33 us (5.3 TB/s),
// a warp per row 84; one token of 64 sequences 2.2.
constexpr int PA_THREADS = 256, PA_ROWS = 4;
__global__ void __launch_bounds__(PA_THREADS)
paged_append_kernel(const __grid_constant__ sk_paged_cache c, const char* k_new, int64_t kn_bs, int64_t kn_ss, int64_t kn_hs, const char* v_new,
                    int64_t vn_bs, int64_t vn_ss, int64_t vn_hs, int S, const int32_t* counts, const int32_t* first, int es, int pieces) {
    pdl_begin();
    // pieces of a row, rounded up to a power of two: lanes of a row and rows of a block
    const int per = 1 << (32 - __clz(pieces - 1)), p = threadIdx.x & (per - 1), step = PA_THREADS / per, shift = 31 - __clz(c.page);
    const int b = blockIdx.y, r0 = blockIdx.x * PA_ROWS * step + threadIdx.x / per, n = counts != nullptr ? min(counts[b], S) : S;
    const int64_t length = max(c.lengths[b], 0);
    // row r is token r / G, head r % G: divided once, then carried along
    const int s0 = r0 / c.G, s_step = step / c.G, g_step = step - s_step * c.G;
    const int64_t cap = (int64_t)c.width * c.page;
    uint4 k[PA_ROWS], v[PA_ROWS];
    int page[PA_ROWS], token[PA_ROWS], head[PA_ROWS];
#pragma unroll
    for (int i = 0, s = s0, g = r0 - s0 * c.G; i < PA_ROWS; ++i) {
        token[i] = s;
        head[i] = g;
        page[i] = -1;
        s += s_step;
        g += g_step;
        if (g >= c.G) {
            g -= c.G;
            ++s;
        }
        if (token[i] >= n) continue;
        if (length + token[i] < cap) page[i] = __ldcg(c.table + b * c.table_ld + ((length + token[i]) >> shift));
        else if (p == 0 && c.status != nullptr) atomicOr(c.status, SK_DEV_POS_OUT_OF_RANGE);
        if (p < pieces) {
            k[i] = __ldcs(reinterpret_cast<const uint4*>(k_new + (b * kn_bs + token[i] * kn_ss + head[i] * kn_hs) * es) + p);
            v[i] = __ldcs(reinterpret_cast<const uint4*>(v_new + (b * vn_bs + token[i] * vn_ss + head[i] * vn_hs) * es) + p);
        }
    }
#pragma unroll
    for (int i = 0; i < PA_ROWS; ++i) {
        const int64_t slot = length + token[i];
        if (token[i] >= n || slot >= cap) continue;
        if (!paged_page_ok(c, page[i])) {
            if (p == 0 && c.status != nullptr) atomicOr(c.status, SK_DEV_INDEX_OUT_OF_RANGE);
            continue;
        }
        const int in = (int)(slot & (c.page - 1)), g = head[i];
        if (p < pieces) {
            reinterpret_cast<uint4*>((char*)c.k + (page[i] * c.k_ps + g * c.k_hs + in * c.k_rs) * es)[p] = k[i];
            reinterpret_cast<uint4*>((char*)c.v + (page[i] * c.v_ps + g * c.v_hs + in * c.v_rs) * es)[p] = v[i];
        }
        if (p == 0) {
            if (c.mass != nullptr) c.mass[b * c.mass_bs + g * c.mass_hs + slot] = 0.f;
            if (c.positions != nullptr) c.positions[b * c.pos_bs + g * c.pos_hs + slot] = (int32_t)(first != nullptr ? (int64_t)first[b] + token[i] : slot);
        }
    }
}

}  // namespace

int launch_paged_append(const sk_paged_cache& c, const void* k_new, int64_t kn_bs, int64_t kn_ss, int64_t kn_hs, const void* v_new,
                        int64_t vn_bs, int64_t vn_ss, int64_t vn_hs, int S, const int32_t* counts, const int32_t* first, cudaStream_t st) {
    const int es = (int)esize(c.dtype), pieces = c.D * es / 16;
    int per = 1;
    while (per < pieces) per *= 2;
    const int64_t rows = (int64_t)S * c.G, of_block = PA_ROWS * (PA_THREADS / per), blocks = (rows + of_block - 1) / of_block;
    if (rows > INT32_MAX - 65536) return fail(SK_ERR_UNSUPPORTED, "sk_paged_append: %lld rows of a sequence in one call", (long long)rows);
    for (int b0 = 0; b0 < c.B; b0 += 65535) {                  // the grid's second dimension
        sk_paged_cache part = c;
        const int n = c.B - b0 < 65535 ? c.B - b0 : 65535;
        part.table += b0 * c.table_ld;
        part.lengths += b0;
        if (part.mass != nullptr) part.mass += b0 * c.mass_bs;
        if (part.positions != nullptr) part.positions += b0 * c.pos_bs;
        const cudaError_t e = launch_after(paged_append_kernel, dim3((unsigned)blocks, n), dim3(PA_THREADS), 0, st, part, (const char*)k_new + b0 * kn_bs * es, kn_bs, kn_ss,
                                           kn_hs, (const char*)v_new + b0 * vn_bs * es, vn_bs, vn_ss, vn_hs, S, counts != nullptr ? counts + b0 : counts,
                                           first != nullptr ? first + b0 : first, es, pieces);
        if (int rc = check_chained(e, "paged_append_kernel")) return rc;
    }
    return SK_OK;
}

namespace {

struct PagedDim {
    int64_t n, s;                                              // entries, elements from one to the next
};
// Rows begin on 16-byte boundaries: v elements are 16 bytes.  The stride of one entry says nothing.
bool paged_aligned(const void* p, int v, PagedDim a, PagedDim b, PagedDim c = {1, 0}) {
    auto on = [v](const PagedDim& x) { return x.n <= 1 || x.s % v == 0; };
    return aligned(p, 16) && on(a) && on(b) && on(c);
}

}  // namespace

// What every call asks of a cache
int paged_check(const sk_paged_cache* c, const char* what) {
    SK_REQUIRE(c != nullptr, "%s: null cache", what);
    SK_REQUIRE(valid_dtype(c->dtype), "%s: bad dtype", what);
    SK_REQUIRE(c->B >= 0 && c->G > 0 && c->D > 0 && c->width >= 0 && c->n_pages >= 0 && c->n_pages <= INT32_MAX, "%s: bad sizes", what);
    if (c->B == 0) return SK_OK;
    SK_REQUIRE(c->lengths && (c->width == 0 || (c->k && c->v && c->table)), "%s: null pointer", what);
    SK_REQUIRE(c->page >= 16 && (c->page & (c->page - 1)) == 0 && (int64_t)c->width * c->page <= 1 << 30, "%s: pages of %d rows, %d a sequence",
               what, c->page, c->width);
    SK_REQUIRE(c->table_ld >= c->width || c->B == 1, "%s: table rows overlap", what);
    const int v = 16 / (int)esize(c->dtype);
    if (c->D % v != 0 || c->D > 256) return fail(SK_ERR_UNSUPPORTED, "%s: head size %d", what, c->D);
    if (!paged_aligned(c->k, v, {c->n_pages, c->k_ps}, {c->G, c->k_hs}, {c->page, c->k_rs}) ||
        !paged_aligned(c->v, v, {c->n_pages, c->v_ps}, {c->G, c->v_hs}, {c->page, c->v_rs}))
        return fail(SK_ERR_MISALIGNED, "%s: pools and their strides must be 16-byte aligned", what);
    // the offset of a page's row is a product of 32-bit numbers
    if (c->k_rs < 0 || c->v_rs < 0 || c->k_rs > INT32_MAX / 4 || c->v_rs > INT32_MAX / 4) return fail(SK_ERR_UNSUPPORTED, "%s: row strides", what);
    return SK_OK;
}

namespace {

// Rows of `inner` elements, n of them s elements apart in every one of three dimensions: no two share an element, where one
// dimension lies inside the other.  What a call writes; what it reads may be expanded.
bool paged_apart(int64_t inner, PagedDim a, PagedDim b, PagedDim c = {1, 0}) {
    PagedDim d[3] = {a, b, c};
    std::sort(d, d + 3, [](const PagedDim& x, const PagedDim& y) { return x.s < y.s; });
    __int128 extent = inner;
    for (const PagedDim& x : d) {
        if (x.n == 0) return true;
        if (x.n == 1) continue;
        if (x.s < extent) return false;
        extent += (__int128)x.s * (x.n - 1);
    }
    return true;
}
bool paged_book_apart(const sk_paged_cache& c, int64_t bs, int64_t hs) {
    return paged_apart((int64_t)c.width * c.page, {c.B, bs}, {c.G, hs});
}
bool paged_pools_apart(const sk_paged_cache& c) {
    return paged_apart(c.D, {c.n_pages, c.k_ps}, {c.G, c.k_hs}, {c.page, c.k_rs}) && paged_apart(c.D, {c.n_pages, c.v_ps}, {c.G, c.v_hs}, {c.page, c.v_rs});
}

}  // namespace
}  // namespace sk

using namespace sk;

extern "C" {

int sk_paged_append(const sk_paged_cache* c, const void* k_new, int64_t kn_bs, int64_t kn_ss, int64_t kn_hs, const void* v_new,
                    int64_t vn_bs, int64_t vn_ss, int64_t vn_hs, int S, const int32_t* counts, const int32_t* first, void* stream) {
    if (int rc = paged_check(c, "sk_paged_append")) return rc;
    SK_REQUIRE(S >= 0, "sk_paged_append: bad sizes");
    if (c->B == 0 || S == 0) return SK_OK;
    SK_REQUIRE(k_new && v_new, "sk_paged_append: null pointer");
    const int v = 16 / (int)esize(c->dtype);
    if (!paged_aligned(k_new, v, {c->B, kn_bs}, {S, kn_ss}, {c->G, kn_hs}) || !paged_aligned(v_new, v, {c->B, vn_bs}, {S, vn_ss}, {c->G, vn_hs}))
        return fail(SK_ERR_MISALIGNED, "sk_paged_append: new rows and their strides must be 16-byte aligned");
    SK_REQUIRE(paged_pools_apart(*c) && (c->mass == nullptr || paged_book_apart(*c, c->mass_bs, c->mass_hs)) &&
               (c->positions == nullptr || paged_book_apart(*c, c->pos_bs, c->pos_hs)), "sk_paged_append: rows of pools, mass or positions overlap");
    return launch_paged_append(*c, k_new, kn_bs, kn_ss, kn_hs, v_new, vn_bs, vn_ss, vn_hs, S, counts, first, (cudaStream_t)stream);
}

size_t sk_paged_attn_workspace_bytes(const sk_paged_cache* c, int H) {
    if (paged_check(c, "sk_paged_attn") != SK_OK || H <= 0 || H % c->G != 0) return 0;
    return paged_attn_workspace(*c, H);
}

int sk_paged_attn(const sk_paged_cache* c, const void* q, int64_t q_bs, int64_t q_hs, void* out, int64_t o_bs, int64_t o_hs, int H,
                  int extra, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = paged_check(c, "sk_paged_attn")) return rc;
    SK_REQUIRE(H > 0 && H % c->G == 0 && extra >= 0, "sk_paged_attn: %d query heads on %d, %d more keys", H, c->G, extra);
    if (c->B == 0) return SK_OK;
    SK_REQUIRE(q && out, "sk_paged_attn: null pointer");
    const int v = 16 / (int)esize(c->dtype);
    if (!paged_aligned(q, v, {c->B, q_bs}, {H, q_hs}) || !paged_aligned(out, v, {c->B, o_bs}, {H, o_hs}))
        return fail(SK_ERR_MISALIGNED, "sk_paged_attn: q, out and their strides must be 16-byte aligned");
    SK_REQUIRE(paged_apart(c->D, {c->B, o_bs}, {H, o_hs}) && (c->mass == nullptr || paged_book_apart(*c, c->mass_bs, c->mass_hs)),
               "sk_paged_attn: rows of out or mass overlap");
    const size_t need = paged_attn_workspace(*c, H);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(SK_ERR_WORKSPACE, "sk_paged_attn: workspace of %zu bytes, %zu needed", workspace == nullptr ? (size_t)0 : workspace_bytes, need);
    if (!aligned(workspace, 16)) return fail(SK_ERR_MISALIGNED, "sk_paged_attn: workspace must be 16-byte aligned");
    return launch_paged_attn(*c, q, q_bs, q_hs, out, o_bs, o_hs, H, extra, scale, workspace, (cudaStream_t)stream);
}

size_t sk_paged_evict_workspace_bytes(const sk_paged_cache* c, int budget) {
    if (paged_check(c, "sk_paged_evict") != SK_OK || budget < 1) return 0;
    return paged_evict_workspace(*c, budget);
}

int sk_paged_evict(const sk_paged_cache* c, int budget, int recent, int sink, float* mass_out, int64_t mo_bs, int64_t mo_hs,
                   int32_t* pos_out, int64_t po_bs, int64_t po_hs, int32_t* lengths_out, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = paged_check(c, "sk_paged_evict")) return rc;
    SK_REQUIRE(budget >= 1 && recent >= 0 && sink >= 0 && (int64_t)recent + sink <= budget, "sk_paged_evict: a budget of %d for %d first and %d last",
               budget, sink, recent);
    if (c->B == 0) return SK_OK;
    SK_REQUIRE(lengths_out && (c->width == 0 || (c->mass && c->positions && mass_out && pos_out)), "sk_paged_evict: null pointer");
    SK_REQUIRE(paged_pools_apart(*c) && paged_book_apart(*c, mo_bs, mo_hs) && paged_book_apart(*c, po_bs, po_hs),
               "sk_paged_evict: rows of pools, mass_out or pos_out overlap");
    const size_t need = paged_evict_workspace(*c, budget);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(SK_ERR_WORKSPACE, "sk_paged_evict: workspace of %zu bytes, %zu needed", workspace == nullptr ? (size_t)0 : workspace_bytes, need);
    if (!aligned(workspace, 16)) return fail(SK_ERR_MISALIGNED, "sk_paged_evict: workspace must be 16-byte aligned");
    return launch_paged_evict(*c, budget, recent, sink, mass_out, mo_bs, mo_hs, pos_out, po_bs, po_hs, lengths_out, workspace,
                              (cudaStream_t)stream);
}

}  // extern "C"
