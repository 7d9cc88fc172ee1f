// Entry points of the paged cache, and the append that fills its pages.
#include "paged.cuh"

namespace sk {
namespace {

// One warp per new row (sequence, token, head): the key's and the value's 16-byte pieces, and the slot's bookkeeping.  Nothing but
// copies: bound by memory.
constexpr int PA_WARPS = 8;
__global__ void __launch_bounds__(PA_WARPS * 32)
paged_append_kernel(const __grid_constant__ sk_paged_cache c, const char* k_new, int64_t kn_bs, int64_t kn_ss, int64_t kn_hs, const char* v_new,
                    int64_t vn_bs, int64_t vn_ss, int64_t vn_hs, int S, const int32_t* counts, const int32_t* first, int es) {
    const int64_t row = (int64_t)blockIdx.x * PA_WARPS + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= (int64_t)c.B * S * c.G) return;
    const int g = (int)(row % c.G), s = (int)(row / c.G % S), b = (int)(row / c.G / S);
    if (counts != nullptr && s >= counts[b]) return;
    const int64_t slot = (int64_t)max(c.lengths[b], 0) + s;
    const int shift = 31 - __clz(c.page);
    int flag = 0;
    if (slot >= (int64_t)c.width * c.page) flag = SK_DEV_POS_OUT_OF_RANGE;
    const int page = flag == 0 ? c.table[b * c.table_ld + (slot >> shift)] : 0;
    if (flag == 0 && !paged_page_ok(c, page)) flag = SK_DEV_INDEX_OUT_OF_RANGE;
    if (flag != 0) {
        if (lane == 0 && c.status != nullptr) atomicOr(c.status, flag);
        return;
    }
    const int r = (int)(slot & (c.page - 1)), pieces = c.D * es / 16;
    const uint4* ks = reinterpret_cast<const uint4*>(k_new + (b * kn_bs + s * kn_ss + g * kn_hs) * es);
    const uint4* vs = reinterpret_cast<const uint4*>(v_new + (b * vn_bs + s * vn_ss + g * vn_hs) * es);
    uint4* kd = reinterpret_cast<uint4*>((char*)c.k + (page * c.k_ps + g * c.k_hs + r * c.k_rs) * es);
    uint4* vd = reinterpret_cast<uint4*>((char*)c.v + (page * c.v_ps + g * c.v_hs + r * c.v_rs) * es);
    for (int i = lane; i < pieces; i += 32) {
        kd[i] = ks[i];
        vd[i] = vs[i];
    }
    if (lane == 0) {
        if (c.mass != nullptr) c.mass[b * c.mass_bs + g * c.mass_hs + slot] = 0.f;
        if (c.positions != nullptr) c.positions[b * c.pos_bs + g * c.pos_hs + slot] = (int32_t)(first != nullptr ? (int64_t)first[b] + s : slot);
    }
}

}  // namespace

int launch_paged_append(const sk_paged_cache& c, const void* k_new, int64_t kn_bs, int64_t kn_ss, int64_t kn_hs, const void* v_new,
                        int64_t vn_bs, int64_t vn_ss, int64_t vn_hs, int S, const int32_t* counts, const int32_t* first, cudaStream_t st) {
    const int64_t rows = (int64_t)c.B * S * c.G, blocks = (rows + PA_WARPS - 1) / PA_WARPS;
    if (blocks > 0x7fffffff) return fail(SK_ERR_UNSUPPORTED, "sk_paged_append: %lld rows in one call", (long long)rows);
    paged_append_kernel<<<(unsigned)blocks, PA_WARPS * 32, 0, st>>>(c, (const char*)k_new, kn_bs, kn_ss, kn_hs, (const char*)v_new, vn_bs,
                                                                    vn_ss, vn_hs, S, counts, first, (int)esize(c.dtype));
    return check_launch("paged_append_kernel");
}

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
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->k_ps % v || c->k_hs % v || c->k_rs % v || c->v_ps % v || c->v_hs % v || c->v_rs % v)
        return fail(SK_ERR_MISALIGNED, "%s: pools and their strides must be 16-byte aligned", what);
    // the offset of a page's row is a product of 32-bit numbers
    if (c->k_rs < 0 || c->v_rs < 0 || c->k_rs > INT32_MAX / 4 || c->v_rs > INT32_MAX / 4) return fail(SK_ERR_UNSUPPORTED, "%s: row strides", what);
    return SK_OK;
}

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
    if (!aligned(k_new, 16) || !aligned(v_new, 16) || kn_bs % v || kn_ss % v || kn_hs % v || vn_bs % v || vn_ss % v || vn_hs % v)
        return fail(SK_ERR_MISALIGNED, "sk_paged_append: new rows and their strides must be 16-byte aligned");
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
    if (!aligned(q, 16) || !aligned(out, 16) || q_bs % v || q_hs % v || o_bs % v || o_hs % v)
        return fail(SK_ERR_MISALIGNED, "sk_paged_attn: q, out and their strides must be 16-byte aligned");
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
    SK_REQUIRE(c->mass && c->positions && mass_out && pos_out && lengths_out, "sk_paged_evict: null pointer");
    const size_t need = paged_evict_workspace(*c, budget);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return fail(SK_ERR_WORKSPACE, "sk_paged_evict: workspace of %zu bytes, %zu needed", workspace == nullptr ? (size_t)0 : workspace_bytes, need);
    if (!aligned(workspace, 16)) return fail(SK_ERR_MISALIGNED, "sk_paged_evict: workspace must be 16-byte aligned");
    return launch_paged_evict(*c, budget, recent, sink, mass_out, mo_bs, mo_hs, pos_out, po_bs, po_hs, lengths_out, workspace,
                              (cudaStream_t)stream);
}

}  // extern "C"
