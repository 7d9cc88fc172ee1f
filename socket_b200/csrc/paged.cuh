// A key-value cache in pages (sk_paged_cache): what its kernels share.
#pragma once
#include "abi_check.cuh"
#include "blocks.cuh"

namespace sk {

// Slots of sequence b in use, `extra` ones behind its length among them; `over`: the length is larger than the table
__device__ __forceinline__ int paged_length(const sk_paged_cache& c, int b, int extra, bool* over = nullptr) {
    const int64_t n = max((int64_t)c.lengths[b], (int64_t)0) + extra, cap = (int64_t)c.width * c.page;
    if (over != nullptr) *over = n > cap;
    return (int)min(n, cap);
}
__device__ __forceinline__ bool paged_page_ok(const sk_paged_cache& c, int page) { return (uint32_t)page < (uint64_t)c.n_pages; }

int paged_check(const sk_paged_cache* c, const char* what);
size_t paged_attn_workspace(const sk_paged_cache& c, int H);
int launch_paged_append(const sk_paged_cache& c, const void* k_new, int64_t kn_bs, int64_t kn_ss, int64_t kn_hs, const void* v_new,
                        int64_t vn_bs, int64_t vn_ss, int64_t vn_hs, int S, const int32_t* counts, const int32_t* first, cudaStream_t st);
int launch_paged_attn(const sk_paged_cache& c, const void* q, int64_t q_bs, int64_t q_hs, void* out, int64_t o_bs, int64_t o_hs, int H,
                      int extra, float scale, void* workspace, cudaStream_t st);
size_t paged_evict_workspace(const sk_paged_cache& c, int budget);
int launch_paged_evict(const sk_paged_cache& c, int budget, int recent, int sink, float* mass_out, int64_t mo_bs, int64_t mo_hs,
                       int32_t* pos_out, int64_t po_bs, int64_t po_hs, int32_t* lengths_out, void* workspace, cudaStream_t st);

}  // namespace sk
