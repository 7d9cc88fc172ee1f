// How likely tokens were: log probabilities, entropy and the likeliest alternatives of rows of logits.
#pragma once
#include "token_rows_body.cuh"

namespace sk {
namespace {

// One block per row: maximum, then sums, then the alternatives one by one, each the first behind the one before.
constexpr int LP_THREADS = 256, LP_TOP = 64;
template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
token_logprobs_kernel(const T* logits, int64_t ld, int vocab, const int64_t* token, int top, float* logprob, float* entropy, float* top_logprob,
                      int64_t* top_token, int32_t* status) {
    __shared__ float red[32], red2[32], best_s[LP_THREADS / 32];
    __shared__ int at_s[LP_THREADS / 32];
    const int64_t r = blockIdx.x;
    const T* x = logits + r * ld;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    // the first of the row behind (after, i_after) in the order of picks
    auto next = [&](float after, int i_after, float& best, int& at) {
        best = -INFINITY;
        at = vocab;
        for (int i = t; i < vocab; i += LP_THREADS) {
            const float v = to_f32(x[i]);
            if ((i_after < 0 || picked(after, i_after, v, i)) && (at == vocab || picked(v, i, best, at))) {
                best = v;
                at = i;
            }
        }
        auto join = [&](float v, int i) {
            if (i < vocab && (at == vocab || picked(v, i, best, at))) {
                best = v;
                at = i;
            }
        };
        for (int o = 16; o >= 1; o >>= 1) {
            const float v = __shfl_xor_sync(FULL, best, o);
            const int i = __shfl_xor_sync(FULL, at, o);
            join(v, i);
        }
        __syncthreads();
        if (lane == 0) {
            best_s[warp] = best;
            at_s[warp] = at;
        }
        __syncthreads();
        for (int w = 0; w < LP_THREADS / 32; ++w) join(best_s[w], at_s[w]);
    };
    float m;
    int at;
    next(0.f, -1, m, at);
    float z = 0.f, zd = 0.f;
    for (int i = t; i < vocab; i += LP_THREADS) {
        const float d = to_f32(x[i]) - m, e = expf(d);
        z += e;
        zd += e == 0.f ? 0.f : e * d;
    }
    z = block_sum(z, red);
    zd = block_sum(zd, red2);
    const float lz = logf(z);
    if (t == 0) {
        if (entropy != nullptr) entropy[r] = lz - zd / z;
        if (token != nullptr) {
            const int64_t i = token[r];
            const bool in = i >= 0 && i < vocab;
            logprob[r] = in ? to_f32(x[i]) - m - lz : NAN;
            if (!in && status != nullptr) atomicOr(status, SK_DEV_INDEX_OUT_OF_RANGE);
        }
    }
    float v = m;
    for (int k = 0; k < top; ++k) {
        if (k > 0) {
            float w;
            next(v, at, w, at);
            v = w;
        }
        if (t == 0) {
            top_logprob[r * top + k] = v - m - lz;
            top_token[r * top + k] = at;
        }
    }
}

}  // namespace

int token_logprobs(const void* logits, int dtype, int64_t ld, int64_t rows, int vocab, const int64_t* token, int top, float* logprob,
                   float* entropy, float* top_logprob, int64_t* top_token, int32_t* status, cudaStream_t st) {
    SK_REQUIRE(valid_dtype(dtype) && rows >= 0 && vocab > 0, "token_logprobs: bad sizes or dtype");
    SK_REQUIRE(top >= 0 && top <= LP_TOP && top <= vocab, "token_logprobs: %d alternatives of %d", top, vocab);
    if (rows == 0) return SK_OK;
    SK_REQUIRE(logits && (ld >= vocab || rows == 1) && (!token || logprob) && (top == 0 || (top_logprob && top_token)),
               "token_logprobs: null pointer or overlapping rows");
    if (rows > 0x7fffffff) return fail(SK_ERR_UNSUPPORTED, "token_logprobs: %lld rows", (long long)rows);
    auto go = [&](auto t) {
        using T = decltype(t);
        token_logprobs_kernel<T><<<(unsigned)rows, LP_THREADS, 0, st>>>((const T*)logits, ld, vocab, token, top, logprob, entropy, top_logprob,
                                                                        top_token, status);
    };
    if (dtype == SK_F32) go(float{});
    else if (dtype == SK_BF16) go(__nv_bfloat16{});
    else go(__half{});
    return check_launch("token_logprobs_kernel");
}

}  // namespace sk
