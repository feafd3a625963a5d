// What the write into the 8-bit paged cache and the attention over it share: how a block of threads finds its request.
#pragma once

#include "ctb_common.cuh"
#include "ctb_kv_index.h"

namespace ctb {

__device__ __forceinline__ KvSeq kv_seq(const ctb_kv_batch &t, int64_t capacity, int b) {
    return kv_seq(t.query_start[b], t.query_start[b + 1], t.seq_lens[b], t.tokens, capacity);
}

// Exclusive scan of `mine` over a block of THREADS threads; `total` gets the sum.  `tmp`: THREADS / 32 shared words.
template <int THREADS>
__device__ __forceinline__ int64_t block_exclusive(int64_t mine, int64_t *tmp, int64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t v = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) tmp[warp] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += tmp[w];
        total += tmp[w];
    }
    __syncthreads();
    return before + v - mine;
}

// host: what every entry point refuses
int kv_check(const ctb_kv_cache *c, const ctb_kv_batch *t, int32_t dtype);

// ctb_kv_attention.cu: the attention for few query rows per cache head; whether it takes a call, its scratch, the call
bool kv_attention_takes(const ctb_kv_cache &c, const ctb_kv_batch &t, int q_heads, const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *out);
int64_t kv_attention_workspace(const ctb_kv_cache &c, const ctb_kv_batch &t, int q_heads);
int kv_attention_launch(const ctb_kv_cache &c, const ctb_kv_batch &t, const void *q, int dtype, int64_t q_token_stride, int64_t q_head_stride, int q_heads,
                        float softmax_scale, int causal, void *out, float *lse, void *workspace, cudaStream_t st);

}  // namespace ctb
