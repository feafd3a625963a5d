// What the write into the 8-bit paged cache and the attention over it share: how a block of threads finds its request.
#pragma once

#include "ctb_common.cuh"
#include "ctb_kv_index.h"

namespace ctb {

__device__ __forceinline__ KvSeq kv_seq(const ctb_kv_batch &t, int64_t capacity, int b) {
    return kv_seq(t.query_start[b], t.query_start[b + 1], t.seq_lens[b], t.tokens, capacity);
}

__device__ __forceinline__ uint32_t warp_inclusive(uint32_t v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += u;
    }
    return v;
}

// Every warp walks the requests for itself, one per lane and 32 at a time; `first` is this lane's of the first 32.
__device__ __forceinline__ KvSeq kv_lane_seq(const ctb_kv_batch &t, int64_t capacity, int base) {
    const int b = base + (threadIdx.x & 31);
    return b < t.batch ? kv_seq(t, capacity, b) : KvSeq{0, 0, 0, 0};
}

// The request that `pos` falls into when weigh(request) numbers are counted off for each in turn, -1 behind the last; its KvSeq and the
// number it begins at, in all lanes.  The numbers of all requests stay below 2^32.
template <class F>
__device__ __forceinline__ int kv_locate(const ctb_kv_batch &t, int64_t capacity, const KvSeq &first, uint32_t pos, F weigh, KvSeq &s, uint32_t &begin) {
    uint32_t run = 0;
    for (int base = 0; base < t.batch; base += 32) {
        const KvSeq q = base == 0 ? first : kv_lane_seq(t, capacity, base);
        const uint32_t n = weigh(q), upto = run + warp_inclusive(n);
        const uint32_t hit = __ballot_sync(0xffffffffu, pos < upto);
        if (hit) {
            const int src = __ffs(hit) - 1;
            s.first_row = __shfl_sync(0xffffffffu, q.first_row, src);
            s.rows = __shfl_sync(0xffffffffu, q.rows, src);
            s.len = __shfl_sync(0xffffffffu, q.len, src);
            s.start = __shfl_sync(0xffffffffu, q.start, src);
            begin = __shfl_sync(0xffffffffu, upto - n, src);
            return base + src;
        }
        run = __shfl_sync(0xffffffffu, upto, 31);
    }
    s = KvSeq{0, 0, 0, 0};
    begin = run;
    return -1;
}

// host: what every entry point refuses
int kv_check(const ctb_kv_cache *c, const ctb_kv_batch *t, int32_t dtype);

// ctb_kv_attention.cu: the attention for few query rows per cache head; whether it takes a call, its scratch, the call
bool kv_attention_takes(const ctb_kv_cache &c, const ctb_kv_batch &t, int q_heads, const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *out);
int64_t kv_attention_workspace(const ctb_kv_cache &c, const ctb_kv_batch &t, int q_heads);
int kv_attention_launch(const ctb_kv_cache &c, const ctb_kv_batch &t, const void *q, int dtype, int64_t q_token_stride, int64_t q_head_stride, int q_heads,
                        float softmax_scale, int causal, void *out, float *lse, void *workspace, cudaStream_t st);

}  // namespace ctb
