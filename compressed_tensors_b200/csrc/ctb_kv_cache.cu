// The 8-bit paged cache: quantized writes, and the attention over it for any head size and block size.
#include "ctb_kv_common.cuh"

namespace ctb {

int kv_check(const ctb_kv_cache *c, const ctb_kv_batch *t, int32_t dtype) {
    if (!c || !t) return fail(CTB_EINVAL_NULL, "null descriptor");
    if (c->dtype != CTB_I8 && c->dtype != CTB_E4M3) return fail(CTB_EINVAL_DTYPE, "the cache holds int8 or e4m3 codes");
    if (dtype != CTB_BF16 && dtype != CTB_F16) return fail(CTB_EINVAL_DTYPE, "queries, keys and values must be bf16 or f16");
    if (c->heads < 1 || c->block_size < 1 || c->num_blocks < 0 || c->num_blocks > INT32_MAX || t->batch < 0 || t->tokens < 0 || t->tokens > INT32_MAX ||
        t->table_width < 0 || t->table_stride < 0)
        return fail(CTB_EINVAL_SHAPE, "invalid cache or batch sizes");
    if (c->head_dim < 1 || c->head_dim > 256) return fail(CTB_EUNSUPPORTED, "head sizes up to 256 are built, got %d", c->head_dim);
    if (t->table_width * c->block_size > INT32_MAX) return fail(CTB_EUNSUPPORTED, "a block table row covers more than 2^31 tokens");
    if (t->batch > 0 && (!t->seq_lens || !t->query_start || (t->table_width > 0 && !t->block_table))) return fail(CTB_EINVAL_NULL, "null block table, lengths or row offsets");
    if (c->num_blocks > 0 && (!c->k || !c->v || !c->k_scale || !c->v_scale)) return fail(CTB_EINVAL_NULL, "null cache buffer");
    return CTB_OK;
}

// ---------------------------------------------------------------- writing
// One block of threads per (written cache block, head, keys or values): the absolute maximum over the rows that this
// call writes there, the scale, the older codes again where the scale grew, the new codes.
//
// A code is the grid value nearest to the exact quotient x / scale.  An fp32 quotient may round onto a tie that the
// exact one is not on, so the quotient is rounded to odd (toward zero, last bit set when inexact): with 24 bits
// against the grid's 4 (e4m3) or 8 (int8) the second rounding is then the only one.
__device__ __forceinline__ float quotient_to_odd(float x, float s) {
    const float q = __fdiv_rz(x, s);
    const float r = fmaf(-q, s, x);
    return r != 0.0f ? __uint_as_float(__float_as_uint(q) | 1u) : q;
}

template <bool INT8>
__device__ __forceinline__ uint8_t cache_code(float q) {
    if (q != q) return 0;  // then the scale is an infinity or NaN: it alone marks the block, so that queries that do not see it stay clean
    if constexpr (INT8) return (uint8_t)(int8_t)(int)fminf(fmaxf(rintf(q), -128.0f), 127.0f);
    else return f32_to_e4m3(q);
}

template <bool INT8>
__device__ __forceinline__ uint8_t cache_recode(uint8_t code, float before, float now) {
    // the product of a code and a scale is exact in fp64, and its quotient cannot come within 2^-53 of a tie without being one
    const double v = (INT8 ? (double)(int8_t)code : (double)e4m3_to_f32(code)) * (double)before / (double)now;
    float f = __double2float_rz(v);
    if ((double)f != v) f = __uint_as_float(__float_as_uint(f) | 1u);
    return cache_code<INT8>(f);
}

constexpr int kAppendThreads = 128;

template <int DT, bool INT8>
__global__ void __launch_bounds__(kAppendThreads)
kv_append_kernel(const ctb_kv_cache c, const ctb_kv_batch t, const void *k, const void *v, int64_t k_token_stride, int64_t k_head_stride,
                 int64_t v_token_stride, int64_t v_head_stride) {
    __shared__ int64_t tmp[kAppendThreads / 32];
    __shared__ int s_request, s_block;
    __shared__ uint32_t s_max[kAppendThreads / 32];
    const int bs = c.block_size;
    const int64_t capacity = t.table_width * bs;
    // which request and which of its blocks: the written blocks of all requests are numbered in order
    const int per = (t.batch + kAppendThreads - 1) / kAppendThreads;
    const int b0 = threadIdx.x * per;
    if (threadIdx.x == 0) s_request = -1;
    auto written = [&](int b, int &first_block) { return kv_written_blocks(kv_seq(t, capacity, b), bs, first_block); };
    int64_t mine = 0, total;
    int fb;
    for (int b = b0; b < b0 + per && b < t.batch; ++b) mine += written(b, fb);
    int64_t at = block_exclusive<kAppendThreads>(mine, tmp, total);
    const int64_t slot = blockIdx.x;
    if (slot >= total) return;
    if (slot >= at && slot < at + mine) {
        for (int b = b0; b < b0 + per && b < t.batch; ++b) {
            const int n = written(b, fb);
            if (slot < at + n) {
                s_request = b;
                s_block = fb + (int)(slot - at);
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    const int b = s_request;
    if (b < 0) return;
    const KvSeq s = kv_seq(t, capacity, b);
    const int page = t.block_table[b * t.table_stride + s_block];
    if (page < 0 || page >= c.num_blocks) return;
    const int p0 = max(max(s.start, 0), s_block * bs), p1 = min(s.len, (s_block + 1) * bs);
    const int kept = p0 - s_block * bs;  // tokens of this request already in the block
    const int head = blockIdx.y, dim = c.head_dim, n = (p1 - p0) * dim;
    const bool values = blockIdx.z != 0;
    const int64_t ts = values ? v_token_stride : k_token_stride;
    const int64_t x0 = (int64_t)(s.first_row + (p0 - s.start)) * ts + (int64_t)head * (values ? v_head_stride : k_head_stride);
    const void *x = values ? v : k;
    uint8_t *codes = (uint8_t *)(values ? c.v : c.k) + (int64_t)page * (values ? c.v_block_stride : c.k_block_stride) +
                     (int64_t)head * (values ? c.v_head_stride : c.k_head_stride);
    const int64_t cs = values ? c.v_token_stride : c.k_token_stride;
    float *scale = (values ? c.v_scale : c.k_scale) + (int64_t)page * c.heads + head;

    uint32_t most = 0;  // bits of |x|: as integers they order like the numbers, with infinity and NaN on top
    for (int i = threadIdx.x; i < n; i += kAppendThreads)
        most = max(most, __float_as_uint(load_f32(x, DT, x0 + (int64_t)(i / dim) * ts + i % dim)) & 0x7fffffffu);
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = most;
    const float before = kept > 0 ? *scale : 0.0f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) most = max(most, s_max[w]);
    float now = __fdiv_rn(__uint_as_float(most), INT8 ? 127.5f : 448.0f);
    now = now != now ? now : fmaxf(now, 1.1920928955078125e-07f);
    if (kept > 0) now = (before > now || before != before) ? before : now;
    if (threadIdx.x == 0) *scale = now;
    if (kept > 0 && now > before)
        for (int i = threadIdx.x; i < kept * dim; i += kAppendThreads) {
            uint8_t *p = codes + (int64_t)(i / dim) * cs + i % dim;
            *p = cache_recode<INT8>(*p, before, now);
        }
    for (int i = threadIdx.x; i < n; i += kAppendThreads)
        codes[(int64_t)(kept + i / dim) * cs + i % dim] =
            cache_code<INT8>(quotient_to_odd(load_f32(x, DT, x0 + (int64_t)(i / dim) * ts + i % dim), now));
}

// ---------------------------------------------------------------- attention, any head size
// One block per (query row, query head): four warps take every fourth cached token with a running maximum and sum
// each, a lane holds every 32nd element of the head, and the four partial results are joined at the end.
constexpr int kAnyWarps = 4;

template <int DT, bool INT8>
__global__ void __launch_bounds__(kAnyWarps * 32)
kv_attention_any_kernel(const ctb_kv_cache c, const ctb_kv_batch t, const void *q, int64_t q_token_stride, int64_t q_head_stride, int q_heads,
                        float scale, int causal, void *out, float *lse) {
    __shared__ float s_o[kAnyWarps][256], s_m[kAnyWarps], s_l[kAnyWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x;
    const int h = blockIdx.y, kvh = h / (q_heads / c.heads), dim = c.head_dim, bs = c.block_size;
    // the request that holds this row: the last one that begins at or before it
    int lo = 0, hi = t.batch;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (t.query_start[mid] <= row) lo = mid + 1;
        else hi = mid;
    }
    int end = 0;
    const int b = lo - 1;
    if (b >= 0) {
        const KvSeq s = kv_seq(t, t.table_width * bs, b);
        const int64_t i = row - s.first_row;
        if (i >= 0 && i < s.rows) end = kv_end(s, i, causal != 0);
    }
    float qr[8], o[8], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int d = lane + 32 * e;
        qr[e] = d < dim ? load_f32(q, DT, row * q_token_stride + h * q_head_stride + d) : 0.0f;
        o[e] = 0.0f;
    }
    for (int p = warp; p < end; p += kAnyWarps) {
        const int page = t.block_table[b * t.table_stride + p / bs];
        if (page < 0 || page >= c.num_blocks) continue;
        const uint8_t *kr = (const uint8_t *)c.k + (int64_t)page * c.k_block_stride + (int64_t)kvh * c.k_head_stride + (int64_t)(p % bs) * c.k_token_stride;
        const uint8_t *vr = (const uint8_t *)c.v + (int64_t)page * c.v_block_stride + (int64_t)kvh * c.v_head_stride + (int64_t)(p % bs) * c.v_token_stride;
        const float ks = c.k_scale[(int64_t)page * c.heads + kvh], vs = c.v_scale[(int64_t)page * c.heads + kvh];
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = lane + 32 * e;
            if (d < dim) dot = fmaf(qr[e], INT8 ? (float)(int8_t)kr[d] : e4m3_to_f32(kr[d]), dot);
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, x);
        const float score = dot * (ks * scale);
        const float mn = fmaxf(m, score);
        const float keep = mn == -INFINITY ? 1.0f : expf(m - mn), w = mn == -INFINITY ? (score != score ? score : 0.0f) : expf(score - mn);
        l = l * keep + w;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = lane + 32 * e;
            if (d < dim) o[e] = o[e] * keep + w * vs * (INT8 ? (float)(int8_t)vr[d] : e4m3_to_f32(vr[d]));
        }
        m = mn;
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s_o[warp][lane + 32 * e] = o[e];
    __syncthreads();
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kAnyWarps; ++w) mm = fmaxf(mm, s_m[w]);
    float ll = 0.0f, f[kAnyWarps];
#pragma unroll
    for (int w = 0; w < kAnyWarps; ++w) {
        f[w] = s_m[w] == -INFINITY ? (s_l[w] != s_l[w] ? s_l[w] : 0.0f) : expf(s_m[w] - mm);
        ll += f[w] * s_l[w];
    }
    for (int d = threadIdx.x; d < dim; d += kAnyWarps * 32) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kAnyWarps; ++w) v += f[w] * s_o[w][d];
        store_f32(out, DT, (row * q_heads + h) * dim + d, ll == 0.0f ? 0.0f : v / ll);
    }
    if (threadIdx.x == 0) lse[row * q_heads + h] = ll == 0.0f ? -INFINITY : mm + logf(ll);
}

}  // namespace ctb

extern "C" int ctb_kv_cache_append(const ctb_kv_cache *c, const ctb_kv_batch *t, const void *k, const void *v, int32_t dtype,
                                   int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride, void *stream) {
    using namespace ctb;
    int rc = kv_check(c, t, dtype);
    if (rc) return rc;
    if (t->batch == 0 || t->tokens == 0 || c->num_blocks == 0) return CTB_OK;
    if (!k || !v) return fail(CTB_EINVAL_NULL, "null keys or values");
    if (c->heads > 65535) return fail(CTB_EUNSUPPORTED, "too many heads");
    const int64_t slots = kv_most_written(t->tokens, t->batch, c->block_size);
    const dim3 grid((unsigned)slots, (unsigned)c->heads, 2);
    const cudaStream_t st = as_stream(stream);
#define CTB_APPEND(DT, I8) kv_append_kernel<DT, I8><<<grid, kAppendThreads, 0, st>>>(*c, *t, k, v, k_token_stride, k_head_stride, v_token_stride, v_head_stride)
    if (dtype == CTB_BF16) {
        if (c->dtype == CTB_I8) CTB_APPEND(CTB_BF16, true);
        else CTB_APPEND(CTB_BF16, false);
    } else {
        if (c->dtype == CTB_I8) CTB_APPEND(CTB_F16, true);
        else CTB_APPEND(CTB_F16, false);
    }
#undef CTB_APPEND
    return after_launch("kv_append_kernel");
}

extern "C" int64_t ctb_kv_cache_attention_workspace_bytes(const ctb_kv_cache *c, const ctb_kv_batch *t, int32_t q_heads) {
    using namespace ctb;
    if (kv_check(c, t, CTB_BF16) || q_heads < 1 || q_heads % c->heads || t->tokens == 0) return 0;
    return kv_attention_workspace(*c, *t, q_heads);
}

extern "C" int ctb_kv_cache_attention(const ctb_kv_cache *c, const ctb_kv_batch *t, const void *q, int32_t dtype, int64_t q_token_stride,
                                      int64_t q_head_stride, int32_t q_heads, float softmax_scale, int32_t causal, void *out, float *lse,
                                      void *workspace, void *stream) {
    using namespace ctb;
    int rc = kv_check(c, t, dtype);
    if (rc) return rc;
    if (q_heads < 1 || q_heads % c->heads) return fail(CTB_EINVAL_SHAPE, "%d query heads are no multiple of %d cache heads", q_heads, c->heads);
    if (q_heads > 65535) return fail(CTB_EUNSUPPORTED, "too many heads");
    if (t->tokens == 0) return CTB_OK;
    if (!q || !out || !lse) return fail(CTB_EINVAL_NULL, "null queries or outputs");
    const cudaStream_t st = as_stream(stream);
    if (kv_attention_takes(*c, *t, q_heads, q, q_token_stride, q_head_stride, out)) {
        if (!workspace) return fail(CTB_EINVAL_NULL, "null workspace");
        return kv_attention_launch(*c, *t, q, dtype, q_token_stride, q_head_stride, q_heads, softmax_scale, causal, out, lse, workspace, st);
    }
    const dim3 grid((unsigned)t->tokens, (unsigned)q_heads);
#define CTB_ATT(DT, I8) kv_attention_any_kernel<DT, I8><<<grid, kAnyWarps * 32, 0, st>>>(*c, *t, q, q_token_stride, q_head_stride, q_heads, softmax_scale, causal, out, lse)
    if (dtype == CTB_BF16) {
        if (c->dtype == CTB_I8) CTB_ATT(CTB_BF16, true);
        else CTB_ATT(CTB_BF16, false);
    } else {
        if (c->dtype == CTB_I8) CTB_ATT(CTB_F16, true);
        else CTB_ATT(CTB_F16, false);
    }
#undef CTB_ATT
    return after_launch("kv_attention_any_kernel");
}
