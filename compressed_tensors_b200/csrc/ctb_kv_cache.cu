// The 8-bit paged cache: quantized writes, and the attention over it for any head size and block size.
#include <type_traits>

#include "ctb_fastdiv.h"
#include "ctb_kv_common.cuh"
#include "ctb_mma.cuh"

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
// What bounds it: two bytes read and one written per element, from and to HBM; for single tokens, the latency of a launch and
// of four dependent loads (lengths, block number, rows and old scale, codes where the scale grew).  Four prompts of up to 4096 tokens,
// 8 heads of 128: 26 us, 3.1 TB/s; one row each of 64 requests: 4.3 us.
//
// A unit is one (written cache block, head, keys or values): the absolute maximum over the rows that the call writes
// there, the scale, the older codes again where the scale grew, the new codes.  A unit is taken by a warp where the call
// has about one row per request, else by a block of four; rows of 16-byte pieces stay in registers between the maximum and the
// codes (up to PIECES of them per thread, which covers 64 x 128), what exceeds that is read again from the cache lines just read.
//
// A code is the grid value nearest to the exact quotient x / scale.  An fp32 quotient may round onto a tie that the
// exact one is not on, so the quotient is rounded to odd (where it is inexact, to the neighbour whose last bit is set): with 24 bits
// against the grid's 4 (e4m3) or 8 (int8) the second rounding is then the only one.  `r` is 1 / s rounded; product, residual and
// correction give the nearest quotient, and the sign of its own residual says on which side the exact one lies.
//
// Where the scale was just made from the rows themselves, s = round(m / h) with m their largest magnitude and h = 448 or 127.5, one
// product replaces that.  x and m have at most 11 significant bits, a tie of the grid at most 9, h at most 8: x h and m tie are
// integers of at most 20 bits times powers of two, equal or 2^-20 apart.  So a quotient is 2^-20 away from every tie, or it would be on
// one if s were exactly m / h: then it lies on the side that the rounding of s puts all of them on, and a factor of 1 -+ 2^-22, which
// the roundings of the quotient and the product (2^-24 each) cannot undo, moves it there.  Where m / h needs no rounding the factor is 1.
__device__ __forceinline__ float quotient_to_odd(float x, float s, float r) {
    const float q0 = x * r, q = fmaf(fmaf(-q0, s, x), r, q0), e = fmaf(-q, s, x);
    const int bits = __float_as_int(q);
    // the residual has the quotient's sign where the exact magnitude is larger (the scale is positive)
    const int step = (__float_as_int(e) ^ bits) < 0 ? -1 : 1;
    return e != 0.0f && !(bits & 1) ? __int_as_float(bits + step) : q;
}

// two quotients -> two codes in the low bytes
template <bool INT8>
__device__ __forceinline__ uint32_t cache_codes2(float a, float b) {
    if constexpr (INT8) {
        // 1.5 * 2^23 + v has the integer nearest to v, ties to even, in its low byte
        const float m = 12582912.0f;
        return __byte_perm(__float_as_uint(fminf(fmaxf(a, -128.0f), 127.0f) + m), __float_as_uint(fminf(fmaxf(b, -128.0f), 127.0f) + m), 0x0040);
    } else {
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
        return r;
    }
}

template <bool INT8>
__device__ __forceinline__ uint8_t cache_recode(uint8_t code, float before, float now) {
    // the product of a code and a scale is exact in fp64, and its quotient cannot come within 2^-53 of a tie without being one
    const double v = (INT8 ? (double)(int8_t)code : (double)e4m3_to_f32(code)) * (double)before / (double)now;
    float f = __double2float_rz(v);
    if ((double)f != v) f = __uint_as_float(__float_as_uint(f) | 1u);
    return (uint8_t)cache_codes2<INT8>(f, 0.0f);
}

constexpr int kAppendThreads = 128;

struct AppendArgs {
    ctb_kv_cache c;
    ctb_kv_batch t;
    const void *x[2];                              // keys, values
    int64_t token_stride[2], head_stride[2];
    int64_t capacity;
    FastDiv by_row;                                // pieces of a row
    FastDiv by_groups;                             // groups of `per` units that the 2 * heads of a block make
    uint32_t groups, per, total;                   // total: all groups that there may be
};

// W: warps of a unit (1 or 4); V: elements that are loaded at once (8, or 1 for rows off the 16-byte grid)
template <int DT, bool INT8, int W, int V>
__global__ void __launch_bounds__(kAppendThreads, 6) kv_append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int T = W * 32, PIECES = 8;
    __shared__ uint32_t s_max[kAppendThreads / 32];
    const int lane = threadIdx.x & 31, i0 = threadIdx.x & (T - 1);
    const uint32_t group = W == 4 ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 5);
    if (group >= a.total) return;  // (with W == 4 for the whole block)
    const uint32_t slot = fastdiv(group, a.by_groups);
    const int first_unit = (int)((group - slot * a.groups) * a.per), bs = a.c.block_size, dim = a.c.head_dim;
    // the written blocks of all requests are numbered in order
    KvSeq s;
    uint32_t begin;
    int fb;
    const int b = kv_locate(a.t, a.capacity, kv_lane_seq(a.t, a.capacity, 0), slot, [&](const KvSeq &q) { return (uint32_t)kv_written_blocks(q, bs, fb); }, s, begin);
    if (b < 0) return;
    kv_written_blocks(s, bs, fb);
    const int block = fb + (int)(slot - begin);
    const int page = a.t.block_table[b * a.t.table_stride + block];
    if (page < 0 || page >= a.c.num_blocks) return;
    const int p0 = max(max(s.start, 0), block * bs), p1 = min(s.len, (block + 1) * bs);
    const int kept = p0 - block * bs;  // tokens of this request already in the block
    const int row = dim / V, n = (p1 - p0) * row;
    for (int u = first_unit; u < min(first_unit + (int)a.per, 2 * a.c.heads); ++u) {
        const int values = u & 1, head = u >> 1;
        const int64_t ts = a.token_stride[values], cs = values ? a.c.v_token_stride : a.c.k_token_stride;
        const uint16_t *x = (const uint16_t *)a.x[values] + (int64_t)(s.first_row + (p0 - s.start)) * ts + (int64_t)head * a.head_stride[values];
        uint8_t *codes = (uint8_t *)(values ? a.c.v : a.c.k) + (int64_t)page * (values ? a.c.v_block_stride : a.c.k_block_stride) +
                         (int64_t)head * (values ? a.c.v_head_stride : a.c.k_head_stride);
        float *scale = (values ? a.c.v_scale : a.c.k_scale) + (int64_t)page * a.c.heads + head;
        const float before = kept > 0 ? *scale : 0.0f;

        // pieces i0, i0 + T, ... of the rows in order
        auto load = [&](int i) {
            const int tk = (int)fastdiv((uint32_t)i, a.by_row), d = (i - tk * row) * V;
            if constexpr (V == 8) return __ldg((const uint4 *)(x + tk * ts + d));
            else return make_uint4(x[tk * ts + d], 0, 0, 0);
        };
        uint4 held[PIECES];
        uint32_t most = 0;  // |x|, two at a time
        auto weigh = [&](const uint4 &v) {
            most = max2_nan<DT>(most, max2_nan<DT>(max2_nan<DT>(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), max2_nan<DT>(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
        };
#pragma unroll
        for (int k = 0; k < PIECES; ++k) held[k] = i0 + k * T < n ? load(i0 + k * T) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < PIECES; ++k) weigh(held[k]);
        for (int i = i0 + PIECES * T; i < n; i += T) weigh(load(i));
        most = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
        if constexpr (W > 1) {
            __syncthreads();  // the unit before has been read
            if (lane == 0) s_max[threadIdx.x >> 5] = most;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < W; ++w) most = max(most, s_max[w]);
        }
        const float top = DT == CTB_BF16 ? bf16_bits_to_f32(most) : __half2float(__ushort_as_half((unsigned short)most));
        constexpr float half_range = INT8 ? 127.5f : 448.0f;
        float now = __fdiv_rn(top, half_range);
        const float off = fmaf(now, half_range, -top);  // how the rounding went
        float side = off > 0.0f ? 1.0f - 0x1p-22f : off < 0.0f ? 1.0f + 0x1p-22f : 1.0f;
        if (now < 1.1920928955078125e-07f) now = 1.1920928955078125e-07f, side = 1.0f;  // a power of two: quotients are exact
        const bool fresh = kept == 0 || now > before;
        if (kept > 0) now = (before > now || before != before) ? before : now;
        __syncwarp();
        if (i0 == 0) *scale = now;
        // an infinity or NaN marks its block by the scale alone (codes of zero), so that queries that do not see it stay clean
        const bool finite = now - now == 0.0f;
        if (kept > 0 && now > before)
            for (int i = i0; i < kept * row; i += T) {
                uint8_t *p = codes + (int64_t)(i / row) * cs + (i % row) * V;
                if constexpr (V == 8) {
                    uint2 w = *(const uint2 *)p;
                    uint8_t(&c)[8] = reinterpret_cast<uint8_t(&)[8]>(w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) c[e] = finite ? cache_recode<INT8>(c[e], before, now) : 0;
                    *(uint2 *)p = w;
                } else {
                    *p = finite ? cache_recode<INT8>(*p, before, now) : 0;
                }
            }
        const float r = __frcp_rn(now);
        auto half = [](uint32_t h) { return DT == CTB_BF16 ? bf16_bits_to_f32(h) : __half2float(__ushort_as_half((unsigned short)h)); };
        auto store = [&](int i, const uint4 &v) {
            const int tk = (int)fastdiv((uint32_t)i, a.by_row), d = (i - tk * row) * V;
            uint8_t *p = codes + (int64_t)(kept + tk) * cs + d;
            const uint32_t h[4] = {v.x, v.y, v.z, v.w};
            float q[8];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float f = half(e & 1 ? h[e >> 1] >> 16 : h[e >> 1] & 0xffffu);
                if (fresh) {
                    const float q0 = f * r;
                    q[e] = fmaf(fmaf(-q0, now, f), r, q0) * side;
                } else {
                    q[e] = quotient_to_odd(f, now, r);
                }
            }
            if constexpr (V == 8) {
                uint2 w = make_uint2(__byte_perm(cache_codes2<INT8>(q[0], q[1]), cache_codes2<INT8>(q[2], q[3]), 0x5410),
                                     __byte_perm(cache_codes2<INT8>(q[4], q[5]), cache_codes2<INT8>(q[6], q[7]), 0x5410));
                if (!finite) w = make_uint2(0, 0);
                *(uint2 *)p = w;
            } else {
                *p = finite ? (uint8_t)cache_codes2<INT8>(q[0], 0.0f) : 0;
            }
        };
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
            if (i0 + k * T < n) store(i0 + k * T, held[k]);
        for (int i = i0 + PIECES * T; i < n; i += T) store(i, load(i));
    }
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
    const int64_t units = kv_most_written(t->tokens, t->batch, c->block_size) * 2 * c->heads;
    if (units > INT32_MAX - 4) return fail(CTB_EUNSUPPORTED, "too many tokens and heads for one call");
    AppendArgs a;
    a.c = *c;
    a.t = *t;
    a.x[0] = k, a.x[1] = v;
    a.token_stride[0] = k_token_stride, a.token_stride[1] = v_token_stride;
    a.head_stride[0] = k_head_stride, a.head_stride[1] = v_head_stride;
    a.capacity = t->table_width * c->block_size;
    const cudaStream_t st = as_stream(stream);
    const bool wide = c->head_dim % 8 == 0 && aligned16(k) && aligned16(v) && (k_token_stride | k_head_stride | v_token_stride | v_head_stride) % 8 == 0 &&
                      (((uintptr_t)c->k | (uintptr_t)c->v) & 7) == 0 &&
                      (c->k_block_stride | c->k_head_stride | c->k_token_stride | c->v_block_stride | c->v_head_stride | c->v_token_stride) % 8 == 0;
    // a warp per unit where its rows fit the warp's registers: about one row per request, or small blocks; else a block of four
    const bool single = t->tokens <= 2 * (int64_t)t->batch || (int64_t)c->block_size * c->head_dim <= 2048;
    // Several units of a cache block in turn, once there are enough of them to fill the GPU: the search for the request is made
    // once for all.
    a.per = units >= 16 * (int64_t)sm_count() * (single ? 4 : 1) ? 4 : 1;
    a.by_row = make_fastdiv((uint32_t)(wide ? c->head_dim / 8 : c->head_dim));
    a.groups = (uint32_t)cdiv(2 * c->heads, a.per);
    a.by_groups = make_fastdiv(a.groups);
    a.total = (uint32_t)(kv_most_written(t->tokens, t->batch, c->block_size) * a.groups);
    auto go = [&](auto dt, auto i8) {
        constexpr int DT = decltype(dt)::value;
        constexpr bool I8 = decltype(i8)::value;
        const unsigned blocks = (unsigned)(single ? cdiv(a.total, 4) : a.total);
        if (wide && single) kv_append_kernel<DT, I8, 1, 8><<<blocks, kAppendThreads, 0, st>>>(a);
        else if (wide) kv_append_kernel<DT, I8, 4, 8><<<blocks, kAppendThreads, 0, st>>>(a);
        else if (single) kv_append_kernel<DT, I8, 1, 1><<<blocks, kAppendThreads, 0, st>>>(a);
        else kv_append_kernel<DT, I8, 4, 1><<<blocks, kAppendThreads, 0, st>>>(a);
    };
    using B = std::integral_constant<int, CTB_BF16>;
    using H = std::integral_constant<int, CTB_F16>;
    if (dtype == CTB_BF16) c->dtype == CTB_I8 ? go(B{}, std::true_type{}) : go(B{}, std::false_type{});
    else c->dtype == CTB_I8 ? go(H{}, std::true_type{}) : go(H{}, std::false_type{});
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
