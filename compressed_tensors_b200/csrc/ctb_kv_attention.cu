// Attention over the 8-bit paged cache for few query rows per cache head (decoding): head sizes 64, 128 and 256, blocks of
// a multiple of 16 tokens.
//
// What bounds it: every cached byte is read once per row tile and used for a handful of query rows, so the call takes the
// time of reading the cache from HBM: 64 requests of up to 8192 tokens, 8 cache heads of 128: 101 us, 5.4 TB/s.  A single request of
// 32768 takes 24 us, of which 8 go to the search, the first loads and the results, and 5 to the second kernel.
//
// A step is 16 cached tokens of one head, which lie in one block: one key scale, one value scale.  With query rows as
// the 8 columns of mma.m16n8k16,
//     S^T [16 tokens, 8 rows] = K [16, D] Q^T,      O^T [D, 8 rows] += V^T [D, 16] P^T,
// both products take the cache as the 16-row operand, so the codes go from 16-byte loads into operand registers without a
// transpose through shared memory: the order of the contracted index is free (d in the first product, tokens in the second),
// and so is the order of the rows of O^T.  Only P^T changes layout (movmatrix, one 8 x 8 tile each).
//
// Number formats.  Codes become f16 exactly (e4m3 and int8 both fit).  A query row is scaled by a power of two to a
// largest element in [128, 256) and held in f16: bf16 elements are exact down to 2^-24 of the largest one.  Weights are f16 as
// well: P' = 2^(s + log2 v_scale - m), where m follows the maximum of s + log2 v_scale (of what a token weighs with its
// scale), so the tokens that matter have f16's 11 bits whatever the scales of their blocks are; the denominator is the fp32
// sum of P' / v_scale before that rounding.  Scores, m, sums and O are fp32.
//
// m is raised only where a score passes it by more than 2^8, which f16 has room for: in nearly every step the decision is
// one vote, and nothing is exchanged between lanes or rescaled.
//
// Work.  The steps of all (request, row tile, head) items form one line that is cut into equal pieces, one per
// block, whatever the lengths are; a piece's parts of an item that other pieces share go to scratch as (O, m, sum), and the
// second kernel joins them.  The warps of a block take every fourth step and join in shared memory.  Each warp keeps
// several steps in flight with cp.async.
#include <atomic>

#include "ctb_fastdiv.h"
#include "ctb_kv_common.cuh"
#include "ctb_mma.cuh"

namespace ctb {

constexpr int kAttWarps = 4, kAttThreads = kAttWarps * 32, kAttMinPiece = 16;

// What the second kernel has to know of the item that begins in a piece and ends behind it: written by the piece's block.
struct AttJoin {
    int64_t row;               // row of out and lse of the item's first query row's head 0 within the cache head
    int64_t slot;              // of the first part; the others follow at slots 2p (p on a padded line), p = piece + 1 .. last
    uint32_t last;             // last piece; 0: there is no such item
    int32_t rows, first;       // query rows of the tile; which of the cache head's query heads the first one is
    int32_t padded;
};

struct AttArgs {
    ctb_kv_cache c;
    ctb_kv_batch t;
    const void *q;
    void *out;
    float *lse, *part;  // part: [slot][8 * NT rows][D + 2]
    int64_t q_token_stride, q_head_stride;
    float scale_log2;   // softmax scale * log2(e)
    int64_t slots;      // of `part`
    int64_t capacity;   // tokens of a row of the block table
    FastDiv block_steps, by_group, by_grid;  // step -> block, row -> query, steps -> pieces
    AttJoin *join;      // [piece]
    uint32_t *pieces;   // how many there are
    int32_t q_heads, group, causal, grid;
};

// How the line of steps is cut.  `padded`: every item begins a piece of its own (short lines: no item is split for nothing).
struct AttCut {
    uint32_t total;  // steps of the line
    uint32_t per;    // steps of a piece
    bool padded;
};

template <int NT>
__device__ __forceinline__ int att_tiles(const AttArgs &a, const KvSeq &s) {
    return (s.rows * a.group + NT * 8 - 1) / (NT * 8);
}
// steps of row tile `tile`: up to the last position that its last row sees
template <int NT>
__device__ __forceinline__ uint32_t att_steps(const AttArgs &a, const KvSeq &s, int tile) {
    const int last = min(s.rows - 1, (int)fastdiv((uint32_t)((tile + 1) * NT * 8 - 1), a.by_group));
    return (uint32_t)(kv_end(s, last, a.causal != 0) + 15) >> 4;
}
// Places that an item takes on the line: its steps, and some for what every item costs besides (rows, first copies, results: about as
// long as kAttItemSteps steps); an item without a step has its place too, and is written there.  On a padded line: whole pieces.
constexpr uint32_t kAttItemSteps = 8;
__device__ __forceinline__ uint32_t att_span(const AttCut &cut, uint32_t n) {
    static_assert(kAttMinPiece == 16, "pieces of a padded line");
    return cut.padded ? (max(n, 1u) + 15) & ~15u : n + kAttItemSteps;
}

// steps of all tiles of a request, for one head
template <int NT>
__device__ __forceinline__ uint32_t att_request_steps(const AttArgs &a, const KvSeq &s, const AttCut &cut) {
    uint32_t n = 0;
    const int tiles = att_tiles<NT>(a, s);
    for (int i = 0; i < tiles; ++i) n += att_span(cut, att_steps<NT>(a, s, i));
    return n;
}

__device__ __forceinline__ KvSeq att_lane_seq(const AttArgs &a, const KvSeq &first, int base) {
    return base == 0 ? first : kv_lane_seq(a.t, a.capacity, base);
}

// The whole line, over all requests and heads.  The host admits only calls whose line stays below 2^31 steps; row offsets
// that decrease can make it longer, and then nothing is on it.
template <int NT>
__device__ __forceinline__ uint32_t att_total(const AttArgs &a, const KvSeq &first, const AttCut &cut) {
    uint64_t n = 0;
    for (int base = 0; base < a.t.batch; base += 32) n += att_request_steps<NT>(a, att_lane_seq(a, first, base), cut);
    n = __reduce_add_sync(0xffffffffu, (uint32_t)(n & 0xffffu)) + ((uint64_t)__reduce_add_sync(0xffffffffu, (uint32_t)min(n >> 16, (uint64_t)0xffffffu)) << 16);
    n *= (uint32_t)a.c.heads;
    return n < 0x80000000ull ? (uint32_t)n : 0;
}

template <int NT>
__device__ __forceinline__ AttCut att_cut(const AttArgs &a, const KvSeq &first) {
    AttCut cut{0, 0, false};
    cut.total = att_total<NT>(a, first, cut);
    cut.per = fastdiv(cut.total + a.grid - 1, a.by_grid);
    if (cut.per <= kAttMinPiece) {
        cut.per = kAttMinPiece;
        cut.padded = true;
        cut.total = att_total<NT>(a, first, cut);
    }
    return cut;
}

struct AttItem {
    KvSeq s;
    int b, tile, head;
    uint32_t begin, steps, span;  // first step on the line; real steps; places on the line
};

// The item that holds position `pos` of the line.
template <int NT>
__device__ __forceinline__ AttItem att_find(const AttArgs &a, const AttCut &cut, const KvSeq &first, uint32_t pos) {
    AttItem it = {};
    const uint32_t heads = (uint32_t)a.c.heads;
    it.b = kv_locate(a.t, a.capacity, first, pos, [&](const KvSeq &q) { return att_request_steps<NT>(a, q, cut) * heads; }, it.s, it.begin);
    const int tiles = it.b < 0 ? 0 : att_tiles<NT>(a, it.s);
    for (it.tile = 0; it.tile < tiles; ++it.tile) {
        it.steps = att_steps<NT>(a, it.s, it.tile);
        it.span = att_span(cut, it.steps);
        if (pos < it.begin + it.span * heads) break;
        it.begin += it.span * heads;
    }
    it.head = heads == 1 || it.span == 0 ? 0 : (int)((pos - it.begin) / it.span);
    it.begin += it.head * it.span;
    return it;
}

// The item behind `it` on the line.
template <int NT>
__device__ __forceinline__ void att_next(const AttArgs &a, const AttCut &cut, const KvSeq &first, AttItem &it) {
    it.begin += it.span;
    if (++it.head < a.c.heads) return;
    it.head = 0;
    if (++it.tile < att_tiles<NT>(a, it.s)) {
        it.steps = att_steps<NT>(a, it.s, it.tile);
        it.span = att_span(cut, it.steps);
    } else {
        it = att_find<NT>(a, cut, first, it.begin);
    }
}

// A step in shared memory: 16 key rows, then 16 value rows.  Rows are copied whole and in order, 16 bytes per lane (with a
// warp instruction spread over many rows the cache was read a quarter slower), and land where the reads below find them without
// two lanes of a phase in one bank:
//   keys: lane (g, t) reads bytes 64 h + 16 t of rows g and g + 8: odd rows have their 64-byte halves exchanged;
//   values: lane (g, t) reads D / 8 bytes at g of rows 2t, 2t + 1, 2t + 8, 2t + 9: the 16-byte pieces of a row are permuted by
//   bits 1 and 2 of its number; rows of 64 bytes are also reordered, so that rows 2t fill whole lines.
template <int D>
struct AttShape {
    static constexpr int HALVES = D / 64;              // 64-byte parts of a key row
    static constexpr int PIECES = D / 16, ROWS = 32 / PIECES;  // 16-byte pieces of a row; rows that a warp instruction copies
    static constexpr int VB = D / 8 < 16 ? D / 8 : 16; // bytes of a value row that a lane reads at once
    static constexpr int VP = D / 8 / VB;              // such reads per row
    static constexpr int STAGE = 16 * D * 2;           // bytes of a step
    static constexpr int STAGES = D == 64 ? 6 : D == 128 ? 4 : 2;  // an even number: two steps are computed at a time
    static __device__ __forceinline__ uint32_t key_at(int row, int piece) { return row * D + (piece ^ (D == 64 ? 0 : (row & 1) << 2)) * 16; }
    static __device__ __forceinline__ uint32_t value_at(int row, int piece) {
        if (D == 64) return ((row & ~3) | (row & 1) << 1 | (row >> 1 & 1)) * 64 + (piece ^ (row >> 1 & 2)) * 16;
        return row * D + (piece ^ (row & 6)) * 16;
    }
};

// two codes in the low (H = 0) or high half of a word -> f16x2
template <bool INT8, int H>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
    if constexpr (INT8) return sub2<CTB_F16>(__byte_perm(w, 0x64646464u, H ? 0x4342 : 0x4140), 0x64806480u);  // 1024 + (code ^ 128) - 1152
    else return f16x2_from_e4m3x2<H>(w);
}
template <bool INT8>
__device__ __forceinline__ uint32_t code_word(uint32_t w) {
    return INT8 ? w ^ 0x80808080u : w;
}

// Rows in front of the first request and behind the last one: zeros.
template <int DT, int D, int THREADS>
__device__ __forceinline__ void att_idle_rows(const AttArgs &a) {
    const int64_t lo = a.t.batch > 0 ? min(max((int64_t)a.t.query_start[0], (int64_t)0), a.t.tokens) : 0;
    const int64_t hi = a.t.batch > 0 ? min(max((int64_t)a.t.query_start[a.t.batch], lo), a.t.tokens) : 0;
    for (int64_t i = blockIdx.x; i < lo + a.t.tokens - hi; i += gridDim.x) {
        const int64_t row = (i < lo ? i : hi + i - lo) * a.q_heads;
        for (int j = threadIdx.x; j < a.q_heads * (D / 2); j += THREADS) store_half2<DT>((uint16_t *)a.out + row * D + 2 * j, 0.0f, 0.0f);
        for (int j = threadIdx.x; j < a.q_heads; j += THREADS) a.lse[row + j] = -INFINITY;
    }
}

// Blocks that an SM holds: what shared memory (head size 256) and registers (two row tiles at 128) leave room for.
__host__ __device__ constexpr int att_blocks(int head_dim, int nt) { return nt == 16 ? 1 : head_dim == 256 || (head_dim == 128 && nt == 2) ? 2 : 3; }

template <int DT, bool INT8, int D, int NT>
__global__ void __launch_bounds__(kAttThreads, att_blocks(D, NT)) kv_attention_kernel(const __grid_constant__ AttArgs a) {
    using S = AttShape<D>;
    constexpr int ROWS = NT * 8, MT = D / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_m[kAttWarps][ROWS], s_l[kAttWarps][ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const KvSeq first = kv_lane_seq(a.t, a.capacity, 0);
    grid_next();
    const AttCut cut = att_cut<NT>(a, first);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.pieces = (cut.total + cut.per - 1) / cut.per;
    const uint32_t ring = smem_u32(smem) + warp * (S::STAGES * S::STAGE);
    const int block_steps = a.c.block_size >> 4;
    // what this lane copies of a step: piece c of rows r, r + ROWS, ...
    const int copy_row = lane / S::PIECES, copy_piece = lane % S::PIECES;
    const int64_t k_lane = copy_row * a.c.k_token_stride + copy_piece * 16, v_lane = copy_row * a.c.v_token_stride + copy_piece * 16;

    for (uint32_t piece = blockIdx.x; (uint64_t)piece * cut.per < cut.total; piece += a.grid) {
        const uint32_t p0 = piece * cut.per, p1 = min(cut.total, p0 + cut.per);
        bool open = false;  // an item begins here and ends behind the piece
        AttItem it = att_find<NT>(a, cut, first, p0);
        for (uint32_t pos = p0; pos < p1; att_next<NT>(a, cut, first, it)) {
            if (it.b < 0 || pos - it.begin >= it.span) break;  // (not with row offsets in order)
            const KvSeq sq = it.s;
            const int steps = (int)it.steps, s0 = (int)(pos - it.begin), s1 = min(steps, (int)(p1 - it.begin));
            pos = min(p1, it.begin + it.span);
            if (s0 > 0 && s0 >= steps) continue;  // nothing but the end of its place is in this piece
            // this warp's steps: s0 + warp, + 4, ...; what has to be known of 32 of them at a time, one per lane
            const int mine = s1 - s0 > warp ? (s1 - s0 - warp + kAttWarps - 1) / kAttWarps : 0;
            const int32_t *table = a.t.block_table + (int64_t)it.b * a.t.table_stride;
            auto look_up = [&](int j) { return j < mine ? __ldg(table + fastdiv((uint32_t)(s0 + warp + j * kAttWarps), a.block_steps)) : -1; };
            int page_next = look_up(lane);
            const int rows = sq.rows * a.group, row0 = it.tile * ROWS;
            const int last_end = kv_end(sq, min(sq.rows - 1, (int)fastdiv((uint32_t)(row0 + ROWS - 1), a.by_group)), a.causal != 0);
            const int first_end = kv_end(sq, fastdiv((uint32_t)row0, a.by_group), a.causal != 0);

            // query rows: lane (g, t) has row g of every tile of eight, elements 16 t .. 16 t + 15 of every 64
            uint4 qraw[NT][D / 32];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int r = row0 + n * 8 + g, i = (int)fastdiv((uint32_t)r, a.by_group);
                const bool in = r < rows;
                const uint16_t *qr = (const uint16_t *)a.q + (int64_t)(sq.first_row + i) * a.q_token_stride + (int64_t)(it.head * a.group + r - i * a.group) * a.q_head_stride;
#pragma unroll
                for (int k = 0; k < D / 32; ++k) qraw[n][k] = in ? __ldg((const uint4 *)(qr + (k >> 1) * 64 + t * 16 + (k & 1) * 8)) : make_uint4(0, 0, 0, 0);
            }
            // for the 32 steps that are fetched, then for those that are computed: key and value scale; which blocks exist
            float ks_next = 0.0f, vs_next = 1.0f, ks = 0.0f, lv = 0.0f, iv = 0.0f;
            uint32_t ok_next = 0, ok = 0, some = 0;
            const int pairs = (mine + 1) & ~1;  // two steps at a time; a missing second one reads as zeros and is masked
            int issued = 0;
            uint32_t put = 0;
            const uint8_t *k0 = (const uint8_t *)a.c.k + (int64_t)it.head * a.c.k_head_stride + k_lane;
            const uint8_t *v0 = (const uint8_t *)a.c.v + (int64_t)it.head * a.c.v_head_stride + v_lane;
            int64_t k_at = 0, v_at = 0;  // of this lane's step
            auto fetch = [&]() {
                if (issued < pairs) {
                    if ((issued & 31) == 0) {
                        const bool there = (uint32_t)page_next < (uint32_t)a.c.num_blocks;  // (a number below zero is a large one)
                        ok_next = __ballot_sync(0xffffffffu, there);
                        const int64_t page = there ? page_next : 0;
                        const uint32_t step = s0 + warp + (issued + lane) * kAttWarps;
                        const int slot = (int)(step - fastdiv(step, a.block_steps) * block_steps) * 16;
                        k_at = page * a.c.k_block_stride + slot * a.c.k_token_stride;
                        v_at = page * a.c.v_block_stride + slot * a.c.v_token_stride;
                        ks_next = __ldg(a.c.k_scale + page * a.c.heads + it.head);
                        vs_next = __ldg(a.c.v_scale + page * a.c.heads + it.head);
                        page_next = look_up(issued + 32 + lane);
                    }
                    const uint8_t *kp = k0 + __shfl_sync(0xffffffffu, k_at, issued & 31), *vp = v0 + __shfl_sync(0xffffffffu, v_at, issued & 31);
                    // tokens of the step that any row sees; the others read as zeros
                    const int seen = (ok_next >> (issued & 31)) & 1 ? last_end - (s0 + warp + issued * kAttWarps) * 16 : 0;
                    const int64_t kr = S::ROWS * a.c.k_token_stride, vr = S::ROWS * a.c.v_token_stride;
                    const uint32_t dst = ring + put, vdst = dst + 16 * D;
                    if (seen >= 16) {
#pragma unroll
                        for (int r = 0; r < 16; r += S::ROWS) {
                            cp_async16(dst + S::key_at(copy_row + r, copy_piece), kp);
                            kp += kr;
                        }
#pragma unroll
                        for (int r = 0; r < 16; r += S::ROWS) {
                            cp_async16(vdst + S::value_at(copy_row + r, copy_piece), vp);
                            vp += vr;
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; r += S::ROWS) {
                            const int n = copy_row + r < seen ? 16 : 0;
                            cp_async16_some(dst + S::key_at(copy_row + r, copy_piece), kp, n);
                            cp_async16_some(vdst + S::value_at(copy_row + r, copy_piece), vp, n);
                            kp += kr;
                            vp += vr;
                        }
                    }
                }
                ++issued;
                put = put == (S::STAGES - 1) * S::STAGE ? 0 : put + S::STAGE;
                cp_async_commit();
            };
#pragma unroll 1
            for (int i = 0; i < S::STAGES; ++i) fetch();

            uint32_t qf[NT][D / 16][2];
            float f[NT][2];   // score factors of rows 2t, 2t + 1: softmax scale * log2 e * the row's power of two
            int end[NT][2];   // positions that rows 2t, 2t + 1 see
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t most = 0;
#pragma unroll
                for (int k = 0; k < D / 32; ++k)
                    most = max2_nan<DT>(most, max2_nan<DT>(max2_nan<DT>(qraw[n][k].x & 0x7fff7fffu, qraw[n][k].y & 0x7fff7fffu),
                                                           max2_nan<DT>(qraw[n][k].z & 0x7fff7fffu, qraw[n][k].w & 0x7fff7fffu)));
                most = max2_nan<DT>(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = max2_nan<DT>(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const float top = half_f32<DT>(max(most & 0xffffu, most >> 16));
                const int e = max((int)(__float_as_uint(top) >> 23), 8);
                const float up = __uint_as_float((uint32_t)(261 - e) << 23);  // the largest element comes to [128, 256)
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {  // k = 4 h + i: elements 16 t + 4 i .. + 3 of half h
                    const uint4 v = qraw[n][k >> 1];
                    const uint32_t x0 = k & 1 ? v.z : v.x, x1 = k & 1 ? v.w : v.y;
                    qf[n][k][0] = pack_f16x2(half_f32<DT>(x0 & 0xffffu) * up, half_f32<DT>(x0 >> 16) * up);
                    qf[n][k][1] = pack_f16x2(half_f32<DT>(x1 & 0xffffu) * up, half_f32<DT>(x1 >> 16) * up);
                }
                const float own = a.scale_log2 * __uint_as_float((uint32_t)max(e - 7, 1) << 23);
#pragma unroll
                for (int i = 0; i < 2; ++i) {  // lane 4 (2t + i) has row 2t + i
                    f[n][i] = __shfl_sync(0xffffffffu, own, (2 * t + i) * 4);
                    const int rr = row0 + n * 8 + 2 * t + i;
                    end[n][i] = rr < rows ? kv_end(sq, fastdiv((uint32_t)rr, a.by_group), a.causal != 0) : 0;
                }
            }

            float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                m[n][0] = m[n][1] = -3.402823466e38f;
                l[n][0] = l[n][1] = 0.0f;
#pragma unroll
                for (int j = 0; j < MT; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
            }

            uint32_t get = 0;
            for (int j = 0; j < pairs; j += 2) {
                if ((j & 31) == 0) {  // (those after these are looked up later than this)
                    // a zero scale has no logarithm: 2^-120 stands for it in the weights, and the values of its block are left out
                    const float vsafe = vs_next < 0x1p-120f ? 0x1p-120f : vs_next;
                    some = __ballot_sync(0xffffffffu, vs_next != 0.0f);
                    ks = ks_next, ok = ok_next, lv = log2f(vsafe), iv = 1.0f / vsafe;
                }
                cp_async_wait<S::STAGES - 2>();
                __syncwarp();
                const uint8_t *st0 = smem + warp * (S::STAGES * S::STAGE) + get;
                float sc[2][NT][4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint8_t *st = st0 + u * S::STAGE;
#pragma unroll
                    for (int h = 0; h < S::HALVES; ++h) {
                        const uint32_t at = S::key_at(g, 4 * h + t);
                        const uint4 ka = *(const uint4 *)(st + at), kb = *(const uint4 *)(st + at + 8 * D);
                        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t xa = code_word<INT8>(wa[i]), xb = code_word<INT8>(wb[i]);
                            const uint32_t a0 = code_pair<INT8, 0>(xa), a1 = code_pair<INT8, 0>(xb), a2 = code_pair<INT8, 1>(xa), a3 = code_pair<INT8, 1>(xb);
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                if (h == 0 && i == 0) mma16816_first<CTB_F16>(sc[u][n], a0, a1, a2, a3, qf[n][0][0], qf[n][0][1]);
                                else mma16816<CTB_F16>(sc[u][n], a0, a1, a2, a3, qf[n][h * 4 + i][0], qf[n][h * 4 + i][1]);
                            }
                        }
                    }
                }
                bool over = false;
                float ivj[2];
                uint32_t keep[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float ksj = __shfl_sync(0xffffffffu, ks, (j & 31) + u), lvj = __shfl_sync(0xffffffffu, lv, (j & 31) + u);
                    ivj[u] = __shfl_sync(0xffffffffu, iv, (j & 31) + u);
                    const bool there = (ok >> ((j & 31) + u)) & 1;
                    keep[u] = (some >> ((j & 31) + u)) & 1 ? 0xffffffffu : 0;
                    const int tok = (s0 + warp + (j + u) * kAttWarps) * 16;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[u][n][i] = fmaf(sc[u][n][i], ksj * f[n][i & 1], lvj);
                        if (tok + 16 > first_end || !there) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (!there || tok + g + (i >> 1) * 8 >= end[n][i & 1]) sc[u][n][i] = -INFINITY;
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) over |= sc[u][n][i] > m[n][i & 1] + 8.0f;
                    }
                }
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float x = fmaxf(fmaxf(sc[0][n][i], sc[0][n][i + 2]), fmaxf(sc[1][n][i], sc[1][n][i + 2]));
#pragma unroll
                            for (int s = 4; s < 32; s <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, s));
                            const float mn = fmaxf(m[n][i], x), down = ex2(m[n][i] - mn);
                            m[n][i] = mn;
                            l[n][i] *= down;
#pragma unroll
                            for (int k = 0; k < MT; ++k) {
                                o[n][k][i] *= down;
                                o[n][k][i + 2] *= down;
                            }
                        }
                }
                uint32_t pb[2][NT][2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            sc[u][n][i] = ex2(sc[u][n][i] - m[n][i & 1]);
                            l[n][i & 1] = fmaf(sc[u][n][i], ivj[u], l[n][i & 1]);
                        }
                        pb[u][n][0] = movmatrix_trans(pack_f16x2(sc[u][n][0], sc[u][n][1]) & keep[u]);
                        pb[u][n][1] = movmatrix_trans(pack_f16x2(sc[u][n][2], sc[u][n][3]) & keep[u]);
                    }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint8_t *sv = st0 + u * S::STAGE + 16 * D;
#pragma unroll
                    for (int c = 0; c < S::VP; ++c) {
                        uint32_t v[4][S::VB / 4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int row = 2 * t + (r & 1) + (r >> 1) * 8;
                            if constexpr (S::VB == 16) {
                                const uint4 x = *(const uint4 *)(sv + S::value_at(row, 8 * c + g));
                                v[r][0] = code_word<INT8>(x.x), v[r][1] = code_word<INT8>(x.y), v[r][2] = code_word<INT8>(x.z), v[r][3] = code_word<INT8>(x.w);
                            } else {
                                const uint2 x = *(const uint2 *)(sv + S::value_at(row, g >> 1) + (g & 1) * 8);
                                v[r][0] = code_word<INT8>(x.x), v[r][1] = code_word<INT8>(x.y);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < S::VB / 2; ++k) {  // d = 2k and 2k + 1 of the lane's bytes are rows g and g + 8 of a tile
                            const uint32_t sel = k & 1 ? 0x7362 : 0x5140;
                            const uint32_t x = __byte_perm(v[0][k >> 1], v[1][k >> 1], sel), y = __byte_perm(v[2][k >> 1], v[3][k >> 1], sel);
                            const uint32_t a0 = code_pair<INT8, 0>(x), a1 = code_pair<INT8, 1>(x), a2 = code_pair<INT8, 0>(y), a3 = code_pair<INT8, 1>(y);
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma16816<CTB_F16>(o[n][c * (S::VB / 2) + k], a0, a1, a2, a3, pb[u][n][0], pb[u][n][1]);
                        }
                    }
                }
                get = get == (S::STAGES - 2) * S::STAGE ? 0 : get + 2 * S::STAGE;
                __syncwarp();
                fetch();
                fetch();
            }
            cp_async_wait<0>();

            // the four warps' results: sums over the lanes of a row, then over the warps in order
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int s = 4; s < 32; s <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], s);
                    if (g == 0) {
                        s_m[warp][n * 8 + 2 * t + i] = m[n][i];
                        s_l[warp][n * 8 + 2 * t + i] = l[n][i];
                    }
                }
            __syncthreads();  // (every ring is idle from here on: the sums go where it was)
            float *so = reinterpret_cast<float *>(smem);
            constexpr int OS = D + 4;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = n * 8 + 2 * t + i;
                    float top = s_m[0][r];
#pragma unroll
                    for (int w = 1; w < kAttWarps; ++w) top = fmaxf(top, s_m[w][r]);
                    const float down = ex2(m[n][i] - top);
                    float *row = so + ((size_t)warp * ROWS + r) * OS;
#pragma unroll
                    for (int c = 0; c < S::VP; ++c)
#pragma unroll
                        for (int k = 0; k < S::VB / 2; ++k) {
                            const float(&x)[4] = o[n][c * (S::VB / 2) + k];
                            *(float2 *)(row + c * 128 + g * S::VB + 2 * k) = make_float2(x[i] * down, x[i + 2] * down);
                        }
                }
            __syncthreads();
            const bool whole = s0 == 0 && s1 == steps;
            const int64_t slot = cut.padded ? piece : 2 * (int64_t)piece + (p0 < it.begin ? 1 : 0);
            float *part = a.part + slot * ROWS * (D + 2);
            for (int i = threadIdx.x; i < ROWS * (D / 2); i += kAttThreads) {
                const int r = i / (D / 2), d = (i % (D / 2)) * 2;
                if (row0 + r >= rows) break;
                float top = s_m[0][r], sum = 0.0f;
#pragma unroll
                for (int w = 1; w < kAttWarps; ++w) top = fmaxf(top, s_m[w][r]);
#pragma unroll
                for (int w = 0; w < kAttWarps; ++w) sum += s_l[w][r] * ex2(s_m[w][r] - top);
                float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kAttWarps; ++w) {
                    const float2 x = *(const float2 *)(so + ((size_t)w * ROWS + r) * OS + d);
                    v.x += x.x, v.y += x.y;
                }
                if (whole) {
                    const int qi = (int)fastdiv((uint32_t)(row0 + r), a.by_group);
                    const int64_t row = (int64_t)(sq.first_row + qi) * a.q_heads + it.head * a.group + row0 + r - qi * a.group;
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // nothing seen: zeros
                    store_half2<DT>((uint16_t *)a.out + row * D + d, v.x * inv, v.y * inv);
                    if (d == 0) a.lse[row] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
                } else if (slot < a.slots) {  // (row offsets that decrease may ask for more than there are)
                    *(float2 *)(part + r * (D + 2) + d) = v;
                    if (d == 0) *(float2 *)(part + r * (D + 2) + D) = make_float2(top, sum);
                }
            }
            if (threadIdx.x == 0 && s1 < steps && it.begin >= p0 && piece < a.slots) {
                const int qi = (int)fastdiv((uint32_t)row0, a.by_group);
                a.join[piece] = AttJoin{(int64_t)(sq.first_row + qi) * a.q_heads + it.head * a.group, slot, (it.begin + (uint32_t)steps - 1) / cut.per,
                                        min(ROWS, rows - row0), row0 - qi * a.group, cut.padded};
                open = true;
            }
            __syncthreads();  // the next item's copies go where the sums are
        }
        if (threadIdx.x == 0 && !open && piece < a.slots) a.join[piece].last = 0;
    }
    att_idle_rows<DT, D, kAttThreads>(a);
}

// ---------------------------------------------------------------- many query rows per cache head (prompts)
// A row tile is 128 query rows, 16 for each of eight warps; 64 cached tokens at a time are converted to f16 once for all of them in
// shared memory and taken from there as the column operand of mma.m16n8k16 (S = Q K^T, O += P V, the weights staying in registers between
// the two).  Number formats, scales and the lazily raised maximum are those of the kernel above, and so are the line of steps,
// its pieces, and the second kernel that joins them.
//
// What bounds it: the matrix instructions (4 D operations per row and token); the codes are read and converted once per 128 rows.
// 512 queries against 4096 tokens, two requests, 32 query heads of 128: 227 us, 190 TFLOP/s, a third of what mma.sync does here.
// While a tile is computed the codes of the next one are on their way in registers, its block numbers and scales one tile ahead of that.
constexpr int kTileWarps = 8, kTileThreads = kTileWarps * 32, kTileTokens = 64;

template <int DT, bool INT8, int D>
__global__ void __launch_bounds__(kTileThreads, 1) kv_attention_tile_kernel(const __grid_constant__ AttArgs a) {
    constexpr int NT = 16, ROWS = 128, KS = D / 16, PIECES = D / 16, PASS = kTileThreads / PIECES, LOADS = kTileTokens / PASS;
    static_assert(LOADS * PASS == kTileTokens && PASS % 16 == 0, "rows that a pass of the block loads are whole steps");
    constexpr int PITCH = D * 2;  // bytes of a converted row; its 16-byte pieces are permuted by the row's low bits
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float4 s_meta[2][4];  // per step of the tile: key scale, log2 and inverse of the value scale, flags (1: there, 2: values count)
    uint8_t *sk = smem, *sv = smem + kTileTokens * PITCH;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const KvSeq first = kv_lane_seq(a.t, a.capacity, 0);
    grid_next();
    const AttCut cut = att_cut<NT>(a, first);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.pieces = (cut.total + cut.per - 1) / cut.per;
    const int block_steps = a.c.block_size >> 4, copy_row = threadIdx.x / PIECES, copy_piece = threadIdx.x % PIECES;

    for (uint32_t piece = blockIdx.x; (uint64_t)piece * cut.per < cut.total; piece += a.grid) {
        const uint32_t p0 = piece * cut.per, p1 = min(cut.total, p0 + cut.per);
        bool open = false;  // an item begins here and ends behind the piece
        AttItem it = att_find<NT>(a, cut, first, p0);
        for (uint32_t pos = p0; pos < p1; att_next<NT>(a, cut, first, it)) {
            if (it.b < 0 || pos - it.begin >= it.span) break;  // (not with row offsets in order)
            const KvSeq sq = it.s;
            const int steps = (int)it.steps, s0 = (int)(pos - it.begin), s1 = min(steps, (int)(p1 - it.begin));
            pos = min(p1, it.begin + it.span);
            if (s0 > 0 && s0 >= steps) continue;  // nothing but the end of its place is in this piece
            const int32_t *table = a.t.block_table + (int64_t)it.b * a.t.table_stride;
            const int rows = sq.rows * a.group, row0 = it.tile * ROWS;
            const int last_end = kv_end(sq, min(sq.rows - 1, (int)fastdiv((uint32_t)(row0 + ROWS - 1), a.by_group)), a.causal != 0);
            const int first_end = kv_end(sq, fastdiv((uint32_t)row0, a.by_group), a.causal != 0);

            // copies: this thread's piece of rows copy_row, + PASS, ... of a tile of four steps
            uint4 kc[LOADS], vc[LOADS];
            int page[LOADS];
            float4 next_meta = make_float4(0, 0, 0, 0);
            int meta_page = -1;
            auto block_of = [&](int step) { return step < s1 ? __ldg(table + fastdiv((uint32_t)step, a.block_steps)) : -1; };
            auto there = [&](int p) { return (uint32_t)p < (uint32_t)a.c.num_blocks; };
            auto look_up = [&](int s) {  // of the tile that begins at step s
#pragma unroll
                for (int i = 0; i < LOADS; ++i) page[i] = block_of(s + (copy_row + i * PASS) / 16);
                if (threadIdx.x < 4) meta_page = block_of(s + threadIdx.x);
            };
            auto load = [&](int s) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int row = copy_row + i * PASS, step = s + row / 16;
                    kc[i] = vc[i] = make_uint4(0, 0, 0, 0);
                    if (there(page[i]) && s * 16 + row < last_end) {  // what no row sees reads as zeros
                        const int slot = (int)((uint32_t)step - fastdiv((uint32_t)step, a.block_steps) * block_steps) * 16 + row % 16;
                        kc[i] = __ldg((const uint4 *)((const uint8_t *)a.c.k + (int64_t)page[i] * a.c.k_block_stride + (int64_t)it.head * a.c.k_head_stride + slot * a.c.k_token_stride) + copy_piece);
                        vc[i] = __ldg((const uint4 *)((const uint8_t *)a.c.v + (int64_t)page[i] * a.c.v_block_stride + (int64_t)it.head * a.c.v_head_stride + slot * a.c.v_token_stride) + copy_piece);
                    }
                }
                if (threadIdx.x < 4) {
                    const bool in = there(meta_page);
                    next_meta.x = in ? __ldg(a.c.k_scale + (int64_t)meta_page * a.c.heads + it.head) : 0.0f;
                    next_meta.y = in ? __ldg(a.c.v_scale + (int64_t)meta_page * a.c.heads + it.head) : 1.0f;
                    next_meta.w = __int_as_float(in ? 1 : 0);
                }
            };
            if (s0 < s1) {
                look_up(s0);
                load(s0);
                look_up(s0 + 4);
            }

            // query rows 16 warp + g and + 8: row operand, elements 2t, 2t + 1 and 2t + 8, 2t + 9 of every 16
            uint32_t qf[KS][4];
            float f[2];   // score factors
            int end[2];   // positions seen
            const bool busy = row0 + warp * 16 < rows;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = row0 + warp * 16 + g + 8 * h, qi = (int)fastdiv((uint32_t)r, a.by_group);
                const bool in = r < rows;
                const uint32_t *qr = (const uint32_t *)((const uint16_t *)a.q + (int64_t)(sq.first_row + (in ? qi : 0)) * a.q_token_stride +
                                                        (int64_t)(it.head * a.group + (in ? r - qi * a.group : 0)) * a.q_head_stride);
                uint32_t most = 0;
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t v = in ? __ldg(qr + k * 8 + t + 4 * j) : 0;
                        qf[k][h + 2 * j] = v;
                        most = max2_nan<DT>(most, v & 0x7fff7fffu);
                    }
                most = max2_nan<DT>(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = max2_nan<DT>(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const float top = half_f32<DT>(max(most & 0xffffu, most >> 16));
                const int e = max((int)(__float_as_uint(top) >> 23), 8);
                const float up = __uint_as_float((uint32_t)(261 - e) << 23);  // the largest element comes to [128, 256)
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t v = qf[k][h + 2 * j];
                        qf[k][h + 2 * j] = pack_f16x2(half_f32<DT>(v & 0xffffu) * up, half_f32<DT>(v >> 16) * up);
                    }
                f[h] = a.scale_log2 * __uint_as_float((uint32_t)max(e - 7, 1) << 23);
                end[h] = in ? kv_end(sq, qi, a.causal != 0) : 0;
            }

            float o[D / 8][4], m[2] = {-3.402823466e38f, -3.402823466e38f}, l[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;

            int buf = 0;
            for (int s = s0; s < s1; s += 4, buf ^= 1) {
                __syncthreads();  // the tile before has been read
                // eight codes -> eight f16 in order
                auto spread = [](uint32_t x, uint32_t y) {
                    const uint32_t u = code_word<INT8>(x), v = code_word<INT8>(y);
                    return make_uint4(code_pair<INT8, 0>(u), code_pair<INT8, 1>(u), code_pair<INT8, 0>(v), code_pair<INT8, 1>(v));
                };
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int row = copy_row + i * PASS, x = row & 7;
                    uint8_t *kr = sk + row * PITCH, *vr = sv + row * PITCH;
                    *(uint4 *)(kr + (((2 * copy_piece) ^ x) << 4)) = spread(kc[i].x, kc[i].y);
                    *(uint4 *)(kr + (((2 * copy_piece + 1) ^ x) << 4)) = spread(kc[i].z, kc[i].w);
                    *(uint4 *)(vr + (((2 * copy_piece) ^ x) << 4)) = spread(vc[i].x, vc[i].y);
                    *(uint4 *)(vr + (((2 * copy_piece + 1) ^ x) << 4)) = spread(vc[i].z, vc[i].w);
                }
                if (threadIdx.x < 4) {
                    const float vs = next_meta.y, vsafe = vs < 0x1p-120f ? 0x1p-120f : vs;  // as in the kernel above
                    s_meta[buf][threadIdx.x] = make_float4(next_meta.x, log2f(vsafe), 1.0f / vsafe, __int_as_float(__float_as_int(next_meta.w) | (vs != 0.0f ? 2 : 0)));
                }
                if (s + 4 < s1) {
                    load(s + 4);
                    look_up(s + 8);
                }
                __syncthreads();
                if (!busy) continue;
                // scores of 16 rows x 64 tokens
                float sc[8][4];
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {  // 16 tokens: two column tiles
                        uint32_t b[4];
                        const int row = j * 16 + (lane & 7) + ((lane >> 4) << 3);
                        ldmatrix4(b, smem_u32(sk + row * PITCH + (((2 * k + ((lane >> 3) & 1)) ^ (row & 7)) << 4)));
                        if (k == 0) {
                            mma16816_first<CTB_F16>(sc[2 * j], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[0], b[1]);
                            mma16816_first<CTB_F16>(sc[2 * j + 1], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[2], b[3]);
                        } else {
                            mma16816<CTB_F16>(sc[2 * j], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[0], b[1]);
                            mma16816<CTB_F16>(sc[2 * j + 1], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[2], b[3]);
                        }
                    }
                bool over = false;
                float iv[4];
                uint32_t keep[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 mt = s_meta[buf][j];
                    const int flags = __float_as_int(mt.w), tok = (s + j) * 16;
                    iv[j] = mt.z;
                    keep[j] = flags & 2 ? 0xffffffffu : 0;
                    const bool mask = !(flags & 1) || tok + 16 > first_end;
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float &x = sc[2 * j + c][i];
                            x = fmaf(x, mt.x * f[i >> 1], mt.y);
                            if (mask && (!(flags & 1) || tok + c * 8 + 2 * t + (i & 1) >= end[i >> 1])) x = -INFINITY;
                            over |= x > m[i >> 1] + 8.0f;
                        }
                }
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x = -INFINITY;
#pragma unroll
                        for (int c = 0; c < 8; ++c) x = fmaxf(x, fmaxf(sc[c][2 * h], sc[c][2 * h + 1]));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                        const float mn = fmaxf(m[h], x), down = ex2(m[h] - mn);
                        m[h] = mn;
                        l[h] *= down;
#pragma unroll
                        for (int j = 0; j < D / 8; ++j) {
                            o[j][2 * h] *= down;
                            o[j][2 * h + 1] *= down;
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // 16 tokens of weights: the row operand of the second product
                    uint32_t p[4];
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float x = ex2(sc[2 * j + c][2 * h] - m[h]), y = ex2(sc[2 * j + c][2 * h + 1] - m[h]);
                            l[h] = fmaf(x + y, iv[j], l[h]);
                            p[2 * c + h] = pack_f16x2(x, y) & keep[j];
                        }
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        uint32_t b[4];
                        const int row = j * 16 + (lane & 15);
                        ldmatrix4_trans(b, smem_u32(sv + row * PITCH + (((2 * d + (lane >> 4)) ^ (row & 7)) << 4)));
                        mma16816<CTB_F16>(o[2 * d], p[0], p[1], p[2], p[3], b[0], b[1]);
                        mma16816<CTB_F16>(o[2 * d + 1], p[0], p[1], p[2], p[3], b[2], b[3]);
                    }
                }
            }

            const bool whole = s0 == 0 && s1 == steps;
            const int64_t slot = cut.padded ? piece : 2 * (int64_t)piece + (p0 < it.begin ? 1 : 0);
            float *part = a.part + slot * ROWS * (D + 2);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                const int r = warp * 16 + g + 8 * h, qi = (int)fastdiv((uint32_t)(row0 + r), a.by_group);
                if (row0 + r >= rows) continue;
                if (whole) {
                    const int64_t row = (int64_t)(sq.first_row + qi) * a.q_heads + it.head * a.group + row0 + r - qi * a.group;
                    const float inv = l[h] == 0.0f ? 0.0f : 1.0f / l[h];  // nothing seen: zeros
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) store_half2<DT>((uint16_t *)a.out + row * D + j * 8 + 2 * t, o[j][2 * h] * inv, o[j][2 * h + 1] * inv);
                    if (t == 0) a.lse[row] = l[h] == 0.0f ? -INFINITY : (m[h] + log2f(l[h])) * 0.6931471805599453f;
                } else if (slot < a.slots) {
                    float *pr = part + r * (D + 2);
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) *(float2 *)(pr + j * 8 + 2 * t) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
                    if (t == 0) *(float2 *)(pr + D) = make_float2(m[h], l[h]);
                }
            }
            if (threadIdx.x == 0 && s1 < steps && it.begin >= p0 && piece < a.slots) {
                const int qi = (int)fastdiv((uint32_t)row0, a.by_group);
                a.join[piece] = AttJoin{(int64_t)(sq.first_row + qi) * a.q_heads + it.head * a.group, slot, (it.begin + (uint32_t)steps - 1) / cut.per,
                                        min(ROWS, rows - row0), row0 - qi * a.group, cut.padded};
                open = true;
            }
        }
        if (threadIdx.x == 0 && !open && piece < a.slots) a.join[piece].last = 0;
    }
    att_idle_rows<DT, D, kTileThreads>(a);
}

// Joins what the pieces of an item left in scratch: block c takes the item that begins in piece c and ends behind it.
constexpr int kJoinWarps = 16;

template <int DT, int D, int NT>
__global__ void __launch_bounds__(kJoinWarps * 32) kv_attention_join_kernel(const __grid_constant__ AttArgs a) {
    constexpr int ROWS = NT * 8, E = D / 32, B = D == 256 ? 2 : 4;  // B: pieces in flight per warp
    __shared__ float s_v[kJoinWarps][D], s_top[kJoinWarps], s_sum[kJoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_wait();
    const uint32_t pieces = (uint32_t)min((int64_t)__ldcg(a.pieces), a.slots);
    for (uint32_t c0 = blockIdx.x; c0 < pieces; c0 += 32 * gridDim.x)
      for (uint32_t todo = __ballot_sync(0xffffffffu, c0 + lane * gridDim.x < pieces && __ldcg(&a.join[min(c0 + lane * gridDim.x, pieces - 1)].last) != 0); todo;
           todo &= todo - 1) {
        const uint32_t c = c0 + (__ffs(todo) - 1) * gridDim.x;
        const AttJoin it = a.join[c];
        const uint32_t last = it.last;
        const int base = blockIdx.y * kJoinWarps, n = min(it.rows - base, kJoinWarps);  // rows base .. base + n of the tile
        if (n <= 0) continue;
        // all warps on the rows: 16 / (n rounded up to a power of two) of them on each, every one with its share of the pieces
        const int log_rows = n <= 1 ? 0 : 32 - __clz(n - 1), log_warps = 4 - log_rows, r = warp & ((1 << log_rows) - 1);
        float top = -3.402823466e38f, sum = 0.0f, v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0.0f;
        if (r < n) {
            for (uint32_t p0 = c + (warp >> log_rows); p0 <= last; p0 += B << log_warps) {
                float x[B][E];
                float2 ml[B];
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    const uint32_t p = p0 + ((uint32_t)i << log_warps);
                    ml[i] = make_float2(-INFINITY, 0.0f);
#pragma unroll
                    for (int e = 0; e < E; ++e) x[i][e] = 0.0f;
                    const int64_t slot = p == c ? it.slot : it.padded ? p : 2 * (int64_t)p;
                    if (p <= last && slot < a.slots) {
                        const float *part = a.part + (slot * ROWS + base + r) * (D + 2);
                        ml[i] = __ldcg((const float2 *)(part + D));
#pragma unroll
                        for (int e = 0; e < E; e += 2) *(float2 *)&x[i][e] = __ldcg((const float2 *)(part + lane * E + e));
                    }
                }
                float mn = top;
#pragma unroll
                for (int i = 0; i < B; ++i) mn = fmaxf(mn, ml[i].x);
                const float w0 = ex2(top - mn);
                sum *= w0;
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] *= w0;
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    const float w = ex2(ml[i].x - mn);
                    sum = fmaf(ml[i].y, w, sum);
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] = fmaf(x[i][e], w, v[e]);
                }
                top = mn;
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) s_v[warp][lane * E + e] = v[e];
        if (lane == 0) s_top[warp] = top, s_sum[warp] = sum;
        __syncthreads();
        for (int i = threadIdx.x; i < n * (D / 2); i += kJoinWarps * 32) {
            const int q = i / (D / 2), d = (i % (D / 2)) * 2;
            float all = -3.402823466e38f, total = 0.0f, x0 = 0.0f, x1 = 0.0f;
            for (int w = 0; w < 1 << log_warps; ++w) all = fmaxf(all, s_top[(w << log_rows) + q]);
            for (int w = 0; w < 1 << log_warps; ++w) {
                const int k = (w << log_rows) + q;
                const float down = ex2(s_top[k] - all);
                total = fmaf(s_sum[k], down, total);
                x0 = fmaf(s_v[k][d], down, x0);
                x1 = fmaf(s_v[k][d + 1], down, x1);
            }
            const int rr = it.first + base + q, qi = (int)fastdiv((uint32_t)rr, a.by_group);
            const int64_t row = it.row + (int64_t)qi * a.q_heads + rr - qi * a.group;
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            store_half2<DT>((uint16_t *)a.out + row * D + d, x0 * inv, x1 * inv);
            if (d == 0) a.lse[row] = total == 0.0f ? -INFINITY : (all + log2f(total)) * 0.6931471805599453f;
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host side

static int64_t att_items(const ctb_kv_cache &c, const ctb_kv_batch &t, int group, int rows) {
    return (int64_t)c.heads * ((t.tokens * group + rows - 1) / rows + t.batch);  // a tile for every `rows` query rows, and one more per request
}

// Row tiles of a call, in eights: 128 rows on average from 48 rows per request on, where the conversions that the tile kernel saves
// outweigh the rows that it computes for nothing; two eights from nine rows on; head size 256 has registers for one eight only.
static int att_nt(const ctb_kv_cache &c, const ctb_kv_batch &t, int group) {
    const int64_t rows = t.tokens * group;
    if (c.head_dim == 256) return 1;
    return rows > 48 * (int64_t)t.batch ? 16 : rows > 8 * (int64_t)t.batch ? 2 : 1;
}

static int att_grid(int head_dim, int nt) { return sm_count() * att_blocks(head_dim, nt); }

bool kv_attention_takes(const ctb_kv_cache &c, const ctb_kv_batch &t, int q_heads, const void *q, int64_t q_token_stride, int64_t q_head_stride, const void *out) {
    const int64_t strides = c.k_block_stride | c.k_head_stride | c.k_token_stride | c.v_block_stride | c.v_head_stride | c.v_token_stride;
    return (c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256) && c.num_blocks > 0 && c.block_size % 16 == 0 && strides % 16 == 0 && aligned16(c.k) && aligned16(c.v) &&
           // positions on the line of steps are 32-bit numbers
           (double)att_items(c, t, q_heads / c.heads, 8) * ((double)t.table_width * c.block_size / 16 + 16) < 2147483648.0 &&
           aligned16(q) && (q_token_stride | q_head_stride) % 8 == 0 && ((uintptr_t)out & 3) == 0;
}

// Scratch: 32 bytes, what is to be joined, the parts.  A slot per short item, two per piece of a long line.
static int64_t att_slots(const ctb_kv_cache &c, const ctb_kv_batch &t, int group, int nt) {
    return att_items(c, t, group, 8 * nt) + 2 * (int64_t)att_grid(c.head_dim, nt);
}

int64_t kv_attention_workspace(const ctb_kv_cache &c, const ctb_kv_batch &t, int q_heads) {
    const int group = q_heads / c.heads, nt = att_nt(c, t, group);
    return 32 + att_slots(c, t, group, nt) * ((int64_t)sizeof(AttJoin) + 8 * nt * (c.head_dim + 2) * 4);
}

template <int DT, int D, int NT>
static int att_finish(const AttArgs &a, cudaStream_t st) {
    // no request is longer than the shortest piece, and so few that the line is a padded one: nothing to join
    if (a.capacity <= kAttMinPiece * 16 && att_items(a.c, a.t, a.group, NT * 8) * (kAttMinPiece + (int)kAttItemSteps) <= (int64_t)kAttMinPiece * a.grid) return CTB_OK;
    return launch_dependent("kv_attention_join_kernel", kv_attention_join_kernel<DT, D, NT>, dim3((unsigned)sm_count(), (NT * 8 + kJoinWarps - 1) / kJoinWarps),
                            kJoinWarps * 32, 0, st, a);
}

template <int DT, bool INT8, int D, int NT>
static int att_launch(const AttArgs &a, cudaStream_t st) {
    auto kernel = kv_attention_kernel<DT, INT8, D, NT>;
    constexpr size_t ring = (size_t)kAttWarps * AttShape<D>::STAGES * AttShape<D>::STAGE, sums = (size_t)kAttWarps * NT * 8 * (D + 4) * 4;
    constexpr size_t bytes = ring > sums ? ring : sums;
    static std::atomic<bool> ready[64];
    int rc = allow_smem(kernel, bytes, ready);
    if (rc) return rc;
    kernel<<<a.grid, kAttThreads, bytes, st>>>(a);
    rc = after_launch("kv_attention_kernel");
    return rc ? rc : att_finish<DT, D, NT>(a, st);
}

template <int DT, bool INT8, int D>
static int att_tile_launch(const AttArgs &a, cudaStream_t st) {
    auto kernel = kv_attention_tile_kernel<DT, INT8, D>;
    constexpr size_t bytes = (size_t)2 * kTileTokens * D * 2;
    static std::atomic<bool> ready[64];
    int rc = allow_smem(kernel, bytes, ready);
    if (rc) return rc;
    kernel<<<a.grid, kTileThreads, bytes, st>>>(a);
    rc = after_launch("kv_attention_tile_kernel");
    return rc ? rc : att_finish<DT, D, 16>(a, st);
}

int kv_attention_launch(const ctb_kv_cache &c, const ctb_kv_batch &t, const void *q, int dtype, int64_t q_token_stride, int64_t q_head_stride, int q_heads,
                        float softmax_scale, int causal, void *out, float *lse, void *workspace, cudaStream_t st) {
    const int group = q_heads / c.heads, nt = att_nt(c, t, group);
    AttArgs a;
    a.c = c;
    a.t = t;
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.slots = att_slots(c, t, group, nt);
    a.pieces = (uint32_t *)workspace;
    a.join = (AttJoin *)((char *)workspace + 32);
    a.part = (float *)(a.join + a.slots);
    a.q_token_stride = q_token_stride;
    a.q_head_stride = q_head_stride;
    a.scale_log2 = softmax_scale * 1.4426950408889634f;
    a.capacity = t.table_width * c.block_size;
    a.grid = att_grid(c.head_dim, nt);
    a.block_steps = make_fastdiv((uint32_t)(c.block_size / 16));
    a.by_group = make_fastdiv((uint32_t)group);
    a.by_grid = make_fastdiv((uint32_t)a.grid);
    a.q_heads = q_heads;
    a.group = group;
    a.causal = causal;
    auto go = [&](auto dt, auto i8) {
        constexpr int DT = decltype(dt)::value;
        constexpr bool I8 = decltype(i8)::value;
        if (nt == 16) return c.head_dim == 64 ? att_tile_launch<DT, I8, 64>(a, st) : att_tile_launch<DT, I8, 128>(a, st);
        if (c.head_dim == 64) return nt == 1 ? att_launch<DT, I8, 64, 1>(a, st) : att_launch<DT, I8, 64, 2>(a, st);
        if (c.head_dim == 128) return nt == 1 ? att_launch<DT, I8, 128, 1>(a, st) : att_launch<DT, I8, 128, 2>(a, st);
        return att_launch<DT, I8, 256, 1>(a, st);
    };
    using B = std::integral_constant<int, CTB_BF16>;
    using H = std::integral_constant<int, CTB_F16>;
    if (dtype == CTB_BF16) return c.dtype == CTB_I8 ? go(B{}, std::true_type{}) : go(B{}, std::false_type{});
    return c.dtype == CTB_I8 ? go(H{}, std::true_type{}) : go(H{}, std::false_type{});
}

}  // namespace ctb
