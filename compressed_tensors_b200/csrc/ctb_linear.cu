// Product with a 4-bit weight: out[t][n] = sum_k x[t][k] * (code[n][k] - zp) * scale (+ bias[n]), for few tokens.
//
// What bounds it: a weight code is used once per token, so at a few tokens the call takes the time of reading the
// packed weight (half a byte per weight) from HBM.  128256 x 4096 by one token: 60 us, 4.5 TB/s of weight; 14336 x 4096: 13 us by one
// token, 15 by 8, 19 by 16, 36 by 32; below about 30 MB the ramp and the instructions (about 170 per 2048 weights and warp) show.
#include <atomic>

#include "ctb_fastdiv.h"
#include "ctb_mma.cuh"

namespace ctb {

struct LinearArgs {
    const void *x, *q, *scale, *bias;
    const int8_t *zp;
    const float *gs;
    void *out;
    int64_t tokens, rows, cols;      // x [tokens, cols], weight [rows, cols], out [tokens, rows]
    int64_t q_row_bytes;             // bytes of one packed row
    int64_t col_group, scale_row_stride;
    int32_t scale_dtype;
};

__device__ __forceinline__ float e2m1_to_f32(uint32_t code) {
    const uint32_t m = code & 7u;  // 0, .5, 1, 1.5, 2, 3, 4, 6: exponent field m >> 1 with bias 1, one fraction bit
    const float v = m < 2 ? 0.5f * (float)m : __uint_as_float(((126u + (m >> 1)) << 23) | ((m & 1u) << 22));
    return code & 8u ? -v : v;
}

// ---------------------------------------------------------------- any sizes
// A warp takes one weight row and up to 8 tokens; a lane takes every 32nd byte of the row (two codes).
template <int DT, bool FP4>
__global__ void __launch_bounds__(256) linear4_any_kernel(const LinearArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (n >= a.rows) return;
    const int64_t t0 = (int64_t)blockIdx.y * 8;
    const int nt = (int)(a.tokens - t0 < 8 ? a.tokens - t0 : 8);
    const uint8_t *row = (const uint8_t *)a.q + n * a.q_row_bytes;
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int64_t k = 2 * lane; k < a.cols; k += 64) {
        const uint32_t b = row[k >> 1];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t c = k + h;
            if (c >= a.cols) break;
            const int64_t si = n * a.scale_row_stride + c / a.col_group;
            const uint32_t code = (b >> (4 * h)) & 15u;
            float w = FP4 ? e2m1_to_f32(code) : (float)((int)code - 8 - (a.zp ? (int)a.zp[si] : 0));
            w *= load_f32(a.scale, a.scale_dtype, si);
#pragma unroll
            for (int t = 0; t < 8; ++t)
                if (t < nt) acc[t] = fmaf(load_f32(a.x, DT, (t0 + t) * a.cols + c), w, acc[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
        float v = acc[t];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0 && t < nt) {
            if (FP4 && a.gs) v = __fdiv_rn(v, *a.gs);
            if (a.bias) v += load_f32(a.bias, DT, n);
            store_f32(a.out, DT, (t0 + t) * a.rows + n, v);
        }
    }
}

// ---------------------------------------------------------------- few tokens, 16-byte rows
// The weight is the 16-row operand of mma.m16n8k16 and the tokens are its 8 columns, so a packed word becomes operand
// registers with a shift, a mask and one exact 16-bit subtraction per two codes, and no weight is ever rounded:
//   int4   (w >> 4i) & 0x000f000f is codes i and i + 4; with 0x4300 (bf16) or 0x6400 (f16) above them they read 128 + c or
//          1024 + c, and 136 + zp or 1032 + zp is subtracted.  The products of a scale group are summed by the tensor
//          core in fp32 and multiplied by the fp32 scale once per group.
//   NVFP4  the three magnitude bits moved to where exponent and fraction meet read value * 2^-126 (bf16) or 2^-14 (f16);
//          times scale * 2^118 or scale * 2^7 they are value * scale * 2^-8 or 2^-7 exactly (2 + 4 significant bits).
// The order of k inside a product is free as long as both operands share it: the activations are stored in the order in
// which the codes leave the word (0 4 1 5 2 6 3 7).
//
// A block takes WARPS * 16 rows and one share of the columns; the blocks of a cluster take the shares of the same
// rows and add their sums through distributed shared memory, in rank order.  Every warp streams its 16 rows through a ring
// of its own (cp.async, 2 KB for 256 columns, swizzled for ldmatrix), so there is no block barrier in the loop and
// 2 * kLinStages KB per warp are in flight.
constexpr int kLinStages = 3;
constexpr int kLinXBytes = 64 * 1024;  // activations held at a time

template <int DT, bool FP4>
struct Code4 {
    static __device__ __forceinline__ uint32_t pair(uint32_t w, int i, uint32_t k) {
        if constexpr (!FP4) {
            return sub2<DT>(and_or(w >> (4 * i), 0x000f000fu, DT == CTB_BF16 ? 0x43004300u : 0x64006400u), k);
        } else {
            constexpr int M = DT == CTB_BF16 ? 6 : 9;  // bit that the fraction bit of the code goes to
            constexpr uint32_t mask = 0x00070007u << M;
            const uint32_t mag = (4 * i <= M ? w << (M - 4 * i) : w >> (4 * i - M)) & mask;
            return mul2<DT>(and_or(w << (12 - 4 * i), 0x80008000u, mag), k);
        }
    }
};

struct LinearPlan {
    int log_shares;  // blocks of a cluster, 1 << log_shares: shares of the columns
    int x_cols;      // columns of activations held at a time, a multiple of 256
    FastDiv group;   // columns, in units of 128 / NS -> scale group
};

// NS: scales per 128 columns and row (1: groups are multiples of 128; 4: multiples of 32); FP4: 8, four of them a lane's
// SB: bytes of a scale
template <int DT, bool FP4, bool ZP, int NS, int SB, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) linear4_mma_kernel(const __grid_constant__ LinearArgs a, const LinearPlan p) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int ROWS = WARPS * 16, TOK = NT * 8, RING = kLinStages * 2048;
    uint8_t *xs = smem + WARPS * RING;
    const int xstride = p.x_cols * 2 + 64;  // 64 mod 128: the 8 lanes of a phase hit 8 groups of banks
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * RING;
    const int shares = 1 << p.log_shares, share = blockIdx.x & (shares - 1);
    const int64_t row0 = (int64_t)(blockIdx.x >> p.log_shares) * ROWS + warp * 16;
    const int64_t t0 = (int64_t)blockIdx.y * TOK;
    const int nt = (int)(a.tokens - t0 < TOK ? a.tokens - t0 : TOK);
    const int cols = (int)a.cols, units = (cols + 255) / 256;
    const int u0 = (units * share) >> p.log_shares, u1 = (units * (share + 1)) >> p.log_shares;

    // activations of columns [x0, x1) * 256: every thread's pieces of eight
    auto each_x = [&](int x0, int x1, auto &&f) {
        for (int m = 0; m < nt; ++m) {
            const uint16_t *xr = (const uint16_t *)a.x + (t0 + m) * a.cols + x0 * 256;
#pragma unroll 4
            for (int c = threadIdx.x; c < (x1 - x0) * 32; c += WARPS * 32) f(xs + m * xstride + c * 16, x0 * 256 + c * 8 < cols ? xr + c * 8 : nullptr);
        }
    };
    auto fetch_x = [&](int x0, int x1) {
        each_x(x0, x1, [&](uint8_t *at, const uint16_t *from) {
            if (from) cp_async16(smem_u32(at), from);
            else *(uint4 *)at = make_uint4(0, 0, 0, 0);
        });
        cp_async_commit();
    };
    fetch_x(u0, min(u1, u0 + p.x_cols / 256));

    // this lane's 16-byte pieces of every stage (16 rows of 128 bytes): piece lane & 7 of rows lane >> 3, + 4, + 8, + 12, so that a
    // warp instruction reads whole lines.  Pieces are permuted by the row's low bits: ldmatrix reads eight rows without a conflict.
    const int64_t row_a = row0 + g < a.rows ? row0 + g : a.rows - 1;  // rows behind the last one: read again, dropped at the end
    const int64_t row_b = row0 + g + 8 < a.rows ? row0 + g + 8 : a.rows - 1;
    const uint8_t *src[4];
    uint32_t dst[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = (lane >> 3) + 4 * i;
        src[i] = (const uint8_t *)a.q + (row0 + r < a.rows ? row0 + r : a.rows - 1) * a.q_row_bytes + (lane & 7) * 16 + (int64_t)u0 * 128;
        dst[i] = ring + r * 128 + (((lane & 7) ^ (r & 7)) << 4);
    }
    int left = u1 - u0;  // units that are not fetched yet
    const int last_cols = cols - (u1 - 1) * 256;  // columns of this share's last unit (more than there are: all 256)
    uint32_t put = 0;
    auto fetch = [&]() {
        if (left > 0) {
            if (left > 1 || (lane & 7) * 32 < last_cols) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    cp_async16(dst[i] + put, src[i]);
                    src[i] += 128;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) st_shared16_zero(dst[i] + put);
            }
            --left;
        }
        put = put == RING - 2048 ? 0 : put + 2048;
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kLinStages; ++s) fetch();

    // scales of rows g and g + 8, 128 columns ahead of their use
    const char *sca = (const char *)a.scale + row_a * a.scale_row_stride * SB, *scb = (const char *)a.scale + row_b * a.scale_row_stride * SB;
    const int8_t *zpa = ZP ? a.zp + row_a * a.scale_row_stride : nullptr, *zpb = ZP ? a.zp + row_b * a.scale_row_stride : nullptr;
    constexpr int NR = FP4 ? 4 : NS;
    uint32_t rawa[NR], rawb[NR];
    int za[ZP ? NR : 1], zb[ZP ? NR : 1];
    auto load_scale = [&](const char *q) -> uint32_t {
        if constexpr (SB == 4) return __ldg((const uint32_t *)q);
        else if constexpr (SB == 2) return __ldg((const uint16_t *)q);
        else return __ldg((const uint8_t *)q);
    };
    auto scales = [&](int ch) {  // ch: chunk of 128 columns
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            rawa[j] = rawb[j] = 0;
            if constexpr (ZP) za[j] = zb[j] = 0;
            if (ch * 128 + j * (128 / NR) < cols) {
                const uint32_t i = FP4 ? (uint32_t)(ch * 8 + j * 2 + (t >> 1)) : fastdiv((uint32_t)(ch * NR + j), p.group);
                rawa[j] = load_scale(sca + i * SB);
                rawb[j] = load_scale(scb + i * SB);
                if constexpr (ZP) {
                    za[j] = __ldg(zpa + i);
                    zb[j] = __ldg(zpb + i);
                }
            }
        }
    };
    const bool scale_bf16 = a.scale_dtype == CTB_BF16;
    auto scale_value = [&](uint32_t r) {
        if constexpr (SB == 4) return __uint_as_float(r);
        return scale_bf16 ? bf16_bits_to_f32(r) : __half2float(__ushort_as_half((unsigned short)r));
    };
    scales(2 * u0);

    const uint32_t ldrow = (lane & 7) + ((lane >> 3) & 1) * 8;
    uint32_t ld[4];  // 64 columns of 16 rows each
#pragma unroll
    for (int i = 0; i < 4; ++i) ld[i] = ring + ldrow * 128 + (((2 * i + (lane >> 4)) ^ (ldrow & 7)) << 4);
    float fin[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) fin[n][i] = 0.0f;
    constexpr float mid = DT == CTB_BF16 ? 136.0f : 1032.0f;

    // tokens that do not fill a tile of eight read a row of zeros
    const uint8_t *xr0[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xr0[n] = xs + (n * 8 + g < nt ? n * 8 + g : nt) * xstride + t * 16;
    if (nt < TOK)
        for (int c = threadIdx.x; c < p.x_cols / 8; c += WARPS * 32) *(uint4 *)(xs + nt * xstride + c * 16) = make_uint4(0, 0, 0, 0);

    uint32_t get = 0;
    for (int x0 = u0; x0 < u1; x0 += p.x_cols / 256) {
        const int x1 = min(u1, x0 + p.x_cols / 256);
        if (x0 > u0) {
            __syncthreads();
            fetch_x(x0, x1);
            cp_async_wait<0>();
        } else {
            cp_async_wait<kLinStages>();  // behind them the first stages of weights are on their way
        }
        each_x(x0, x1, [&](uint8_t *at, const uint16_t *) {  // every thread puts its own pieces into the codes' order
            const uint4 v = *(const uint4 *)at;
            *(uint4 *)at = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                                      __byte_perm(v.y, v.w, 0x7632));
        });
        __syncthreads();
        uint32_t xo = 0;
        for (int u = x0; u < x1; ++u) {
            cp_async_wait<kLinStages - 1>();
            __syncwarp();
            uint32_t w[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) ldmatrix4(w[i], ld[i] + get);
            get = get == RING - 2048 ? 0 : get + 2048;
            __syncwarp();
            fetch();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t ka[NR], kb[NR];  // what the pair conversion takes: the subtrahend, or the scale
                float sa[NR], sb[NR];
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    if constexpr (FP4) {
                        const float up = DT == CTB_BF16 ? 0x1p118f : 128.0f;
                        ka[j] = dup2<DT>(e4m3_to_f32((uint8_t)rawa[j]) * up);
                        kb[j] = dup2<DT>(e4m3_to_f32((uint8_t)rawb[j]) * up);
                    } else {
                        ka[j] = dup2<DT>(ZP ? mid + (float)za[ZP ? j : 0] : mid);
                        kb[j] = dup2<DT>(ZP ? mid + (float)zb[ZP ? j : 0] : mid);
                        sa[j] = scale_value(rawa[j]);
                        sb[j] = scale_value(rawb[j]);
                    }
                }
                scales(2 * u + h + 1);
                float acc[NT][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // 32 columns: one word of each row
                    const uint32_t wa = w[2 * h + (j >> 1)][(j & 1) * 2], wb = w[2 * h + (j >> 1)][(j & 1) * 2 + 1];
                    const int q = NR == 4 ? j : 0;
                    uint32_t pa[4], pb[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        pa[i] = Code4<DT, FP4>::pair(wa, i, ka[q]);
                        pb[i] = Code4<DT, FP4>::pair(wb, i, kb[q]);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 b = *(const uint4 *)(xr0[n] + xo + h * 256 + j * 64);
                        if constexpr (FP4) {
                            mma16816<DT>(fin[n], pa[0], pb[0], pa[1], pb[1], b.x, b.y);
                            mma16816<DT>(fin[n], pa[2], pb[2], pa[3], pb[3], b.z, b.w);
                        } else {
                            if (NR == 4 || j == 0) mma16816_first<DT>(acc[n], pa[0], pb[0], pa[1], pb[1], b.x, b.y);
                            else mma16816<DT>(acc[n], pa[0], pb[0], pa[1], pb[1], b.x, b.y);
                            mma16816<DT>(acc[n], pa[2], pb[2], pa[3], pb[3], b.z, b.w);
                            if (NR == 4 || j == 3) {
                                fin[n][0] = fmaf(sa[q], acc[n][0], fin[n][0]);
                                fin[n][1] = fmaf(sa[q], acc[n][1], fin[n][1]);
                                fin[n][2] = fmaf(sb[q], acc[n][2], fin[n][2]);
                                fin[n][3] = fmaf(sb[q], acc[n][3], fin[n][3]);
                            }
                        }
                    }
                }
            }
            xo += 512;
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    // sums of this share, [token][row], where the rings were
    float *red = reinterpret_cast<float *>(smem);
    constexpr int RS = ROWS + 4;
    static_assert(TOK * RS * 4 <= WARPS * RING, "the sums fit where the rings were");
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[(n * 8 + 2 * t + (i & 1)) * RS + warp * 16 + g + (i >> 1) * 8] = fin[n][i];
    if (shares > 1) cluster_sync();
    else __syncthreads();
    constexpr int LOG_ROWS = WARPS == 4 ? 6 : WARPS == 8 ? 7 : 8;
    static_assert(1 << LOG_ROWS == ROWS, "rows of a tile");
    const int log_part = LOG_ROWS - p.log_shares;  // rows of the tile that this block finishes
    const int64_t r0 = (int64_t)(blockIdx.x >> p.log_shares) * ROWS + (share << log_part);
    float gs = 1.0f;
    if (FP4 && a.gs) gs = *a.gs;
    for (int i = threadIdx.x; i < nt << log_part; i += WARPS * 32) {
        const int m = i >> log_part, r = i & ((1 << log_part) - 1);
        if (r0 + r >= a.rows) continue;
        const float *at = red + m * RS + (share << log_part) + r;
        float v = 0.0f;
        if (shares > 1) {
#pragma unroll 8
            for (int s = 0; s < shares; ++s) v += ld_cluster(smem_u32(at), s);
        } else {
            v = *at;
        }
        if constexpr (FP4) v = __fdiv_rn(v * (DT == CTB_BF16 ? 256.0f : 128.0f), gs);
        if (a.bias) v += load_f32(a.bias, DT, r0 + r);
        store_f32(a.out, DT, (t0 + m) * a.rows + r0 + r, v);
    }
    if (shares > 1) cluster_leave();  // nobody leaves while its sums are still read
}

template <int DT, bool FP4, bool ZP, int NS, int SB, int NT, int WARPS>
static int linear_mma_launch(const LinearArgs &a, cudaStream_t st) {
    constexpr int TOK = NT * 8;
    constexpr size_t RINGS = WARPS * kLinStages * 2048;
    // Shares of the columns: as many blocks as the GPU holds at once, each with two stages at least.
    const int64_t tiles = cdiv(a.rows, WARPS * 16) * cdiv(a.tokens, TOK), units = cdiv(a.cols, 256);
    const int nt = (int)(a.tokens < TOK ? a.tokens : TOK);
    const int64_t held = kLinXBytes / (2 * nt) / 256 * 256;
    LinearPlan p;
    size_t bytes = 0;
    for (int log_shares = 0; log_shares <= 3; ++log_shares) {
        const int shares = 1 << log_shares;
        const int64_t slice = cdiv(units, shares) * 256;
        const int64_t x_cols = slice < held ? slice : held;
        const size_t need = RINGS + (size_t)(nt < TOK ? nt + 1 : nt) * (x_cols * 2 + 64);
        const int64_t at_once = (int64_t)(227 * 1024 / (need + 1024)) * sm_count();
        if (shares > 1 && (tiles * shares > at_once || units < 2 * shares)) break;
        p.log_shares = log_shares;
        p.x_cols = (int)x_cols;
        bytes = need;
    }
    p.group = make_fastdiv((uint32_t)(FP4 ? 1 : a.col_group / (128 / NS)));
    auto kernel = linear4_mma_kernel<DT, FP4, ZP, NS, SB, NT, WARPS>;
    static std::atomic<bool> ready[64];
    int rc = allow_smem(kernel, RINGS + 2 * kLinXBytes + (TOK + 1) * 64, ready);
    if (rc) return rc;
    const int64_t gx = cdiv(a.rows, WARPS * 16) << p.log_shares, gy = cdiv(a.tokens, TOK);
    if (gx > INT32_MAX || gy > 65535) return fail(CTB_EUNSUPPORTED, "too many rows or tokens for one call");
    return launch_cluster("linear4_mma_kernel", kernel, dim3((unsigned)gx, (unsigned)gy), WARPS * 32, bytes, 1u << p.log_shares, st, a, p);
}

template <int DT, bool FP4>
static int linear_launch(const LinearArgs &a, cudaStream_t st) {
    // Rows of 16-byte pieces, and scale groups that the tensor-core kernel can keep apart; the rest goes one code at a time.
    const bool rows16 = a.cols > 0 && a.cols % 32 == 0 && a.cols <= INT32_MAX / 2 && aligned16(a.q) && aligned16(a.x);
    const bool groups = FP4 ? a.col_group == 16 && a.scale_dtype == CTB_E4M3 : a.col_group % 32 == 0 && a.scale_dtype != CTB_E4M3;
    if (!rows16 || !groups) {
        const int64_t gx = cdiv(a.rows, 8), gy = cdiv(a.tokens, 8);
        if (gx > INT32_MAX || gy > 65535) return fail(CTB_EUNSUPPORTED, "too many rows or tokens for one call");
        linear4_any_kernel<DT, FP4><<<dim3((unsigned)gx, (unsigned)gy), 256, 0, st>>>(a);
        return after_launch("linear4_any_kernel");
    }
    auto go = [&](auto zp, auto ns, auto sb) {
        constexpr bool Z = decltype(zp)::value;
        constexpr int N = decltype(ns)::value, S = decltype(sb)::value;
        // Every block prepares its columns of x for itself, so the more tokens, the more rows a block should take, as long as there are
        // blocks for all SMs: 16 tokens, 14336 rows: 22.8 us with 128 rows a block, 18.9 with 256; 4096 rows: 10.3 and 19.2.
        const bool tall = a.rows >= 8192;
        if (a.tokens <= 8) return linear_mma_launch<DT, FP4, Z, N, S, 1, 4>(a, st);
        if (a.tokens <= 16) return tall ? linear_mma_launch<DT, FP4, Z, N, S, 2, 16>(a, st) : linear_mma_launch<DT, FP4, Z, N, S, 2, 8>(a, st);
        return tall ? linear_mma_launch<DT, FP4, Z, N, S, 4, 16>(a, st) : linear_mma_launch<DT, FP4, Z, N, S, 4, 8>(a, st);
    };
    using T = std::true_type;
    using F = std::false_type;
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    using Four = std::integral_constant<int, 4>;
    if constexpr (FP4) {
        return go(F{}, One{}, One{});
    } else {
        auto width = [&](auto zp, auto ns) { return a.scale_dtype == CTB_F32 ? go(zp, ns, Four{}) : go(zp, ns, Two{}); };
        if (a.col_group % 128 == 0) return a.zp ? width(T{}, One{}) : width(F{}, One{});
        return a.zp ? width(T{}, Four{}) : width(F{}, Four{});
    }
}

}  // namespace ctb

extern "C" int ctb_dequantize_linear(const ctb_qdesc *d, const void *x, int64_t tokens, const void *q, const void *scale,
                                     const void *zero_point, const float *global_scale, const void *bias, void *out, void *stream) {
    using namespace ctb;
    if (!d) return fail(CTB_EINVAL_NULL, "null descriptor");
    if (d->rows < 0 || d->cols < 0 || tokens < 0) return fail(CTB_EINVAL_SHAPE, "negative size");
    const bool fp4 = d->codec == CTB_CODE_FP4X2;
    if (d->codec != CTB_CODE_FP4X2 && d->codec != CTB_CODE_PACK32) return fail(CTB_EUNSUPPORTED, "the product takes packed codes (PACK32 or FP4X2)");
    if (d->num_bits != 4 || d->qtype != (fp4 ? CTB_QFLOAT : CTB_QINT)) return fail(CTB_EUNSUPPORTED, "the product is built for 4-bit codes: int in PACK32, float in FP4X2");
    if (d->row_group != 1) return fail(CTB_EUNSUPPORTED, "the product takes one scale row per weight row (row_group 1)");
    if (d->x_dtype != CTB_BF16 && d->x_dtype != CTB_F16) return fail(CTB_EINVAL_DTYPE, "x must be bf16 or f16");
    if (!is_float_dtype(d->scale_dtype) && d->scale_dtype != CTB_E4M3) return fail(CTB_EINVAL_DTYPE, "scales must be bf16, f16, f32 or e4m3");
    if (fp4 && zero_point) return fail(CTB_EUNSUPPORTED, "fp4 codes have no zero point");
    if (zero_point && d->zp_dtype != CTB_I8) return fail(CTB_EINVAL_DTYPE, "zero points must be int8");
    if (!fp4 && global_scale) return fail(CTB_EUNSUPPORTED, "a global scale belongs to fp4 codes");
    if (fp4 && d->cols % 2) return fail(CTB_EINVAL_SHAPE, "fp4 codes come in pairs: cols must be even");
    if (d->rows == 0 || tokens == 0) return CTB_OK;
    if (d->cols > 0 && (d->col_group < 1 || d->cols % d->col_group)) return fail(CTB_EINVAL_SHAPE, "tensor column shape must be divisble by the given group_size");
    if (d->scale_row_stride < 0) return fail(CTB_EINVAL_SHAPE, "negative scale stride");
    if (!out || (d->cols > 0 && (!x || !q || !scale))) return fail(CTB_EINVAL_NULL, "null buffer");
    if (((uintptr_t)x | (uintptr_t)out | (uintptr_t)bias) & 1) return fail(CTB_EINVAL_ALIGN, "x, bias and out must be aligned to their element size");
    LinearArgs a{x, q, scale, bias, (const int8_t *)zero_point, global_scale, out, tokens, d->rows, d->cols,
                 fp4 ? d->cols / 2 : cdiv(d->cols, 8) * 4, d->cols > 0 ? d->col_group : 1, d->scale_row_stride, d->scale_dtype};
    const cudaStream_t st = as_stream(stream);
    if (d->x_dtype == CTB_BF16) return fp4 ? linear_launch<CTB_BF16, true>(a, st) : linear_launch<CTB_BF16, false>(a, st);
    return fp4 ? linear_launch<CTB_F16, true>(a, st) : linear_launch<CTB_F16, false>(a, st);
}
