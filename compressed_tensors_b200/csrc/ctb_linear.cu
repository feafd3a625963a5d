// Product with a 4-bit weight: out[t][n] = sum_k x[t][k] * (code[n][k] - zp) * scale (+ bias[n]), for few tokens.
//
// What bounds it: a weight code is used once per token, so at a few tokens the call takes the time of reading the
// packed weight (half a byte per weight) from HBM.
#include "ctb_common.cuh"

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

template <int DT, bool FP4>
static int linear_launch(const LinearArgs &a, cudaStream_t st) {
    const int64_t gx = cdiv(a.rows, 8), gy = cdiv(a.tokens, 8);
    if (gx > INT32_MAX || gy > 65535) return fail(CTB_EUNSUPPORTED, "too many rows or tokens for one call");
    linear4_any_kernel<DT, FP4><<<dim3((unsigned)gx, (unsigned)gy), 256, 0, st>>>(a);
    return after_launch("linear4_any_kernel");
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
