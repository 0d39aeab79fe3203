// Products with 4-bit weights for DenseMatrix<float>: res = x t(W), W given as codes in [-8, 7] and one scale per group of
// columns, x as floats or as 8-bit rows with one scale each.
//
//   res[i][o] = sum over groups g of scale[o][g] * sum over k in g of code[o][k] x[i][k]      (x = x_scale[i] * code, if 8 bits)
//
// Few rows of x read every weight once, half a byte each: bound by memory. Codes are two to a byte, row by row, the even
// column in the low half.
#include "common.h"

namespace dh_q4 {

constexpr int THREADS = 256;

// One wavefront per result, a lane per byte of codes and step.
template <typename X>
__global__ __launch_bounds__(THREADS) void matvec_plain_kernel(float *res, size_t ld_res, const X *x, size_t rows, size_t cols, size_t ld_x,
                                                               const float *x_scale, const unsigned char *codes, size_t outs, size_t ld_codes,
                                                               const float *scales, size_t ld_scales, size_t group) {
    const size_t o = static_cast<size_t>(blockIdx.x) * (THREADS / DH_WAVE) + threadIdx.x / DH_WAVE;
    if (o >= outs)
        return;
    const size_t i = blockIdx.y;
    const unsigned lane = threadIdx.x % DH_WAVE;
    const unsigned char *w = codes + o * ld_codes;
    const X *xi = x + i * ld_x;
    float acc = 0.f;
    for (size_t b = lane; 2 * b < cols; b += DH_WAVE) {
        const int lo = static_cast<int>(static_cast<unsigned>(w[b]) << 28) >> 28, hi = static_cast<int>(static_cast<unsigned>(w[b]) << 24) >> 28;
        float s = static_cast<float>(lo) * static_cast<float>(xi[2 * b]);
        if (2 * b + 1 < cols)
            s += static_cast<float>(hi) * static_cast<float>(xi[2 * b + 1]);
        acc += s * scales[o * ld_scales + 2 * b / group]; // groups are whole pairs of columns
    }
    dh_butterfly(DH_WAVE, [&](auto peer) { acc += peer(acc); });
    if (lane == 0)
        res[i * ld_res + o] = x_scale ? acc * x_scale[i] : acc;
}

template <typename X>
dh_status matvec(dh_ctx *ctx, float *res, size_t ld_res, const X *x, size_t rows, size_t cols, size_t ld_x, const float *x_scale,
                 const unsigned char *codes, size_t outs, size_t ld_codes, const float *scales, size_t ld_scales, size_t group) {
    constexpr const char *what = "matVecQ4";
    if (group == 0 || group % 32 != 0)
        return dh_fail(DH_ERR_INVALID_ARG, "%s - the group of %zu columns is not a multiple of 32", what, group);
    if (ld_res < outs || ld_x < cols || ld_codes < dh_ceil_div(cols, 2) || ld_scales < dh_ceil_div(cols, group))
        return dh_fail(DH_ERR_RUNTIME, "%s - a leading dimension is smaller than its column count", what);
    if (rows > 0 && outs > 0 &&
        (res == nullptr || (cols > 0 && (x == nullptr || codes == nullptr || scales == nullptr)) || (sizeof(X) == 1 && x_scale == nullptr)))
        return dh_fail(DH_ERR_RUNTIME, "%s - a matrix is null", what);
    DH_REQUIRE_CTX(ctx);
    if (rows == 0 || outs == 0)
        return DH_OK;
    const size_t gx = dh_ceil_div(outs, THREADS / DH_WAVE);
    if (gx >= (size_t(1) << 31) || rows >= 65536)
        return dh_fail(DH_ERR_RUNTIME, "%s - extents exceed one launch", what);
    hipLaunchKernelGGL((matvec_plain_kernel<X>), dim3(static_cast<unsigned>(gx), static_cast<unsigned>(rows)), dim3(THREADS), 0, ctx->stream,
                       res, ld_res, x, rows, cols, ld_x, x_scale, codes, outs, ld_codes, scales, ld_scales, group);
    DH_CHECK_LAUNCH();
    return DH_OK;
}

// One wavefront per group: its largest magnitude becomes 7, values are rounded to the nearest code (ties to even).
static __global__ __launch_bounds__(THREADS) void quantize_kernel(unsigned char *codes, size_t ld_codes, float *scales, size_t ld_scales,
                                                                  const float *w, size_t rows, size_t cols, size_t ld, size_t group,
                                                                  size_t groups) {
    const size_t job = static_cast<size_t>(blockIdx.x) * (THREADS / DH_WAVE) + threadIdx.x / DH_WAVE;
    if (job >= rows * groups)
        return;
    const size_t r = job / groups, g = job % groups, c0 = g * group, c1 = c0 + group < cols ? c0 + group : cols;
    const unsigned lane = threadIdx.x % DH_WAVE;
    const float *row = w + r * ld;
    float most = 0.f;
    for (size_t c = c0 + lane; c < c1; c += DH_WAVE) {
        const float v = fabsf(row[c]);
        most = most != most ? most : (v != v || v > most ? v : most);
    }
    dh_butterfly(DH_WAVE, [&](auto peer) {
        const float o = peer(most);
        most = most != most ? most : (o != o || o > most ? o : most);
    });
    const bool finite = most <= 3.402823466e38f;
    const float scale = finite ? most / 7.0f : dh_nan<float>();
    if (lane == 0)
        scales[r * ld_scales + g] = scale;
    // in 64 bits: the quotient of two floats is never rounded onto a border between two codes
    const double to_code = finite && most > 0.f ? 7.0 / static_cast<double>(most) : 0.0;
    for (size_t b = c0 / 2 + lane; 2 * b < c1; b += DH_WAVE) {
        const int lo = finite ? static_cast<int>(rint(static_cast<double>(row[2 * b]) * to_code)) : 0;
        const int hi = finite && 2 * b + 1 < cols ? static_cast<int>(rint(static_cast<double>(row[2 * b + 1]) * to_code)) : 0;
        codes[r * ld_codes + b] = static_cast<unsigned char>((lo & 15) | ((hi & 15) << 4));
    }
}

} // namespace dh_q4

extern "C" dh_status dh_matvec_q4_f32(dh_ctx *ctx, float *res, size_t ld_res, const float *x, size_t rows, size_t cols, size_t ld_x,
                                      const uint8_t *codes, size_t outs, size_t ld_codes, const float *scales, size_t ld_scales, size_t group) {
    return dh_q4::matvec<float>(ctx, res, ld_res, x, rows, cols, ld_x, nullptr, codes, outs, ld_codes, scales, ld_scales, group);
}

extern "C" dh_status dh_matvec_q4_q8_f32(dh_ctx *ctx, float *res, size_t ld_res, const int8_t *x, size_t rows, size_t cols, size_t ld_x,
                                         const float *x_scale, const uint8_t *codes, size_t outs, size_t ld_codes, const float *scales,
                                         size_t ld_scales, size_t group) {
    return dh_q4::matvec<int8_t>(ctx, res, ld_res, x, rows, cols, ld_x, x_scale, codes, outs, ld_codes, scales, ld_scales, group);
}

extern "C" dh_status dh_quantize_q4_f32(dh_ctx *ctx, uint8_t *codes, size_t ld_codes, float *scales, size_t ld_scales, const float *w,
                                        size_t rows, size_t cols, size_t ld, size_t group) {
    if (group == 0 || group % 32 != 0)
        return dh_fail(DH_ERR_INVALID_ARG, "quantizeQ4 - the group of %zu columns is not a multiple of 32", group);
    if (ld < cols || ld_codes < dh_ceil_div(cols, 2) || ld_scales < dh_ceil_div(cols, group))
        return dh_fail(DH_ERR_RUNTIME, "quantizeQ4 - a leading dimension is smaller than its column count");
    if (rows > 0 && cols > 0 && (codes == nullptr || scales == nullptr || w == nullptr))
        return dh_fail(DH_ERR_RUNTIME, "quantizeQ4 - a matrix is null");
    DH_REQUIRE_CTX(ctx);
    if (rows == 0 || cols == 0)
        return DH_OK;
    const size_t groups = dh_ceil_div(cols, group), gx = dh_ceil_div(rows * groups, dh_q4::THREADS / DH_WAVE);
    if (gx >= (size_t(1) << 31))
        return dh_fail(DH_ERR_RUNTIME, "quantizeQ4 - extents exceed one launch");
    hipLaunchKernelGGL(dh_q4::quantize_kernel, dim3(static_cast<unsigned>(gx)), dim3(dh_q4::THREADS), 0, ctx->stream, codes, ld_codes, scales,
                       ld_scales, w, rows, cols, ld, group, groups);
    DH_CHECK_LAUNCH();
    return DH_OK;
}
