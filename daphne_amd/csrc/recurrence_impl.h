// Gated linear recurrence over packed sequences for DenseMatrix<float|double>, forward and backward.
//
//   f_t = sigmoid(z_t)      h_t = f_t h_{t-1} + (1 - f_t) x_t                 for every channel of every sequence,
//   G_t = d_out_t + f_{t+1} G_{t+1}  (the last row adds d_last),
//   d_x_t = (1 - f_t) G_t   d_z_t = G_t (h_{t-1} - x_t) f_t (1 - f_t)         d_h0 = f_0 G_0.
//
// Rows are tokens: the sequences lie one behind the other, sequence s in rows [offsets[s], offsets[s + 1]).
#pragma once

#include "common.h"

namespace dh_rec {

constexpr int THREADS = 256;

// f = 1 / (1 + exp(-z)) and 1 - f, each to full relative precision: both from e = exp(-|z|), which never overflows.
template <typename T> __device__ __forceinline__ void gates(T z, T &f, T &w) {
    const T e = sizeof(T) == 4 ? static_cast<T>(__expf(-fabsf(static_cast<float>(z)))) : static_cast<T>(exp(-fabs(static_cast<double>(z))));
    const T r = T(1) / (T(1) + e), er = e * r;
    f = z >= T(0) ? r : er;
    w = z >= T(0) ? er : r;
}

// Rows of sequence s, clamped to the tokens that exist; equal lengths without offsets.
struct Spans {
    const long long *offsets; // nullptr: every sequence has `even` rows
    size_t ld;
    size_t even, tokens;
    __device__ __forceinline__ size_t at(size_t s) const {
        if (offsets == nullptr)
            return s * even;
        const long long o = offsets[s * ld];
        return o < 0 ? 0 : static_cast<unsigned long long>(o) > tokens ? tokens : static_cast<size_t>(o);
    }
};

// Raises if the offsets fall or leave [0, tokens]; every thread of the launch takes a share.
__device__ __forceinline__ void check_offsets(const Spans &sp, size_t num_seq, size_t i, size_t stride, int *rec) {
    if (sp.offsets == nullptr)
        return;
    for (; i <= num_seq; i += stride) {
        const long long o = sp.offsets[i * sp.ld], before = i ? sp.offsets[(i - 1) * sp.ld] : 0;
        if (o < before || o < 0 || static_cast<unsigned long long>(o) > sp.tokens)
            dh_raise(rec, DH_DEFERRED_OFFSETS, 0, o, static_cast<long long>(sp.tokens));
    }
}

// One thread per sequence and channel, one row after the other.
template <typename T>
__global__ __launch_bounds__(THREADS) void forward_serial_kernel(T *res, size_t ld_res, T *last, size_t ld_last, const T *x, size_t ld_x,
                                                                 const T *z, size_t ld_z, const T *h0, size_t ld_h0, Spans sp,
                                                                 size_t num_seq, size_t channels, int *rec) {
    const size_t c = static_cast<size_t>(blockIdx.x) * THREADS + threadIdx.x, s = blockIdx.y;
    if (s == 0)
        check_offsets(sp, num_seq, c, static_cast<size_t>(gridDim.x) * THREADS, rec);
    if (c >= channels)
        return;
    T h = h0 ? h0[s * ld_h0 + c] : T(0);
    const size_t end = sp.at(s + 1);
    for (size_t t = sp.at(s); t < end; t++) {
        T f, w;
        gates(z[t * ld_z + c], f, w);
        h = f * h + w * x[t * ld_x + c];
        res[t * ld_res + c] = h;
    }
    if (last)
        last[s * ld_last + c] = h;
}

template <typename T>
__global__ __launch_bounds__(THREADS) void backward_serial_kernel(T *d_x, size_t ld_dx, T *d_z, size_t ld_dz, T *d_h0, size_t ld_dh0,
                                                                  const T *x, size_t ld_x, const T *z, size_t ld_z, const T *h, size_t ld_h,
                                                                  const T *h0, size_t ld_h0, const T *d_out, size_t ld_do, const T *d_last,
                                                                  size_t ld_dl, Spans sp, size_t num_seq, size_t channels, int *rec) {
    const size_t c = static_cast<size_t>(blockIdx.x) * THREADS + threadIdx.x, s = blockIdx.y;
    if (s == 0)
        check_offsets(sp, num_seq, c, static_cast<size_t>(gridDim.x) * THREADS, rec);
    if (c >= channels)
        return;
    T carry = d_last ? d_last[s * ld_dl + c] : T(0); // f_{t+1} G_{t+1}
    const size_t begin = sp.at(s);
    for (size_t t = sp.at(s + 1); t > begin;) {
        t--;
        T f, w;
        gates(z[t * ld_z + c], f, w);
        const T g = d_out[t * ld_do + c] + carry;
        const T before = t > begin ? h[(t - 1) * ld_h + c] : h0 ? h0[s * ld_h0 + c] : T(0);
        const T xv = x[t * ld_x + c];
        d_x[t * ld_dx + c] = w * g;
        d_z[t * ld_dz + c] = g * (before - xv) * f * w;
        carry = f * g;
    }
    if (d_h0)
        d_h0[s * ld_dh0 + c] = carry;
}

// What every entry point checks of its sequences.
static inline dh_status check_sequences(const char *what, const long long *offsets, size_t ld_offsets, size_t num_seq, size_t tokens) {
    if (offsets != nullptr)
        return ld_offsets < 1 ? dh_fail(DH_ERR_RUNTIME, "%s - a leading dimension is smaller than its column count", what) : DH_OK;
    if (num_seq == 0 ? tokens != 0 : tokens % num_seq != 0)
        return dh_fail(DH_ERR_RUNTIME, "%s - %zu rows do not divide into %zu sequences of equal length (offsets are needed)", what, tokens,
                       num_seq);
    return DH_OK;
}

template <typename T> size_t workspace(size_t, size_t, size_t) { return 0; }

template <typename T>
dh_status forward(dh_ctx *ctx, T *res, size_t ld_res, T *last, size_t ld_last, const T *x, size_t tokens, size_t channels, size_t ld_x,
                  const T *z, size_t ld_z, const T *h0, size_t ld_h0, const long long *offsets, size_t ld_offsets, size_t num_seq, void *ws,
                  size_t ws_bytes) {
    constexpr const char *what = "gatedRecurrenceForward";
    if (ld_res < channels || ld_x < channels || ld_z < channels || (last && ld_last < channels) || (h0 && ld_h0 < channels))
        return dh_fail(DH_ERR_RUNTIME, "%s - a leading dimension is smaller than its column count", what);
    if (dh_status st = check_sequences(what, offsets, ld_offsets, num_seq, tokens); st != DH_OK)
        return st;
    if (channels > 0 && num_seq > 0 && tokens > 0 && (res == nullptr || x == nullptr || z == nullptr))
        return dh_fail(DH_ERR_RUNTIME, "%s - a matrix is null", what);
    DH_REQUIRE_CTX(ctx);
    if (channels == 0 || num_seq == 0)
        return DH_OK;
    int *rec = nullptr;
    if (offsets)
        if (dh_status st = dh_checked_begin(ctx, what, &rec); st != DH_OK)
            return st;
    void *work = nullptr;
    if (dh_status st = dh_call_workspace(ctx, what, ws, ws_bytes, workspace<T>(tokens, num_seq, channels), &work); st != DH_OK)
        return st;
    const size_t gx = dh_ceil_div(channels, THREADS);
    if (gx >= (size_t(1) << 31) || num_seq >= 65536)
        return dh_fail(DH_ERR_RUNTIME, "%s - extents exceed one launch", what);
    const Spans sp{offsets, ld_offsets, tokens / num_seq, tokens};
    hipLaunchKernelGGL((forward_serial_kernel<T>), dim3(static_cast<unsigned>(gx), static_cast<unsigned>(num_seq)), dim3(THREADS), 0,
                       ctx->stream, res, ld_res, last, ld_last, x, ld_x, z, ld_z, h0, ld_h0, sp, num_seq, channels, rec);
    DH_CHECK_LAUNCH();
    return offsets ? dh_checked_end(ctx) : DH_OK;
}

template <typename T>
dh_status backward(dh_ctx *ctx, T *d_x, size_t ld_dx, T *d_z, size_t ld_dz, T *d_h0, size_t ld_dh0, const T *x, size_t tokens,
                   size_t channels, size_t ld_x, const T *z, size_t ld_z, const T *h, size_t ld_h, const T *h0, size_t ld_h0,
                   const T *d_out, size_t ld_do, const T *d_last, size_t ld_dl, const long long *offsets, size_t ld_offsets, size_t num_seq,
                   void *ws, size_t ws_bytes) {
    constexpr const char *what = "gatedRecurrenceBackward";
    if (ld_dx < channels || ld_dz < channels || ld_x < channels || ld_z < channels || ld_h < channels || ld_do < channels ||
        (d_h0 && ld_dh0 < channels) || (h0 && ld_h0 < channels) || (d_last && ld_dl < channels))
        return dh_fail(DH_ERR_RUNTIME, "%s - a leading dimension is smaller than its column count", what);
    if (dh_status st = check_sequences(what, offsets, ld_offsets, num_seq, tokens); st != DH_OK)
        return st;
    if (channels > 0 && num_seq > 0 && tokens > 0 && (d_x == nullptr || d_z == nullptr || x == nullptr || z == nullptr || h == nullptr || d_out == nullptr))
        return dh_fail(DH_ERR_RUNTIME, "%s - a matrix is null", what);
    DH_REQUIRE_CTX(ctx);
    if (channels == 0 || num_seq == 0)
        return DH_OK;
    int *rec = nullptr;
    if (offsets)
        if (dh_status st = dh_checked_begin(ctx, what, &rec); st != DH_OK)
            return st;
    void *work = nullptr;
    if (dh_status st = dh_call_workspace(ctx, what, ws, ws_bytes, workspace<T>(tokens, num_seq, channels), &work); st != DH_OK)
        return st;
    const size_t gx = dh_ceil_div(channels, THREADS);
    if (gx >= (size_t(1) << 31) || num_seq >= 65536)
        return dh_fail(DH_ERR_RUNTIME, "%s - extents exceed one launch", what);
    const Spans sp{offsets, ld_offsets, tokens / num_seq, tokens};
    hipLaunchKernelGGL((backward_serial_kernel<T>), dim3(static_cast<unsigned>(gx), static_cast<unsigned>(num_seq)), dim3(THREADS), 0,
                       ctx->stream, d_x, ld_dx, d_z, ld_dz, d_h0, ld_dh0, x, ld_x, z, ld_z, h, ld_h, h0, ld_h0, d_out, ld_do, d_last, ld_dl,
                       sp, num_seq, channels, rec);
    DH_CHECK_LAUNCH();
    return offsets ? dh_checked_end(ctx) : DH_OK;
}

} // namespace dh_rec
