// Token embeddings for DenseMatrix<float|double>: rows of a table by token number, scaled, and the gradient of the table.
//
//   forward   res[i] = scale * table[ids[i]]
//   backward  d_table[v] = scale * sum over { i : ids[i] = v } of d_out[i]   (+ d_table[v])
//
// The forward pass is ExtractRow with a factor: it moves n rows in and n rows out and is bound by memory. Token numbers
// are checked by the kernels that read them; a number outside the table reads and writes nothing and is reported.
// The backward pass adds a token's rows in the order of their positions, in 64 bits, without floating-point atomics:
// results do not depend on timing.
#pragma once

#include "common.h"

namespace dh_embed {

constexpr int THREADS = 256;

// One 16-byte vector (VEC values) per thread and step; LPR lanes share a row, a power of two up to THREADS. blockIdx.y
// takes UN * LPR vectors of a row each.
template <typename T, int VEC, int UN>
__global__ __launch_bounds__(THREADS) void forward_kernel(T *res, size_t ld_res, const T *table, size_t ld_table, long long vocab,
                                                          size_t width_vecs, const long long *ids, size_t ld_ids, size_t n, T scale,
                                                          unsigned lpr, int *rec) {
    const unsigned lane = threadIdx.x % lpr;
    const size_t row = static_cast<size_t>(blockIdx.x) * (THREADS / lpr) + threadIdx.x / lpr;
    if (row >= n)
        return;
    const long long id = ids[row * ld_ids];
    const size_t v0 = static_cast<size_t>(blockIdx.y) * UN * lpr + lane;
    if (id < 0 || id >= vocab) {
        if (v0 == 0)
            dh_raise(rec, DH_DEFERRED_TOKEN_ID, 0, id, vocab);
        return;
    }
    const T *src = table + static_cast<size_t>(id) * ld_table;
    T *dst = res + row * ld_res;
    T v[UN][VEC];
#pragma unroll
    for (int u = 0; u < UN; u++) {
        const size_t j = v0 + static_cast<size_t>(u) * lpr;
        dh_load_vec<T, VEC>(src + (j < width_vecs ? j : width_vecs - 1) * VEC, v[u]); // beyond the row: its last vector, never stored
    }
#pragma unroll
    for (int u = 0; u < UN; u++) {
        const size_t j = v0 + static_cast<size_t>(u) * lpr;
        if (j >= width_vecs)
            break;
#pragma unroll
        for (int e = 0; e < VEC; e++)
            v[u][e] *= scale;
        dh_store_vec<T, VEC>(dst + j * VEC, v[u]);
    }
}

template <typename T>
dh_status forward(dh_ctx *ctx, T *res, size_t ld_res, const T *table, size_t vocab, size_t width, size_t ld_table, const long long *ids,
                  size_t n, size_t ld_ids, T scale) {
    if (ld_res < width || ld_table < width || ld_ids < 1)
        return dh_fail(DH_ERR_RUNTIME, "embeddingForward - a leading dimension is smaller than its column count");
    if (n > 0 && width > 0 && (res == nullptr || ids == nullptr || (table == nullptr && vocab > 0)))
        return dh_fail(DH_ERR_RUNTIME, "embeddingForward - a matrix is null");
    DH_REQUIRE_CTX(ctx);
    if (n == 0 || width == 0)
        return DH_OK;
    int *rec = nullptr;
    if (dh_status st = dh_checked_begin(ctx, "embeddingForward", &rec); st != DH_OK)
        return st;
    constexpr int V = dh_vec<T>::N;
    const bool vec = width % V == 0 && ld_res % V == 0 && ld_table % V == 0 && dh_aligned(res, 16) && dh_aligned(table, 16);
    const size_t wv = vec ? width / V : width;
    unsigned lpr = 1;
    while (lpr < THREADS && lpr < wv)
        lpr <<= 1;
    const size_t gx = dh_ceil_div(n, THREADS / lpr);
    const bool four = gx * dh_ceil_div(wv, lpr) >= 4096; // several vectors in flight a thread once the workgroups fill the device
    const size_t gy = dh_ceil_div(wv, static_cast<size_t>(lpr) * (four ? 4 : 1));
    if (gx >= (size_t(1) << 31) || gy >= 65536)
        return dh_fail(DH_ERR_RUNTIME, "embeddingForward - extents exceed one launch");
    const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy));
#define DH_EMBED_FORWARD(VEC, UN)                                                                                                          \
    hipLaunchKernelGGL((forward_kernel<T, VEC, UN>), grid, dim3(THREADS), 0, ctx->stream, res, ld_res, table, ld_table,                   \
                       static_cast<long long>(vocab), wv, ids, ld_ids, n, scale, lpr, rec)
    if (vec && four)
        DH_EMBED_FORWARD(V, 4);
    else if (vec)
        DH_EMBED_FORWARD(V, 1);
    else if (four)
        DH_EMBED_FORWARD(1, 4);
    else
        DH_EMBED_FORWARD(1, 1);
#undef DH_EMBED_FORWARD
    DH_CHECK_LAUNCH();
    return dh_checked_end(ctx);
}

// One workgroup per table row and slice of THREADS columns: the positions of its token are picked out of every THREADS
// token numbers in order, and their rows added.
template <typename T>
__global__ __launch_bounds__(THREADS) void backward_scan_kernel(T *d_table, size_t ld, long long vocab, size_t width, const T *d_out,
                                                                size_t ld_out, const long long *ids, size_t ld_ids, size_t n, T scale,
                                                                int accumulate, int *rec) {
    __shared__ unsigned hits[THREADS];
    __shared__ unsigned count[THREADS / DH_WAVE];
    const long long v = static_cast<long long>(blockIdx.x);
    const size_t col = static_cast<size_t>(blockIdx.y) * THREADS + threadIdx.x;
    const unsigned wave = threadIdx.x / DH_WAVE, lane = threadIdx.x % DH_WAVE;
    double acc = 0.0;
    bool any = false;
    for (size_t base = 0; base < n; base += THREADS) {
        const size_t i = base + threadIdx.x;
        const long long id = i < n ? ids[i * ld_ids] : -1;
        if (blockIdx.x == 0 && blockIdx.y == 0 && i < n && (id < 0 || id >= vocab))
            dh_raise(rec, DH_DEFERRED_TOKEN_ID, 0, id, vocab);
        const bool hit = i < n && id == v;
        const unsigned long long mask = __ballot(hit);
        if (lane == 0)
            count[wave] = __popcll(mask);
        __syncthreads();
        unsigned at = __popcll(mask & ((1ull << lane) - 1)), total = 0;
        for (unsigned w = 0; w < THREADS / DH_WAVE; w++) {
            at += w < wave ? count[w] : 0;
            total += count[w];
        }
        if (hit)
            hits[at] = threadIdx.x;
        __syncthreads();
        any |= total != 0;
        if (col < width)
            for (unsigned k = 0; k < total; k++)
                acc += static_cast<double>(d_out[(base + hits[k]) * ld_out + col]);
        __syncthreads();
    }
    if (col < width && (any || !accumulate)) {
        T *p = d_table + static_cast<size_t>(v) * ld + col;
        const double s = acc * static_cast<double>(scale);
        *p = static_cast<T>(accumulate ? s + static_cast<double>(*p) : s);
    }
}

template <typename T> size_t backward_workspace(size_t, size_t, size_t) { return 0; }

template <typename T>
dh_status backward(dh_ctx *ctx, T *d_table, size_t vocab, size_t width, size_t ld, const T *d_out, size_t ld_out, const long long *ids,
                   size_t n, size_t ld_ids, T scale, int accumulate, void *ws, size_t ws_bytes) {
    if (ld < width || ld_out < width || ld_ids < 1)
        return dh_fail(DH_ERR_RUNTIME, "embeddingBackward - a leading dimension is smaller than its column count");
    if (width > 0 && ((d_table == nullptr && vocab > 0) || (n > 0 && (d_out == nullptr || ids == nullptr))))
        return dh_fail(DH_ERR_RUNTIME, "embeddingBackward - a matrix is null");
    DH_REQUIRE_CTX(ctx);
    if (width == 0 || (vocab == 0 && n == 0))
        return DH_OK;
    int *rec = nullptr;
    if (dh_status st = dh_checked_begin(ctx, "embeddingBackward", &rec); st != DH_OK)
        return st;
    void *work = nullptr;
    if (dh_status st = dh_call_workspace(ctx, "embeddingBackward", ws, ws_bytes, backward_workspace<T>(n, vocab, width), &work); st != DH_OK)
        return st;
    const size_t gy = dh_ceil_div(width, THREADS), gx = vocab ? vocab : 1;
    if (gx >= (size_t(1) << 31) || gy >= 65536)
        return dh_fail(DH_ERR_RUNTIME, "embeddingBackward - extents exceed one launch");
    hipLaunchKernelGGL((backward_scan_kernel<T>), dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), dim3(THREADS), 0, ctx->stream,
                       d_table, ld, static_cast<long long>(vocab), vocab ? width : 0, d_out, ld_out, ids, ld_ids, n, scale, accumulate, rec);
    DH_CHECK_LAUNCH();
    return dh_checked_end(ctx);
}

} // namespace dh_embed
