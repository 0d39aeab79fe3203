// Sequence-model kernels, double instantiation. See embed_impl.h, rmsnorm_impl.h and recurrence_impl.h for the mathematics.
#include "embed_impl.h"
#include "recurrence_impl.h"
#include "rmsnorm_impl.h"

static inline const long long *as_ll(const int64_t *p) { return reinterpret_cast<const long long *>(p); }

extern "C" dh_status dh_embedding_forward_f64(dh_ctx *ctx, double *res, size_t ld_res, const double *table, size_t vocab, size_t width,
                                              size_t ld_table, const int64_t *ids, size_t n, size_t ld_ids, double scale) {
    return dh_embed::forward<double>(ctx, res, ld_res, table, vocab, width, ld_table, as_ll(ids), n, ld_ids, scale);
}
extern "C" size_t dh_embedding_backward_workspace_f64(size_t n, size_t vocab, size_t width) {
    return dh_embed::backward_workspace<double>(n, vocab, width);
}
extern "C" dh_status dh_embedding_backward_f64(dh_ctx *ctx, double *d_table, size_t vocab, size_t width, size_t ld_table, const double *d_out,
                                               size_t ld_out, const int64_t *ids, size_t n, size_t ld_ids, double scale, int accumulate,
                                               void *workspace, size_t workspace_bytes) {
    return dh_embed::backward<double>(ctx, d_table, vocab, width, ld_table, d_out, ld_out, as_ll(ids), n, ld_ids, scale, accumulate, workspace,
                                   workspace_bytes);
}

extern "C" dh_status dh_rmsnorm_forward_f64(dh_ctx *ctx, double *res, size_t ld_res, double *sum, size_t ld_sum, double *inv_rms, const double *x,
                                            size_t rows, size_t cols, size_t ld_x, const double *residual, size_t ld_residual,
                                            const double *gamma, double eps) {
    return dh_rms::forward<double, false>(ctx, {res, nullptr, nullptr, ld_res, sum, ld_sum, inv_rms, x, ld_x, residual, ld_residual, gamma, rows,
                                             cols, static_cast<double>(eps)});
}
extern "C" size_t dh_rmsnorm_backward_workspace_f64(size_t rows, size_t cols) { return dh_rms::backward_workspace<double>(rows, cols); }
extern "C" dh_status dh_rmsnorm_backward_f64(dh_ctx *ctx, double *dx, size_t ld_dx, double *d_gamma, const double *h, size_t rows, size_t cols,
                                             size_t ld_h, const double *inv_rms, const double *gamma, const double *d_res, size_t ld_dres,
                                             const double *d_sum, size_t ld_dsum, void *workspace, size_t workspace_bytes) {
    return dh_rms::backward<double>(ctx, {dx, ld_dx, d_gamma, h, ld_h, inv_rms, gamma, d_res, ld_dres, d_sum, ld_dsum, rows, cols}, workspace,
                                 workspace_bytes);
}

extern "C" size_t dh_gated_recurrence_workspace_f64(size_t tokens, size_t num_seq, size_t channels) {
    return dh_rec::workspace<double>(tokens, num_seq, channels);
}
extern "C" dh_status dh_gated_recurrence_forward_f64(dh_ctx *ctx, double *res, size_t ld_res, double *last, size_t ld_last, const double *x,
                                                     size_t tokens, size_t channels, size_t ld_x, const double *z, size_t ld_z,
                                                     const double *h0, size_t ld_h0, const int64_t *offsets, size_t ld_offsets,
                                                     size_t num_seq, void *workspace, size_t workspace_bytes) {
    return dh_rec::forward<double>(ctx, res, ld_res, last, ld_last, x, tokens, channels, ld_x, z, ld_z, h0, ld_h0, as_ll(offsets), ld_offsets,
                                num_seq, workspace, workspace_bytes);
}
extern "C" dh_status dh_gated_recurrence_backward_f64(dh_ctx *ctx, double *d_x, size_t ld_dx, double *d_z, size_t ld_dz, double *d_h0,
                                                      size_t ld_dh0, const double *x, size_t tokens, size_t channels, size_t ld_x,
                                                      const double *z, size_t ld_z, const double *h, size_t ld_h, const double *h0, size_t ld_h0,
                                                      const double *d_res, size_t ld_dres, const double *d_last, size_t ld_dlast,
                                                      const int64_t *offsets, size_t ld_offsets, size_t num_seq, void *workspace,
                                                      size_t workspace_bytes) {
    return dh_rec::backward<double>(ctx, d_x, ld_dx, d_z, ld_dz, d_h0, ld_dh0, x, tokens, channels, ld_x, z, ld_z, h, ld_h, h0, ld_h0, d_res,
                                 ld_dres, d_last, ld_dlast, as_ll(offsets), ld_offsets, num_seq, workspace, workspace_bytes);
}
