// Internal interface between the C ABI (api.cu) and the RMSNorm kernels (rmsnorm.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace pg {

struct RmsFwdArgs {
    void *y;
    const void *x;
    const float *gamma;
    int64_t rows, h;
    float eps;
    bool bf16;
};

struct RmsBwdArgs {
    void *dx;
    float *dgamma;
    const void *dy;
    const void *x;
    const float *gamma;
    int64_t rows, h;
    float eps;
    bool bf16;
    void *workspace;   // [ctas, h] fp32
};

// Largest h the backward kernel supports.
int64_t rmsnorm_max_h();

// fp32 partial rows of dgamma the backward kernel writes for this shape on the current device.
cudaError_t rmsnorm_bwd_ctas(int64_t rows, int64_t h, bool bf16, int *ctas);

cudaError_t rmsnorm_fwd_launch(const RmsFwdArgs &a, cudaStream_t stream);
cudaError_t rmsnorm_bwd_launch(const RmsBwdArgs &a, int ctas, cudaStream_t stream);

// rstd[r] = rsqrt(mean(x[r,:]^2) + eps), fp32 (rmsnorm_rstd.cu).
cudaError_t rmsnorm_rstd_launch(float *rstd, const void *x, int64_t rows, int64_t h, float eps, bool bf16,
                                cudaStream_t stream);

// The norms around a block, its gate and the scaled residual (rmsnorm_residual.cu).  Null pointers: the term is absent.
struct RmsResidualTerms {
    const float *gamma_post;   // [h]: norm of the block's output u; null: u itself
    const void *gate;          // [gate_rows, h] 16-bit, consecutive rows / gate_rows rows share one; null: 1
    int64_t gate_rows;
    const float *res_scale;    // [h] or [1]; null: 1
    bool res_scale_one;        // res_scale has one element
    const float *gamma_pre;    // [h]: norm of the new residual stream s; null: no y
    int64_t rows, h;
    float eps;
    bool bf16;
};
struct RmsResidualFwdArgs {
    RmsResidualTerms t;
    void *s, *y;
    const void *u, *residual;
};
struct RmsResidualBwdArgs {
    RmsResidualTerms t;
    void *du, *dresidual;
    float *dgamma_post;
    void *dgate;
    float *dres_scale, *dgamma_pre;
    const void *dy, *ds, *s, *u, *residual;
    void *workspace;
};
cudaError_t rmsnorm_residual_fwd_launch(const RmsResidualFwdArgs &a, cudaStream_t stream);
// Scratch of the backward pass for this shape on the current device.
cudaError_t rmsnorm_residual_bwd_bytes(int64_t rows, int64_t h, int64_t gate_rows, size_t *bytes);
cudaError_t rmsnorm_residual_bwd_launch(const RmsResidualBwdArgs &a, cudaStream_t stream);

// Backward, sums over rows: the rows are cut into `workers` consecutive runs; worker w's fp32 part of dgamma_post,
// dgamma_pre and dres_scale is row w of its table.  A gate whose rows lie in one run gets its gradient from that worker;
// one whose rows lie in several gets a part from each: a run holds at most two such gates, its first (row 2w of `gate`)
// and its last (row 2w + 1).
struct RmsResidualParts {
    float *post, *pre, *scale, *gate;
    double *scale_one;      // n_one of them, where res_scale has one element
    uint32_t workers, n_one;
};
// Clusters of C CTAs, one to an SM, that the device holds at once (C a power of two up to 8).
int rmsnorm_residual_clusters(int C, int sms);
// Bulk-copy staged forward kernel (rmsnorm_residual_staged_fwd.cu), where it has the width and every worker a row.
bool rmsnorm_residual_staged_fwd_supported(const RmsResidualTerms &t, int sms);
cudaError_t rmsnorm_residual_staged_fwd(const RmsResidualFwdArgs &a, cudaStream_t stream);
// Bulk-copy staged backward kernel (rmsnorm_residual_staged.cu), for the widths where `workers` is not 0; a row is
// shared by ctas_per_row CTAs, each of which writes a scale_one of its own.
uint32_t rmsnorm_residual_staged_workers(int64_t rows, int64_t h, int sms, uint32_t *ctas_per_row);
cudaError_t rmsnorm_residual_staged_bwd(const RmsResidualBwdArgs &a, const RmsResidualParts &parts, cudaStream_t stream);

// Bulk-copy staged variants (rmsnorm_staged.cu), used for 2048 <= h <= 16384.
bool rmsnorm_staged_supported(int64_t h, bool bwd);
cudaError_t rmsnorm_staged_ctas(int64_t rows, int64_t h, bool bwd, int *ctas, int *partial_rows);
cudaError_t rmsnorm_staged_fwd(const RmsFwdArgs &a, cudaStream_t stream);
cudaError_t rmsnorm_staged_bwd(const RmsBwdArgs &a, cudaStream_t stream);   // writes the partial rows only
// SM count of the current device and the staged kernels' status word there.
cudaError_t rmsnorm_device(int *sms, int **status);
// Synchronises the stream, returns and clears the staged kernels' device status word.
cudaError_t rmsnorm_device_status(int *out, cudaStream_t stream);

}  // namespace pg
