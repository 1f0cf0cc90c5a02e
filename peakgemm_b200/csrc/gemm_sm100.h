// Internal interface between the C ABI (api.cu) and the GEMM kernels (gemm_sm100.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace pg {

// Rank elements of a block of V's rows, which hold each block twice (lora_epilogue.cuh), and the elements of such a row.
constexpr uint32_t lora_width(int64_t rank) { return rank <= 16 ? 16u : 32u; }
constexpr int64_t lora_v_cols(int64_t rank) {
    return (rank + lora_width(rank) - 1) / lora_width(rank) * (2 * lora_width(rank));
}

// What the GEMM kernels need to add the adapters' up projections (see lora_epilogue.cuh).
struct LoraGemm {
    const int32_t *ids, *table;
    const void *v, *b;
    int64_t adapters, rank, max_slots, group_rows, slot_rows, table_stride, mask_off;
};

struct GemmArgs {
    void *c;
    const void *a;
    const void *b;
    int64_t m, n, k;
    int64_t lda, ldb, ldc;   // row pitches in elements
    bool bf16;               // false: fp16
    int n_extra_dst = 0;     // further destinations of C (same extents and pitch as c), at most 7
    void *extra_dst[7] = {};
    // Fused epilogue, every term optional (null = absent):
    //   C[i,j] = round(row_scale[i] * sum_k A[i,k] B[j,k] + bias[j] + residual[i,j])
    const float *row_scale = nullptr;   // [m] fp32
    const void *bias = nullptr;         // [n], the matrices' element type
    const void *residual = nullptr;     // [m, n] with row pitch ldr, the matrices' element type; may be c itself
    int64_t ldr = 0;
    bool pdl_wait = false;              // the epilogue waits for the preceding kernel of the stream before it reads
                                        // row_scale (programmatic dependent launch); the main loop does not wait
    void *mc_dst = nullptr;             // non-null: C is written through this multicast address (row pitch ldc) with
                                        // multimem.st instead of TMA stores to c; c must still be a local address
    void *workspace = nullptr;          // optional scratch for the tail split of the 256-wide CTA-pair kernel
    size_t workspace_bytes = 0;
    const LoraGemm *lora = nullptr;     // adapters beside b (hgemm_launch_with_lora only)
};

enum LaunchResult { kLaunchOk = 0, kLaunchCuda = 1, kLaunchNotSm100 = 2, kLaunchBadConfig = 3 };

// variant: 0 auto, 1 = one CTA per tile, 2 = CTA pair per tile, 3 = cluster split-K, 4 = skinny,
// 5 = CTA pair with two row blocks per CTA (512 x 256 tiles); block_n: 0 auto, 64, 128, 256.
// max_sms: 0 = all SMs, else an upper bound on the SMs the persistent grid occupies.
int hgemm_launch(const GemmArgs &g, int variant, int block_n, int max_sms, cudaStream_t stream,
                 cudaError_t *cuda_err);

// g's product and terms with the adapters of g.lora, whose v and table the previous launch on the stream writes: the
// product's own k-blocks run beside that launch.  lora_group_rows: the rows that share a slot table, for a device with
// `sms` SMs.
int hgemm_launch_with_lora(const GemmArgs &g, cudaStream_t stream, cudaError_t *cuda_err);
int lora_group_rows(int64_t m, int64_t n, int64_t k, int sms);

// SM count, compute capability and status word of the current device; a tensor map of a row-major 16-bit matrix with
// a box of box_rows x 64 elements, 128-byte swizzle.
cudaError_t gemm_device(int *sm_count, int *cc_major, int **status);
bool gemm_operand_map(CUtensorMap *tm, const void *base, int64_t rows, int64_t cols, int64_t ld, uint32_t box_rows,
                      bool bf16);

// Resolves variant/block_n == 0 to concrete values for a device with sm_count SMs.
void choose_config(const GemmArgs &g, int sm_count, int *variant, int *block_n);

// Workspace (bytes) that lets hgemm_launch split the last, partial wave of this shape over idle SM pairs; 0 if none.
size_t hgemm_workspace_bytes(int64_t m, int64_t n, int64_t k, int sm_count);

// Synchronises the stream, returns and clears the kernels' device status word.
int gemm_device_status(int *out, cudaStream_t stream, cudaError_t *cuda_err);

}  // namespace pg
