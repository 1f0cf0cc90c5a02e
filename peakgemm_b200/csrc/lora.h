// Internal interface between the C ABI (api.cu) and the adapter projection (lora.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "gemm_sm100.h"

namespace pg {

struct LoraArgs {
    const void *a;         // [adapters, rank, k], the matrices' element type
    const void *b;         // [adapters, n, rank]
    const int32_t *ids;    // [m]; outside 0 .. adapters-1: the row has no adapter
    const float *scale;    // [adapters] fp32 or null (1)
    int64_t adapters, rank;
    void *workspace;
};

// Scratch for this shape on the current device.
cudaError_t lora_workspace_bytes(int64_t m, int64_t n, int64_t k, int64_t adapters, int64_t rank, size_t *bytes);

// g's product and epilogue terms plus the adapters' contribution; a LaunchResult.
int hgemm_lora_launch(const GemmArgs &g, const LoraArgs &l, cudaStream_t stream, cudaError_t *cuda_err);

}  // namespace pg
