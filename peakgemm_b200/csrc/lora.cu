// A projection with low-rank adapters of many requests at once: row t of the batch uses adapter i = ids[t],
//     d[t] = row_scale[t] * (a[t] * b^T + scale[i] * (a[t] * A_i^T) * B_i^T) + bias + residual[t].
// First form, plain: v = scale * a * A^T (one warp per element, fp32), then one thread per element of d.

#include <cuda_runtime.h>
#include <stdint.h>

#include "host_util.h"
#include "lora.h"
#include "rms_vec.cuh"

namespace pg {
namespace {

// v[t, r] = scale * sum_k a[t, k] A[ids[t], r, k], 0 without an adapter.
template <bool BF16>
__global__ void __launch_bounds__(256)
lora_shrink_kernel(float *v, const uint4 *a, int64_t lda8, const LoraArgs l, int64_t m, int k8) {
    const int64_t warp = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    if (warp >= m * l.rank) return;
    const int lane = threadIdx.x & 31;
    const int64_t t = warp / l.rank, r = warp - t * l.rank;
    const int id = l.ids[t];
    float sum = 0.f;
    if (id >= 0 && id < l.adapters) {
        const uint4 *x = a + t * lda8, *w = static_cast<const uint4 *>(l.a) + (static_cast<int64_t>(id) * l.rank + r) * k8;
        for (int i = lane; i < k8; i += 32) {
            float f[8], g[8];
            vec_unpack<BF16>(x[i], f);
            vec_unpack<BF16>(w[i], g);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(f[e], g[e], sum);
        }
        if (l.scale) sum *= l.scale[id];
    }
    sum = warp_sum_f32(sum);
    if (lane == 0) v[warp] = sum;
}

// d[t, j] = row_scale * (sum_k a[t, k] b[j, k] + sum_r v[t, r] B[ids[t], j, r]) + bias[j] + residual[t, j].
template <bool BF16>
__global__ void __launch_bounds__(256)
lora_expand_kernel(const GemmArgs g, const LoraArgs l, const float *v) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= g.m * g.n) return;
    const int64_t t = i / g.n, j = i - t * g.n;
    const int id = l.ids[t];
    float sum = 0.f, unused, x;
    {
        const uint4 *p = static_cast<const uint4 *>(g.a) + t * (g.lda / 8), *q = static_cast<const uint4 *>(g.b) + j * (g.ldb / 8);
        for (int64_t c = 0; c < g.k / 8; ++c) {
            float f[8], w[8];
            vec_unpack<BF16>(p[c], f);
            vec_unpack<BF16>(q[c], w);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(f[e], w[e], sum);
        }
    }
    if (id >= 0 && id < l.adapters) {
        const uint4 *w = static_cast<const uint4 *>(l.b) + (static_cast<int64_t>(id) * g.n + j) * (l.rank / 8);
        for (int r = 0; r < l.rank / 8; ++r) {
            float f[8];
            vec_unpack<BF16>(w[r], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(f[e], v[t * l.rank + 8 * r + e], sum);
        }
    }
    if (g.row_scale) sum *= g.row_scale[t];
    if (g.bias) {
        ptx::unpack2<BF16>(static_cast<const uint16_t *>(g.bias)[j], x, unused);
        sum += x;
    }
    if (g.residual) {
        ptx::unpack2<BF16>(static_cast<const uint16_t *>(g.residual)[t * g.ldr + j], x, unused);
        sum += x;
    }
    static_cast<uint16_t *>(g.c)[t * g.ldc + j] = static_cast<uint16_t>(ptx::pack2<BF16>(sum, 0.f) & 0xffffu);
}

}  // namespace

size_t lora_workspace_bytes(int64_t m, int64_t, int64_t, int64_t, int64_t rank) {
    return (static_cast<size_t>(m) * rank * sizeof(float) + 255) / 256 * 256;
}

int hgemm_lora_launch(const GemmArgs &g, const LoraArgs &l, cudaStream_t stream, cudaError_t *cuda_err) {
    float *v = static_cast<float *>(l.workspace);
    const int64_t warps = g.m * l.rank, elements = g.m * g.n;
    if ((warps + 7) / 8 > 2147483647 || (elements + 255) / 256 > 2147483647) return kLaunchBadConfig;
    const unsigned gs = static_cast<unsigned>((warps + 7) / 8), ge = static_cast<unsigned>((elements + 255) / 256);
    const int k8 = static_cast<int>(g.k / 8);
    if (g.bf16) {
        lora_shrink_kernel<true><<<gs, 256, 0, stream>>>(v, static_cast<const uint4 *>(g.a), g.lda / 8, l, g.m, k8);
        lora_expand_kernel<true><<<ge, 256, 0, stream>>>(g, l, v);
    } else {
        lora_shrink_kernel<false><<<gs, 256, 0, stream>>>(v, static_cast<const uint4 *>(g.a), g.lda / 8, l, g.m, k8);
        lora_expand_kernel<false><<<ge, 256, 0, stream>>>(g, l, v);
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) { *cuda_err = e; return kLaunchCuda; }
    return kLaunchOk;
}

}  // namespace pg
