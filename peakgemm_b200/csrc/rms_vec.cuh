// 16-byte vectors of eight 16-bit elements <-> fp32, and the warp sum, for the kernels of rmsnorm_residual*.cu.
#pragma once

#include <stdint.h>

#include "ptx.cuh"

namespace pg {

template <bool BF16>
__device__ __forceinline__ void vec_unpack(const uint4 &v, float (&f)[8]) {
    ptx::unpack2<BF16>(v.x, f[0], f[1]);
    ptx::unpack2<BF16>(v.y, f[2], f[3]);
    ptx::unpack2<BF16>(v.z, f[4], f[5]);
    ptx::unpack2<BF16>(v.w, f[6], f[7]);
}

template <bool BF16>
__device__ __forceinline__ uint4 vec_pack(const float (&f)[8]) {
    return make_uint4(ptx::pack2<BF16>(f[0], f[1]), ptx::pack2<BF16>(f[2], f[3]), ptx::pack2<BF16>(f[4], f[5]),
                      ptx::pack2<BF16>(f[6], f[7]));
}

// Eight consecutive fp32 values, 16-byte aligned.
__device__ __forceinline__ void vec_load_f32(const float *p, float (&f)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p));
    const float4 b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void vec_store_f32(float *p, const float (&f)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

__device__ __forceinline__ float warp_sum_f32(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

}  // namespace pg
