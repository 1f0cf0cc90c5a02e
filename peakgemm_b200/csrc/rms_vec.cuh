// Pieces of the RMSNorm kernels: bulk row copies and the voting group barrier (rmsnorm_staged.cu, rmsnorm_residual_staged.cu),
// 16-byte vectors of eight 16-bit elements <-> fp32, and the warp sum.
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

// First row of the c-th of n runs that share `rows` rows evenly.
__host__ __device__ __forceinline__ uint32_t rms_run_begin(uint32_t c, uint32_t n, uint32_t rows) {
    return static_cast<uint32_t>(static_cast<uint64_t>(c) * rows / n);
}

// Two fp32 values in one register pair: the packed instructions issue half as often, which is what bounds the kernels
// that do much arithmetic per byte (rmsnorm_residual_staged.cu).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)),
          "l"(reinterpret_cast<const unsigned long long &>(c)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)));
    return d;
}
template <bool BF16>
__device__ __forceinline__ void vec_unpack2(const uint4 &v, float2 (&f)[4]) {
    ptx::unpack2<BF16>(v.x, f[0].x, f[0].y);
    ptx::unpack2<BF16>(v.y, f[1].x, f[1].y);
    ptx::unpack2<BF16>(v.z, f[2].x, f[2].y);
    ptx::unpack2<BF16>(v.w, f[3].x, f[3].y);
}
template <bool BF16>
__device__ __forceinline__ uint4 vec_pack2(const float2 (&f)[4]) {
    return make_uint4(ptx::pack2<BF16>(f[0].x, f[0].y), ptx::pack2<BF16>(f[1].x, f[1].y),
                      ptx::pack2<BF16>(f[2].x, f[2].y), ptx::pack2<BF16>(f[3].x, f[3].y));
}
// Eight fp32 values from shared memory, the upper four `half` bytes behind the lower ones.
__device__ __forceinline__ void vec_load2(uint32_t s, uint32_t half, float2 (&f)[4]) {
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f[0].x), "=f"(f[0].y), "=f"(f[1].x), "=f"(f[1].y) : "r"(s));
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f[2].x), "=f"(f[2].y), "=f"(f[3].x), "=f"(f[3].y) : "r"(s + half));
}
__device__ __forceinline__ void vec_store2(float *p, const float2 (&f)[4]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
    reinterpret_cast<float4 *>(p)[1] = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
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

// 1-D bulk copy global -> shared; both addresses 16-byte aligned, bytes % 16 == 0.
__device__ __forceinline__ void bulk_load(uint32_t dst_smem, const void *src, uint32_t bytes, uint32_t bar,
                                          uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint "
                 "[%0], [%1], %2, [%3], %4;"
                 ::"r"(dst_smem), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar), "l"(policy)
                 : "memory");
}

// A warp's sums to the buffer place `at` of every CTA of the cluster, arriving on the barrier at `bar` there.
__device__ __forceinline__ void send_sums(uint32_t at, uint32_t bar, uint32_t cta, float x, float y, float z) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
                 ::"r"(ptx::mapa(at, cta)), "f"(x), "f"(y), "f"(z), "f"(0.f), "r"(ptx::mapa(bar, cta)) : "memory");
}

// Named barrier `id` over `nthreads` consumer threads that also ORs a predicate across
// them, so that "somebody abandoned a wait" is decided identically by the whole group.
__device__ __forceinline__ bool group_barrier_or(uint32_t id, uint32_t nthreads, bool pred) {
    uint32_t r;
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.u32 q, %1, 0;\n\t"
        "bar.red.or.pred p, %2, %3, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}\n"
        : "=r"(r)
        : "r"(static_cast<uint32_t>(pred)), "r"(id), "r"(nthreads)
        : "memory");
    return r != 0;
}

}  // namespace pg
