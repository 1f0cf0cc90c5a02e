// The boundary between two blocks of a network in one pass: norm of a block's output, its gate, the scaled residual,
// and the norm in front of the next block.  For every row
//     p = u * rstd(u) * gamma_post           (without gamma_post: p = u)
//     s = res_scale * residual + gate * p
//     y = s * rstd(s) * gamma_pre             (optional),      rstd(v) = 1 / sqrt(mean(v^2) + eps)
// All sums and products in fp32; s and y are each rounded once, and y is computed from the unrounded s.
// Backward, with D the whole gradient of s, shat = s * rstd(s), uhat = u * rstd(u), w = dy * gamma_pre:
//     D = ds + rstd(s) * (w - shat * mean(w * shat))            dgamma_pre  = sum_r dy * shat
//     dresidual = res_scale * D                                  dres_scale  = sum_r D * residual
//     e = gate * D                                               dgate       = sum over the gate's rows of D * p
//     du = rstd(u) * (e * gamma_post - uhat * mean(e * gamma_post * uhat))     dgamma_post = sum_r e * uhat
// rstd is computed again from s and u: no saved statistics cross the interface.

#include <cuda_runtime.h>
#include <stdint.h>

#include "host_util.h"
#include "rms_vec.cuh"
#include "rmsnorm.h"

namespace pg {
namespace {

// Sum over the block's threads, the same value in every thread.  `red`: one float per warp, not in use by an earlier
// sum that some thread may still be reading.
__device__ __forceinline__ float block_sum(float v, float *red) {
    v = warp_sum_f32(v);
    if (blockDim.x == 32) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
    for (uint32_t w = 0; w < blockDim.x / 32; ++w) t += red[w];
    return t;
}

__device__ __forceinline__ float dot8(const float (&a)[8], const float (&b)[8]) {
    float t = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) t = fmaf(a[e], b[e], t);
    return t;
}

struct Row {
    const uint4 *gate;     // the row's gate, or null
    __device__ __forceinline__ Row(const RmsResidualTerms &t, uint32_t row, uint32_t rows_per_gate) {
        gate = t.gate ? static_cast<const uint4 *>(t.gate) + static_cast<int64_t>(row / rows_per_gate) * (t.h / 8) : nullptr;
    }
};

__device__ __forceinline__ void load_scale(const RmsResidualTerms &t, int idx, float (&f)[8]) {
    if (t.res_scale && !t.res_scale_one) {
        vec_load_f32(t.res_scale + 8 * idx, f);
    } else {
        const float v = t.res_scale ? __ldg(t.res_scale) : 1.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = v;
    }
}

// ---------------------------------------------------------------- forward ----

// One block per row, thread t owns the vectors t, t + blockDim.x, ... (at most VPT) and holds the row in registers.
// For few rows of h <= 16384 (with one for every worker of the staged kernel that one runs).  Bound by latency (loads, two
// block sums): replayed in a graph, [1, 4096] 3.3 us, [64, 8192] 4.5 us with a launch of about 2.5 us.
template <int VPT, bool BF16>
__global__ void __launch_bounds__(1024)
rms_residual_fwd_kernel(const RmsResidualFwdArgs a, uint32_t rows_per_gate) {
    __shared__ float red[2][32];
    const int h8 = static_cast<int>(a.t.h / 8);
    const float inv_h = 1.f / static_cast<float>(a.t.h);
    const uint32_t row = blockIdx.x;
    const int64_t base = static_cast<int64_t>(row) * h8;
    const Row r(a.t, row, rows_per_gate);
    uint4 uv[VPT], rv[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int idx = threadIdx.x + blockDim.x * j;
        const bool in = idx < h8;
        uv[j] = in ? static_cast<const uint4 *>(a.u)[base + idx] : make_uint4(0, 0, 0, 0);
        rv[j] = in ? static_cast<const uint4 *>(a.residual)[base + idx] : make_uint4(0, 0, 0, 0);
    }
    float rstd_u = 1.f;
    if (a.t.gamma_post) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            float f[8];
            vec_unpack<BF16>(uv[j], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(f[e], f[e], ss);
        }
        rstd_u = 1.f / sqrtf(block_sum(ss, red[0]) * inv_h + a.t.eps);
    }
    float s[VPT][8], ss = 0.f;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int idx = threadIdx.x + blockDim.x * j;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j][e] = 0.f;
        if (idx < h8) {
            float f[8], g[8];
            vec_unpack<BF16>(uv[j], f);
            if (a.t.gamma_post) {
                vec_load_f32(a.t.gamma_post + 8 * idx, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = (f[e] * rstd_u) * g[e];
            }
            if (r.gate) {
                vec_unpack<BF16>(__ldg(r.gate + idx), g);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= g[e];
            }
            float x[8];
            vec_unpack<BF16>(rv[j], x);
            load_scale(a.t, idx, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s[j][e] = fmaf(g[e], x[e], f[e]);
                ss = fmaf(s[j][e], s[j][e], ss);
            }
            static_cast<uint4 *>(a.s)[base + idx] = vec_pack<BF16>(s[j]);
        }
    }
    if (a.y) {
        const float rstd_s = 1.f / sqrtf(block_sum(ss, red[1]) * inv_h + a.t.eps);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int idx = threadIdx.x + blockDim.x * j;
            if (idx < h8) {
                float g[8];
                vec_load_f32(a.t.gamma_pre + 8 * idx, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] *= s[j][e] * rstd_s;
                static_cast<uint4 *>(a.y)[base + idx] = vec_pack<BF16>(g);
            }
        }
    }
}

// Any h: the row is read three times (the second and third reads hit L2); [2048, 65536] 384-416 us, 0.4-0.5 of the copy
// bandwidth.  Nothing is written before the last pass, so s may be the residual and y may be u here too.  A thread's sums
// of eight squares are added in 64 bits: their number grows with h.
template <bool BF16>
__global__ void __launch_bounds__(1024)
rms_residual_fwd_wide_kernel(const RmsResidualFwdArgs a, uint32_t rows_per_gate) {
    __shared__ float red[2][32];
    const int h8 = static_cast<int>(a.t.h / 8);
    const float inv_h = 1.f / static_cast<float>(a.t.h);
    for (uint32_t row = blockIdx.x; row < a.t.rows; row += gridDim.x) {
        const int64_t base = static_cast<int64_t>(row) * h8;
        const Row r(a.t, row, rows_per_gate);
        const uint4 *u = static_cast<const uint4 *>(a.u) + base, *res = static_cast<const uint4 *>(a.residual) + base;
        float rstd_u = 1.f, rstd_s = 1.f;
        for (int pass = a.t.gamma_post ? 0 : 1; pass < 3; ++pass) {
            if (pass == 1 && !a.y) continue;
            double ss = 0.0;
            for (int idx = threadIdx.x; idx < h8; idx += blockDim.x) {
                float f[8], g[8], x[8];
                vec_unpack<BF16>(u[idx], f);
                if (pass > 0) {
                    if (a.t.gamma_post) {
                        vec_load_f32(a.t.gamma_post + 8 * idx, g);
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] = (f[e] * rstd_u) * g[e];
                    }
                    if (r.gate) {
                        vec_unpack<BF16>(__ldg(r.gate + idx), g);
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] *= g[e];
                    }
                    vec_unpack<BF16>(res[idx], x);
                    load_scale(a.t, idx, g);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = fmaf(g[e], x[e], f[e]);
                }
                if (pass < 2) {
                    ss += static_cast<double>(dot8(f, f));
                } else {
                    static_cast<uint4 *>(a.s)[base + idx] = vec_pack<BF16>(f);
                    if (a.y) {
                        vec_load_f32(a.t.gamma_pre + 8 * idx, g);
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] = (f[e] * rstd_s) * g[e];
                        static_cast<uint4 *>(a.y)[base + idx] = vec_pack<BF16>(f);
                    }
                }
            }
            if (pass == 0) rstd_u = 1.f / sqrtf(block_sum(static_cast<float>(ss), red[0]) * inv_h + a.t.eps);
            if (pass == 1) rstd_s = 1.f / sqrtf(block_sum(static_cast<float>(ss), red[1]) * inv_h + a.t.eps);
        }
        __syncthreads();
    }
}

// --------------------------------------------------------------- backward ----

// What a row contributes to its elements' gradients: D = ds + rstd_s * w - ms * s, du = rstd_u * e * gamma_post - mu * u.
struct RowStats {
    float rstd_s, ms;     // rstd(s), rstd(s)^3 * mean(w * s)
    float rstd_u, mu;     // rstd(u), rstd(u)^3 * mean(e * gamma_post * u)
};

// D of one vector.
template <bool BF16>
__device__ __forceinline__ void load_stream_grad(const RmsResidualBwdArgs &a, int64_t at, int idx, const RowStats &st,
                                                 float (&D)[8], float (&dy)[8], float (&s)[8]) {
    if (a.ds) {
        vec_unpack<BF16>(static_cast<const uint4 *>(a.ds)[at], D);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) D[e] = 0.f;
    }
    if (a.dy) {
        float g[8];
        vec_unpack<BF16>(static_cast<const uint4 *>(a.dy)[at], dy);
        vec_unpack<BF16>(static_cast<const uint4 *>(a.s)[at], s);
        vec_load_f32(a.t.gamma_pre + 8 * idx, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) D[e] += st.rstd_s * (dy[e] * g[e]) - st.ms * s[e];
    }
}

template <bool BF16>
__global__ void __launch_bounds__(256)
rms_residual_bwd_stats_kernel(const RmsResidualBwdArgs a, RowStats *stats, uint32_t rows_per_gate) {
    __shared__ float red[4][8];
    const int h8 = static_cast<int>(a.t.h / 8);
    const float inv_h = 1.f / static_cast<float>(a.t.h);
    for (uint32_t row = blockIdx.x; row < a.t.rows; row += gridDim.x) {
        const int64_t base = static_cast<int64_t>(row) * h8;
        const Row r(a.t, row, rows_per_gate);
        RowStats st = {1.f, 0.f, 1.f, 0.f};
        double ss = 0.0, ws = 0.0, uu = 0.0;           // of sums of eight: their number grows with h
        for (int idx = threadIdx.x; idx < h8; idx += blockDim.x) {
            float f[8], g[8], d[8];
            if (a.dy) {
                vec_unpack<BF16>(static_cast<const uint4 *>(a.s)[base + idx], f);
                vec_unpack<BF16>(static_cast<const uint4 *>(a.dy)[base + idx], d);
                vec_load_f32(a.t.gamma_pre + 8 * idx, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] *= g[e];
                ss += static_cast<double>(dot8(f, f));
                ws += static_cast<double>(dot8(d, f));
            }
            if (a.t.gamma_post) {
                vec_unpack<BF16>(static_cast<const uint4 *>(a.u)[base + idx], f);
                uu += static_cast<double>(dot8(f, f));
            }
        }
        if (a.dy) {
            st.rstd_s = 1.f / sqrtf(block_sum(static_cast<float>(ss), red[0]) * inv_h + a.t.eps);
            st.ms = block_sum(static_cast<float>(ws), red[1]) * inv_h * st.rstd_s * (st.rstd_s * st.rstd_s);
        }
        if (a.t.gamma_post) {
            st.rstd_u = 1.f / sqrtf(block_sum(static_cast<float>(uu), red[2]) * inv_h + a.t.eps);
            double eu = 0.0;
            for (int idx = threadIdx.x; idx < h8; idx += blockDim.x) {
                float D[8], f[8], g[8], x[8];
                load_stream_grad<BF16>(a, base + idx, idx, st, D, x, g);
                vec_unpack<BF16>(static_cast<const uint4 *>(a.u)[base + idx], f);
                vec_load_f32(a.t.gamma_post + 8 * idx, g);
                if (r.gate) {
                    vec_unpack<BF16>(__ldg(r.gate + idx), x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) g[e] *= x[e];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) D[e] *= g[e];
                eu += static_cast<double>(dot8(D, f));
            }
            st.mu = block_sum(static_cast<float>(eu), red[3]) * inv_h * st.rstd_u * (st.rstd_u * st.rstd_u);
        }
        if (threadIdx.x == 0) stats[row] = st;
        __syncthreads();
    }
}

constexpr int kColThreads = 64;

// Thread = one vector of eight columns over the rows of one chunk.
template <bool BF16>
__global__ void __launch_bounds__(kColThreads)
rms_residual_bwd_cols_kernel(const RmsResidualBwdArgs a, const RowStats *stats, const RmsResidualParts parts,
                             uint32_t rows_per_gate) {
    const int h8 = static_cast<int>(a.t.h / 8), idx = blockIdx.x * kColThreads + threadIdx.x;
    const uint32_t rows = static_cast<uint32_t>(a.t.rows);
    const uint32_t r0 = rms_run_begin(blockIdx.y, parts.workers, rows), r1 = rms_run_begin(blockIdx.y + 1, parts.workers, rows);
    float gp[8], sc[8], gate[8], q[8], post[8], pre[8], scale[8];
    double one = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        gp[e] = gate[e] = 1.f;
        q[e] = post[e] = pre[e] = scale[e] = sc[e] = 0.f;
    }
    if (idx < h8) {
        if (a.t.gamma_post) vec_load_f32(a.t.gamma_post + 8 * idx, gp);
        load_scale(a.t, idx, sc);
        for (uint32_t row = r0; row < r1; ++row) {
            const int64_t at = static_cast<int64_t>(row) * h8 + idx;
            const RowStats st = stats[row];
            if (a.t.gate && (row == r0 || row % rows_per_gate == 0))
                vec_unpack<BF16>(__ldg(static_cast<const uint4 *>(a.t.gate) + static_cast<int64_t>(row / rows_per_gate) * h8 + idx), gate);
            float D[8], f[8], g[8];
            load_stream_grad<BF16>(a, at, idx, st, D, f, g);
            if (a.dy) {
#pragma unroll
                for (int e = 0; e < 8; ++e) pre[e] = fmaf(f[e], g[e] * st.rstd_s, pre[e]);
            }
            if (a.dres_scale) {
                vec_unpack<BF16>(static_cast<const uint4 *>(a.residual)[at], f);
                float part = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (a.t.res_scale_one) part = fmaf(D[e], f[e], part);
                    else scale[e] = fmaf(D[e], f[e], scale[e]);
                }
                one += static_cast<double>(part);
            }
            if (a.t.gamma_post || a.dgate) vec_unpack<BF16>(static_cast<const uint4 *>(a.u)[at], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = D[e] * sc[e];
            static_cast<uint4 *>(a.dresidual)[at] = vec_pack<BF16>(g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                q[e] = fmaf(D[e], f[e] * st.rstd_u, q[e]);
                g[e] = D[e] * gate[e];
                if (a.t.gamma_post) g[e] = st.rstd_u * (g[e] * gp[e]) - st.mu * f[e];
            }
            static_cast<uint4 *>(a.du)[at] = vec_pack<BF16>(g);
            // the sum over D * uhat gives both gradients: dgate = gamma_post * q, dgamma_post = sum of gate * q
            if (row + 1 == r1 || (a.t.gate && (row + 1) % rows_per_gate == 0)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    post[e] = fmaf(gate[e], q[e], post[e]);
                    q[e] *= gp[e];
                }
                if (a.dgate) {
                    const uint32_t gi = row / rows_per_gate, g_first = gi * rows_per_gate;
                    if (g_first >= r0 && g_first + rows_per_gate <= r1)
                        static_cast<uint4 *>(a.dgate)[static_cast<int64_t>(gi) * h8 + idx] = vec_pack<BF16>(q);
                    else
                        vec_store_f32(parts.gate + (2 * static_cast<int64_t>(blockIdx.y) + (gi == r0 / rows_per_gate ? 0 : 1)) * a.t.h + 8 * idx, q);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) q[e] = 0.f;
            }
        }
        const int64_t at = static_cast<int64_t>(blockIdx.y) * a.t.h + 8 * idx;
        if (a.dgamma_post) vec_store_f32(parts.post + at, post);
        if (a.dgamma_pre) vec_store_f32(parts.pre + at, pre);
        if (a.dres_scale && !a.t.res_scale_one) vec_store_f32(parts.scale + at, scale);
    }
    if (a.dres_scale && a.t.res_scale_one) {
        __shared__ double red[kColThreads];
        red[threadIdx.x] = one;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 1; i < kColThreads; ++i) one += red[i];
            parts.scale_one[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = one;
        }
    }
}

// The gates whose rows lie in several runs, found through the gates (by_run false: count = the gates) or through the
// runs' borders (count = the borders: the gate that begins in the run and reaches past its end); of a block's 32 slices of
// threads a power of two add the runs of one gate: as many as it has runs, at most 32.
struct SharedGates {
    uint32_t count, slices_log2;
    bool by_run;
};

// Adds the parts in a fixed order.  Block = 32 groups of four columns x 32 slices.  blockIdx.y: 0 dgamma_post,
// 1 dgamma_pre, 2 dres_scale; from 3 on 32 / slices of the shared gates each (with one gate to a block most slices had
// no run to read, and [40, 16384] with 8 gates took 24.3 us instead of 17.4, [32768, 4096] with 4096 gates
// 402 instead of 328).
template <bool BF16>
__global__ void __launch_bounds__(1024)
rms_residual_bwd_reduce_kernel(const RmsResidualBwdArgs a, const RmsResidualParts parts, uint32_t rows_per_gate, const SharedGates gates) {
    __shared__ float4 red[32][33];
    // launched under programmatic stream serialisation, as the staged kernel in front of it
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int cx = threadIdx.x & 31, sl = threadIdx.x >> 5;
    const int64_t h4 = a.t.h / 4, col = static_cast<int64_t>(blockIdx.x) * 32 + cx;
    const uint32_t rows = static_cast<uint32_t>(a.t.rows);
    if (blockIdx.y == 2 && a.dres_scale && a.t.res_scale_one) {
        if (blockIdx.x != 0) return;
        double *rd = reinterpret_cast<double *>(&red[0][0]);
        double v = 0.0;
        for (uint32_t i = threadIdx.x; i < parts.n_one; i += 1024) v += __ldcg(parts.scale_one + i);
        rd[threadIdx.x] = v;
        __syncthreads();
        for (int s = 512; s > 0; s >>= 1) {
            if (static_cast<int>(threadIdx.x) < s) rd[threadIdx.x] += rd[threadIdx.x + s];
            __syncthreads();
        }
        if (threadIdx.x == 0) a.dres_scale[0] = static_cast<float>(rd[0]);
        return;
    }
    const float *src = blockIdx.y == 0 ? parts.post : blockIdx.y == 1 ? parts.pre : parts.scale;
    float *dst = blockIdx.y == 0 ? a.dgamma_post : blockIdx.y == 1 ? a.dgamma_pre : a.dres_scale;
    uint32_t c0 = 0, c1 = parts.workers, gi = 0, slices = 32;
    bool active = col < h4;
    if (blockIdx.y >= 3) {
        slices = 1u << gates.slices_log2;
        const uint32_t i = (((blockIdx.y - 3) << 5) + sl) >> gates.slices_log2;
        active = active && i < gates.count;
        gi = min(i, gates.count - 1);
        if (gates.by_run) {
            const uint32_t border = rms_run_begin(gi + 1, parts.workers, rows);
            active = active && border % rows_per_gate != 0;
            gi = border / rows_per_gate;
        }
        // first and last run that hold rows of the gate: run c begins at floor(c * rows / workers)
        const uint64_t first = static_cast<uint64_t>(gi) * rows_per_gate, last = first + rows_per_gate - 1;
        c0 = static_cast<uint32_t>(((first + 1) * parts.workers - 1) / rows);
        c1 = static_cast<uint32_t>(((last + 1) * parts.workers - 1) / rows) + 1;
        active = active && c1 - c0 >= 2 && (!gates.by_run || c0 == i);
    } else if (!dst) {
        return;
    }
    const uint32_t slice = sl & (slices - 1);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&v](const float4 p) { v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w; };
    if (active && blockIdx.y < 3) {
#pragma unroll 4
        for (uint32_t c = sl; c < c1; c += 32) add(__ldcg(reinterpret_cast<const float4 *>(src) + c * h4 + col));
    } else if (active) {
        for (uint32_t c = c0 + slice; c < c1; c += slices) {
            const uint32_t slot = gi == rms_run_begin(c, parts.workers, rows) / rows_per_gate ? 0u : 1u;
            add(__ldcg(reinterpret_cast<const float4 *>(parts.gate) + (2 * static_cast<int64_t>(c) + slot) * h4 + col));
        }
    }
    red[sl][cx] = v;
    __syncthreads();
#pragma unroll
    for (uint32_t s = 16; s > 0; s >>= 1) {
        if (s >= slices) continue;
        if (slice < s) {
            const float4 o = red[sl + s][cx];
            float4 m = red[sl][cx];
            m.x += o.x; m.y += o.y; m.z += o.z; m.w += o.w;
            red[sl][cx] = m;
        }
        __syncthreads();
    }
    if (slice != 0 || !active) return;
    v = red[sl][cx];
    if (blockIdx.y < 3) reinterpret_cast<float4 *>(dst)[col] = v;
    else reinterpret_cast<uint2 *>(a.dgate)[gi * h4 + col] = make_uint2(ptx::pack2<BF16>(v.x, v.y), ptx::pack2<BF16>(v.z, v.w));
}

uint32_t col_blocks(int64_t h) { return static_cast<uint32_t>((h / 8 + kColThreads - 1) / kColThreads); }

// How the backward pass of a shape runs: the staged kernel where it has the width, else the statistics and column
// kernels with about 16 blocks of the latter per SM; and its workspace: [parts][statistics of the rows].
struct BwdPlan {
    bool staged;
    uint32_t workers, n_one;
    size_t post, pre, scale, one, gate, stats, total;
};
BwdPlan bwd_plan(int64_t rows, int64_t h, int64_t gate_rows, int sms) {
    const auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    BwdPlan p;
    uint32_t ctas_per_row = 1;
    p.workers = rmsnorm_residual_staged_workers(rows, h, sms, &ctas_per_row);
    p.staged = p.workers > 0;
    if (!p.staged) {
        const int64_t c = (static_cast<int64_t>(sms) * 16 + col_blocks(h) - 1) / col_blocks(h);
        p.workers = static_cast<uint32_t>(c < rows ? c : rows);
    }
    p.n_one = p.staged ? p.workers * ctas_per_row : p.workers * col_blocks(h);
    const size_t table = up(static_cast<size_t>(p.workers) * h * sizeof(float));
    p.post = 0;
    p.pre = p.post + table;
    p.scale = p.pre + table;
    p.one = p.scale + table;
    p.gate = p.one + up(p.n_one * sizeof(double));
    p.stats = p.gate + (gate_rows ? 2 * table : 0);
    p.total = p.stats + (p.staged ? 0 : up(static_cast<size_t>(rows) * sizeof(RowStats)));
    return p;
}

uint32_t rows_per_gate(const RmsResidualTerms &t) {
    return static_cast<uint32_t>(t.gate_rows ? t.rows / t.gate_rows : t.rows);
}

}  // namespace

cudaError_t rmsnorm_residual_fwd_launch(const RmsResidualFwdArgs &a, cudaStream_t stream) {
    int sms = 0;
    cudaError_t e = current_device_sm_count(&sms);
    if (e != cudaSuccess) return e;
    if (rmsnorm_residual_staged_fwd_supported(a.t, sms)) return rmsnorm_residual_staged_fwd(a, stream);
    const int64_t h8 = a.t.h / 8;
    const uint32_t rpg = rows_per_gate(a.t);
    if (h8 <= 2048) {
        const unsigned g = static_cast<unsigned>(a.t.rows);
        const int vpt = h8 <= 64 ? 1 : 2;
        int threads = static_cast<int>((h8 + vpt - 1) / vpt + 31) / 32 * 32;
        if (vpt == 1) {
            if (a.t.bf16) rms_residual_fwd_kernel<1, true><<<g, threads, 0, stream>>>(a, rpg);
            else rms_residual_fwd_kernel<1, false><<<g, threads, 0, stream>>>(a, rpg);
        } else {
            if (a.t.bf16) rms_residual_fwd_kernel<2, true><<<g, threads, 0, stream>>>(a, rpg);
            else rms_residual_fwd_kernel<2, false><<<g, threads, 0, stream>>>(a, rpg);
        }
    } else {
        const int64_t most = static_cast<int64_t>(sms) * 16;
        const unsigned g = static_cast<unsigned>(a.t.rows < most ? a.t.rows : most);
        if (a.t.bf16) rms_residual_fwd_wide_kernel<true><<<g, 1024, 0, stream>>>(a, rpg);
        else rms_residual_fwd_wide_kernel<false><<<g, 1024, 0, stream>>>(a, rpg);
    }
    return cudaGetLastError();
}

cudaError_t rmsnorm_residual_bwd_bytes(int64_t rows, int64_t h, int64_t gate_rows, size_t *bytes) {
    int sms = 0;
    const cudaError_t e = current_device_sm_count(&sms);
    if (e != cudaSuccess) return e;
    *bytes = bwd_plan(rows, h, gate_rows, sms).total;
    return cudaSuccess;
}

cudaError_t rmsnorm_residual_bwd_launch(const RmsResidualBwdArgs &a, cudaStream_t stream) {
    int sms = 0;
    cudaError_t e = current_device_sm_count(&sms);
    if (e != cudaSuccess) return e;
    const BwdPlan p = bwd_plan(a.t.rows, a.t.h, a.t.gate_rows, sms);
    const uint32_t rpg = rows_per_gate(a.t);
    uint8_t *ws = static_cast<uint8_t *>(a.workspace);
    RmsResidualParts parts = {reinterpret_cast<float *>(ws + p.post), reinterpret_cast<float *>(ws + p.pre),
                              reinterpret_cast<float *>(ws + p.scale), reinterpret_cast<float *>(ws + p.gate),
                              reinterpret_cast<double *>(ws + p.one), p.workers, p.n_one};
    if (p.staged) {
        e = rmsnorm_residual_staged_bwd(a, parts, stream);
        if (e != cudaSuccess) return e;
    } else {
        RowStats *stats = reinterpret_cast<RowStats *>(ws + p.stats);
        int64_t grid = static_cast<int64_t>(sms) * 8;
        if (grid > a.t.rows) grid = a.t.rows;
        const dim3 cols(col_blocks(a.t.h), p.workers);
        if (a.t.bf16) {
            rms_residual_bwd_stats_kernel<true><<<static_cast<unsigned>(grid), 256, 0, stream>>>(a, stats, rpg);
            rms_residual_bwd_cols_kernel<true><<<cols, kColThreads, 0, stream>>>(a, stats, parts, rpg);
        } else {
            rms_residual_bwd_stats_kernel<false><<<static_cast<unsigned>(grid), 256, 0, stream>>>(a, stats, rpg);
            rms_residual_bwd_cols_kernel<false><<<cols, kColThreads, 0, stream>>>(a, stats, parts, rpg);
        }
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    // gates whose rows lie in several runs exist only where a gate has several rows; there are at most as many of them
    // as gates, and as borders between runs
    SharedGates gates = {0, 0, false};
    if (a.dgate && rpg > 1) {
        gates.by_run = a.t.gate_rows > static_cast<int64_t>(p.workers) - 1;
        gates.count = gates.by_run ? p.workers - 1 : static_cast<uint32_t>(a.t.gate_rows);
        const int64_t runs = (static_cast<int64_t>(rpg) * p.workers + a.t.rows - 1) / a.t.rows + 1;      // of a gate, at most
        while (gates.slices_log2 < 5 && 1 << gates.slices_log2 < runs) ++gates.slices_log2;
    }
    if (!(a.dgamma_post || a.dgamma_pre || a.dres_scale || gates.count)) return cudaSuccess;
    const unsigned per_block = 32u >> gates.slices_log2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((a.t.h / 4 + 31) / 32), 3 + (gates.count + per_block - 1) / per_block, 1);
    cfg.blockDim = dim3(1024, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, a.t.bf16 ? rms_residual_bwd_reduce_kernel<true> : rms_residual_bwd_reduce_kernel<false>,
                              a, parts, rpg, gates);
}

}  // namespace pg
