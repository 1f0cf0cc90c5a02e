// Forward pass of the norms around a gated residual (formulas: rmsnorm_residual.cu) for many rows of h <= 32768.
// HBM-bound: two or three rows of 2h bytes come in and one or two go out for every row.
//   * The threads of a CTA form G groups of T threads, each a worker that takes every W-th row; a thread owns two
//     vectors of eight columns.  Operand rows (u, residual, the row's gate) arrive by cp.async.bulk in a ring of
//     shared-memory slots per group, issued by the group's first thread for a slot that the group has just left.
//   * A row needs the sum over u^2 (A) before s can be formed (B), and the sum over s^2 before y (C).  The second sum
//     of a row is joined with the first of the next one: per row one barrier, behind it C of the row before, B, and A
//     of the row after.
//   * Rows of more than 8192 columns are shared by a cluster of 4 or 8 CTAs, at most 4096 columns each; the warps of all of
//     them send their two sums to every CTA with st.async, in two buffers in turn: who sends the sums of a row has those
//     of the row before from everyone, and everyone sent them after reading the ones before.
//   * The gains are kept in shared memory, the lower and upper halves of the vectors apart (no bank conflicts).
// In a CUDA graph: [32768, 4096] bf16, 8 gates: 181 us, 0.91 of the copy bandwidth; [65536, 2048] 0.95, [26112, 5120] 0.91-0.97,
// [16384, 8192] 0.83-0.98, with res_scale per column 0.75; [8192, 16384] 222-244 us, 0.73-0.84 (280-316 with one block per
// row), [4096, 32768] 259-284 us, 0.60-0.72 (398-436 with three passes).  A run of a few rows is bound by the latency of its first
// loads and of the gains': [1003, 5120] fp16 13.8 us where its bytes take 6.3.

#include <cuda_runtime.h>
#include <stdint.h>

#include "gemm_common.cuh"
#include "host_util.h"
#include "ptx.cuh"
#include "rms_vec.cuh"
#include "rmsnorm.h"

namespace pg {

using namespace ptx;

namespace {

enum : int { kStRmsConsumer = 12 };      // status code: a consumer gave up waiting for its row

constexpr int kVpt = 2;
constexpr int kMaxThreads = 768;         // 80 registers a thread
constexpr int kMaxGroups = 8, kMaxPerGroup = 4;
constexpr uint32_t kSmemMost = 232448;

struct FwdPlan {
    int T, G, per_group;          // threads of a group, groups, slots of a group; T = 0: the width is not supported
    int C, cols8, clusters;       // CTAs that share a row, vectors a CTA owns (the last may own fewer), clusters of the grid
    bool staged_gate;             // the row's gate comes through the ring
    uint32_t row_bytes, slot_bytes, off_slot, off_red, off_bar, smem;
};

// GATE: 0 none, 1 read by the threads, 2 through the ring.  FULL: gamma_post and y are there.
template <bool CLUSTER, bool BF16, int GATE, bool SCALE_COL, bool FULL>
__global__ void __launch_bounds__(kMaxThreads, 1)
rms_residual_fwd_staged_kernel(const RmsResidualFwdArgs a, const FwdPlan p, uint32_t workers, uint32_t rows_per_gate,
                               int *status) {
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int VPT = kVpt;
    const uint32_t sbase = smem_u32(smem);
    const int row8 = static_cast<int>(a.t.h / 8);                   // a whole row, in vectors
    const uint32_t C = CLUSTER ? p.C : 1u, cta = CLUSTER ? cluster_ctarank() : 0u;
    const int col0 = static_cast<int>(cta) * p.cols8;               // this CTA's columns, in vectors
    const int h8 = CLUSTER ? min(p.cols8, row8 - col0) : row8;
    const uint32_t row_bytes = h8 * 16, pitch = CLUSTER ? p.row_bytes : row_bytes, half = pitch;
    const float inv_h = 1.f / static_cast<float>(a.t.h);
    const uint32_t rows = static_cast<uint32_t>(a.t.rows);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group_warps = p.T >> 5, g = threadIdx.x / p.T, t = threadIdx.x - g * p.T, gw = warp - g * group_warps;
    const uint32_t bar_full = sbase + p.off_bar + g * p.per_group * 8;
    const uint32_t bar_sums = sbase + p.off_bar + (kMaxGroups * kMaxPerGroup + 2 * g) * 8;      // CLUSTER: [parity]
    volatile uint32_t *abort_flag =
        reinterpret_cast<volatile uint32_t *>(smem + p.off_bar + (kMaxGroups * kMaxPerGroup + 2 * kMaxGroups) * 8);
    const WaitCtx ctx{abort_flag, status};
    const bool has_post = FULL || a.t.gamma_post, has_y = FULL || a.y;
    // the next launch orders itself with griddepcontrol.wait, as this one does
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.G * p.per_group; ++s) mbar_init(sbase + p.off_bar + s * 8, 1);
        if constexpr (CLUSTER)
            for (int i = 0; i < 2 * p.G; ++i) mbar_init(sbase + p.off_bar + (kMaxGroups * kMaxPerGroup + i) * 8, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t ring0 = p.off_slot + g * p.per_group * p.slot_bytes;
    const uint32_t first = blockIdx.x / C * p.G + g;
    const auto issue = [&](uint32_t row, int at) {
        const uint64_t pol = l2_policy_evict_first();
        const uint32_t dst = sbase + ring0 + at * p.slot_bytes, bar = bar_full + at * 8;
        mbar_arrive_expect_tx(bar, CLUSTER ? p.slot_bytes / p.row_bytes * row_bytes : p.slot_bytes);
        bulk_load(dst, static_cast<const uint4 *>(a.u) + static_cast<int64_t>(row) * row8 + col0, row_bytes, bar, pol);
        bulk_load(dst + pitch, static_cast<const uint4 *>(a.residual) + static_cast<int64_t>(row) * row8 + col0, row_bytes, bar,
                  pol);
        if constexpr (GATE == 2)
            bulk_load(dst + 2 * pitch, static_cast<const uint4 *>(a.t.gate) + static_cast<int64_t>(row / rows_per_gate) * row8 + col0,
                      row_bytes, bar, rows_per_gate == 1 ? pol : l2_policy_evict_last());
    };
    // rows first, first + workers, ...; the first of them are on their way while the gains are copied
    if (t == 0)
        for (int i = 0; i < p.per_group && first + static_cast<uint64_t>(i) * workers < rows; ++i) issue(first + i * workers, i);
    {
        const float *src[3] = {has_post ? a.t.gamma_post : nullptr, has_y ? a.t.gamma_pre : nullptr,
                               SCALE_COL ? a.t.res_scale : nullptr};
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (src[k])
                for (int i = threadIdx.x; i < 2 * h8; i += blockDim.x)
                    reinterpret_cast<float4 *>(smem)[(2 * k + (i & 1)) * (pitch / 16) + (i >> 1)] =
                        __ldg(reinterpret_cast<const float4 *>(src[k]) + 2 * col0 + i);
    }
    __syncthreads();
    if constexpr (CLUSTER) {                   // every CTA's barriers exist before anyone signals them
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }

    float4 *red = reinterpret_cast<float4 *>(smem + p.off_red);
    float2 *sums = reinterpret_cast<float2 *>(red) + g * 2 * group_warps;          // [parity][warps]
    const uint32_t n_sums = C * group_warps;                                       // CLUSTER: [parity][CTAs][warps] of 16 bytes
    red += g * 2 * n_sums;
    const float one_scale = a.t.res_scale && a.t.res_scale_one ? __ldg(a.t.res_scale) : 1.f;
    const float2 scale_one = make_float2(one_scale, one_scale), zero = make_float2(0.f, 0.f);
    float2 s[VPT][4];
    float uu = 0.f, ss = 0.f;
    int ring = 0, ring_prev = 0;
    uint32_t phase = 0, parity = 0, sums_phase = 0;
    bool ok = true;
    const auto operand = [&](int at, int o, int idx) {
        return reinterpret_cast<const uint4 *>(smem + ring0 + at * p.slot_bytes + o * pitch)[idx];
    };
    // A: this thread's part of the sum over u^2 of the row at `at`
    const auto sum_of = [&](int at) {
        ok = __all_sync(0xffffffffu, wait_bar(bar_full + at * 8, phase, ctx, kStRmsConsumer));
        float2 x = zero;
        if (has_post) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int idx = t + p.T * j;
                if (ok && idx < h8) {
                    float2 u[4];
                    vec_unpack2<BF16>(operand(at, 0, idx), u);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x = fma2(u[e], u[e], x);
                }
            }
        }
        uu = x.x + x.y;
    };
    sum_of(0);
    const uint64_t stride = workers;
    for (uint64_t row = first;; row += stride, parity ^= 1u) {
        uint4 gate[GATE == 1 ? VPT : 1];
        if constexpr (GATE == 1) {
            if (row < rows) {
#pragma unroll
                for (int j = 0; j < VPT; ++j) {
                    const int idx = t + p.T * j;
                    if (idx < h8) gate[j] = __ldg(static_cast<const uint4 *>(a.t.gate) + static_cast<int64_t>(static_cast<uint32_t>(row) / rows_per_gate) * row8 + col0 + idx);
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            uu += __shfl_xor_sync(0xffffffffu, uu, o);
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
        }
        if constexpr (CLUSTER) {
            if (!ok) break;                    // the others run out of patience in turn
            const uint32_t bar = bar_sums + 8 * parity;
            if (t == 0) mbar_arrive_expect_tx(bar, n_sums * 16);
            if (static_cast<uint32_t>(lane) < C)
                send_sums(sbase + p.off_red + ((g * 2 + parity) * n_sums + cta * group_warps + gw) * 16, bar, lane, uu, ss, 0.f);
            ok = __all_sync(0xffffffffu, wait_bar(bar, sums_phase, ctx, kStRmsConsumer));
            if (!ok) break;
            sums_phase ^= parity;
            uu = ss = 0.f;
            for (uint32_t w = 0; w < n_sums; ++w) {
                const float4 x = red[parity * n_sums + w];
                uu += x.x;
                ss += x.y;
            }
        } else {
            if (lane == 0) sums[parity * group_warps + gw] = make_float2(uu, ss);
            if (group_barrier_or(1 + g, p.T, !ok || *abort_flag != 0)) break;
            uu = ss = 0.f;
            for (int w = 0; w < group_warps; ++w) {
                const float2 x = sums[parity * group_warps + w];
                uu += x.x;
                ss += x.y;
            }
        }
        if (row != first) {
            const uint64_t before = row - stride;
            // the group has left the slot of the row before
            if (t == 0 && before + p.per_group * stride < rows) issue(static_cast<uint32_t>(before + p.per_group * stride), ring_prev);
            if (has_y) {
                // C (rsqrt.approx is within 2 ulp of fp32; y is rounded to 16 bits)
                const float r = rsqrtf(fmaf(ss, inv_h, a.t.eps));
                const float2 r2 = make_float2(r, r);
#pragma unroll
                for (int j = 0; j < VPT; ++j) {
                    const int idx = t + p.T * j;
                    if (idx < h8) {
                        float2 gm[4];
                        vec_load2(sbase + 2 * half + 16 * idx, half, gm);
#pragma unroll
                        for (int e = 0; e < 4; ++e) gm[e] = mul2(mul2(s[j][e], r2), gm[e]);
                        __stcs(static_cast<uint4 *>(a.y) + static_cast<int64_t>(before) * row8 + col0 + idx, vec_pack2<BF16>(gm));
                    }
                }
            }
        }
        if (row >= rows) break;
        // B: s, its sum of squares
        const float r = has_post ? rsqrtf(fmaf(uu, inv_h, a.t.eps)) : 1.f;
        const float2 r2 = make_float2(r, r);
        float2 ss2 = zero;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int idx = t + p.T * j;
            if (idx < h8) {
                float2 u[4], x[4];
                vec_unpack2<BF16>(operand(ring, 0, idx), u);
                if (has_post) {
                    vec_load2(sbase + 16 * idx, half, x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[e] = mul2(mul2(u[e], r2), x[e]);
                }
                if constexpr (GATE != 0) {
                    if constexpr (GATE == 1) vec_unpack2<BF16>(gate[j], x);
                    else vec_unpack2<BF16>(operand(ring, 2, idx), x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[e] = mul2(u[e], x[e]);
                }
                vec_unpack2<BF16>(operand(ring, 1, idx), x);
                if constexpr (SCALE_COL) {
                    float2 sc[4];
                    vec_load2(sbase + 4 * half + 16 * idx, half, sc);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[j][e] = fma2(sc[e], x[e], u[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[j][e] = fma2(scale_one, x[e], u[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) ss2 = fma2(s[j][e], s[j][e], ss2);
                __stcs(static_cast<uint4 *>(a.s) + static_cast<int64_t>(row) * row8 + col0 + idx, vec_pack2<BF16>(s[j]));
            }
        }
        ss = ss2.x + ss2.y;
        uu = 0.f;
        ring_prev = ring;
        if (++ring == p.per_group) { ring = 0; phase ^= 1u; }
        if (row + stride < rows) sum_of(ring);
    }
    __syncthreads();
    if (*abort_flag) __nanosleep(50000);       // let bulk copies still in flight land
    if constexpr (CLUSTER) {                   // nobody leaves while a peer may still send sums here
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
}

FwdPlan make_plan(const RmsResidualTerms &t, int sms) {
    FwdPlan p = {};
    const int64_t row8 = t.h / 8;
    p.C = 1;
    if (row8 > 1024)
        while (p.C < 8 && row8 > 512 * p.C) p.C *= 2;
    if (row8 > 1024 && row8 > 512 * p.C) return p;
    p.clusters = rmsnorm_residual_clusters(p.C, sms);
    const int64_t h8 = (row8 + p.C - 1) / p.C;
    p.cols8 = static_cast<int>(h8);
    p.row_bytes = static_cast<uint32_t>(h8) * 16;
    const int T = static_cast<int>(((h8 + kVpt - 1) / kVpt + 31) / 32 * 32);
    p.G = kMaxThreads / T;
    if (p.G > kMaxGroups) p.G = kMaxGroups;
    p.off_slot = static_cast<uint32_t>(h8) * 32 * (t.res_scale && !t.res_scale_one ? 3 : 2);
    const uint32_t red_bytes = p.G * (T / 32) * 2 * (p.C > 1 ? 16 * p.C : 8);
    const uint32_t bar_bytes = (kMaxGroups * kMaxPerGroup + 2 * kMaxGroups) * 8 + 16, fixed = red_bytes + 16 + bar_bytes;
    // About 112 KiB of rows in flight from HBM, at least two slots for a group and three for a lone one (whose next row
    // has to be there while it works).  [rows, h] bf16, 134 M elements, us with 2 / 3 / 4 slots: h = 1024 (8 groups)
    // 196 / 180 / 192, 2048 (6) 171 / 192 / 193, 5120 (2) 202 / 163-181 / 167-188, with a gate per row 224 / 236 / 234,
    // 8192 (1) 281 / 174 / 166, with a gate per row 302 / 200 / 203.
    const bool token_gate = t.gate && t.gate_rows == t.rows;
    const int hbm_row = static_cast<int>(h8) * 16 * (token_gate ? 3 : 2) * p.G;
    const int least = p.G == 1 ? 3 : 2;
    int want = (112 * 1024 + hbm_row / 2) / hbm_row;
    if (want < least) want = least;
    if (want > kMaxPerGroup) want = kMaxPerGroup;
    const auto slots_of = [&](int operands) {
        const int n = static_cast<int>((kSmemMost - p.off_slot - fixed) / (static_cast<uint32_t>(h8) * 16 * operands)) / p.G;
        return n > want ? want : n;
    };
    // A gate of several rows is staged with each of them where the ring keeps the least number of slots; else the threads
    // read it from L2 themselves, unless the runs are short.  [16384, 8192], 8 gates, us staged / read: res_scale per column
    // (two slots) 261 / 218, a single one (three) 189 / 207; [32768, 4096] 182 / 194, [131072, 1024] 176 / 190; short runs:
    // [1003, 5120] 13.8 / 14.8.
    p.staged_gate = t.gate && (token_gate || slots_of(3) >= least || t.rows < static_cast<int64_t>(p.clusters) * p.G * 6);
    p.per_group = slots_of(p.staged_gate ? 3 : 2);
    if (p.per_group < 1) return p;
    p.slot_bytes = static_cast<uint32_t>(h8) * 16 * (p.staged_gate ? 3 : 2);
    p.T = T;
    p.off_red = p.off_slot + p.G * p.per_group * p.slot_bytes;
    p.off_bar = (p.off_red + red_bytes + 15) / 16 * 16;
    p.smem = p.off_bar + bar_bytes;
    return p;
}

template <bool CLUSTER, bool BF16, int GATE, bool SCALE_COL, bool FULL>
cudaError_t launch_fwd(const RmsResidualFwdArgs &a, const FwdPlan &p, int *status, cudaStream_t stream) {
    auto kernel = rms_residual_fwd_staged_kernel<CLUSTER, BF16, GATE, SCALE_COL, FULL>;
    static DeviceOnce once;
    const cudaError_t e = allow_dynamic_smem(once, kernel, static_cast<int>(kSmemMost));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.clusters * p.C), 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(p.T * p.G), 1, 1);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(p.C);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CLUSTER ? 2 : 1;
    const uint32_t rpg = static_cast<uint32_t>(a.t.gate_rows ? a.t.rows / a.t.gate_rows : a.t.rows);
    return cudaLaunchKernelEx(&cfg, kernel, a, p, static_cast<uint32_t>(p.clusters * p.G), rpg, status);
}

template <bool CLUSTER, bool BF16>
cudaError_t launch_terms(const RmsResidualFwdArgs &a, const FwdPlan &p, int *status, cudaStream_t stream) {
    const bool col = a.t.res_scale && !a.t.res_scale_one, full = a.t.gamma_post && a.y;
#define PG_FWD(GATE, COL)                                                             \
    (full ? launch_fwd<CLUSTER, BF16, GATE, COL, true>(a, p, status, stream)          \
          : launch_fwd<CLUSTER, BF16, GATE, COL, false>(a, p, status, stream))
    if (!a.t.gate) return col ? PG_FWD(0, true) : PG_FWD(0, false);
    if (!p.staged_gate) return col ? PG_FWD(1, true) : PG_FWD(1, false);
    return col ? PG_FWD(2, true) : PG_FWD(2, false);
#undef PG_FWD
}

}  // namespace

bool rmsnorm_residual_staged_fwd_supported(const RmsResidualTerms &t, int sms) {
    const FwdPlan p = make_plan(t, sms);
    // Every worker has a row (a CTA's groups begin with one each).  One block per row does rows of more than 8192 columns
    // sooner while each has an SM of its own: [104, 16384] 6.2 us, here 9.1; [160, 16384] 10.5, here 9.3.
    return p.T != 0 && t.rows >= static_cast<int64_t>(p.clusters) * p.G && (p.C == 1 || t.rows > sms);
}

cudaError_t rmsnorm_residual_staged_fwd(const RmsResidualFwdArgs &a, cudaStream_t stream) {
    int sms = 0, *status = nullptr;
    const cudaError_t e = rmsnorm_device(&sms, &status);
    if (e != cudaSuccess) return e;
    const FwdPlan p = make_plan(a.t, sms);
    if (p.C > 1) return a.t.bf16 ? launch_terms<true, true>(a, p, status, stream) : launch_terms<true, false>(a, p, status, stream);
    return a.t.bf16 ? launch_terms<false, true>(a, p, status, stream) : launch_terms<false, false>(a, p, status, stream);
}

}  // namespace pg
