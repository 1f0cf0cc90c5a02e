// Backward pass of the norms around a gated residual (formulas: rmsnorm_residual.cu) in one pass over the rows, for
// h <= 32768.  HBM-bound: 4 to 6 rows of 2h bytes come in and 2 or 3 go out for every row.
//   * The threads of a CTA form G groups of T threads, each a worker with a run of consecutive rows and a ring of
//     shared-memory slots; a thread owns VPT vectors of eight columns for the whole run.
//   * Operand rows (dy, s, ds, u, residual, a token's gate) arrive by cp.async.bulk, so that the bytes in flight do not
//     depend on registers.  A group's first thread issues them itself, for a slot that its group has just emptied: a
//     producer warp would be the 17th and cost every thread a quarter of its registers.
//   * Per row: the sums over s, dy, u -> one barrier -> D, dresidual and the column sums, the sum over
//     e * gamma_post * u -> second barrier, after which the slot is refilled -> du.
//   * dgate and dgamma_post both come from q = sum of D * uhat over the rows of a gate: dgate = gamma_post * q,
//     dgamma_post = sum over the gates of gate * q, so that one set of accumulators in registers serves both
//     (where every row has a gate of its own, q is a row's and the accumulators hold dgamma_post).
//   * Rows of more than 4096 columns are shared by a cluster of 2, 4 or 8 CTAs, at most 4096 columns each: the gains and
//     a few rows fit into shared memory, and two or more rows are in work per SM, which hides the sums' latency.  The
//     warps of all CTAs send their sums to every CTA with st.async (data and arrival in one, no fence).
// In a CUDA graph: [32768, 4096] bf16, 8 gates, one res_scale: 330 us, 0.87 of the copy bandwidth; [4099, 5120] fp16, a gate per token, 75 us;
// [16384, 8192], 8 gates, res_scale per column, 437 us (0.66); [8192, 16384] 481-550 us (0.52-0.65).  What bounds it now is
// issue and latency at 16 warps an SM (half of the issue slots busy, DRAM at 55 %): 128 registers a thread hold the column sums.
// The workers' parts of the column sums go to tables that rmsnorm_residual.cu adds up in a fixed order.

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

constexpr int kMaxSlots = 2 * 8;     // two for each group
constexpr int kMaxGroups = 8;
constexpr uint32_t kSmemMost = 232448;

// The operand rows of a slot, in this order; -1: not staged.
enum { kDy, kS, kDs, kU, kRes, kGate, kOperands };

struct StagedPlan {
    int T, G, C, slots;           // threads of a group, groups, CTAs that share a row; T = 0: the width is not supported
    int cols8;                    // vectors of eight columns a CTA owns (the last one of a cluster may own fewer)
    int place[kOperands];         // position of an operand's row in a slot
    uint32_t row_bytes, slot_bytes, off_slot, off_red, off_bar, smem;
};

struct Group {
    int T, G, C, cols8, clusters;      // clusters: that fit the GPU at once
};
constexpr int kVpt = 2;                // vectors a thread owns: 128 registers a thread, 512 threads
constexpr int kMaxThreads = 512;

Group make_group(int64_t rows, int64_t h, int sms) {
    const int64_t h8 = h / 8;
    Group g = {0, 0, 1, 0, 0};
    while (g.C < 8 && h8 > 512 * g.C) g.C *= 2;
    if (h8 > 512 * g.C) return g;
    g.cols8 = static_cast<int>((h8 + g.C - 1) / g.C);
    g.T = ((g.cols8 + kVpt - 1) / kVpt + 31) / 32 * 32;
    g.G = kMaxThreads / g.T;
    if (g.G > kMaxGroups) g.G = kMaxGroups;
    g.clusters = rmsnorm_residual_clusters(g.C, sms);
    const int64_t per_cluster = (rows + g.clusters - 1) / g.clusters;
    if (g.G > per_cluster) g.G = static_cast<int>(per_cluster);
    return g;
}

// Which terms a call has, where the kernel is compiled for them: gate 0 none, 1 one for several rows, 2 one for each row;
// a res_scale per column or not; FULL: dy, ds and gamma_post are all there.  GATE 3: whatever the call has.
template <bool CLUSTER, bool BF16, int GATE, bool SCALE_COL, bool FULL>
__global__ void __launch_bounds__(kMaxThreads, 1)
rms_residual_bwd_staged_kernel(const RmsResidualBwdArgs a, const RmsResidualParts parts, const StagedPlan p,
                               uint32_t rows_per_gate, int *status) {
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t sbase = smem_u32(smem);
    constexpr int VPT = kVpt;
    const int row8 = static_cast<int>(a.t.h / 8);                   // a whole row, in vectors
    const uint32_t C = CLUSTER ? p.C : 1u, cta = CLUSTER ? cluster_ctarank() : 0u;
    const int col0 = static_cast<int>(cta) * p.cols8;               // this CTA's columns, in vectors
    const int h8 = CLUSTER ? min(p.cols8, row8 - col0) : row8;
    const uint32_t row_bytes = h8 * 16;
    const float inv_h = 1.f / static_cast<float>(a.t.h);
    const uint32_t rows = static_cast<uint32_t>(a.t.rows);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group_warps = p.T >> 5, per_group = p.slots / p.G;
    const uint32_t bar_full = sbase + p.off_bar;
    const uint32_t bar_sums = bar_full + p.slots * 8;               // CLUSTER: [group][A, B]
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + p.off_bar + (p.slots + 2 * kMaxGroups) * 8);
    const WaitCtx ctx{abort_flag, status};
    // the next launch orders itself with griddepcontrol.wait, as this one does
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.slots; ++s) mbar_init(bar_full + s * 8, 1);
        if constexpr (CLUSTER)
            for (int i = 0; i < 2 * p.G; ++i) mbar_init(bar_sums + i * 8, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool has_dy = FULL || a.dy, has_ds = FULL || a.ds, has_post = FULL || a.t.gamma_post;
    {
        const float *src[3] = {has_dy ? a.t.gamma_pre : nullptr, has_post ? a.t.gamma_post : nullptr,
                               SCALE_COL ? a.t.res_scale : nullptr};
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (src[k])
                for (int i = threadIdx.x; i < 2 * h8; i += blockDim.x)
                    reinterpret_cast<float4 *>(smem)[(2 * k + (i & 1)) * p.cols8 + (i >> 1)] =
                        __ldg(reinterpret_cast<const float4 *>(src[k]) + 2 * col0 + i);
    }
    __syncthreads();
    if constexpr (CLUSTER) {                   // every CTA's barriers exist before anyone signals them
        cluster_arrive();
        cluster_wait();
    }
    // the lower and upper halves of the vectors apart: a warp's 16-byte loads are consecutive
    const uint32_t half = 16 * p.cols8;
    const auto gamma_pre = [&](int idx, float2 (&f)[4]) { vec_load2(sbase + 16 * idx, half, f); };
    const auto gamma_post = [&](int idx, float2 (&f)[4]) { vec_load2(sbase + 2 * half + 16 * idx, half, f); };

    const int g = threadIdx.x / p.T, t = threadIdx.x - g * p.T;
    const uint32_t worker = blockIdx.x / C * p.G + g;
    const uint32_t r0 = rms_run_begin(worker, parts.workers, rows), r1 = rms_run_begin(worker + 1, parts.workers, rows);
    // row sums of the group: [parity][A, B][warps]; CLUSTER: [A, B][CTAs][warps]
    float4 *red = reinterpret_cast<float4 *>(smem + p.off_red) + g * (CLUSTER ? 2 * C : 4u) * group_warps;
    const uint32_t red_s = sbase + p.off_red + g * (CLUSTER ? 2 * C : 4u) * group_warps * 16;
    const uint32_t gw = warp - g * group_warps, sums = C * group_warps;
    // one thread: the copies of `row` into the group's ring place `at`
    const auto issue = [&](uint32_t row, int at) {
        const int slot = at * p.G + g;
        const uint64_t pol = l2_policy_evict_first();              // every row is read once
        const void *src[kOperands] = {a.dy, a.s, a.ds, a.u, a.residual, a.t.gate};
        mbar_arrive_expect_tx(bar_full + slot * 8, CLUSTER ? p.slot_bytes / p.row_bytes * row_bytes : p.slot_bytes);
#pragma unroll
        for (int o = 0; o < kOperands; ++o)
            if (p.place[o] >= 0)
                bulk_load(sbase + p.off_slot + slot * p.slot_bytes + p.place[o] * p.row_bytes,
                          static_cast<const uint4 *>(src[o]) + static_cast<int64_t>(row) * row8 + col0, row_bytes,
                          bar_full + slot * 8, pol);
    };
    if (t == 0)
        for (int i = 0; i < per_group && r0 + i < r1; ++i) issue(r0 + i, i);

    const bool token_gate = GATE == 2 || (GATE == 3 && p.place[kGate] >= 0);
    const bool group_gate = GATE == 1 || (GATE == 3 && a.t.gate && !token_gate);
    const bool needs_u = FULL || a.t.gamma_post || a.dgate;
    const float one_scale = a.t.res_scale && a.t.res_scale_one ? __ldg(a.t.res_scale) : 1.f;
    const float2 scale_one = make_float2(one_scale, one_scale), zero = make_float2(0.f, 0.f);

    float2 q[VPT][4], pre[VPT][4], scale[SCALE_COL ? VPT : 1][4];
    uint4 gate[VPT];
    double one = 0.0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        gate[j] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            q[j][e] = pre[j][e] = zero;
            if constexpr (SCALE_COL) scale[j][e] = zero;
        }
    }
    uint32_t gi = group_gate ? r0 / rows_per_gate : 0u;
    uint32_t gate_end = group_gate ? (gi + 1) * rows_per_gate : rows;
    bool fresh_gate = group_gate, first_flush = true;
    int ring = 0;
    uint32_t phase = 0, parity = 0;
    for (uint32_t row = r0; row < r1; ++row, parity ^= 1u) {
        if (fresh_gate) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int idx = t + p.T * j;
                if (idx < h8) gate[j] = __ldg(static_cast<const uint4 *>(a.t.gate) + static_cast<int64_t>(gi) * row8 + col0 + idx);
            }
            fresh_gate = false;
        }
        const int slot = ring * p.G + g;
        bool ok = wait_bar(bar_full + slot * 8, phase, ctx, kStRmsConsumer);
        ok = __all_sync(0xffffffffu, ok);
        if constexpr (CLUSTER) {
            if (!ok) break;                        // the others run out of patience in turn
            if (t == 0) {
                mbar_arrive_expect_tx(bar_sums + 16 * g, sums * 16);
                mbar_arrive_expect_tx(bar_sums + 16 * g + 8, sums * 16);
            }
        }
        const uint8_t *base = smem + p.off_slot + slot * p.slot_bytes;
        const auto operand = [&](int o, int idx) {
            return reinterpret_cast<const uint4 *>(base + p.place[o] * p.row_bytes)[idx];
        };
        // A: sums over the row
        uint4 dyv[VPT], sv[VPT], uv[VPT];
        float2 ss2 = zero, ws2 = zero, uu2 = zero;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int idx = t + p.T * j;
            dyv[j] = sv[j] = uv[j] = make_uint4(0, 0, 0, 0);
            if (ok && idx < h8) {
                if (has_dy) {
                    dyv[j] = operand(kDy, idx);
                    sv[j] = operand(kS, idx);
                    float2 s[4], d[4], gm[4];
                    vec_unpack2<BF16>(sv[j], s);
                    vec_unpack2<BF16>(dyv[j], d);
                    gamma_pre(idx, gm);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        ss2 = fma2(s[e], s[e], ss2);
                        ws2 = fma2(mul2(d[e], gm[e]), s[e], ws2);
                    }
                }
                if (needs_u) {
                    uv[j] = operand(kU, idx);
                    float2 u[4];
                    vec_unpack2<BF16>(uv[j], u);
#pragma unroll
                    for (int e = 0; e < 4; ++e) uu2 = fma2(u[e], u[e], uu2);
                }
            }
        }
        float ss = warp_sum_f32(ss2.x + ss2.y), ws = warp_sum_f32(ws2.x + ws2.y), uu = warp_sum_f32(uu2.x + uu2.y);
        if constexpr (CLUSTER) {
            if (static_cast<uint32_t>(lane) < C)
                send_sums(red_s + (cta * group_warps + gw) * 16, bar_sums + 16 * g, lane, ss, ws, uu);
            ok = __all_sync(0xffffffffu, wait_bar(bar_sums + 16 * g, parity, ctx, kStRmsConsumer));
            if (!ok) break;
        } else {
            if (lane == 0) red[parity * 2 * group_warps + gw] = make_float4(ss, ws, uu, 0.f);
            if (group_barrier_or(1 + g, p.T, !ok || *abort_flag != 0)) break;
        }
        ss = ws = uu = 0.f;
        for (uint32_t w = 0; w < sums; ++w) {
            const float4 v = red[(CLUSTER ? 0 : parity * 2 * group_warps) + w];
            ss += v.x;
            ws += v.y;
            uu += v.z;
        }
        // rsqrt.approx is within 2 ulp of fp32; the gradients are rounded to 16 bits or bounded by 2^-17
        const float rs = rsqrtf(fmaf(ss, inv_h, a.t.eps)), ru = has_post ? rsqrtf(fmaf(uu, inv_h, a.t.eps)) : 1.f;
        const float ms = -(ws * inv_h * rs * (rs * rs));
        const float2 rs2 = make_float2(rs, rs), ms2 = make_float2(ms, ms), ru2 = make_float2(ru, ru);
        // B: D and all that needs no further sum.  v = rstd(u) * e * gamma_post, so that du = v - rstd(u)^2 mean(v u) u.
        float2 v[VPT][4], eu2 = zero, part = zero;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int idx = t + p.T * j;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j][e] = zero;
            if (idx < h8) {
                float2 D[4], f[4], x[4];
                const int64_t at = static_cast<int64_t>(row) * row8 + col0 + idx;
                if (has_ds) {
                    vec_unpack2<BF16>(operand(kDs, idx), D);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) D[e] = zero;
                }
                if (has_dy) {
                    float2 gm[4];
                    vec_unpack2<BF16>(dyv[j], x);
                    vec_unpack2<BF16>(sv[j], f);
                    gamma_pre(idx, gm);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = mul2(x[e], rs2);
                        pre[j][e] = fma2(x[e], f[e], pre[j][e]);
                        D[e] = fma2(ms2, f[e], fma2(x[e], gm[e], D[e]));
                    }
                }
                if (a.dres_scale) {
                    vec_unpack2<BF16>(operand(kRes, idx), f);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (SCALE_COL) scale[j][e] = fma2(D[e], f[e], scale[j][e]);
                        else part = fma2(D[e], f[e], part);
                    }
                }
                if constexpr (SCALE_COL) {
                    vec_load2(sbase + 4 * half + 16 * idx, half, x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = mul2(x[e], D[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = mul2(D[e], scale_one);
                }
                __stcs(static_cast<uint4 *>(a.dresidual) + at, vec_pack2<BF16>(x));
                vec_unpack2<BF16>(uv[j], f);
                float2 gp[4];
                if (has_post) gamma_post(idx, gp);
                if (token_gate) {
                    vec_unpack2<BF16>(operand(kGate, idx), x);
                    if (a.dgate) {
                        float2 dg[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            dg[e] = mul2(mul2(D[e], ru2), f[e]);
                            if (has_post) dg[e] = mul2(dg[e], gp[e]);
                        }
                        __stcs(static_cast<uint4 *>(a.dgate) + at, vec_pack2<BF16>(dg));
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) D[e] = mul2(D[e], x[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    D[e] = mul2(D[e], ru2);
                    q[j][e] = fma2(D[e], f[e], q[j][e]);
                }
                if (group_gate) {
                    vec_unpack2<BF16>(gate[j], x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) D[e] = mul2(D[e], x[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[j][e] = has_post ? mul2(D[e], gp[e]) : D[e];
                    eu2 = fma2(v[j][e], f[e], eu2);
                }
            }
        }
        if constexpr (!SCALE_COL) one += static_cast<double>(part.x + part.y);
        // C: du
        float eu = warp_sum_f32(eu2.x + eu2.y);
        const float4 *rb = red + (CLUSTER ? sums : (parity * 2 + 1) * group_warps);
        if constexpr (CLUSTER) {
            if (static_cast<uint32_t>(lane) < C)
                send_sums(red_s + (sums + cta * group_warps + gw) * 16, bar_sums + 16 * g + 8, lane, eu, 0.f, 0.f);
            ok = __all_sync(0xffffffffu, wait_bar(bar_sums + 16 * g + 8, parity, ctx, kStRmsConsumer));
            if (!ok) break;
        } else {
            if (lane == 0) red[(parity * 2 + 1) * group_warps + gw].x = eu;
            if (group_barrier_or(1 + g, p.T, *abort_flag != 0)) break;
        }
        // the whole group has the rest of the row in registers: its slot takes the next one
        if (t == 0 && row + per_group < r1) issue(row + per_group, ring);
        if (++ring == per_group) { ring = 0; phase ^= 1u; }
        float2 mu2 = zero;
        if (has_post) {
            eu = 0.f;
            for (uint32_t w = 0; w < sums; ++w) eu += rb[w].x;
            const float mu = -(eu * inv_h * ru * ru);
            mu2 = make_float2(mu, mu);
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int idx = t + p.T * j;
            if (idx < h8) {
                float2 u[4];
                vec_unpack2<BF16>(uv[j], u);
#pragma unroll
                for (int e = 0; e < 4; ++e) u[e] = has_post ? fma2(mu2, u[e], v[j][e]) : v[j][e];
                __stcs(static_cast<uint4 *>(a.du) + static_cast<int64_t>(row) * row8 + col0 + idx, vec_pack2<BF16>(u));
            }
        }
        // the end of a gate's rows, or of the run
        if (group_gate && (row + 1 == gate_end || row + 1 == r1)) {
            const uint32_t g_first = gi * rows_per_gate;
            const bool whole = g_first >= r0 && gate_end <= r1;
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int idx = t + p.T * j;
                if (idx < h8) {
                    float2 x[4], o[4];
                    float *post = parts.post + static_cast<int64_t>(worker) * a.t.h + 8 * (col0 + idx);
                    if (a.dgamma_post) {
                        vec_unpack2<BF16>(gate[j], x);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o[e] = fma2(x[e], q[j][e], first_flush ? zero : reinterpret_cast<const float2 *>(post)[e]);
                        vec_store2(post, o);
                    }
                    if (a.dgate) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] = q[j][e];
                        if (has_post) {
                            gamma_post(idx, x);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[e] = mul2(o[e], x[e]);
                        }
                        if (whole)
                            static_cast<uint4 *>(a.dgate)[static_cast<int64_t>(gi) * row8 + col0 + idx] = vec_pack2<BF16>(o);
                        else
                            vec_store2(parts.gate + (2 * static_cast<int64_t>(worker) + (g_first <= r0 ? 0 : 1)) * a.t.h + 8 * (col0 + idx), o);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) q[j][e] = zero;
                }
            }
            first_flush = false;
            ++gi;
            gate_end += rows_per_gate;
            fresh_gate = true;
        }
    }
    const int64_t at = static_cast<int64_t>(worker) * a.t.h + 8 * col0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int idx = t + p.T * j;
        if (idx < h8) {
            if (a.dgamma_post && !group_gate) vec_store2(parts.post + at + 8 * idx, q[j]);
            if (a.dgamma_pre) vec_store2(parts.pre + at + 8 * idx, pre[j]);
            if constexpr (SCALE_COL)
                if (a.dres_scale) vec_store2(parts.scale + at + 8 * idx, scale[j]);
        }
    }
    if constexpr (!SCALE_COL) {
        if (a.dres_scale) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
            double *rd = reinterpret_cast<double *>(smem + p.off_slot + g * p.slot_bytes);     // the group's ring is idle
            group_barrier_or(1 + g, p.T, false);
            if (lane == 0) rd[gw] = one;
            group_barrier_or(1 + g, p.T, false);
            if (t == 0) {
                double sum = 0.0;
                for (int w = 0; w < group_warps; ++w) sum += rd[w];
                parts.scale_one[worker * C + cta] = sum;
            }
        }
    }
    __syncthreads();
    if (*abort_flag) __nanosleep(50000);       // let bulk copies still in flight land
    if constexpr (CLUSTER) {                   // nobody leaves while a peer may still send sums here
        __syncwarp();
        cluster_arrive();
        cluster_wait();
    }
}

// Slots and shared memory: the gains (and a res_scale per column), the ring, row sums, barriers, abort flag.
StagedPlan make_staged_plan(const RmsResidualBwdArgs &a, int sms) {
    const Group g = make_group(a.t.rows, a.t.h, sms);
    StagedPlan p = {};
    p.T = g.T;
    p.G = g.G;
    p.C = g.C;
    p.cols8 = g.cols8;
    if (g.T == 0) return p;
    const bool token_gate = a.t.gate && a.t.gate_rows == a.t.rows;
    const bool staged[kOperands] = {a.dy != nullptr, a.dy != nullptr, a.ds != nullptr, a.t.gamma_post || a.dgate,
                                    a.dres_scale != nullptr, token_gate};
    int n = 0;
    for (int o = 0; o < kOperands; ++o) p.place[o] = staged[o] ? n++ : -1;
    p.row_bytes = static_cast<uint32_t>(g.cols8) * 16;
    p.slot_bytes = n * p.row_bytes;
    p.off_slot = static_cast<uint32_t>(g.cols8) * 32 * (a.t.res_scale && !a.t.res_scale_one ? 3 : 2);
    const uint32_t red_bytes = g.G * (g.T / 32) * 16 * (g.C > 1 ? 2 * g.C : 4);
    const uint32_t bar_bytes = (kMaxSlots + 2 * kMaxGroups) * 8 + 16;
    int slots = static_cast<int>((kSmemMost - p.off_slot - red_bytes - bar_bytes) / p.slot_bytes);
    // Two rows per group, the one in work and the next: with three, [32768, 4096] bf16 without a gate takes 316 us
    // instead of 278, [16384, 8192] 417 instead of 347; with one, 490 instead of 402 with a gate per token.
    if (slots > 2 * p.G) slots = 2 * p.G;
    p.slots = slots / p.G * p.G;                // one or more for each group (six operands of 8 KiB: three in all)
    p.off_red = p.off_slot + p.slots * p.slot_bytes;
    p.off_bar = p.off_red + red_bytes;
    p.smem = p.off_bar + bar_bytes;
    return p;
}

template <bool CLUSTER, bool BF16, int GATE, bool SCALE_COL, bool FULL>
cudaError_t launch_staged(const RmsResidualBwdArgs &a, const RmsResidualParts &parts, const StagedPlan &p, int *status,
                          cudaStream_t stream) {
    auto kernel = rms_residual_bwd_staged_kernel<CLUSTER, BF16, GATE, SCALE_COL, FULL>;
    static DeviceOnce once;
    const cudaError_t e = allow_dynamic_smem(once, kernel, static_cast<int>(kSmemMost));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(parts.workers / p.G * p.C, 1, 1);
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
    return cudaLaunchKernelEx(&cfg, kernel, a, parts, p, rpg, status);
}

// Kernels compiled for the terms a training step has (dy, ds and gamma_post there); one for all other combinations.
template <bool CLUSTER, bool BF16>
cudaError_t launch_terms(const RmsResidualBwdArgs &a, const RmsResidualParts &parts, const StagedPlan &p, int *status,
                         cudaStream_t stream) {
    const bool col = a.t.res_scale && !a.t.res_scale_one;
    if (!(a.dy && a.ds && a.t.gamma_post))
        return col ? launch_staged<CLUSTER, BF16, 3, true, false>(a, parts, p, status, stream)
                   : launch_staged<CLUSTER, BF16, 3, false, false>(a, parts, p, status, stream);
    const int gate = !a.t.gate ? 0 : p.place[kGate] >= 0 ? 2 : 1;
    if (gate == 0) return col ? launch_staged<CLUSTER, BF16, 0, true, true>(a, parts, p, status, stream)
                              : launch_staged<CLUSTER, BF16, 0, false, true>(a, parts, p, status, stream);
    if (gate == 1) return col ? launch_staged<CLUSTER, BF16, 1, true, true>(a, parts, p, status, stream)
                              : launch_staged<CLUSTER, BF16, 1, false, true>(a, parts, p, status, stream);
    return col ? launch_staged<CLUSTER, BF16, 2, true, true>(a, parts, p, status, stream)
               : launch_staged<CLUSTER, BF16, 2, false, true>(a, parts, p, status, stream);
}

}  // namespace

// Clusters of C CTAs that the device holds at once: fewer than sms / C, since a cluster's CTAs share a GPC.  With one
// that has to wait for another to end, a call takes almost twice as long: [8192, 16384] bf16, 8 gates, 806 us with sms / 4
// clusters of 4, 481 with those that fit.
int rmsnorm_residual_clusters(int C, int sms) {
    if (C == 1) return sms;
    static DeviceOnce once;
    static int table[kMaxDevices][3] = {};
    int dev = 0;
    const auto fill = [&]() {
        auto kernel = rms_residual_bwd_staged_kernel<true, true, 3, true, false>;       // they differ in nothing that counts here
        for (int i = 0; i < 3; ++i) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(static_cast<unsigned>(sms / (2 << i) * (2 << i)), 1, 1);
            cfg.blockDim = dim3(kMaxThreads, 1, 1);
            cfg.dynamicSmemBytes = kSmemMost;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 2u << i;
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMost));
            if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&table[dev][i], kernel, &cfg);
            if (e != cudaSuccess) return e;
        }
        return cudaSuccess;
    };
    int n = 0;
    if (current_device(&dev) == cudaSuccess && once.run(dev, fill) == cudaSuccess) n = table[dev][C == 2 ? 0 : C == 4 ? 1 : 2];
    else cudaGetLastError();
    return n < 1 ? 1 : n;
}

uint32_t rmsnorm_residual_staged_workers(int64_t rows, int64_t h, int sms, uint32_t *ctas_per_row) {
    const Group g = make_group(rows, h, sms);
    *ctas_per_row = static_cast<uint32_t>(g.C);
    if (g.T == 0) return 0;
    int64_t clusters = rows / g.G;                  // every worker has a row
    if (clusters > g.clusters) clusters = g.clusters;
    return static_cast<uint32_t>(clusters * g.G);
}

cudaError_t rmsnorm_residual_staged_bwd(const RmsResidualBwdArgs &a, const RmsResidualParts &parts, cudaStream_t stream) {
    int sms = 0, *status = nullptr;
    const cudaError_t e = rmsnorm_device(&sms, &status);
    if (e != cudaSuccess) return e;
    const StagedPlan p = make_staged_plan(a, sms);
    if (p.T == 0 || p.slots == 0 || parts.workers % p.G != 0) return cudaErrorInvalidValue;
    if (p.C > 1)
        return a.t.bf16 ? launch_terms<true, true>(a, parts, p, status, stream) : launch_terms<true, false>(a, parts, p, status, stream);
    return a.t.bf16 ? launch_terms<false, true>(a, parts, p, status, stream) : launch_terms<false, false>(a, parts, p, status, stream);
}

}  // namespace pg
