// Backward pass of the norms around a gated residual (formulas: rmsnorm_residual.cu) in one pass over the rows, for
// h <= 8192.  HBM-bound: 4 to 6 rows of 2h bytes come in and 2 or 3 go out for every row.
//   * The threads of a CTA form G groups of T threads, each a worker with a run of consecutive rows and a ring of
//     shared-memory slots; a thread owns VPT vectors of eight columns for the whole run.
//   * Operand rows (dy, s, ds, u, residual, a token's gate) arrive by cp.async.bulk, so that the bytes in flight do not
//     depend on registers.  A group's first thread issues them itself, for a slot that its group has just emptied: a
//     producer warp would be the 17th (21st) and cost every thread a quarter of its registers.
//   * Per row: the sums over s, dy, u -> one barrier -> D, dresidual and the column sums, the sum over
//     e * gamma_post * u -> second barrier, after which the slot is refilled -> du.
//   * dgate and dgamma_post both come from q = sum of D * uhat over the rows of a gate: dgate = gamma_post * q,
//     dgamma_post = sum over the gates of gate * q, so that one set of accumulators in registers serves both
//     (where every row has a gate of its own, q is a row's and the accumulators hold dgamma_post).
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

constexpr int kMaxSlots = 16;
constexpr int kMaxGroups = 8;
constexpr uint32_t kSmemMost = 232448;
constexpr uint32_t kRedBytes = 4 * 20 * 16;       // row sums: [parity][A, B] x the CTA's warps (at most 20) x 16 bytes

// The operand rows of a slot, in this order; -1: not staged.
enum { kDy, kS, kDs, kU, kRes, kGate, kOperands };

struct StagedPlan {
    int vpt, T, G, slots;         // T = 0: the width is not supported
    bool gamma_smem;              // gamma_pre and gamma_post are copied to shared memory
    int place[kOperands];         // position of an operand's row in a slot
    uint32_t row_bytes, slot_bytes, off_slot, off_red, off_bar, smem;
};

struct Group {
    int vpt, T, G;
};
// VPT * T vectors cover a row.  Two vectors a thread and 512 consumers (128 registers) up to h = 4096 and from 5128 on;
// between them one vector a thread (half of the second one would be empty).
Group make_group(int64_t rows, int64_t h, int sms) {
    const int64_t h8 = h / 8;
    Group g = {0, 0, 0};
    if (h8 > 1024) return g;
    g.vpt = h8 > 512 && h8 <= 640 ? 1 : 2;
    g.T = static_cast<int>(((h8 + g.vpt - 1) / g.vpt + 31) / 32 * 32);
    g.G = g.vpt == 1 ? 1 : 512 / g.T;
    if (g.G > kMaxGroups) g.G = kMaxGroups;
    const int64_t per_sm = (rows + sms - 1) / sms;
    if (g.G > per_sm) g.G = static_cast<int>(per_sm);
    return g;
}

template <int VPT> constexpr int max_threads() { return VPT == 1 ? 640 : 512; }

// Which terms a call has, where the kernel is compiled for them: gate 0 none, 1 one for several rows, 2 one for each row;
// a res_scale per column or not; FULL: dy, ds and gamma_post are all there.  GATE 3: whatever the call has.
template <int VPT, bool BF16, int GATE, bool SCALE_COL, bool FULL>
__global__ void __launch_bounds__(max_threads<VPT>(), 1)
rms_residual_bwd_staged_kernel(const RmsResidualBwdArgs a, const RmsResidualParts parts, const StagedPlan p,
                               uint32_t rows_per_gate, int *status) {
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t sbase = smem_u32(smem);
    const int h = static_cast<int>(a.t.h), h8 = h / 8;
    const float inv_h = 1.f / static_cast<float>(h);
    const uint32_t rows = static_cast<uint32_t>(a.t.rows);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group_warps = p.T >> 5, per_group = p.slots / p.G;
    const uint32_t bar_full = sbase + p.off_bar;
    volatile uint32_t *abort_flag = reinterpret_cast<volatile uint32_t *>(smem + p.off_bar + p.slots * 8);
    const WaitCtx ctx{abort_flag, status};
    // the next launch orders itself with griddepcontrol.wait, as this one does
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.slots; ++s) mbar_init(bar_full + s * 8, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool has_dy = FULL || a.dy, has_ds = FULL || a.ds, has_post = FULL || a.t.gamma_post;
    if (p.gamma_smem) {
        float *d = reinterpret_cast<float *>(smem);
        for (int i = threadIdx.x; i < h / 4; i += blockDim.x) {
            if (has_dy) reinterpret_cast<float4 *>(d)[i] = __ldg(reinterpret_cast<const float4 *>(a.t.gamma_pre) + i);
            if (has_post) reinterpret_cast<float4 *>(d + h)[i] = __ldg(reinterpret_cast<const float4 *>(a.t.gamma_post) + i);
        }
    }
    __syncthreads();
    const auto gamma_pre = [&](int idx, float2 (&f)[4]) {
        vec_load2(p.gamma_smem, sbase + 32 * idx, a.t.gamma_pre + 8 * idx, f);
    };
    const auto gamma_post = [&](int idx, float2 (&f)[4]) {
        vec_load2(p.gamma_smem, sbase + 4 * h + 32 * idx, a.t.gamma_post + 8 * idx, f);
    };

    const int g = threadIdx.x / p.T, t = threadIdx.x - g * p.T;
    const uint32_t worker = blockIdx.x * p.G + g;
    const uint32_t r0 = rms_run_begin(worker, parts.workers, rows), r1 = rms_run_begin(worker + 1, parts.workers, rows);
    float4 *red = reinterpret_cast<float4 *>(smem + p.off_red) + g * 4 * group_warps;       // [parity][A, B][warps]
    // one thread: the copies of `row` into the group's ring place `at`
    const auto issue = [&](uint32_t row, int at) {
        const int slot = at * p.G + g;
        const uint64_t pol = l2_policy_evict_first();              // every row is read once
        const void *src[kOperands] = {a.dy, a.s, a.ds, a.u, a.residual, a.t.gate};
        mbar_arrive_expect_tx(bar_full + slot * 8, p.slot_bytes);
#pragma unroll
        for (int o = 0; o < kOperands; ++o)
            if (p.place[o] >= 0)
                bulk_load(sbase + p.off_slot + slot * p.slot_bytes + p.place[o] * p.row_bytes,
                          static_cast<const uint4 *>(src[o]) + static_cast<int64_t>(row) * h8, p.row_bytes,
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
                if (idx < h8) gate[j] = __ldg(static_cast<const uint4 *>(a.t.gate) + static_cast<int64_t>(gi) * h8 + idx);
            }
            fresh_gate = false;
        }
        const int slot = ring * p.G + g;
        bool ok = wait_bar(bar_full + slot * 8, phase, ctx, kStRmsConsumer);
        ok = __all_sync(0xffffffffu, ok);
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
        float4 *ra = red + parity * 2 * group_warps;
        if (lane == 0) ra[warp - g * group_warps] = make_float4(ss, ws, uu, 0.f);
        if (group_barrier_or(1 + g, p.T, !ok || *abort_flag != 0)) break;
        ss = ws = uu = 0.f;
        for (int w = 0; w < group_warps; ++w) {
            const float4 v = ra[w];
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
                const int64_t at = static_cast<int64_t>(row) * h8 + idx;
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
                    vec_load2(false, 0u, a.t.res_scale + 8 * idx, x);
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
        float *rb = reinterpret_cast<float *>(red + (parity * 2 + 1) * group_warps);
        if (lane == 0) rb[warp - g * group_warps] = eu;
        if (group_barrier_or(1 + g, p.T, *abort_flag != 0)) break;
        // the whole group has the rest of the row in registers: its slot takes the next one
        if (t == 0 && row + per_group < r1) issue(row + per_group, ring);
        if (++ring == per_group) { ring = 0; phase ^= 1u; }
        float2 mu2 = zero;
        if (has_post) {
            eu = 0.f;
            for (int w = 0; w < group_warps; ++w) eu += rb[w];
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
                __stcs(static_cast<uint4 *>(a.du) + static_cast<int64_t>(row) * h8 + idx, vec_pack2<BF16>(u));
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
                    float *post = parts.post + static_cast<int64_t>(worker) * h + 8 * idx;
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
                            static_cast<uint4 *>(a.dgate)[static_cast<int64_t>(gi) * h8 + idx] = vec_pack2<BF16>(o);
                        else
                            vec_store2(parts.gate + (2 * static_cast<int64_t>(worker) + (g_first <= r0 ? 0 : 1)) * h + 8 * idx, o);
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
    const int64_t at = static_cast<int64_t>(worker) * h;
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
            // the row sums' buffers are free once the group has met again
            group_barrier_or(1 + g, p.T, false);
            double *rd = reinterpret_cast<double *>(red);
            if (lane == 0) rd[warp - g * group_warps] = one;
            group_barrier_or(1 + g, p.T, false);
            if (t == 0) {
                double sum = 0.0;
                for (int w = 0; w < group_warps; ++w) sum += rd[w];
                parts.scale_one[worker] = sum;
            }
        }
    }
    __syncthreads();
    if (*abort_flag) __nanosleep(50000);       // let bulk copies still in flight land
}

// Slots and shared memory; slots = 0 where not even two rows fit (it never happens at the widths of make_group).
StagedPlan make_staged_plan(const RmsResidualBwdArgs &a, int sms) {
    const Group g = make_group(a.t.rows, a.t.h, sms);
    StagedPlan p = {};
    p.vpt = g.vpt;
    p.T = g.T;
    p.G = g.G;
    const bool token_gate = a.t.gate && a.t.gate_rows == a.t.rows;
    const bool staged[kOperands] = {a.dy != nullptr, a.dy != nullptr, a.ds != nullptr, a.t.gamma_post || a.dgate,
                                    a.dres_scale != nullptr, token_gate};
    int n = 0;
    for (int o = 0; o < kOperands; ++o) p.place[o] = staged[o] ? n++ : -1;
    p.row_bytes = static_cast<uint32_t>(a.t.h) * 2;
    p.slot_bytes = n * p.row_bytes;
    const uint32_t fixed = kRedBytes + kMaxSlots * 8 + 16;    // sums, barriers, abort flag
    for (p.gamma_smem = true;; p.gamma_smem = false) {
        p.off_slot = p.gamma_smem ? static_cast<uint32_t>(a.t.h) * 8 : 0;
        const uint32_t room = kSmemMost - fixed - p.off_slot;
        int slots = p.slot_bytes ? static_cast<int>(room / p.slot_bytes) : 2 * p.G;
        if (slots > kMaxSlots) slots = kMaxSlots;
        p.slots = slots / p.G * p.G;
        if (p.slots >= 2 * p.G || !p.gamma_smem) break;
    }
    p.off_red = p.off_slot + p.slots * p.slot_bytes;
    p.off_bar = p.off_red + kRedBytes;
    p.smem = p.off_bar + p.slots * 8 + 16;
    return p;
}

template <int VPT, bool BF16, int GATE, bool SCALE_COL, bool FULL>
cudaError_t launch_staged(const RmsResidualBwdArgs &a, const RmsResidualParts &parts, const StagedPlan &p, int *status,
                          cudaStream_t stream) {
    auto kernel = rms_residual_bwd_staged_kernel<VPT, BF16, GATE, SCALE_COL, FULL>;
    static DeviceOnce once;
    const cudaError_t e = allow_dynamic_smem(once, kernel, static_cast<int>(kSmemMost));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(parts.workers / p.G, 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(p.T * p.G), 1, 1);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const uint32_t rpg = static_cast<uint32_t>(a.t.gate_rows ? a.t.rows / a.t.gate_rows : a.t.rows);
    return cudaLaunchKernelEx(&cfg, kernel, a, parts, p, rpg, status);
}

// Kernels compiled for the terms a training step has (dy, ds and gamma_post there); one for all other combinations.
template <int VPT, bool BF16>
cudaError_t launch_terms(const RmsResidualBwdArgs &a, const RmsResidualParts &parts, const StagedPlan &p, int *status,
                         cudaStream_t stream) {
    const bool col = a.t.res_scale && !a.t.res_scale_one;
    if (!(a.dy && a.ds && a.t.gamma_post))
        return col ? launch_staged<VPT, BF16, 3, true, false>(a, parts, p, status, stream)
                   : launch_staged<VPT, BF16, 3, false, false>(a, parts, p, status, stream);
    const int gate = !a.t.gate ? 0 : p.place[kGate] >= 0 ? 2 : 1;
    if (gate == 0) return col ? launch_staged<VPT, BF16, 0, true, true>(a, parts, p, status, stream)
                              : launch_staged<VPT, BF16, 0, false, true>(a, parts, p, status, stream);
    if (gate == 1) return col ? launch_staged<VPT, BF16, 1, true, true>(a, parts, p, status, stream)
                              : launch_staged<VPT, BF16, 1, false, true>(a, parts, p, status, stream);
    return col ? launch_staged<VPT, BF16, 2, true, true>(a, parts, p, status, stream)
               : launch_staged<VPT, BF16, 2, false, true>(a, parts, p, status, stream);
}

}  // namespace

uint32_t rmsnorm_residual_staged_workers(int64_t rows, int64_t h, int sms) {
    const Group g = make_group(rows, h, sms);
    if (g.T == 0) return 0;
    int64_t ctas = rows / g.G;                  // every worker has a row
    if (ctas > sms) ctas = sms;
    return static_cast<uint32_t>(ctas * g.G);
}

cudaError_t rmsnorm_residual_staged_bwd(const RmsResidualBwdArgs &a, const RmsResidualParts &parts, cudaStream_t stream) {
    int sms = 0, *status = nullptr;
    const cudaError_t e = rmsnorm_device(&sms, &status);
    if (e != cudaSuccess) return e;
    const StagedPlan p = make_staged_plan(a, sms);
    if (p.T == 0 || p.slots < p.G) return cudaErrorInvalidValue;
    if (p.vpt == 1)
        return a.t.bf16 ? launch_terms<1, true>(a, parts, p, status, stream) : launch_terms<1, false>(a, parts, p, status, stream);
    return a.t.bf16 ? launch_terms<2, true>(a, parts, p, status, stream) : launch_terms<2, false>(a, parts, p, status, stream);
}

}  // namespace pg
