// A projection with low-rank adapters of many requests at once: row t of the batch uses adapter i = ids[t],
//     d[t] = row_scale[t] * (a[t] * b^T + scale[i] * (a[t] * A_i^T) * B_i^T) + bias + residual[t].
//
// Two launches.  This file's kernel is the down projection, v[t] = scale * a[t] * A_i^T; the GEMM kernels of
// gemm_sm100.cu run the product and take the up projection along as further k-blocks (lora_epilogue.cuh).  The GEMM is
// launched under programmatic stream serialisation: it streams the shared weights while this kernel runs and waits for
// it only in front of the tile's last block.
//
// Few tokens, or few rank elements of many adapters, take plain fp32 dot products (lora_dot_kernel): blocks without
// set-up, a few microseconds, beside which the GEMM's CTAs fit on the same SMs.  Otherwise the tensor cores:
//
// Down projection, per 128 rows of a (one tile): the adapters that occur in the tile's group of rows are listed in the
// order of their first row; their A_i, `rank` rows of k elements each, stand below one another as the second operand,
// cut into chunks of 64 to 128 rows, as many as the grid has clusters.  A cluster computes 128 rows x a chunk with
// tcgen05 (every row of a against every listed adapter: the tensor pipe has time to spare, a and A_i are what costs),
// each CTA of the cluster a slice of k; the partial sums meet through distributed shared memory in rank order.  Each CTA
// then writes its rows of V: the scaled value as two 16-bit terms (the next product's operand type) for the
// rows that use the adapter; where V is stored for each slot, zeros for the others (selected, not multiplied: a row's NaN
// stays its own).
//
// Bound by latency and by what one SM pulls from HBM, about 55 GB/s whatever the ring's depth: some 9 us of launch, first
// loads, exchange and V, and 0.4 us per 24 KiB k-block.  128 x 4096 x 14336, 20 adapters of rank 64: 25 us alone (40 MB
// from DRAM), both launches 52 us in a CUDA graph where the product alone takes 27; 1003 x 4104 x 5128, 5 of rank 24: 55 of 41.

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gemm_common.cuh"
#include "host_util.h"
#include "lora.h"
#include "ptx.cuh"
#include "rms_vec.cuh"

namespace pg {

using namespace ptx;

namespace {

constexpr uint32_t kXBytes = kBM * kBK * 2;
constexpr uint32_t kMaxGroup = 512;

constexpr uint32_t kStages = 4;
constexpr uint32_t kMinChunk = 64, kMaxChunk = 128;             // columns (adapter rows) of a cluster's tile
constexpr uint32_t kWBytes = kMaxChunk * kBK * 2;
constexpr uint32_t kOffX = 0;
constexpr uint32_t kOffW = kOffX + kStages * kXBytes;
constexpr uint32_t kOffRecv = kOffW + kStages * kWBytes;        // [S senders][columns / 4][128 / S rows][4] fp32
constexpr uint32_t kOffBar = kOffRecv + kBM * kMaxChunk * 4;    // full[], empty[], acc_full
constexpr uint32_t kOffMisc = kOffBar + (2 * kStages + 1) * 8;  // tensor-memory slot, abort flag, slot count
constexpr uint32_t kOffPiece = kOffMisc + 16;                   // first row of A of each piece of the chunk
constexpr uint32_t kOffIds = kOffPiece + 16 * 4;                // the group's adapter ids, -1: none
constexpr uint32_t kOffSlots = kOffIds + kMaxGroup * 4;         // the adapters that occur
constexpr uint32_t kSmem = kOffSlots + kMaxGroup * 4 + 1024;
static_assert(kSmem <= 232448, "exceeds 227 KiB of shared memory");

// Eight values as two 16-bit terms: hi = round(f), lo = round(f - hi); what hi cannot hold (infinity, NaN) is hi's alone.
template <bool BF16>
__device__ __forceinline__ void split_terms(const float (&f)[8], uint4 &hi, uint4 &lo) {
    float h[8], l[8];
    hi = vec_pack<BF16>(f);
    vec_unpack<BF16>(hi, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) l[e] = fabsf(h[e]) < __int_as_float(0x7f800000) ? f[e] - h[e] : 0.f;
    lo = vec_pack<BF16>(l);
}

// The distinct ids that are not negative among `rows` rows, in the order of their first row, by one warp: 32 rows at a
// time, first against each other, then against the list so far.  Returns their number.
template <class IdAt>
__device__ __forceinline__ uint32_t list_slots(uint32_t rows, uint32_t lane, int32_t *slots, const IdAt &id_at) {
    uint32_t n = 0;
    for (uint32_t r = 0; r < rows; r += 32) {
        const int32_t id = r + lane < rows ? id_at(r + lane) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, id);       // every lane takes part
        bool fresh = id >= 0 && __ffs(same) - 1 == static_cast<int>(lane);
        for (uint32_t e = 0; e < n; ++e) fresh = fresh && slots[e] != id;
        const uint32_t who = __ballot_sync(0xffffffffu, fresh);
        if (fresh) slots[n + __popc(who & ((1u << lane) - 1u))] = id;
        n += __popc(who);
        __syncwarp();
    }
    return n;
}

struct Shrink {
    const int32_t *ids;
    const float *scale;
    int32_t *table;
    uint4 *v;
    uint32_t m, k, adapters, rank, max_slots, group_rows, slot_rows, table_stride, mask_off;      // see LoraDev
    uint32_t width, v_cols8;       // of a block of V's rows, elements; of a row, vectors of eight
    uint32_t piece;                // rows of A per load: 8 .. 64, divides rank

    // The mask word of row r of the group, and the 31 behind it, for a slot.
    __device__ __forceinline__ int32_t &mask(uint32_t group, uint32_t slot, uint32_t r) const {
        return table[static_cast<size_t>(group) * table_stride + mask_off + slot * (group_rows / 32) + r / 32];
    }
    // Where rank elements 8 r8 .. 8 r8 + 7 of V's row stand, in vectors; their lo terms are width / 8 behind.
    __device__ __forceinline__ int64_t v_at(int64_t row, uint32_t r8) const {
        const uint32_t w8 = width / 8;
        return row * v_cols8 + r8 / w8 * (2 * w8) + r8 % w8;
    }
    // The last eight of an odd number of them: the MMA reads sixteen, so eight zeros follow.
    __device__ __forceinline__ bool ends_odd(uint32_t r8) const { return (rank & 8u) && 8 * r8 + 8 == rank; }
};

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
lora_shrink_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_a, const Shrink p,
                   int *status) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t S = cluster_nctarank(), rank = cluster_ctarank();
    const uint32_t own_rows = kBM / S;                                 // rows of the tile this CTA finally owns
    const uint32_t bar_full = smem_base + kOffBar, bar_empty = bar_full + kStages * 8, bar_acc = bar_empty + kStages * 8;
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(smem + kOffMisc);
    volatile uint32_t *abort_flag = misc + 1;
    const WaitCtx ctx{abort_flag, status};
    int32_t *piece_row = reinterpret_cast<int32_t *>(smem + kOffPiece);
    int32_t *ids = reinterpret_cast<int32_t *>(smem + kOffIds), *slots = reinterpret_cast<int32_t *>(smem + kOffSlots);

    const uint32_t row0 = blockIdx.x / S * kBM;                        // the tile's first row
    const uint32_t group = row0 / p.group_rows, group0 = group * p.group_rows;
    const uint32_t k_blocks = (p.k + kBK - 1) / kBK, per = (k_blocks + S - 1) / S;
    const uint32_t kb0 = min(k_blocks, rank * per), kb1 = min(k_blocks, kb0 + per);
    const bool has_k = kb1 > kb0;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(bar_full + s * 8, 1);
            mbar_init(bar_empty + s * 8, 1);
        }
        mbar_init(bar_acc, 1);
        *abort_flag = 0;
        fence_mbar_init();
        prefetch_tensormap(&tm_x);
        prefetch_tensormap(&tm_a);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_base + kOffMisc, kMaxChunk);
        tmem_relinquish<1>();
    }
    // Everything before this launch has completed: the next launch, the GEMM, may read what they wrote at once.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // The rows of a do not depend on the list: the first of them are on their way while it is made.
    const uint32_t early = blockIdx.y == 0 ? min(kStages, kb1 - kb0) : 0u;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < early; ++i) {
            mbar_expect_tx(bar_full + i * 8, kXBytes);
            tma_load_2d_hint(smem_base + kOffX + i * kXBytes, &tm_x, bar_full + i * 8, static_cast<int32_t>((kb0 + i) * kBK),
                             static_cast<int32_t>(row0), l2_policy_evict_last());
        }
    }
    for (uint32_t i = threadIdx.x; i < p.group_rows; i += kThreads) {
        const int32_t id = group0 + i < p.m ? p.ids[group0 + i] : -1;
        ids[i] = id >= 0 && static_cast<uint32_t>(id) < p.adapters ? id : -1;
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = misc[0];
    if (warp == 2) {
        const uint32_t n = list_slots(p.group_rows, lane, slots, [&](uint32_t r) { return ids[r]; });
        if (lane == 0) misc[2] = n;
    }
    __syncthreads();
    const uint32_t n_slots = misc[2], a_rows = n_slots * p.rank;
    // The narrowest chunk (a multiple of 16, and of the pieces A comes in) with which the grid's clusters take one each:
    // 128 x 4096 x 14336 with 20 adapters of rank 64, 16 chunks of 80 on 128 CTAs instead of 20 of 64 on 160.
    const uint32_t step = max(16u, p.piece);
    const uint32_t chunk = min(kMaxChunk, max(kMinChunk, ((a_rows + gridDim.y - 1) / gridDim.y + step - 1) / step * step));
    const uint32_t chunks = (a_rows + chunk - 1) / chunk;
    if (rank == 0 && blockIdx.y == 0 && row0 == group0) {
        int32_t *t = p.table + static_cast<size_t>(group) * p.table_stride;
        if (threadIdx.x == 0) t[0] = static_cast<int32_t>(n_slots);
        for (uint32_t i = threadIdx.x; i < n_slots; i += kThreads) t[1 + i] = slots[i];
    }
    if (warp >= 2 && rank == 0 && p.slot_rows == 0) {
        // which of the tile's rows do not use a slot's adapter; the last tile answers for the rest of its group too
        const uint32_t in_group = row0 - group0, end = row0 + kBM >= p.m ? p.group_rows : in_group + kBM;
        for (uint32_t s = blockIdx.y + gridDim.y * (warp - 2); s < n_slots; s += gridDim.y * 4)
            for (uint32_t r = in_group; r < end; r += 32) {
                const uint32_t off = __ballot_sync(0xffffffffu, ids[r + lane] != slots[s]);
                if (lane == 0) p.mask(group, s, r) = off;
            }
    }
    __syncwarp();              // the cluster barrier wants whole warps
    cluster_arrive();          // every CTA of the cluster is running before anyone writes into its shared memory
    cluster_wait();

    if (chunks == 0 && threadIdx.x == 0) {             // no row of the group has an adapter: let the early loads land
        for (uint32_t i = 0; i < early; ++i) mbar_arrive(bar_full + i * 8);
        for (uint32_t i = 0; i < early; ++i)
            if (!wait_bar(bar_full + i * 8, 0, ctx, kStProducerEmpty)) break;
    }
    uint32_t stage = 0, phase = 0, acc_phase = 0;
    for (uint32_t c = blockIdx.y; c < chunks; c += gridDim.y, acc_phase ^= 1u) {
        const uint32_t live = min(chunk, a_rows - c * chunk);       // columns of this chunk that exist
        if (warp == 0) {
            if (lane == 0) {
                const uint32_t pieces = live / p.piece;
                for (uint32_t i = 0; i < pieces; ++i) {
                    const uint32_t at = c * chunk + i * p.piece, slot = at / p.rank;
                    piece_row[i] = slots[slot] * static_cast<int32_t>(p.rank) + static_cast<int32_t>(at - slot * p.rank);
                }
                const uint64_t keep = l2_policy_evict_last(), stream = l2_policy_evict_first();
                for (uint32_t kb = kb0; kb < kb1; ++kb) {
                    if (!wait_bar(bar_empty + stage * 8, phase ^ 1u, ctx, kStProducerEmpty)) break;
                    const uint32_t full = bar_full + stage * 8;
                    const bool there = c == 0 && kb - kb0 < early;
                    mbar_arrive_expect_tx(full, (there ? 0u : kXBytes) + live * kBK * 2);
                    const int32_t kx = static_cast<int32_t>(kb * kBK);
                    if (!there)
                        tma_load_2d_hint(smem_base + kOffX + stage * kXBytes, &tm_x, full, kx, static_cast<int32_t>(row0), keep);
                    for (uint32_t i = 0; i < pieces; ++i)
                        tma_load_2d_hint(smem_base + kOffW + stage * kWBytes + i * p.piece * kBK * 2, &tm_a, full, kx,
                                         piece_row[i], stream);
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
            }
            __syncwarp();
        } else if (warp == 1) {
            if (lane == 0 && has_k) {
                // columns that do not exist hold what was in shared memory; they are not stored
                const uint32_t idesc = instr_desc_f16(BF16, kBM, chunk);
                bool ok = true;
                for (uint32_t kb = kb0; kb < kb1; ++kb) {
                    ok = wait_bar(bar_full + stage * 8, phase, ctx, kStMmaFull);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint64_t dx = smem_desc_k_sw128(smem_base + kOffX + stage * kXBytes);
                    const uint64_t dw = smem_desc_k_sw128(smem_base + kOffW + stage * kWBytes);
#pragma unroll
                    for (uint32_t k = 0; k < kBK / kUmmaK; ++k)
                        umma_f16<1>(tmem, dx + 2 * k, dw + 2 * k, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
                    umma_commit<1>(bar_empty + stage * 8);
                    if (++stage == kStages) { stage = 0; phase ^= 1u; }
                }
                if (ok) umma_commit<1>(bar_acc);
            }
            __syncwarp();
        } else {
            // my partial sums of a row go to the CTA that owns it
            const uint32_t q = warp & 3u, row = q * 32u + lane;
            bool ok = has_k;
            if (has_k) {
                ok = wait_bar(bar_acc, acc_phase, ctx, kStEpiAccFull);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after_sync();
            }
            const uint32_t owner = row / own_rows;
            const uint32_t recv = mapa(smem_base + kOffRecv + (rank * (chunk / 4) * own_rows + row - owner * own_rows) * 16u, owner);
#pragma unroll 1
            for (uint32_t h = 0; h < (live + 31) / 32; ++h) {
                uint32_t v[32];
                if (ok) {
                    tmem_ld_32x32b_x32(tmem + ((q * 32u) << 16) + h * 32u, v);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0u;
                }
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j)
                    if (h * 32u + 4u * j < live)
                        st_cluster_v4(recv + (h * 8u + j) * own_rows * 16u, __uint_as_float(v[4 * j]),
                                      __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3]));
            }
            tc_fence_before_sync();
        }
        __syncwarp();
        cluster_arrive();          // all parts delivered
        cluster_wait();
        if (warp >= 2) {
            const float4 *recv = reinterpret_cast<const float4 *>(smem + kOffRecv);
            for (uint32_t i = threadIdx.x - 64; i < own_rows * (live / 8); i += 128) {
                const uint32_t g = i / own_rows, r_own = i - g * own_rows, row = row0 + rank * own_rows + r_own;
                const uint32_t in_group = row - group0;
                if (in_group >= p.group_rows || row >= p.m) continue;
                const int32_t id = ids[in_group];
                const uint32_t at = c * chunk + 8 * g, slot = at / p.rank, r = at - slot * p.rank;
                uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
                if (slots[slot] != id && p.slot_rows == 0) continue;
                if (slots[slot] == id) {
                    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    for (uint32_t s = 0; s < S; ++s) {
                        const float4 *src = recv + (s * (chunk / 4) + 2 * g) * own_rows + r_own;
                        const float4 a = src[0], b = src[own_rows];
                        f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w;
                        f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
                    }
                    const float scale = p.scale ? p.scale[id] : 1.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= scale;
                    split_terms<BF16>(f, hi, lo);
                }
                const int64_t v_row = p.slot_rows ? static_cast<int64_t>(slot) * p.slot_rows + row : row;
                uint4 *out = p.v + p.v_at(v_row, r / 8);
                out[0] = hi;
                out[p.width / 8] = lo;
                if (p.ends_odd(r / 8)) out[1] = out[p.width / 8 + 1] = make_uint4(0, 0, 0, 0);
            }
        }
        if (c + gridDim.y < chunks) {      // the receive buffer and the accumulator are free again everywhere
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            tc_fence_after_sync();
        }
    }
    __syncthreads();
    if (*abort_flag) __nanosleep(50000);
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<1>(tmem, kMaxChunk);
    }
}

constexpr uint32_t kDotRanks = 4;        // rank elements of a block: its loads of a token's row serve all of them
constexpr uint32_t kDotWarps = 8;

// v of one token and kDotRanks rank elements.  Bound by latency: every load of a thread is in flight at once for k up to
// 2048, and the row's adapter is read in parallel with the listing of its group's.
template <bool BF16>
__global__ void __launch_bounds__(kDotWarps * 32)
lora_dot_kernel(const uint4 *x, int64_t ldx8, const uint4 *a, const Shrink p) {
    __shared__ int32_t slots[kMaxGroup];
    __shared__ uint32_t s_count;
    __shared__ float red[kDotWarps][kDotRanks];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t t = blockIdx.y, r0 = blockIdx.x * kDotRanks;
    const auto checked = [&](int32_t id) { return id >= 0 && static_cast<uint32_t>(id) < p.adapters ? id : -1; };
    const int32_t id = checked(p.ids[t]);
    const uint32_t group = t / p.group_rows, group0 = group * p.group_rows, group_end = min(p.m, group0 + p.group_rows);
    if (warp == 0) {
        const uint32_t n = list_slots(group_end - group0, lane, slots, [&](uint32_t r) { return checked(p.ids[group0 + r]); });
        if (lane == 0) s_count = n;
    }
    float sum[kDotRanks] = {};
    if (id >= 0) {
        const uint32_t k8 = p.k / 8;
        const uint4 *xr = x + t * ldx8, *ar = a + (static_cast<int64_t>(id) * p.rank + r0) * k8;
#pragma unroll 2
        for (uint32_t i = threadIdx.x; i < k8; i += kDotWarps * 32) {
            const uint4 xv = __ldg(xr + i);
            uint4 av[kDotRanks];
#pragma unroll
            for (uint32_t r = 0; r < kDotRanks; ++r) av[r] = __ldg(ar + static_cast<int64_t>(r) * k8 + i);
            float f[8], g[8];
            vec_unpack<BF16>(xv, f);
#pragma unroll
            for (uint32_t r = 0; r < kDotRanks; ++r) {
                vec_unpack<BF16>(av[r], g);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[r] = fmaf(f[e], g[e], sum[r]);
            }
        }
    }
#pragma unroll
    for (uint32_t r = 0; r < kDotRanks; ++r) sum[r] = warp_sum_f32(sum[r]);
    if (lane == 0)
#pragma unroll
        for (uint32_t r = 0; r < kDotRanks; ++r) red[warp][r] = sum[r];
    __syncthreads();
    const uint32_t n = s_count;
    if (blockIdx.x == 0 && t == group0) {
        int32_t *table = p.table + static_cast<size_t>(group) * p.table_stride;
        if (threadIdx.x == 0) table[0] = static_cast<int32_t>(n);
        for (uint32_t i = threadIdx.x; i < n; i += kDotWarps * 32) table[1 + i] = slots[i];
    }
    if (blockIdx.x == 0 && p.slot_rows == 0) {          // the group's blocks share the slots' masks
        for (uint32_t s = t - group0; s < n; s += group_end - group0)
            for (uint32_t r = warp * 32; r < p.group_rows; r += kDotWarps * 32) {
                const int32_t other = group0 + r + lane < group_end ? checked(p.ids[group0 + r + lane]) : -1;
                const uint32_t off = __ballot_sync(0xffffffffu, other != slots[s]);
                if (lane == 0) p.mask(group, s, r) = off;
            }
    }
    // the scaled value in two terms; V for each slot: in the slot of the row's adapter, zeros in the others
    for (uint32_t slot = threadIdx.x; slot < n; slot += kDotWarps * 32) {
        if (slots[slot] != id && p.slot_rows == 0) continue;
        uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
        if (slots[slot] == id) {
            const float scale = p.scale ? p.scale[id] : 1.f;
            float v[8] = {};
#pragma unroll
            for (uint32_t w = 0; w < kDotWarps; ++w)
#pragma unroll
                for (uint32_t r = 0; r < kDotRanks; ++r) v[r] += red[w][r];
#pragma unroll
            for (uint32_t r = 0; r < kDotRanks; ++r) v[r] *= scale;
            split_terms<BF16>(v, hi, lo);
        }
        const int64_t row = p.slot_rows ? static_cast<int64_t>(slot) * p.slot_rows + t : t;
        uint2 *out = reinterpret_cast<uint2 *>(p.v + p.v_at(row, r0 / 8)) + r0 % 8 / 4;      // half a vector
        const uint32_t to_lo = p.width / 4;
        out[0] = make_uint2(hi.x, hi.y);
        out[to_lo] = make_uint2(lo.x, lo.y);
        if (p.ends_odd(r0 / 8)) out[2] = out[to_lo + 2] = make_uint2(0, 0);
    }
}

struct Plan {
    int64_t group_rows, groups, max_slots, slot_rows, table_stride, mask_off;
    size_t off_v, bytes;
};

Plan make_plan(int64_t m, int64_t n, int64_t k, int64_t adapters, int64_t rank, int sms) {
    Plan p;
    p.group_rows = lora_group_rows(m, n, k, sms);
    p.groups = (m + p.group_rows - 1) / p.group_rows;
    p.max_slots = adapters < p.group_rows ? adapters : p.group_rows;
    p.slot_rows = p.group_rows < kBM ? p.group_rows : 0;      // the kernel for few tokens
    p.mask_off = (1 + p.max_slots + 3) / 4 * 4;
    p.table_stride = p.mask_off + (p.slot_rows ? 0 : p.max_slots * (p.group_rows / 32));
    const int64_t v_rows = p.slot_rows ? p.max_slots * p.slot_rows : m;
    p.off_v = (static_cast<size_t>(p.groups) * p.table_stride * 4 + 255) / 256 * 256;
    p.bytes = p.off_v + static_cast<size_t>(v_rows) * lora_v_cols(rank) * 2;
    return p;
}

// Dot products read an adapter's rows once for every token, a tcgen05 launch once for every tile that uses it, but against
// all rows of the tile.  m x n x k, pool, rank, us of both launches in a CUDA graph with dot products / tcgen05:
//   64 tokens and fewer: 1 x 4096 x 4096, 8, 16 10.8 / 15.9; 64 x 4096 x 4096, 32, 64 32.3 / 44.1; 32 x 4096 x 14336, 4, 64
//   30.9 / 41.0; 16 x 4096 x 16384 (64 MiB of such reads), 16, 128 43.6 / 65.7; 64 x 4096 x 8192 (128 MiB), 1, 128 32.2 / 31.8
//   more, a large pool, mixed: 128 x 4096 x 4096, 32, 16 25.3 / 31.4; 256 x 4096 x 4096, 64, 16 (32 MiB) 39.6 / 49.7;
//   128 x 4096 x 4096 (64 MiB), 64, 64 71.5 / 71.8, 32, 64 52.0 / 46.4
//   more, a small pool: 128 x 4096 x 4096, 1, 16 19.1 / 16.6, 8, 64 31.9 / 28.2, but 256 x 4096 x 4096, 8, 16 26.7 / 29.1
bool dot_pays(int64_t m, int64_t k, int64_t rank, int64_t adapters) {
    const int64_t most = m <= 64 ? 128 : adapters > 16 ? 32 : 0;
    return m * k * rank * 2 <= most << 20;
}

// CTAs of a cluster over k: as many as keep the tiles within one wave and leave every CTA four k-blocks.  Fewer, beside
// which the persistent GEMM kernels could begin, cost more: each occupies half an SM pair, and the tiles of the pairs
// that come free late end late (1003 x 4104 x 5128, us with 1 / 2 / 4 / 8: 75 / 57 / 59 / 56).
int64_t choose_split(int64_t tiles, int64_t k_blocks, int sms) {
    int64_t split = 1;
    while (split < 8 && tiles * split * 2 <= sms && k_blocks >= 8 * split) split *= 2;
    return split;
}

}  // namespace

cudaError_t lora_workspace_bytes(int64_t m, int64_t n, int64_t k, int64_t adapters, int64_t rank, size_t *bytes) {
    int sms = 0;
    const cudaError_t e = current_device_sm_count(&sms);
    if (e != cudaSuccess) return e;
    *bytes = make_plan(m, n, k, adapters, rank, sms).bytes;
    return cudaSuccess;
}

int hgemm_lora_launch(const GemmArgs &g, const LoraArgs &l, cudaStream_t stream, cudaError_t *cuda_err) {
    const auto failed = [cuda_err](cudaError_t e) { *cuda_err = e; return static_cast<int>(kLaunchCuda); };
    int sms = 0, cc = 0, *status = nullptr;
    cudaError_t e = gemm_device(&sms, &cc, &status);
    if (e != cudaSuccess) return failed(e);
    if (cc != 10) return kLaunchNotSm100;
    const Plan p = make_plan(g.m, g.n, g.k, l.adapters, l.rank, sms);
    int32_t *table = static_cast<int32_t *>(l.workspace);
    uint8_t *v = static_cast<uint8_t *>(l.workspace) + p.off_v;

    Shrink s = {l.ids, l.scale, table, reinterpret_cast<uint4 *>(v), static_cast<uint32_t>(g.m), static_cast<uint32_t>(g.k),
                static_cast<uint32_t>(l.adapters), static_cast<uint32_t>(l.rank), static_cast<uint32_t>(p.max_slots),
                static_cast<uint32_t>(p.group_rows), static_cast<uint32_t>(p.slot_rows), static_cast<uint32_t>(p.table_stride),
                static_cast<uint32_t>(p.mask_off), lora_width(l.rank),
                static_cast<uint32_t>(lora_v_cols(l.rank) / 8), 8};
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (g.m <= 65535 && dot_pays(g.m, g.k, l.rank, l.adapters)) {
        cfg.gridDim = dim3(static_cast<unsigned>(l.rank / kDotRanks), static_cast<unsigned>(g.m), 1);
        cfg.blockDim = dim3(kDotWarps * 32, 1, 1);
        if ((e = cudaLaunchKernelEx(&cfg, g.bf16 ? lora_dot_kernel<true> : lora_dot_kernel<false>,
                                    static_cast<const uint4 *>(g.a), g.lda / 8, static_cast<const uint4 *>(l.a), s)) != cudaSuccess)
            return failed(e);
    } else {
        while (s.piece < 64 && l.rank % (2 * s.piece) == 0) s.piece *= 2;
        CUtensorMap tm_x, tm_a;
        if (!gemm_operand_map(&tm_x, g.a, g.m, g.k, g.lda, kBM, g.bf16) ||
            !gemm_operand_map(&tm_a, l.a, l.adapters * l.rank, g.k, g.k, s.piece, g.bf16))
            return failed(cudaErrorInvalidValue);
        const int64_t tiles = (g.m + kBM - 1) / kBM;
        const int64_t split = choose_split(tiles, (g.k + kBK - 1) / kBK, sms);
        // Clusters for as many chunks as there can be, up to one wave of CTAs; those without a chunk leave at once.
        int64_t chunks = (p.max_slots < g.m ? p.max_slots : g.m) * l.rank;
        chunks = (chunks + kMinChunk - 1) / kMinChunk;
        const int64_t most = sms / (tiles * split);
        if (chunks > most) chunks = most < 1 ? 1 : most;

        auto kernel = g.bf16 ? lora_shrink_kernel<true> : lora_shrink_kernel<false>;
        static DeviceOnce once[2];
        if ((e = allow_dynamic_smem(once[g.bf16 ? 1 : 0], kernel, kSmem)) != cudaSuccess) return failed(e);
        cfg.gridDim = dim3(static_cast<unsigned>(tiles * split), static_cast<unsigned>(chunks), 1);
        cfg.blockDim = dim3(kThreads, 1, 1);
        cfg.dynamicSmemBytes = kSmem;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = static_cast<unsigned>(split);
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
        if ((e = cudaLaunchKernelEx(&cfg, kernel, tm_x, tm_a, s, status)) != cudaSuccess) return failed(e);
    }

    const LoraGemm lg = {l.ids, table, v, l.b, l.adapters, l.rank, p.max_slots, p.group_rows, p.slot_rows, p.table_stride,
                         p.mask_off};
    GemmArgs with = g;
    with.lora = &lg;
    return hgemm_launch_with_lora(with, stream, cuda_err);
}

}  // namespace pg
