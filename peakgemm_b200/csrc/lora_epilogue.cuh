// The adapters inside the GEMM kernels of gemm_sm100.cu.
//
// The up projection is more k: with v[t] = scale * x[t] A^T (lora.cu) a tile's accumulator gets, behind the k-blocks of
// x W^T, the rank elements of every adapter that occurs among the tile's rows:
//     acc[t, j] += sum_r v[t, r] B_i[j, r]      for the rows t that use adapter i, and no others.
// The contribution is added in fp32 before the one rounding, and the output is neither read again nor written twice.
// A tile's rows form a group; lora.cu writes the group's adapters in the order of their first row ("slots") into a table.
// Where the tile's rows are the accumulator's lanes, the table holds a mask of the rows that do not use the slot's adapter,
// and the MMA leaves those lanes as they are: V is stored once, and no row meets another one's adapter.  The kernel for few
// tokens has the tokens as columns; there V is stored for each slot, zeros in the rows of other adapters, at most 64 x 64.
// V is a sum and keeps its bits: it goes in as two 16-bit terms, hi = round(v) and lo = round(v - hi), both multiplied with
// the same B_i, which leaves an error of (eps / 2)^2 of itself.  A row of V is `width` elements of hi, the lo of the same,
// and so on; width is 16 for a rank up to 16, else 32.
// A stage of the operand ring takes 64 elements of V's rows: 32 of a rank, or two adapters of a rank up to 16.  Each is a
// part of its own in the stage, with the swizzle of its width (128 or 64 bytes for V, half as many for B_i).
// 64 x 14336 x 4096, rank 16, 32 adapters in the batch: 41.9 us, of which the product alone takes 24.5 (with V as one
// term, four adapters in a stage, 37.3).  What bounds the rest is the rate of a TMA load of short rows, about 1.8 ns for each row
// whatever its width, and the turn of a stage.  Where a tile has few adapters their blocks hide behind the product.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "gemm_common.cuh"
#include "rms_vec.cuh"

namespace pg {
namespace {

struct LoraDev {
    const int32_t *ids;         // [m]
    const int32_t *table;       // per group table_stride words: the number of slots, the slots' adapters; from mask_off on
                                // group_rows / 32 words for each slot, a bit set for every row that does not use it
    const uint16_t *v;          // [m][2 * rank_blocks * width]; slot_rows > 0: [max_slots][slot_rows][...]
    const uint16_t *b;          // [adapters][n][rank]
    const uint16_t *x, *w;      // the product's operands
    int64_t ldx, ldw;
    uint32_t k, n, rank, rank_blocks, width;      // width: rank elements of a part
    uint32_t max_slots, group_rows, slot_rows, table_stride, mask_off;
};

template <bool LORA> struct LoraParam {};
template <> struct LoraParam<true> {
    CUtensorMap tm_v, tm_b;
    LoraDev d;
};

// What a stage holds, written by the producer before it arms the stage: bits 0-2 the 16-element steps of k in a part,
// bit 3 whether the tile ends with the stage, bits 4-6 the number of adapter parts (0: a block of the product).
constexpr uint32_t kLoraLast = 8u;

// The producer's walk over a tile's adapters: slots first, first + step, ..., in `count` stages.
struct LoraBlocks {
    uint32_t count = 0, slot = 0, slot_step = 1, slots = 0, rb = 0, row0 = 0;
    int4 head = {0, 0, 0, 0};          // the table's first words: the number of slots and three adapters
    const int32_t *adapters = nullptr;
    int32_t v_row = 0, b_row = 0;      // of the part that next() returned

    static __device__ __forceinline__ uint32_t pack(const LoraDev &d) { return kBK / (2 * d.width); }      // parts of a full stage

    __device__ __forceinline__ void load(const LoraDev &d, uint32_t group) {
        const int32_t *t = d.table + static_cast<size_t>(group) * d.table_stride;
        head = *reinterpret_cast<const int4 *>(t);
        adapters = t + 1;
        row0 = group * d.group_rows;
    }
    __device__ __forceinline__ void open(const LoraDev &d, uint32_t first = 0, uint32_t step = 1) {
        slots = min(static_cast<uint32_t>(head.x), d.max_slots);
        slot = first;
        slot_step = step;
        rb = 0;
        const uint32_t mine = slots > first ? (slots - first + step - 1) / step : 0u;
        count = d.width < 32 ? (mine + pack(d) - 1) / pack(d) : mine * d.rank_blocks;
    }
    // Parts of the stage that next() will fill.
    __device__ __forceinline__ uint32_t parts(const LoraDev &d) const {
        return min(pack(d), (slots - slot + slot_step - 1) / slot_step);
    }
    // The word of the stage that block kb goes to (block kb1 - 1 is the product's last).
    __device__ __forceinline__ uint32_t info(const LoraDev &d, uint32_t kb, uint32_t kb1) const {
        const uint32_t last = kb + 1 >= kb1 && kb + 1 - kb1 == count ? kLoraLast : 0u;
        if (kb < kb1) return kBK / kUmmaK | last;
        return min(d.width, d.rank - rb * d.width + kUmmaK - 1) / kUmmaK | last | parts(d) << 4;
    }
    // Moves to the next part; returns its first rank element, half of its first column in V.
    __device__ __forceinline__ int32_t next(const LoraDev &d) {
        v_row = static_cast<int32_t>(row0 + slot * d.slot_rows);
        const int32_t adapter = slot == 0 ? head.y : slot == 1 ? head.z : slot == 2 ? head.w : adapters[slot];
        b_row = adapter * static_cast<int32_t>(d.n);
        const int32_t x = static_cast<int32_t>(rb * d.width);
        if (++rb == d.rank_blocks) {
            rb = 0;
            slot += slot_step;
        }
        return x;
    }
};

// Bytes of a part's rows in the stage: of V's, of B_i's.
__device__ __forceinline__ uint32_t lora_v_row_bytes(const LoraDev &d) { return d.width * 4; }
__device__ __forceinline__ uint32_t lora_b_row_bytes(const LoraDev &d) { return d.width * 2; }

// The MMA issuer's walk over the same slots: which rows each stage's parts leave alone.  BLOCKS: uint4 of a slot's mask.
template <int BLOCKS>
struct LoraLanes {
    const uint4 *masks = nullptr;
    uint32_t slot = 0, slot_step = 1, rb = 0;
    uint4 off[2][BLOCKS];              // of the next stage's parts

    __device__ __forceinline__ void open(const LoraDev &d, uint32_t group, uint32_t first = 0, uint32_t step = 1) {
        masks = reinterpret_cast<const uint4 *>(d.table + static_cast<size_t>(group) * d.table_stride + d.mask_off);
        slot = first;
        slot_step = step;
        rb = 0;
    }
    // Ahead of the wait for the stage; a slot behind the last one in use reads what nobody uses.
    __device__ __forceinline__ void load(const LoraDev &d) {
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i) {
            const uint32_t s = slot + i * slot_step;
            if (s >= d.max_slots || (i == 1 && d.width == 32)) continue;
#pragma unroll
            for (uint32_t j = 0; j < BLOCKS; ++j) off[i][j] = __ldcg(masks + static_cast<size_t>(s) * BLOCKS + j);
        }
    }
    __device__ __forceinline__ void step(const LoraDev &d, uint32_t parts) {
        if (d.width == 32 && ++rb < d.rank_blocks) return;
        rb = 0;
        slot += parts * slot_step;
    }
};

// The MMAs of a stage of adapter parts: V's parts from smem_v, v_rows rows each, B_i's from smem_b, b_rows rows each.
// LANES: V's rows are the accumulator's lanes, and part i leaves the lanes of off[i][first ...] alone; else V is the MMA's
// B operand and has zeros in the rows that do not use the adapter.
template <int CTA_GROUP, bool LANES, int BLOCKS>
__device__ __forceinline__ void lora_stage_mma(uint32_t tmem_d, uint32_t smem_v, uint32_t smem_b, uint32_t v_rows,
                                               uint32_t b_rows, uint32_t idesc, uint32_t info, const LoraDev &d,
                                               const uint4 (&off)[2][BLOCKS], uint32_t first) {
    const uint32_t parts = info >> 4, steps = info & 7u;
    const uint32_t v_bytes = lora_v_row_bytes(d), b_bytes = lora_b_row_bytes(d);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        if (i >= parts) break;
        const uint64_t dv = ptx::smem_desc_k(smem_v + i * v_rows * v_bytes, v_bytes);
        const uint64_t db = ptx::smem_desc_k(smem_b + i * b_rows * b_bytes, b_bytes);
        for (uint32_t k = 0; k < 2 * steps; ++k) {               // hi, then lo: 32 bytes = +2 in the >>4 address field
            const uint32_t lo = k >= steps ? 1u : 0u, at = k - lo * steps;
            const uint64_t v = dv + 2 * (lo * d.width / kUmmaK + at), b = db + 2 * at;
            if constexpr (LANES) ptx::umma_f16_lanes<CTA_GROUP>(tmem_d, v, b, idesc, &off[i][first]);
            else ptx::umma_f16<CTA_GROUP>(tmem_d, b, v, idesc, 1u);
        }
    }
}

// Few tokens: a zero of V times an infinity or NaN in another row's adapter is NaN; such an element is computed again from
// its own row's terms alone.  `acc` unless one of the batch's other adapters holds such a value in this column.
template <bool BF16>
__device__ __noinline__ float lora_exact(const LoraDev &d, uint32_t row, uint32_t col, float acc) {
    const int32_t *t = d.table;
    const int32_t slots = t[0], id = d.ids[row];
    int32_t mine = -1;
    bool other = false;
    const uint32_t r8 = d.rank / 8;
    float f[8], g[8];
    for (int32_t s = 0; s < slots; ++s) {
        const int32_t a = t[1 + s];
        if (a == id) {
            mine = s;
            continue;
        }
        const uint4 *b = reinterpret_cast<const uint4 *>(d.b) + (static_cast<int64_t>(a) * d.n + col) * r8;
        for (uint32_t r = 0; r < r8; ++r) {
            vec_unpack<BF16>(b[r], f);
            for (int e = 0; e < 8; ++e) other |= !(fabsf(f[e]) < __int_as_float(0x7f800000));     // infinity or NaN
        }
    }
    if (!other) return acc;
    float sum = 0.f;
    const uint4 *x = reinterpret_cast<const uint4 *>(d.x + static_cast<int64_t>(row) * d.ldx);
    const uint4 *w = reinterpret_cast<const uint4 *>(d.w + static_cast<int64_t>(col) * d.ldw);
    for (uint32_t c = 0; c < d.k / 8; ++c) {
        vec_unpack<BF16>(x[c], f);
        vec_unpack<BF16>(w[c], g);
        for (int e = 0; e < 8; ++e) sum = fmaf(f[e], g[e], sum);
    }
    if (mine >= 0) {
        const uint32_t w8 = d.width / 8;
        const uint4 *v = reinterpret_cast<const uint4 *>(d.v) +
                         (static_cast<int64_t>(mine) * d.slot_rows + row) * (2 * d.rank_blocks * w8);
        const uint4 *b = reinterpret_cast<const uint4 *>(d.b) + (static_cast<int64_t>(id) * d.n + col) * r8;
        for (uint32_t r = 0; r < r8; ++r) {
            const uint4 *hi = v + r / w8 * (2 * w8) + r % w8;
            float lo[8];
            vec_unpack<BF16>(*hi, f);
            vec_unpack<BF16>(hi[w8], lo);
            vec_unpack<BF16>(b[r], g);
            for (int e = 0; e < 8; ++e) sum = fmaf(f[e] + lo[e], g[e], sum);
        }
    }
    return sum;
}

}  // namespace
}  // namespace pg
