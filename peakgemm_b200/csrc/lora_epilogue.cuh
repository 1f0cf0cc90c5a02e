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
// Rows as lanes: a stage of the operand ring brings the tile's rows of V, `width` of the rank, and the B_i of two or four
// slots (64 elements of k); V stays for the following stages, which bring more slots alone.  What bounds many adapters is the
// rate of a TMA load of short rows, about 1.8 ns for each row whatever its width: 100 x 14336 x 4096, 64 adapters of rank 16,
// 71 us with V in every stage, 49 so (48 with V as one term); 128 x 4096 x 4096, 64 of rank 64, 82 and 72 (64).  In large
// batches it is the tensor pipe: each adapter of a tile multiplies all of its rows, hi and lo.  1024 x 4096 x 4096, 64 of
// rank 32 in mixed order, 195 (182), of which the product alone takes 27.  Few adapters to a tile hide behind the product:
// 4096 x 14336 x 4096, 8 of rank 64 in runs, 348 us.  (All in a CUDA graph.)
// Few tokens: a part is a slot's V beside its B_i, two in a stage up to rank 16.  64 x 14336 x 4096, 32 adapters of rank 16:
// 42.4 us a call (with one term, four in a stage, 37.4), of which the product alone takes 24.5.
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
    uint32_t n, rank, rank_blocks, width;         // width: rank elements of a part
    uint32_t max_slots, group_rows, slot_rows, table_stride, mask_off;
};

template <bool LORA> struct LoraParam {};
template <> struct LoraParam<true> {
    CUtensorMap tm_v, tm_b;
    LoraDev d;
};

// What a stage holds, written by the producer before it arms the stage: bits 0-2 the 16-element steps of k in a part,
// bit 3 whether the tile ends with the stage, bits 4-6 the number of adapter parts (0: a block of the product); where V is
// kept for several stages: whether the stage brings V, is the last one to use it, is the last one of its block of the rank.
constexpr uint32_t kLoraLast = 8u, kLoraV = 0x80u, kLoraRelease = 0x100u, kLoraBlockEnd = 0x200u;
__device__ __forceinline__ uint32_t lora_steps(uint32_t info) { return info & 7u; }
__device__ __forceinline__ uint32_t lora_parts(uint32_t info) { return info >> 4 & 7u; }

// Bytes of a part's rows in the stage: of V's, of B_i's.
__device__ __forceinline__ uint32_t lora_v_row_bytes(const LoraDev &d) { return d.width * 4; }
__device__ __forceinline__ uint32_t lora_b_row_bytes(const LoraDev &d) { return d.width * 2; }

// A group's slots as the producers walk through them.
struct LoraSlots {
    int4 head = {0, 0, 0, 0};          // the table's first words: the number of slots and three adapters
    const int32_t *adapters = nullptr;

    __device__ __forceinline__ void load(const LoraDev &d, uint32_t group) {
        const int32_t *t = d.table + static_cast<size_t>(group) * d.table_stride;
        head = *reinterpret_cast<const int4 *>(t);
        adapters = t + 1;
    }
    __device__ __forceinline__ uint32_t number(const LoraDev &d) const { return min(static_cast<uint32_t>(head.x), d.max_slots); }
    __device__ __forceinline__ int32_t b_row(const LoraDev &d, uint32_t slot) const {
        const int32_t adapter = slot == 0 ? head.y : slot == 1 ? head.z : slot == 2 ? head.w : adapters[slot];
        return adapter * static_cast<int32_t>(d.n);
    }
};

// The producer's walk over a tile's adapters, slots first, first + step, ..., in `count` stages; rows are lanes.  V is the
// same for all slots: one block of the rank after the other, each with all slots, and a stage that brings V keeps it for up
// to HOLD stages of B_i's parts (HOLD below the ring's depth, so that its place is not wanted before).
template <int HOLD>
struct LoraTile : LoraSlots {
    uint32_t count = 0, rb = 0;

    __device__ __forceinline__ void open(const LoraDev &d, uint32_t first_slot = 0, uint32_t step = 1) {
        const uint32_t slots = number(d);
        first = slot = first_slot;
        slot_step = step;
        mine = left = slots > first ? (slots - first + step - 1) / step : 0u;
        rb = held = 0;
        count = d.rank_blocks * ((mine + pack(d) - 1) / pack(d));
    }
    __device__ __forceinline__ uint32_t parts(const LoraDev &d) const { return min(pack(d), left); }
    __device__ __forceinline__ bool brings_v() const { return held == 0; }
    // The word of the stage that block kb goes to (block kb1 - 1 is the product's last).
    __device__ __forceinline__ uint32_t info(const LoraDev &d, uint32_t kb, uint32_t kb1) const {
        const uint32_t last = kb + 1 >= kb1 && kb + 1 - kb1 == count ? kLoraLast : 0u;
        if (kb < kb1) return kBK / kUmmaK | last;
        const bool block_end = left <= pack(d);
        return min(d.width, d.rank - rb * d.width + kUmmaK - 1) / kUmmaK | last | parts(d) << 4 | (brings_v() ? kLoraV : 0u) |
               (block_end || held + 1 == HOLD ? kLoraRelease : 0u) | (block_end ? kLoraBlockEnd : 0u);
    }
    // The next part's first row in the up projections.
    __device__ __forceinline__ int32_t next(const LoraDev &d) {
        const int32_t row = b_row(d, slot);
        slot += slot_step;
        --left;
        return row;
    }
    __device__ __forceinline__ void end_stage() {
        if (++held == HOLD) held = 0;
        if (left) return;
        ++rb;
        slot = first;
        left = mine;
        held = 0;
    }

private:
    uint32_t first = 0, slot = 0, slot_step = 1, mine = 0, left = 0, held = 0;
    static __device__ __forceinline__ uint32_t pack(const LoraDev &d) { return kBK / d.width; }      // parts of a full stage
};

// The MMA issuer's walk over the same slots: which rows each stage's parts leave alone.  BLOCKS: uint4 of a slot's mask.
template <int BLOCKS>
struct LoraLanes {
    const uint4 *masks = nullptr;
    uint32_t first = 0, slot = 0, slot_step = 1;
    uint4 off[4][BLOCKS];              // of the next stage's parts

    __device__ __forceinline__ void open(const LoraDev &d, uint32_t group, uint32_t first_slot = 0, uint32_t step = 1) {
        masks = reinterpret_cast<const uint4 *>(d.table + static_cast<size_t>(group) * d.table_stride + d.mask_off);
        first = slot = first_slot;
        slot_step = step;
    }
    // Ahead of the wait for the stage; a slot behind the last one in use reads what nobody uses.
    __device__ __forceinline__ void load(const LoraDev &d) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t s = slot + i * slot_step;
            if (s >= d.max_slots || (i >= 2 && d.width == 32)) continue;
#pragma unroll
            for (uint32_t j = 0; j < BLOCKS; ++j) off[i][j] = __ldcg(masks + static_cast<size_t>(s) * BLOCKS + j);
        }
    }
    __device__ __forceinline__ void step(uint32_t info) {
        slot = info & kLoraBlockEnd ? first : slot + lora_parts(info) * slot_step;
    }
};

// The MMAs of a stage of B_i's parts, b_rows rows each, with V at smem_v: hi, then lo (32 bytes of a row = +2 in the >>4
// address field).  Part i leaves the lanes of off[i][block ...] alone.
template <int CTA_GROUP, int BLOCKS>
__device__ __forceinline__ void lora_stage_mma(uint32_t tmem_d, uint32_t smem_v, uint32_t smem_b, uint32_t b_rows,
                                               uint32_t idesc, uint32_t info, const LoraDev &d,
                                               const uint4 (&off)[4][BLOCKS], uint32_t block) {
    const uint32_t parts = lora_parts(info), steps = lora_steps(info), b_bytes = lora_b_row_bytes(d);
    const uint64_t dv = ptx::smem_desc_k(smem_v, lora_v_row_bytes(d));
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        if (i >= parts) break;
        const uint64_t db = ptx::smem_desc_k(smem_b + i * b_rows * b_bytes, b_bytes);
        for (uint32_t k = 0; k < 2 * steps; ++k) {
            const uint32_t lo = k >= steps ? 1u : 0u, at = k - lo * steps;
            ptx::umma_f16_lanes<CTA_GROUP>(tmem_d, dv + 2 * (lo * d.width / kUmmaK + at), db + 2 * at, idesc, &off[i][block]);
        }
    }
}

// Few tokens: V for each slot, beside its B_i in the stage.  The producer's walk over slots first, first + step, ... but
// those of `skip`, of at most 64 slots.
struct LoraBlocks : LoraSlots {
    uint32_t count = 0, slot = 0, slot_step = 1, left = 0, rb = 0;
    uint64_t skip = 0;
    int32_t v_row = 0, up_row = 0;     // of the part that next() returned

    static __device__ __forceinline__ uint32_t pack(const LoraDev &d) { return kBK / (2 * d.width); }      // parts of a full stage

    __device__ __forceinline__ void open(const LoraDev &d, uint32_t first, uint32_t step) {
        const uint32_t slots = number(d);
        slot = first;
        slot_step = step;
        rb = 0;
        left = slots > first ? (slots - first + step - 1) / step : 0u;
        if (skip) {
            for (uint32_t s = first; s < slots; s += step) left -= skip >> s & 1u;
            if (left) pass_over();
        }
        count = d.width < 32 ? (left + pack(d) - 1) / pack(d) : left * d.rank_blocks;
    }
    __device__ __forceinline__ void pass_over() {
        while (skip >> slot & 1u) slot += slot_step;
    }
    // Parts of the stage that next() will fill.
    __device__ __forceinline__ uint32_t parts(const LoraDev &d) const { return min(pack(d), left); }
    __device__ __forceinline__ uint32_t info(const LoraDev &d, uint32_t kb, uint32_t kb1) const {
        const uint32_t last = kb + 1 >= kb1 && kb + 1 - kb1 == count ? kLoraLast : 0u;
        if (kb < kb1) return kBK / kUmmaK | last;
        return min(d.width, d.rank - rb * d.width + kUmmaK - 1) / kUmmaK | last | parts(d) << 4;
    }
    // Moves to the next part; returns its first rank element, half of its first column in V.
    __device__ __forceinline__ int32_t next(const LoraDev &d) {
        v_row = static_cast<int32_t>(slot * d.slot_rows);
        up_row = b_row(d, slot);
        const int32_t x = static_cast<int32_t>(rb * d.width);
        if (++rb == d.rank_blocks) {
            rb = 0;
            slot += slot_step;
            --left;
            if (left) pass_over();
        }
        return x;
    }
};

// The MMAs of such a stage: B_i is the A operand, its rows the accumulator's; V has zeros in the rows that do not use it.
__device__ __forceinline__ void lora_slot_mma(uint32_t tmem_d, uint32_t smem_v, uint32_t smem_b, uint32_t v_rows,
                                              uint32_t idesc, uint32_t info, const LoraDev &d) {
    const uint32_t steps = lora_steps(info), v_bytes = lora_v_row_bytes(d), b_bytes = lora_b_row_bytes(d);
    for (uint32_t i = 0; i < lora_parts(info); ++i) {
        const uint64_t dv = ptx::smem_desc_k(smem_v + i * v_rows * v_bytes, v_bytes);
        const uint64_t db = ptx::smem_desc_k(smem_b + i * kBM * b_bytes, b_bytes);
        for (uint32_t k = 0; k < 2 * steps; ++k) {
            const uint32_t lo = k >= steps ? 1u : 0u, at = k - lo * steps;
            ptx::umma_f16<1>(tmem_d, db + 2 * at, dv + 2 * (lo * d.width / kUmmaK + at), idesc, 1u);
        }
    }
}

// Few tokens: a zero of V times an infinity or NaN in another row's adapter is NaN.  A CTA in whose sums that may have
// happened makes them again without the slots that hold such values (its "spoilt" slots), and adds those slots' values to
// the rows that use them here: the weights pass by twice, whatever is not finite.  64 x 14336 x 4096, 6 adapters of rank 16,
// 40 us; with one of NaN alone, or with one NaN in it, 65 (each element computed again by a warp took 1700).

// Which of the slots first, first + step, ... (at most 64 in all) are not finite in column `col`.
template <bool BF16>
__device__ __noinline__ uint64_t lora_spoilt_slots(const LoraDev &d, uint32_t col, uint32_t first, uint32_t step) {
    const uint32_t r8 = d.rank / 8, slots = min(static_cast<uint32_t>(d.table[0]), d.max_slots);
    uint64_t spoilt = 0;
    for (uint32_t s = first; s < slots; s += step) {
        const uint4 *b = reinterpret_cast<const uint4 *>(d.b) + (static_cast<int64_t>(d.table[1 + s]) * d.n + col) * r8;
        bool found = false;
#pragma unroll 4
        for (uint32_t r = 0; r < r8; ++r) {
            float g[8];
            vec_unpack<BF16>(__ldg(b + r), g);
#pragma unroll
            for (int e = 0; e < 8; ++e) found |= !(fabsf(g[e]) < __int_as_float(0x7f800000));
        }
        spoilt |= static_cast<uint64_t>(found) << s;
    }
    return spoilt;
}

// The same for a warp's 32 columns, where one of them has a NaN; every lane gets the slots of all.
template <bool BF16, int TOK>
__device__ __forceinline__ uint64_t lora_spoilt(const float (&f)[TOK], const LoraDev &d, uint32_t tokens, uint32_t col,
                                                uint32_t first, uint32_t step) {
    bool bad = false;
#pragma unroll
    for (uint32_t t = 0; t < TOK; ++t) bad |= t < tokens && f[t] != f[t];
    bad = bad && col < d.n;
    if (!__any_sync(0xffffffffu, bad)) return 0;
    const uint64_t mine = bad ? lora_spoilt_slots<BF16>(d, col, first, step) : 0;
    return static_cast<uint64_t>(__reduce_or_sync(0xffffffffu, static_cast<uint32_t>(mine >> 32))) << 32 |
           __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(mine));
}

// What token t gets in column `col` from its adapter's slot.
template <bool BF16>
__device__ __noinline__ float lora_slot_value(const LoraDev &d, uint32_t t, uint32_t col, uint32_t slot) {
    const uint32_t r8 = d.rank / 8, w8 = d.width / 8;
    const uint4 *b = reinterpret_cast<const uint4 *>(d.b) + (static_cast<int64_t>(d.table[1 + slot]) * d.n + col) * r8;
    const uint4 *v = reinterpret_cast<const uint4 *>(d.v) + (static_cast<int64_t>(slot) * d.slot_rows + t) * (2 * d.rank_blocks * w8);
    float sum = 0.f;
    for (uint32_t r = 0; r < r8; ++r) {
        const uint4 *hi = v + r / w8 * (2 * w8) + r % w8;
        float x[8], lo[8], g[8];
        vec_unpack<BF16>(*hi, x);
        vec_unpack<BF16>(hi[w8], lo);
        vec_unpack<BF16>(__ldg(b + r), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(x[e] + lo[e], g[e], sum);
    }
    return sum;
}

// Adds to the tokens' sums in column `col` what they get from those of the slots that they use.
template <bool BF16, int TOK>
__device__ __forceinline__ void lora_add_spoilt(float (&f)[TOK], const LoraDev &d, uint32_t tokens, uint32_t col, uint64_t which) {
    for (; which; which &= which - 1) {
        const uint32_t slot = __ffsll(static_cast<long long>(which)) - 1;
        const int32_t adapter = d.table[1 + slot];
#pragma unroll
        for (uint32_t t = 0; t < TOK; ++t)
            if (t < tokens && col < d.n && d.ids[t] == adapter) f[t] += lora_slot_value<BF16>(d, t, col, slot);
    }
}

}  // namespace
}  // namespace pg
