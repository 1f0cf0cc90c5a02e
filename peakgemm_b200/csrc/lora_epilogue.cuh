// The adapters inside the GEMM kernels of gemm_sm100.cu.
//
// The up projection is more k: with v[t] = scale * x[t] A^T (lora.cu) a tile's accumulator gets, behind the k-blocks of
// x W^T, the rank elements of every adapter that occurs among the tile's rows:
//     acc[t, j] += sum_r V[t, r] B_i[j, r],     V = v for the rows t that use adapter i, zeros for the others.
// The contribution is added in fp32 before the one rounding, and the output is neither read again nor written twice.
// A tile's rows form a group; lora.cu writes the group's adapters in the order of their first row ("slots") into a table
// and the masked V of each slot, [group rows, rank], next to it.
// V is a sum and keeps its bits: it goes in as two 16-bit terms, hi = round(v) and lo = round(v - hi), both multiplied with
// the same B_i, which leaves an error of (eps / 2)^2 of itself.  A row of V is `width` elements of hi, the lo of the same,
// and so on; width is 16 for a rank up to 16, else 32.
// A stage of the operand ring takes 64 elements of V's rows: 32 of a rank, or two adapters of a rank up to 16.  Each is a
// part of its own in the stage, with the swizzle of its width (128 or 64 bytes for V, half as many for B_i).  64 x 14336 x 4096, rank 16, 32 adapters in the batch: 41.9 us, of which the product alone takes 24.5 (with V as one term,
// four adapters in a stage, 37.3).  What bounds the rest is the rate of a TMA load of short rows, about 1.8 ns for each row
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
    const int32_t *table;       // per group table_stride words: the number of slots, then the slots' adapters
    const uint16_t *v;          // [groups][max_slots][group_rows][2 * rank_blocks * width]
    const uint16_t *b;          // [adapters][n][rank]
    const uint16_t *x, *w;      // the product's operands
    int64_t ldx, ldw;
    uint32_t k, n, rank, rank_blocks, width, max_slots, group_rows, table_stride;     // width: rank elements of a part
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
    uint32_t count = 0, slot = 0, slot_step = 1, slots = 0, rb = 0, base = 0;
    int4 head = {0, 0, 0, 0};          // the table's first words: the number of slots and three adapters
    const int32_t *adapters = nullptr;
    int32_t v_row = 0, b_row = 0;      // of the part that next() returned

    static __device__ __forceinline__ uint32_t pack(const LoraDev &d) { return kBK / (2 * d.width); }      // parts of a full stage

    __device__ __forceinline__ void load(const LoraDev &d, uint32_t group) {
        const int32_t *t = d.table + static_cast<size_t>(group) * d.table_stride;
        head = *reinterpret_cast<const int4 *>(t);
        adapters = t + 1;
        base = group * d.max_slots;
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
        v_row = static_cast<int32_t>((base + slot) * d.group_rows);
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

// Bytes of a part in the stage: a row of V's operand, a row of B_i's.
__device__ __forceinline__ uint32_t lora_v_row_bytes(const LoraDev &d) { return d.width * 4; }
__device__ __forceinline__ uint32_t lora_b_row_bytes(const LoraDev &d) { return d.width * 2; }

// The MMAs of a stage of adapter parts: V's parts from smem_v, v_rows rows each, B_i's from smem_b, b_rows rows each.
// V_FIRST: V is the MMA's A operand (its rows are the accumulator's), else its B operand.
template <int CTA_GROUP, bool V_FIRST>
__device__ __forceinline__ void lora_stage_mma(uint32_t tmem_d, uint32_t smem_v, uint32_t smem_b, uint32_t v_rows,
                                               uint32_t b_rows, uint32_t idesc, uint32_t info, const LoraDev &d) {
    const uint32_t parts = info >> 4, steps = info & 7u;
    const uint32_t v_bytes = lora_v_row_bytes(d), b_bytes = lora_b_row_bytes(d);
    for (uint32_t i = 0; i < parts; ++i) {
        const uint64_t dv = ptx::smem_desc_k(smem_v + i * v_rows * v_bytes, v_bytes);
        const uint64_t db = ptx::smem_desc_k(smem_b + i * b_rows * b_bytes, b_bytes);
        for (uint32_t k = 0; k < 2 * steps; ++k) {               // hi, then lo: 32 bytes = +2 in the >>4 address field
            const uint32_t lo = k >= steps ? 1u : 0u, at = k - lo * steps;
            const uint64_t v = dv + 2 * (lo * d.width / kUmmaK + at), b = db + 2 * at;
            ptx::umma_f16<CTA_GROUP>(tmem_d, V_FIRST ? v : b, V_FIRST ? b : v, idesc, 1u);
        }
    }
}

// A zero of V times an infinity or NaN in another row's adapter is NaN: such an element is computed again from its own
// row's terms alone.  `acc` unless one of the group's other adapters holds such a value in this column.
template <bool BF16>
__device__ __noinline__ float lora_exact(const LoraDev &d, uint32_t group, uint32_t row, uint32_t col, float acc) {
    const int32_t *t = d.table + static_cast<size_t>(group) * d.table_stride;
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
        const uint32_t in_group = row - group * d.group_rows;
        const uint32_t w8 = d.width / 8;
        const uint4 *v = reinterpret_cast<const uint4 *>(d.v) +
                         ((static_cast<int64_t>(group) * d.max_slots + mine) * d.group_rows + in_group) * (2 * d.rank_blocks * w8);
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

// N accumulators of row `row`, columns col, col + 1, ...
template <bool BF16, int N>
__device__ __forceinline__ void lora_repair(float (&f)[N], const LoraDev &d, uint32_t group, uint32_t row, uint32_t col,
                                            uint32_t M) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; ++i) bad |= f[i] != f[i];
    if (!bad || row >= M) return;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (f[i] != f[i] && col + i < d.n) f[i] = lora_exact<BF16>(d, group, row, col + i, f[i]);
}
template <bool BF16>
__device__ __forceinline__ void lora_repair(uint32_t (&v)[32], const LoraDev &d, uint32_t group, uint32_t row, uint32_t col,
                                            uint32_t M) {
    lora_repair<BF16, 32>(reinterpret_cast<float(&)[32]>(v), d, group, row, col, M);
}

}  // namespace
}  // namespace pg
