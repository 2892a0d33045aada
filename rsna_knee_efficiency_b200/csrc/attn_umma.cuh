// attn_umma.cuh -- tcgen05 kind::f16 pieces of the attention kernels: tiles of 128 rows x 64 or 128
// elements in shared memory (blocks of 64 elements = 128-byte rows, 128-byte swizzle, as TMA writes
// them), fp32 accumulators and 16-bit left operands in TMEM.
#pragma once
#include "attn_common.cuh"

namespace dn8 {

constexpr int AT_TILE = 128;                       // rows of a query or key tile
constexpr uint32_t AT_BLOCK = AT_TILE * 128;       // bytes of a block: 128 rows x 64 elements

DN8_DEV void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar)) : "memory");
}
// A tile of DP elements: one box of 64 elements x 1 head x 128 rows per block.
template <int DP> DN8_DEV void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int row) {
#pragma unroll
    for (int b = 0; b < DP / 64; ++b) tma_load_3d(dst + b * AT_BLOCK, map, bar, b * 64, head, row);
}

constexpr uint32_t LAYOUT_SW128 = 2;
// Rows along M or N, the 64-element blocks along K: K step kk (16 elements).
DN8_DEV uint64_t desc_rows(uint32_t tile, int kk) {
    return sdesc(tile + (kk >> 2) * AT_BLOCK + (kk & 3) * 32, 16, 1024, LAYOUT_SW128);
}
// Rows along K (16 rows per step, kk), elements along N.
DN8_DEV uint64_t desc_cols(uint32_t tile, int kk) { return sdesc(tile + kk * 2048, AT_BLOCK, 1024, LAYOUT_SW128); }

// Instruction descriptor of kind::f16: D fp32, A and B of type T; `bcols`: B's rows are along K.
template <typename T> DN8_DEV constexpr uint32_t idesc_f16(int M, int N, bool bcols) {
    const uint32_t t = sizeof(T) == 2 && !__is_same(T, __half) ? 1u : 0u;        // 1: bf16, 0: fp16
    return (1u << 4) | (t << 7) | (t << 10) | (static_cast<uint32_t>(bcols) << 16) |
           (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
// ---- issue ------------------------------------------------------------------------------------
// An MMA takes its descriptors and addresses from uniform registers. Where the compiler cannot see that a
// value is the same in the whole warp, it moves it there for every MMA (measured: 80 clocks per MMA, more
// than the MMA's own time). So the issuing warp makes its values uniform once (`uniform`, a reduction whose
// result lives in a uniform register), keeps its control flow uniform (conditions that come from a `vote`),
// and issues four MMAs (64 elements of K) per block with offsets that are constants.
DN8_DEV uint32_t uniform(uint32_t x) { return __reduce_or_sync(0xffffffffu, x); }
DN8_DEV bool vote(bool x) { return __any_sync(0xffffffffu, x) != 0; }

// Issued by a whole converged warp (one elected lane). D (+)= A B^T over 64 elements, 128-byte rows both.
DN8_DEV void umma_f16_ss4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, e, t;\n\t.reg .b32 l;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "setp.eq.b32 t, 0, 0;\n\t"
                 "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
                 "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
                 "elect.sync l|e, 0xffffffff;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// A from TMEM: 64 elements of a row, 16 in each 8 columns (elements 2c and 2c + 1 in column c) from a, a + 8,
// a + STEP, a + STEP + 8 on; B: 64 rows.
template <int STEP> DN8_DEV void umma_f16_ts4(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, e, t;\n\t.reg .b32 l, a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "setp.eq.b32 t, 0, 0;\n\t"
                 "add.s32 a1, %1, 8;\n\tadd.s32 a2, %1, %5;\n\tadd.s32 a3, %1, %6;\n\t"
                 "add.s64 b1, %2, 128;\n\tadd.s64 b2, %2, 256;\n\tadd.s64 b3, %2, 384;\n\t"
                 "elect.sync l|e, 0xffffffff;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "n"(STEP), "n"(STEP + 8) : "memory");
}
// D[128 x 128] = A B^T over DP elements, both tiles in shared memory
template <typename T, int DP> DN8_DEV void mma_scores(uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
    for (int k = 0; k < DP / 64; ++k)
        umma_f16_ss4(d, desc_rows(a, 4 * k), desc_rows(b, 4 * k), idesc_f16<T>(AT_TILE, AT_TILE, false), k > 0);
}
// D[128 x DP] (+)= A B, A [128 x 128] in TMEM, B a tile of 128 rows. A lies over the fp32 tile it was made
// from: each PART columns of it in the first PART / 2 TMEM columns of their own, so that the threads that
// read a part write over nothing else (PART = 32), or all in the first 64 TMEM columns (PART = 128: threads
// that have whole rows).
template <typename T, int DP, int PART> DN8_DEV void mma_values(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
        umma_f16_ts4<PART == 128 ? 16 : 32>(d, a + (PART == 128 ? 32 : 64) * k, desc_cols(b, 4 * k),
                                            idesc_f16<T>(AT_TILE, DP, true), accumulate || k > 0);
}

// Four threads per row: 16 rows x 64 columns of fp32. Thread t's registers 4k .. 4k + 3 are (row t / 4, columns
// 8k + 2 (t % 4) and the next) and the same columns of row t / 4 + 8.
#define DN8_R8(i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), \
                  "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
DN8_DEV void tmem_ld16x256_8(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : DN8_R8(0), DN8_R8(8), DN8_R8(16), DN8_R8(24) : "r"(taddr) : "memory");
}
DN8_DEV void tmem_ld16x256_4(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : DN8_R8(0), DN8_R8(8) : "r"(taddr) : "memory");
}
#undef DN8_R8
DN8_DEV void tmem_st16x256_4(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// 16 rows x 32 columns of packed words: registers 2k, 2k + 1 are column 4k + t % 4 of rows t / 4 and t / 4 + 8.
DN8_DEV void tmem_st16x128_8(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}

// One row per thread: 16 packed words (32 elements of 16 bits) to columns taddr ..
DN8_DEV void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// (see tmem_wait_st(r) in dn8_common.cuh: the registers of a store stay alive until it has read them)
DN8_DEV void tmem_wait_st(const uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::st.sync.aligned;"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}

// ---- work taken over from blocks that have not started ------------------------------------------
// The grid has one block per piece of work; a running block asks the launch hardware for the index of a
// block that has not been launched yet (that one then never is) and does its work too: setup once per
// SM, no tail between pieces, and whoever is free takes the next one. One thread asks; the 16-byte answer
// arrives in shared memory and completes on `bar`. After a refusal nothing may be asked again.
DN8_DEV void ask_for_block(void* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
// The block's index, or -1: there is none left.
DN8_DEV int answered_block(const void* answer) {
    uint32_t ok, x = 0;
    asm volatile("{\n\t.reg .b128 h;\n\t.reg .b64 lo, hi;\n\t.reg .pred p;\n\t"
                 "ld.shared.v2.b64 {lo, hi}, [%2];\n\t"
                 "mov.b128 h, {lo, hi};\n\t"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t"
                 "mov.u32 %1, 0;\n\t"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
                 : "=r"(ok), "=r"(x) : "r"(smem_u32(answer)) : "memory");
    return ok ? static_cast<int>(x) : -1;
}

DN8_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Bits lo .. and .. hi of a row of 128, word w. (shl.b32 gives 0 for counts of 32 and more.)
DN8_DEV uint32_t bits_from(int lo, int w) {
    uint32_t r;
    asm("shl.b32 %0, %1, %2;" : "=r"(r) : "r"(0xFFFFFFFFu), "r"(max(lo - 32 * w, 0)));
    return r;
}
DN8_DEV uint32_t bits_upto(int hi, int w) { return ~bits_from(hi + 1, w); }

// 3-D map over [rows][heads][D] with token / head strides (elements): box 64 elements x 1 head x `box_rows`
// rows. Elements behind D and rows behind the tensor arrive as zeros.
cudaError_t make_head_map(CUtensorMap* map, const void* base, int type, int64_t rows, int heads, int D, int64_t stride_t,
                          int64_t stride_h, int box_rows = AT_TILE);

}  // namespace dn8
