// attn_bwd.cu -- the gradient of attention (attn.cu): with P = exp(scale q k - lse) on the visible pairs
// and delta = sum(dout out) per row and head,
//   dv = P^T dout,  dS = P (dout v^T - delta) scale,  dq = dS k,  dk = dS^T q,
// dk and dv summed over the query heads of a key head's group. A query that sees nothing has lse =
// -inf: its P is zero.
//
// No atomics, so the same inputs give the same bits: a CTA owns 128 rows of dk and dv and walks over the
// query tiles that see them (all heads of the group), or owns 128 rows of dq and walks over the key
// tiles it sees. That is 7 products per pair of tiles instead of the 5 of one walk that adds dq up in
// memory, for which no CTA waits for another. Both walks have one form: two resident tiles R0, R1, two
// streamed ones X0, X1, and per step
//   S = R0 X0^T, dP = R1 X1^T   (tcgen05, 128 x 128 fp32 in TMEM; a TMEM lane is a resident row)
//   dk, dv: R = k, v; X = q, dout: P and dS go back to TMEM in 16 bits over S and dP, and
//           dv += P X1, dk += dS X0
//   dq:     R = q, dout; X = k, v: dS goes back, dq += dS X0
// so no operand is ever transposed or written to shared memory by a thread. Where TMEM has room for two
// S tiles (all but dk, dv with D > 64) S(u + 1) is made while the threads are still on step u, and dP(u + 1)
// while they take the exponentials of S(u + 1); else S(u + 1) is made while they work on dS(u).
//
// A CTA takes one piece (one walk) after the other (ask_for_block). Under a window, the first tokens' key
// tile is seen by every query: its walk is cut into shares, whose sums attn_bwd_join_kernel adds (and where heads are
// few, every long walk of dk and dv).
//
// 2 x 8192 tokens, 16 heads, no mask, in bursts at 1965 MHz: D = 64 2083 us (660 TFLOP/s of the 10 D per pair), D =
// 128 3171 us (867). Bound by the latency of a step's chain: at views of 6160 with windows of 512 to each side, D = 64
// (436 us), issue slots are busy for 0.50 of the time, special function units for 0.38, tensor cores for 0.33, and
// taking work away gained little (from 422 us then: 403 without the exponentials, 378 without the product of dS, 401
// with half of the value products).
#include <type_traits>

#include "attn_umma.cuh"

namespace dn8 {

// ---- delta and the logarithms, head by head -------------------------------------
// work: -lse2 [Hq][Tq] (-inf where the row sees nothing: its P = 2^(s - inf) = 0), then -delta scale
// [Hq][Tq]: so that P = 2^(S c + w0) and dS = P (dP scale + w1), two fused operations on pairs.
// LANES (8 or 16) threads per row of up to 64 or 128 elements; 32 rows of one head per block.
template <typename T, int LANES>
__global__ void __launch_bounds__(32 * LANES) attn_bwd_prep_kernel(const dn8_attention_bwd_args a) {
    griddep_launch_dependents();
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x / LANES;
    const int h = blockIdx.y, d = (threadIdx.x % LANES) * 8;
    float s = 0.0f;
    if (row < a.Tq && d < a.D) {
        float o[8], g[8];
        load_f32(static_cast<const T*>(a.out) + row * a.o_stride_t + h * a.o_stride_h + d, o);
        load_f32(static_cast<const T*>(a.dout) + row * a.do_stride_t + h * a.do_stride_h + d, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(o[e], g[e], s);
    }
#pragma unroll
    for (int k = LANES / 2; k > 0; k >>= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
    if (row < a.Tq && threadIdx.x % LANES == 0) {
        const float lse = a.lse[row * a.Hq + h];
        float* w = static_cast<float*>(a.work) + h * a.Tq + row;
        w[0] = lse == -INFINITY ? -INFINITY : -lse * ATT_LOG2E;
        w[a.Hq * a.Tq] = lse == -INFINITY ? 0.0f : -s * a.scale;
    }
}

// ---- the two walks -----------------------------------------------------------------------------
// Warps 0-15: rows; 16: tcgen05 issue; 17: TMA; 18: statistics and masked rows of the streamed tiles; 19: which
// piece comes next, asked for AB_AHEAD steps before the end of a piece (asked for at its start, a piece waits
// behind a long one while others run out of work).
constexpr int AB_THREADS = 640, AB_AHEAD = 4;
// The launch gives every thread 96 registers: 16 x 32 x 104 + 4 x 32 x 64 = 20 x 32 x 96.
constexpr int AB_REGS_ROWS = 104, AB_REGS_OTHER = 64;
template <int DP> struct BwdCfg {
    // Slots of the streamed tiles. X1 is done with early in a step (dP, dv), X0 at its end (dq, dk) and asked
    // for again at the next one's start (S), so where memory is short X0 has the third slot.
    static constexpr int N0 = 3, N1 = DP == 64 ? 3 : 2;
    static constexpr uint32_t TILE = AT_TILE * DP * 2;
    // (the sequences by blocks of queries and of keys lie behind the state where there is room)
    static constexpr bool TABLES = DP == 64;
    static constexpr uint32_t STATE = 3 << 10, SMEM = TILE * (2 + N0 + N1) + STATE + (TABLES ? 2 * sizeof(SequenceTable) : 0);
    // TMEM columns: dP, then S (one or two tiles), then the sums at the end
    static constexpr uint32_t DPC = 0, S = 128, ACC1 = 512 - DP, ACC0 = 512 - 2 * DP;
};
// S tiles: the sums are dv (ACC0) and dk (ACC1), or dq (ACC1)
template <int DP> DN8_DEV constexpr int s_tiles(bool kv) { return kv && DP == 128 ? 1 : 2; }

// Shares of the walks over key tiles (dk, dv). Under a window, those over the first tokens' tiles are cut
// (split_blocks > 0). Where the keys make few pieces and a key head has several query heads, every walk longer than
// two thirds of an SM's part of all steps is (sms > 0): the lengths are known to the GPU alone, so each CTA adds
// them up. A step of dk, dv counts KV_STEP steps of dq (five products, not three). Uncut and cut, us: 3022 tokens,
// 8 heads in groups of 4, D = 80, left of 479: 220 and 134 (147 in parts of an SM's whole share); 719 tokens, D = 128,
// the same heads: 64 and 43. Walks of dq are never the longest there, and short walks are not cut: 900 tokens, 4
// heads of their own, D = 128, took 30 us uncut and 49 cut.
struct BwdPlan {
    int kv_blocks, split_blocks, tiles, shares, sms;
    int blocks, records;                      // blocks in all; those that may be shares
    float* part;                              // [block][dv, dk][128][DP]
    int4* rec;                                // [block] first key row; rows (0: not a piece's first share) + 256 head;
                                              // shares; blocks from one share to the next
};
constexpr float KV_STEP = 1.5f, AB_SHARE = 8.0f;      // AB_SHARE: steps of a share, at least
constexpr float AB_PARTS = 1.5f;              // parts per SM
// Tiles of 128 that the rows of a tile meet on an axis of n, the first tokens aside (n < 2^28).
template <typename A> DN8_DEV int met_tiles(const A& a, int n) {
    const int met = a.left < 0 || a.right < 0 ? n : min(n, min(a.left, n) + min(a.right, n) + AT_TILE);
    return (met + AT_TILE - 1) / AT_TILE;
}
struct BwdShares {
    const dn8_attention_bwd_args& a;
    float inv;                                // 1 / steps of a part, or 0: nothing is cut
    DN8_DEV int operator()(int nq, int) const { return max(1, __float2int_rn(met_tiles(a, nq) * (a.Hq / a.Hk) * inv)); }
};
DN8_DEV BwdShares bwd_shares(const dn8_attention_bwd_args& a, const BwdPlan& plan) {      // (one whole warp)
    BwdShares s = {a, 0.0f};
    if (plan.sms == 0) return s;
    float total = 0.0f;
    for (int b = threadIdx.x & 31; b < a.B; b += 32) {
        const Sequence q = sequence_of(a, b);
        total += KV_STEP * static_cast<float>((q.nk + AT_TILE - 1) / AT_TILE) * met_tiles(a, q.nq) +
                 static_cast<float>((q.nq + AT_TILE - 1) / AT_TILE) * met_tiles(a, q.nk);
    }
    s.inv = fminf(AB_PARTS * KV_STEP * static_cast<float>(plan.sms) / (warp_sum(total) * static_cast<float>(a.Hq)), 1.0f / AB_SHARE);
    return s;
}

struct BwdPiece {
    Sequence seq;                             // seq.b = -2: no more pieces
    int kv;                                   // dk, dv of a key tile, or dq of a query tile
    int r0;                                   // first resident row, within the sequence
    int h;                                    // key head (kv) or query head
    int steps;
    int share;                                // kv: where a share's sums go, or -1: straight to dk, dv
    // Streamed tiles: `tile0`, then one after the other; after `turn` comes `back` (dk, dv: the next head's first
    // tile; dq: from the first tokens' tiles to the window's). hx: the first step's head.
    int tile0, turn, back, hx;
    // A step whose first column is above `hic`, or below `loc` but above `skc`, or every step, needs a mask.
    int always, hic, loc, skc;
};
struct BwdShared {
    uint64_t answer[2];
    uint64_t answered, pfilled, pread, near, rfull, rempty, fin, aempty, dpfull, dsready;
    // (of even and odd steps: the rows may be done with S(u + 1), where there are two S tiles, before the
    // issuing warp, held up by its own queue, has looked for S(u))
    uint64_t pready[2];
    uint64_t sfull[2], x0full[3], x0empty[3], x0ok[3], x1full[3], x1empty[3], x1ok[3], sempty[2];
    BwdPiece piece[2];
    uint32_t words[2][4];                     // of even and odd steps, as the statistics
    uint32_t tmem;
    int abort;
    alignas(16) float w0[2][AT_TILE], w1[2][AT_TILE];      // the statistics of a step's queries
};

// The 16 row warps on one piece: warp w has the TMEM lanes (resident rows) 32 (w % 4) .. and the columns
// 32 (w / 4) .. of every step. c: steps of this CTA so far; sp: phases of sfull.
template <typename T, int DP, bool KV>
DN8_DEV bool bwd_rows(const dn8_attention_bwd_args& a, BwdShared& sh, const BwdPiece& pc, float* part, uint32_t tmem,
                      uint32_t& c, uint32_t& sp, uint32_t& fp) {
    using C = BwdCfg<DP>;
    constexpr int NS = s_tiles<DP>(KV);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int quarter = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    volatile int* abort_flag = &sh.abort;
    const int left = a.left < 0 ? ATT_FAR : a.left, right = a.right < 0 ? ATT_FAR : a.right;
    const float sc = a.scale * ATT_LOG2E;
    const int r = pc.r0 + row;                                   // key j (KV) or query i
    const bool inside = r < (KV ? pc.seq.nk : pc.seq.nq);
    // KV: the key may be seen at all; dq: the row's statistics
    const bool keep = KV && inside && (a.keep == nullptr || a.keep[pc.seq.k0 + r] != 0);
    float row_w0 = -INFINITY, row_w1 = 0.0f;
    if (!KV && inside) {
        const float* w = static_cast<const float*>(a.work) + pc.h * a.Tq + pc.seq.q0 + r;
        row_w0 = w[0];
        row_w1 = w[a.Hq * a.Tq];
    }
    bool ok = true;
    const int steps = pc.steps, turn = pc.turn, hic = pc.hic, loc = pc.loc, skc = pc.skc;
    const bool always = pc.always != 0;
    int tile = pc.tile0;
    for (int u = 0; u < steps; ++u, ++c) {
        const int c0 = tile * AT_TILE;
        tile = tile == turn ? pc.back : tile + 1;
        const uint32_t sx = c & 1;
        ok = mbar_wait_w(&sh.x0ok[c % C::N0], (c / C::N0) & 1, a.err, abort_flag, ERR_WAIT_FULL | (80 << 4));
        if (!ok) return false;
        uint32_t word = 0xFFFFFFFFu;
        const bool masked = always || c0 > hic || (c0 < loc && c0 > skc);
        if (masked) {
            const int off = pc.seq.nk - pc.seq.nq;
            if (KV) {
                // columns are queries: seen from j - right - off on, up to j + left - off (first tokens: by all).
                // Queries behind the end are zero rows with w0 = -inf.
                const int lo = r - right - off - c0, hi = r < a.sinks ? ATT_FAR : r + left - off - c0;
                word = keep ? bits_from(lo, quarter) & bits_upto(hi, quarter) : 0u;
            } else {
                const int p = r + off, hi = min(pc.seq.nk - 1, p + right) - c0, lo = p - left - c0;
                word = bits_upto(hi, quarter) & sh.words[sx][quarter] &
                       (bits_from(lo, quarter) | bits_upto(a.sinks - 1 - c0, quarter));
            }
        }
        const int sb = NS == 1 ? 0 : u & 1;
        const uint32_t ts = lanes + C::S + sb * 128 + quarter * 32, tp = lanes + C::DPC + quarter * 32;
        ok = mbar_wait_w(&sh.sfull[sb], (sp >> sb) & 1, a.err, abort_flag, ERR_WAIT_ACC | (81 << 4));
        if (!ok) return false;
        sp ^= 1u << sb;
        tc_fence_after();
        uint32_t pr[32];                                         // P of this thread's columns, fp32
        tmem_ld32(ts, pr);
        tmem_wait_ld(pr);
        if (!KV) {                                               // S is in registers: its tile is free
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.pready[c & 1]);
        }
        // (a part of the exponentials by polynomial, to spare the special function units, was slower: the row
        // warps' issue slots are the scarcer of the two)
        const float2 sc2 = f2_pack(sc, sc);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            float4 w = make_float4(row_w0, row_w0, row_w0, row_w0);
            if (KV) w = *reinterpret_cast<const float4*>(sh.w0[sx] + quarter * 32 + e);
            const float2 x = f2_fma(f2_pack(__uint_as_float(pr[e]), __uint_as_float(pr[e + 1])), sc2, f2_pack(w.x, w.y));
            const float2 y = f2_fma(f2_pack(__uint_as_float(pr[e + 2]), __uint_as_float(pr[e + 3])), sc2, f2_pack(w.z, w.w));
            pr[e] = __float_as_uint(ex2(x.x));
            pr[e + 1] = __float_as_uint(ex2(x.y));
            pr[e + 2] = __float_as_uint(ex2(y.x));
            pr[e + 3] = __float_as_uint(ex2(y.y));
        }
        if (masked)
#pragma unroll
            for (int e = 0; e < 32; ++e) pr[e] = (word >> e) & 1u ? pr[e] : 0u;
        if (KV) {
            // P in [0, 1], rounded to the inputs' type for dv
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) pk[e] = pack2(T(), __uint_as_float(pr[2 * e]), __uint_as_float(pr[2 * e + 1]));
            tmem_st16(ts, pk);
            tmem_wait_st(pk);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.pready[c & 1]);
        }
        ok = mbar_wait_w(&sh.dpfull, c & 1, a.err, abort_flag, ERR_WAIT_ACC | (82 << 4));
        if (!ok) return false;
        tc_fence_after();
        uint32_t dp[32], pk[16];
        tmem_ld32(tp, dp);
        tmem_wait_ld(dp);
        // (a masked pair's P is 0, but its dP may be NaN, and 0 * NaN is not 0)
        if (masked)
#pragma unroll
            for (int e = 0; e < 32; ++e) dp[e] = (word >> e) & 1u ? dp[e] : 0u;
        const float2 scale2 = f2_pack(a.scale, a.scale);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            float4 w = make_float4(row_w1, row_w1, row_w1, row_w1);
            if (KV) w = *reinterpret_cast<const float4*>(sh.w1[sx] + quarter * 32 + e);
            const float2 x = f2_fma(f2_pack(__uint_as_float(dp[e]), __uint_as_float(dp[e + 1])), scale2, f2_pack(w.x, w.y));
            const float2 y = f2_fma(f2_pack(__uint_as_float(dp[e + 2]), __uint_as_float(dp[e + 3])), scale2, f2_pack(w.z, w.w));
            const float2 u2 = __fmul2_rn(x, f2_pack(__uint_as_float(pr[e]), __uint_as_float(pr[e + 1])));
            const float2 v2 = __fmul2_rn(y, f2_pack(__uint_as_float(pr[e + 2]), __uint_as_float(pr[e + 3])));
            pk[e / 2] = pack2(T(), u2.x, u2.y);
            pk[e / 2 + 1] = pack2(T(), v2.x, v2.y);
        }
        tmem_st16(tp, pk);
        tmem_wait_st(pk);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&sh.dsready);
            mbar_arrive(&sh.sempty[sx]);
        }
    }
    if (steps > 0) {
        ok = mbar_wait_w(&sh.fin, fp, a.err, abort_flag, ERR_WAIT_ACC | (83 << 4));
        if (!ok) return false;
        fp ^= 1;
        tc_fence_after();
    }
    // the sums: quarters 0, 1 write dv and 2, 3 dk, half of the elements each, or each a quarter of dq's
    constexpr int COLS = KV ? DP / 2 : DP / 4;
    const int d0 = KV ? (quarter & 1) * COLS : quarter * COLS;
    const uint32_t acc = lanes + (KV && quarter < 2 ? C::ACC0 : C::ACC1) + d0;
    const int64_t at = static_cast<int64_t>(KV ? pc.seq.k0 : pc.seq.q0) + r;
    T* dst = KV ? (quarter < 2 ? static_cast<T*>(a.dv) + at * a.dv_stride_t + pc.h * a.dv_stride_h
                               : static_cast<T*>(a.dk) + at * a.dk_stride_t + pc.h * a.dk_stride_h)
                : static_cast<T*>(a.dq) + at * a.dq_stride_t + pc.h * a.dq_stride_h;
    const bool zero = steps == 0 || (!KV && row_w0 == -INFINITY);
#pragma unroll 1
    for (int k = 0; k < COLS; k += 16) {
        uint32_t o[16] = {};
        if (steps > 0) {
            tmem_ld16(acc + k, o);
            tmem_wait_ld(o);
        }
        if (zero)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0u;
        if (KV && pc.share >= 0) {
            float* p = part + ((static_cast<size_t>(pc.share) * 2 + (quarter >> 1)) * AT_TILE + row) * DP + d0 + k;
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<uint4*>(p + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else if (inside) {
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                float v[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) v[x] = __uint_as_float(o[e + x]);
                if (d0 + k + e < a.D) store_f32(dst + d0 + k + e, v);
            }
        }
    }
    if (steps > 0) {                                             // the sums have been read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.aempty);
    }
    return true;
}

template <typename T, int DP, bool CUT>
__global__ void __launch_bounds__(AB_THREADS, 1)
attn_bwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo,
                const dn8_attention_bwd_args a, const BwdPlan plan) {
    using C = BwdCfg<DP>;
    static_assert(sizeof(BwdShared) <= C::STATE, "shared state");
    extern __shared__ __align__(1024) uint8_t smem[];    // (no static shared memory, so it starts aligned)
    uint8_t* sr = smem;                                  // R0, R1
    uint8_t* sx0 = smem + 2 * C::TILE;                   // slots of X0
    uint8_t* sx1 = sx0 + C::N0 * C::TILE;                // slots of X1
    BwdShared& sh = *reinterpret_cast<BwdShared*>(sx1 + C::N1 * C::TILE);
    volatile int* abort_flag = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.Hq / a.Hk;
    if (smem_u32(smem) & 1023u) {                        // the tiles' swizzle needs it; never seen
        if (threadIdx.x == 0 && a.err != nullptr) atomicCAS(a.err, 0, ERR_SHAPE);
        return;
    }
    if (threadIdx.x == 512) {
        mbar_init(&sh.answered, 1);
        mbar_init(&sh.pfilled, 1);
        mbar_init(&sh.pread, 19);
        mbar_init(&sh.near, 1);
        mbar_init(&sh.rfull, 1);
        mbar_init(&sh.rempty, 1);
        mbar_init(&sh.fin, 1);
        mbar_init(&sh.aempty, 16);
        mbar_init(&sh.dpfull, 1);
        mbar_init(&sh.dsready, 16);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sh.sfull[s], 1);
            mbar_init(&sh.pready[s], 16);
            mbar_init(&sh.sempty[s], 16);
        }
        for (int s = 0; s < 3; ++s) {
            mbar_init(&sh.x0full[s], 1);
            mbar_init(&sh.x0empty[s], 1);
            mbar_init(&sh.x0ok[s], 1);
            mbar_init(&sh.x1full[s], 1);
            mbar_init(&sh.x1empty[s], 1);
            mbar_init(&sh.x1ok[s], 1);
        }
        sh.abort = 0;
        mbar_fence_init();
    }
    if (warp == 17) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int left = a.left < 0 ? ATT_FAR : a.left, right = a.right < 0 ? ATT_FAR : a.right;

    // Piece n of this CTA: sh.piece[n % 2], from the moment it is filled until every warp has begun with the
    // next one. Every warp but the last calls this for n = 0, 1, ... when it begins; false: there is
    // none (or a wait gave up).
    auto begin_piece = [&](int n) -> bool {
        if (!mbar_wait_w(&sh.pfilled, n & 1, a.err, abort_flag, ERR_WAIT_FULL | (91 << 4))) return false;
        if (lane == 0) mbar_arrive(&sh.pread);
        return sh.piece[n & 1].seq.b >= 0;
    };
    griddep_wait();                                      // the statistics

    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AB_REGS_OTHER));
        if (warp == 19) {
            // ---------------- pieces ----------------
            int block = blockIdx.x, asked = 0;
            BwdPiece pc;
            const BwdShares shares = CUT ? bwd_shares(a, plan) : BwdShares{a, 0.0f};
            // a block's sequence: from shared memory, from this warp's registers where that is full, or read again
            const bool few = a.B <= (C::TABLES ? SequenceTable::MOST : SequenceLanes::MOST);
            SequenceTable* table = reinterpret_cast<SequenceTable*>(reinterpret_cast<uint8_t*>(&sh) + C::STATE);
            SequenceLanes seqs;
            if (few && C::TABLES) {
                table[0].fill<false>(a, AT_TILE, OneShare());
                table[1].fill<true>(a, AT_TILE, shares);
            } else if (few) {
                seqs.fill(a, AT_TILE, shares);
            }
            auto tile_of = [&](auto keys, int unit) -> Sequence {
                constexpr bool KEYS = decltype(keys)::value;
                if (!few) {
                    if constexpr (KEYS && CUT) return find_block<true>(a, unit, 1, AT_TILE, shares);
                    else return find_block<KEYS>(a, unit, 1, AT_TILE);
                }
                if constexpr (C::TABLES) return table[KEYS].find(a.B, unit);
                else return seqs.template find<KEYS>(unit);
            };
            for (int n = 0;;) {
                pc.seq.b = -2;
                pc.steps = pc.tile0 = pc.hx = 0;
                pc.turn = pc.back = pc.share = -1;
                int cuts = 1, mine = 0;                  // shares, and which one
                if (block >= 0) {
                    pc.kv = block < plan.kv_blocks;
                    if (block < plan.split_blocks) {
                        // share s of the walk over tile t of sequence b and key head h: block = ((b tiles + t) Hk + h)
                        // shares + s
                        const int x = block / plan.shares;
                        cuts = plan.shares;
                        mine = block - x * cuts;
                        pc.seq = sequence_of(a, x / a.Hk / plan.tiles);
                        pc.seq.blk = x / a.Hk % plan.tiles;
                        pc.h = x % a.Hk;
                        if (pc.seq.blk * AT_TILE >= pc.seq.nk) pc.seq.b = -1;
                    } else if (CUT && pc.kv) {
                        pc.seq = tile_of(std::true_type(), block / a.Hk);
                        pc.h = block % a.Hk;
                        if (pc.seq.b >= 0) cuts = shares(pc.seq.nq, pc.seq.nk);
                        mine = pc.seq.blk % cuts;
                        pc.seq.blk /= cuts;
                    } else if (pc.kv) {
                        const int x = block - plan.split_blocks;
                        pc.seq = tile_of(std::true_type(), x / a.Hk);
                        pc.h = x % a.Hk;
                        if (plan.shares > 1 && pc.seq.blk < plan.tiles) pc.seq.b = -1;
                    } else {
                        const int x = block - plan.kv_blocks;
                        pc.seq = tile_of(std::false_type(), x / a.Hq);
                        pc.h = x % a.Hq;
                    }
                    if (cuts > 1) pc.share = block;
                    if (block < plan.records && lane == 0) {
                        const int r0 = pc.seq.blk * AT_TILE;
                        const bool first = pc.seq.b >= 0 && mine == 0 && cuts > 1;
                        plan.rec[block] = make_int4(pc.seq.k0 + r0, (first ? min(AT_TILE, pc.seq.nk - r0) : 0) + 256 * pc.h, cuts,
                                                    CUT ? a.Hk : 1);
                    }
                }
                if (pc.seq.b >= 0) {
                    const int nq = pc.seq.nq, nk = pc.seq.nk, off = nk - nq;
                    if (pc.kv) {
                        // first key tiles first: open left sides make them the longest
                        pc.r0 = pc.seq.blk * AT_TILE;
                        const int jl = min(pc.r0 + AT_TILE, nk) - 1;
                        const int lo = max(0, pc.r0 - right - off);
                        const int hi = pc.r0 < a.sinks ? nq - 1 : min(nq - 1, jl + left - off);
                        const int first = lo / AT_TILE, per = lo <= hi ? hi / AT_TILE - first + 1 : 1;
                        pc.steps = lo <= hi ? per * G : 0;
                        int begin = 0;
                        if (cuts > 1) {                  // steps [s n / shares, (s + 1) n / shares)
                            const int n_ = pc.steps;
                            begin = static_cast<int>(static_cast<int64_t>(mine) * n_ / cuts);
                            pc.steps = static_cast<int>(static_cast<int64_t>(mine + 1) * n_ / cuts) - begin;
                        }
                        pc.tile0 = first + begin % per;
                        pc.hx = pc.h * G + begin / per;
                        pc.turn = first + per - 1;
                        pc.back = first;
                        pc.always = a.keep != nullptr || pc.r0 + AT_TILE > nk;
                        pc.loc = jl - right - off;
                        pc.skc = -1;
                        pc.hic = jl < a.sinks ? ATT_FAR : pc.r0 + left - off - (AT_TILE - 1);
                    } else {
                        pc.r0 = ((nq - 1) / AT_TILE - pc.seq.blk) * AT_TILE;
                        const int il = min(pc.r0 + AT_TILE, nq) - 1;
                        const KeyTiles k = key_tiles(pc.r0 + off, il + off, nk, left, right, a.sinks, AT_TILE);
                        pc.steps = k.count;
                        pc.tile0 = k.tile(0);
                        pc.hx = pc.h / G;
                        pc.turn = k.first - 1;
                        pc.back = k.start;
                        pc.always = a.keep != nullptr;
                        pc.hic = min(nk - 1, pc.r0 + off + right) - (AT_TILE - 1);
                        pc.loc = il + off - left;
                        pc.skc = a.sinks - AT_TILE;
                    }
                }
                if (pc.seq.b != -1) {                    // (-1: nothing there)
                    if (lane == 0) {
                        sh.piece[n & 1] = pc;
                        mbar_arrive(&sh.pfilled);
                    }
                    if (pc.seq.b == -2) break;
                    // (every warp has begun with it: one piece is known ahead, no more)
                    if (!mbar_wait_w(&sh.near, n & 1, a.err, abort_flag, ERR_WAIT_EMPTY | (99 << 4)) ||
                        !mbar_wait_w(&sh.pread, n & 1, a.err, abort_flag, ERR_WAIT_EMPTY | (92 << 4)))
                        break;
                    ++n;
                }
                if (lane == 0) {
                    fence_async_smem();                  // the last answer has been read
                    mbar_expect_tx(&sh.answered, 16);
                    ask_for_block(sh.answer, &sh.answered);
                }
                if (!mbar_wait_w(&sh.answered, asked & 1, a.err, abort_flag, ERR_WAIT_FULL | (93 << 4))) break;
                ++asked;
                block = answered_block(sh.answer);
                __syncwarp();
            }
        } else if (warp == 17) {
            // ---------------- TMA ----------------
            uint32_t c = 0, np = 0;
            for (int n = 0; begin_piece(n); ++n) {
                const BwdPiece& pc = sh.piece[n & 1];
                if (pc.steps == 0) continue;
                if (lane == 0) {
                    const bool kv = pc.kv != 0;
                    bool ok = mbar_wait(&sh.rempty, (np & 1) ^ 1, a.err, abort_flag, ERR_WAIT_EMPTY | (94 << 4));
                    if (ok) {
                        const int r0 = (kv ? pc.seq.k0 : pc.seq.q0) + pc.r0;
                        mbar_expect_tx(&sh.rfull, 2 * C::TILE);
                        load_tile<DP>(sr, kv ? &mk : &mq, &sh.rfull, pc.h, r0);
                        load_tile<DP>(sr + C::TILE, kv ? &mv : &mdo, &sh.rfull, pc.h, r0);
                    }
                    int tile = pc.tile0, hx = pc.hx;
                    for (int u = 0; ok && u < pc.steps; ++u, ++c) {
                        const uint32_t s0 = c % C::N0, s1 = c % C::N1;
                        const int x0 = (kv ? pc.seq.q0 : pc.seq.k0) + tile * AT_TILE;
                        ok = mbar_wait(&sh.x0empty[s0], ((c / C::N0) & 1) ^ 1, a.err, abort_flag, ERR_WAIT_EMPTY | (84 << 4));
                        if (!ok) break;
                        mbar_expect_tx(&sh.x0full[s0], C::TILE);
                        load_tile<DP>(sx0 + s0 * C::TILE, kv ? &mq : &mk, &sh.x0full[s0], hx, x0);
                        ok = mbar_wait(&sh.x1empty[s1], ((c / C::N1) & 1) ^ 1, a.err, abort_flag, ERR_WAIT_EMPTY | (96 << 4));
                        if (!ok) break;
                        mbar_expect_tx(&sh.x1full[s1], C::TILE);
                        load_tile<DP>(sx1 + s1 * C::TILE, kv ? &mdo : &mv, &sh.x1full[s1], hx, x0);
                        if (tile == pc.turn) {
                            tile = pc.back;
                            hx += kv ? 1 : 0;
                        } else {
                            ++tile;
                        }
                    }
                }
                ++np;
                __syncwarp();
            }
        } else if (warp == 18) {
            // ---------------- masked rows of the streamed tiles, statistics of the query rows ----------------
            // Streamed rows are summed over: a row whose weights are all zero must not hold NaN. The next step's
            // statistics are on their way while this one's tiles are waited for.
            uint32_t c = 0;
            bool ok = true;
            for (int n = 0; ok && begin_piece(n); ++n) {
                const BwdPiece& pc = sh.piece[n & 1];
                const bool kv = pc.kv != 0;
                const int steps = pc.steps, q0 = pc.seq.q0, nq = pc.seq.nq, nk = pc.seq.nk;
                const uint32_t hidden = hidden_keys(a, nq, nk);
                int tile = pc.tile0, hx = pc.hx;
                float l2[4], de[4];
                bool live[4];
                auto fetch = [&]() {                     // of the step that `tile` and `hx` stand at
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int x = tile * AT_TILE + w * 32 + lane;
                        l2[w] = -INFINITY;
                        de[w] = 0.0f;
                        live[w] = true;
                        if (kv && x < nq) {
                            const float* ws = static_cast<const float*>(a.work) + static_cast<int64_t>(hx) * a.Tq + q0 + x;
                            l2[w] = ws[0];
                            de[w] = ws[a.Hq * a.Tq];
                        }
                        if (!kv) live[w] = x < nk && behind_hidden(a, x, hidden) && (a.keep == nullptr || a.keep[pc.seq.k0 + x] != 0);
                    }
                    if (tile == pc.turn) {
                        tile = pc.back;
                        hx += kv ? 1 : 0;
                    } else {
                        ++tile;
                    }
                };
                if (steps > 0) fetch();
                if (steps == 0 && lane == 0) mbar_arrive(&sh.near);
                for (int u = 0; u < steps; ++u, ++c) {
                    if (u == max(0, steps - AB_AHEAD) && lane == 0) mbar_arrive(&sh.near);
                    const uint32_t s0 = c % C::N0, s1 = c % C::N1, sx = c & 1;
                    uint32_t word[4];
                    // (the step before the last has been read)
                    ok = mbar_wait_w(&sh.sempty[sx], ((c >> 1) & 1) ^ 1, a.err, abort_flag, ERR_WAIT_EMPTY | (97 << 4));
                    if (!ok) break;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        word[w] = __ballot_sync(0xffffffffu, kv ? l2[w] != -INFINITY : live[w]);
                        if (kv) {
                            sh.w0[sx][w * 32 + lane] = l2[w];
                            sh.w1[sx][w * 32 + lane] = de[w];
                        } else if (lane == w) {
                            sh.words[sx][w] = word[w];
                        }
                    }
                    if (u + 1 < steps) fetch();
                    const bool fix = (word[0] & word[1] & word[2] & word[3]) != 0xFFFFFFFFu;
                    auto zero_rows = [&](uint8_t* x) {
#pragma unroll
                        for (int w = 0; w < 4; ++w)
                            if (!((word[w] >> lane) & 1u))
                                for (int b = 0; b < DP / 64; ++b) {
                                    uint4* row = reinterpret_cast<uint4*>(x + b * AT_BLOCK + (w * 32 + lane) * 128);
#pragma unroll
                                    for (int k = 0; k < 8; ++k) row[k] = make_uint4(0u, 0u, 0u, 0u);
                                }
                        fence_async_smem();
                    };
                    ok = mbar_wait_w(&sh.x0full[s0], (c / C::N0) & 1, a.err, abort_flag, ERR_WAIT_FULL | (85 << 4));
                    if (!ok) break;
                    if (fix) zero_rows(sx0 + s0 * C::TILE);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.x0ok[s0]);
                    ok = mbar_wait_w(&sh.x1full[s1], (c / C::N1) & 1, a.err, abort_flag, ERR_WAIT_FULL | (98 << 4));
                    if (!ok) break;
                    if (fix && kv) zero_rows(sx1 + s1 * C::TILE);      // (dq: V's rows meet no sum over rows)
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.x1ok[s1]);
                }
            }
        } else {
            // ---------------- tcgen05 issue (every value and branch uniform, see attn_umma.cuh) ----------------
            const uint32_t r0 = uniform(smem_u32(sr)), x0b = uniform(smem_u32(sx0)), x1b = uniform(smem_u32(sx1));
            const uint32_t tm = uniform(tmem);
            uint32_t s0 = 0, p0 = 0, s1 = 0, p1 = 0;     // the slots of the next tiles to wait for, their phases
            uint32_t c = 0, np = 0;                      // steps and pieces so far
            bool ok = true;
            // (x0ok and x1ok come after the tiles' own barriers)
            auto wait_x0 = [&]() -> uint32_t {
                const uint32_t s = s0;
                ok = mbar_wait_w(&sh.x0ok[s], p0, a.err, abort_flag, ERR_WAIT_FULL | (86 << 4));
                if (++s0 == C::N0) {
                    s0 = 0;
                    p0 ^= 1;
                }
                return s;
            };
            auto wait_x1 = [&]() -> uint32_t {
                const uint32_t s = s1;
                ok = mbar_wait_w(&sh.x1ok[s], p1, a.err, abort_flag, ERR_WAIT_FULL | (87 << 4));
                if (++s1 == C::N1) {
                    s1 = 0;
                    p1 ^= 1;
                }
                return s;
            };
            for (int n = 0; vote(begin_piece(n)); ++n) {
                const int steps = uniform(sh.piece[n & 1].steps);
                const bool kv = vote(sh.piece[n & 1].kv != 0);
                if (vote(steps == 0)) continue;
                const bool two = !kv || DP == 64;        // two S tiles
                ok = mbar_wait_w(&sh.rfull, np & 1, a.err, abort_flag, ERR_WAIT_FULL | (88 << 4));
                if (!ok) break;
                uint32_t x0 = wait_x0(), x0n = 0;        // slots of step u and of step u + 1
                if (!ok) break;
                tc_fence_after();
                mma_scores<T, DP>(tm + C::S, r0, x0b + x0 * C::TILE);
                umma_commit_w(&sh.sfull[0]);
                uint32_t x1 = wait_x1();
                if (!ok) break;
                tc_fence_after();
                mma_scores<T, DP>(tm + C::DPC, r0 + C::TILE, x1b + x1 * C::TILE);
                umma_commit_w(&sh.dpfull);
                if (!kv) umma_commit_w(&sh.x1empty[x1]);
                if (vote(steps == 1)) umma_commit_w(&sh.rempty);
                for (int u = 0; vote(u < steps); ++u, ++c) {
                    const bool more = vote(u + 1 < steps), first = vote(u == 0);
                    const uint32_t sb = two && (u & 1) ? 1u : 0u, sn = two ? sb ^ 1u : 0u;
                    // the last piece's sums have been read (with D > 64 dv's lie where dq has its second S tile)
                    if (first) {
                        ok = mbar_wait_w(&sh.aempty, (np & 1) ^ 1, a.err, abort_flag, ERR_WAIT_ACC | (95 << 4));
                        if (!ok) break;
                    }
                    if (more && two) {
                        // (its tile: P(u - 1), whose product was issued, or S(u - 1), which has been read)
                        x0n = wait_x0();
                        if (!ok) break;
                        tc_fence_after();
                        mma_scores<T, DP>(tm + C::S + sn * 128, r0, x0b + x0n * C::TILE);
                        umma_commit_w(&sh.sfull[sn]);
                    }
                    ok = mbar_wait_w(&sh.pready[c & 1], (c >> 1) & 1, a.err, abort_flag, ERR_WAIT_ACC | (89 << 4));
                    if (!ok) break;
                    if (kv) {
                        tc_fence_after();
                        mma_values<T, DP, 32>(tm + C::ACC0, tm + C::S + sb * 128, x1b + x1 * C::TILE, !first);
                        umma_commit_w(&sh.x1empty[x1]);
                    }
                    if (more && !two) {
                        x0n = wait_x0();
                        if (!ok) break;
                        tc_fence_after();
                        mma_scores<T, DP>(tm + C::S, r0, x0b + x0n * C::TILE);
                        umma_commit_w(&sh.sfull[0]);
                    }
                    if (more) {
                        x1 = wait_x1();
                        if (!ok) break;
                    }
                    ok = mbar_wait_w(&sh.dsready, c & 1, a.err, abort_flag, ERR_WAIT_ACC | (90 << 4));
                    if (!ok) break;
                    tc_fence_after();
                    mma_values<T, DP, 32>(tm + C::ACC1, tm + C::DPC, x0b + x0 * C::TILE, !first);
                    if (more) {
                        mma_scores<T, DP>(tm + C::DPC, r0 + C::TILE, x1b + x1 * C::TILE);
                        umma_commit_w(&sh.dpfull);
                        if (!kv) umma_commit_w(&sh.x1empty[x1]);
                    }
                    umma_commit_w(&sh.x0empty[x0]);
                    if (vote(u + 2 == steps)) umma_commit_w(&sh.rempty);      // no more products with R
                    x0 = x0n;
                }
                if (!ok) break;
                umma_commit_w(&sh.fin);
                ++np;
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AB_REGS_ROWS));
        uint32_t c = 0, sp = 0, fp = 0;
        for (int n = 0; begin_piece(n); ++n) {
            const BwdPiece& pc = sh.piece[n & 1];
            if (!(pc.kv ? bwd_rows<T, DP, true>(a, sh, pc, plan.part, tmem, c, sp, fp)
                        : bwd_rows<T, DP, false>(a, sh, pc, plan.part, tmem, c, sp, fp)))
                break;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 17) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

// The sums of cut walks: the shares', in order. Every warp reads the records and takes one row in `step` of those
// that they name; a lane holds DP / 32 elements.
constexpr int AB_JOIN_WARPS = 16;
template <typename T, int DP>
__global__ void __launch_bounds__(AB_JOIN_WARPS * 32) attn_bwd_join_kernel(const dn8_attention_bwd_args a, const BwdPlan plan) {
    constexpr int BATCH = 4;                          // 32 records each, loaded together
    const int lane = threadIdx.x & 31, step = gridDim.x * AB_JOIN_WARPS, d = lane * (DP / 32);
    int next = blockIdx.x * AB_JOIN_WARPS + (threadIdx.x >> 5), run = 0;
    griddep_wait();
    for (int base = 0; base < plan.records; base += 32 * BATCH) {
        int4 rec[BATCH];
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
            const int block = base + 32 * x + lane;
            rec[x] = block < plan.records ? plan.rec[block] : make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
            // (offsets that go back and forth may ask for more shares than there is room for, and a kernel that gave
            // up leaves records behind that say nothing: rows and shares are kept inside the tensors)
            const int4 c = rec[x];
            const bool sound = c.x >= 0 && c.y >= 0 && (c.y & 255) <= AT_TILE && c.w >= 1 && (c.y >> 8) < a.Hk &&
                               static_cast<int64_t>(c.x) + (c.y & 255) <= a.Tk;
            const int mine = sound ? c.y & 255 : 0;
            int incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const int total = __shfl_sync(0xffffffffu, incl, 31);
            for (; next < run + total; next += step) {
                const int src = __ffs(__ballot_sync(0xffffffffu, next < run + incl)) - 1;
                const int r = next - run - __shfl_sync(0xffffffffu, incl - mine, src);
                const int64_t row = static_cast<int64_t>(__shfl_sync(0xffffffffu, c.x, src)) + r;
                const int from = __shfl_sync(0xffffffffu, c.w, src), h = __shfl_sync(0xffffffffu, c.y, src) >> 8;
                const int block = base + 32 * x + src;
                const int cuts = min(__shfl_sync(0xffffffffu, c.z, src), (plan.records - 1 - block) / from + 1);
                const float* p = plan.part + (static_cast<size_t>(block) * 2 * AT_TILE + r) * DP + d;
                float s[2][DP / 32] = {};
#pragma unroll 4
                for (int y = 0; y < cuts; ++y) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float v[DP / 32];
                        load_f32(p + (static_cast<size_t>(y) * from * 2 + k) * AT_TILE * DP, v);
#pragma unroll
                        for (int e = 0; e < DP / 32; ++e) s[k][e] += v[e];
                    }
                }
                if (d < a.D) {
                    store_f32(static_cast<T*>(a.dv) + row * a.dv_stride_t + h * a.dv_stride_h + d, s[0]);
                    store_f32(static_cast<T*>(a.dk) + row * a.dk_stride_t + h * a.dk_stride_h + d, s[1]);
                }
            }
            run += total;
        }
    }
}

// Shares: under a window the tiles of the first tokens are walked over by all queries, the others by a few
// tiles of them. They are cut when that makes them the longest by far, into as many shares as leave them
// no longer than the others, or as fill the SMs.
static BwdPlan bwd_plan(const dn8_attention_bwd_args& a, int sms) {
    BwdPlan p = {};
    p.shares = 1;
    p.tiles = 1;
    // bounds on the tiles: every sequence may leave one unfilled
    int64_t kt = a.Tk / AT_TILE + (a.B < a.Tk ? a.B : a.Tk), qt = a.Tq / AT_TILE + (a.B < a.Tq ? a.B : a.Tq);
    const int64_t G = a.Hq / a.Hk, width = a.left < 0 || a.right < 0 ? a.Tq : static_cast<int64_t>(a.left) + a.right + AT_TILE;
    if (G > 1 && 2 * a.Tk * a.Hk < sms * AT_TILE && G * (width < a.Tq ? width : a.Tq) >= 20 * AT_TILE && kt * a.Hk < 4ll * sms) {
        // sum of max(1, steps / part), rounded, <= pieces + AB_PARTS sms / Hk (and one for the rounding of the sums)
        p.sms = sms;
        kt += static_cast<int64_t>(AB_PARTS * sms) / a.Hk + 1;
    } else if (a.left >= 0 && a.sinks > 0 && a.Tk > 0 && a.Tq > 0) {
        const int64_t tiles = (static_cast<int64_t>(a.sinks < a.Tk ? a.sinks : a.Tk) + AT_TILE - 1) / AT_TILE;
        const int64_t all = G * (a.Tq / a.B / AT_TILE + 1);
        const int64_t others = G * ((static_cast<int64_t>(a.left) + (a.right < 0 ? a.Tq / a.B : a.right) + AT_TILE) / AT_TILE + 1);
        const int64_t walks = a.B * tiles * a.Hk;
        int64_t s = (all + others - 1) / others;
        const int64_t fill = (2ll * sms + walks - 1) / walks;
        if (s > fill) s = fill;
        if (s > 1 && all > 2 * others) {
            p.tiles = static_cast<int>(tiles);
            p.shares = static_cast<int>(s < 32 ? s : 32);
            p.split_blocks = static_cast<int>(walks * p.shares);
        }
    }
    const int64_t kv = kt * a.Hk + p.split_blocks, all = kv + qt * a.Hq;
    if (all > 0x7FFFFFFFll) {
        p.blocks = -1;
        return p;
    }
    p.kv_blocks = static_cast<int>(kv);
    p.blocks = static_cast<int>(all);
    p.records = p.sms > 0 ? p.kv_blocks : p.split_blocks;
    return p;
}
static size_t bwd_stat_bytes(const dn8_attention_bwd_args& a) {
    return (static_cast<size_t>(a.Tq) * a.Hq * 2 * sizeof(float) + 255) / 256 * 256;
}

size_t attention_bwd_work(const dn8_attention_bwd_args& a, int sms) {
    const int DP = a.D <= 64 ? 64 : 128;
    return bwd_stat_bytes(a) + static_cast<size_t>(bwd_plan(a, sms).records) * (2 * AT_TILE * DP * sizeof(float) + sizeof(int4));
}

template <typename T, int DP> static cudaError_t bwd_go(const dn8_attention_bwd_args& a, int sms, cudaStream_t st) {
    CUtensorMap mq = {}, mk = {}, mv = {}, mdo = {};
    cudaError_t e = cudaSuccess;
    if (a.Tq > 0) {
        e = make_head_map(&mq, a.q, a.type, a.Tq, a.Hq, a.D, a.q_stride_t, a.q_stride_h);
        if (e == cudaSuccess) e = make_head_map(&mdo, a.dout, a.type, a.Tq, a.Hq, a.D, a.do_stride_t, a.do_stride_h);
    }
    if (e == cudaSuccess && a.Tk > 0) {
        e = make_head_map(&mk, a.k, a.type, a.Tk, a.Hk, a.D, a.k_stride_t, a.k_stride_h);
        if (e == cudaSuccess) e = make_head_map(&mv, a.v, a.type, a.Tk, a.Hk, a.D, a.v_stride_t, a.v_stride_h);
    }
    if (e != cudaSuccess) return e;
    BwdPlan plan = bwd_plan(a, sms);
    const auto kernel = plan.sms > 0 ? attn_bwd_kernel<T, DP, true> : attn_bwd_kernel<T, DP, false>;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdCfg<DP>::SMEM);
    if (e != cudaSuccess) return e;
    if (plan.blocks < 0) return cudaErrorInvalidValue;
    plan.part = reinterpret_cast<float*>(static_cast<uint8_t*>(a.work) + bwd_stat_bytes(a));
    plan.rec = reinterpret_cast<int4*>(plan.part + static_cast<size_t>(plan.records) * 2 * AT_TILE * DP);
    if (a.Tq > 0) {
        e = launch_pdl(false, attn_bwd_prep_kernel<T, DP / 8>, dim3(static_cast<unsigned>((a.Tq + 31) / 32), a.Hq),
                       dim3(32 * (DP / 8)), 0, st, a);
        if (e != cudaSuccess) return e;
    }
    e = launch_pdl(a.Tq > 0, kernel, dim3(static_cast<unsigned>(plan.blocks)), dim3(AB_THREADS),
                   BwdCfg<DP>::SMEM, st, mq, mk, mv, mdo, a, plan);
    if (e != cudaSuccess || plan.records == 0) return e;
    return launch_pdl(true, attn_bwd_join_kernel<T, DP>, dim3(2 * sms), dim3(AB_JOIN_WARPS * 32), 0, st, a, plan);
}

cudaError_t launch_attention_bwd(const dn8_attention_bwd_args& a, int sms, cudaStream_t st) {
    if (a.type == DN8_F16) return a.D <= 64 ? bwd_go<__half, 64>(a, sms, st) : bwd_go<__half, 128>(a, sms, st);
    return a.D <= 64 ? bwd_go<__nv_bfloat16, 64>(a, sms, st) : bwd_go<__nv_bfloat16, 128>(a, sms, st);
}

}  // namespace dn8
