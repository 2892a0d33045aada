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
// so no operand is ever transposed or written to shared memory by a thread. The issue order dv(u),
// S(u + 1), dk(u), dP(u + 1) keeps the tensor cores on one of them while the threads work on the other:
// exponentials of S while dP is made, dS while dv and the next S are made.
#include "attn_umma.cuh"

namespace dn8 {

// ---- delta and the logarithms in units of log2, head by head -------------------------------------
// work: lse2 [Hq][Tq] (+inf where the row sees nothing: its P = 2^(s - inf) = 0), then delta [Hq][Tq].
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
        w[0] = lse == -INFINITY ? INFINITY : lse * ATT_LOG2E;
        w[a.Hq * a.Tq] = lse == -INFINITY ? 0.0f : s;
    }
}

// ---- the two walks -----------------------------------------------------------------------------
constexpr int AB_THREADS = 384;             // warps 0-7: rows; 8: tcgen05 issue; 9: TMA; 10: masked rows
template <int DP> struct BwdCfg {
    static constexpr int ST = DP == 64 ? 3 : 2;
    static constexpr uint32_t TILE = AT_TILE * DP * 2;
    static constexpr uint32_t SMEM = 1024 + TILE * 2 * (1 + ST) + 4096 + 1024;
    static constexpr uint32_t S = 0, DPC = 128, ACC0 = 256, ACC1 = 256 + DP;     // TMEM columns
};
struct BwdShared {
    float lse2[3][AT_TILE], delta[3][AT_TILE];
    uint32_t words[3][4];
    uint64_t rfull, fin, sfull, dpfull, pready, dsready;
    uint64_t xfull[3], xempty[3], xok[3];
    uint32_t tmem;
    int abort;
    Sequence seq;
};

// What a CTA does: its resident rows and the tiles it walks over.
struct BwdWalk {
    bool kv;                 // dk, dv of a key tile, or dq of a query tile
    int r0;                  // first resident row, within the sequence
    int h;                   // key head (kv) or query head
    int steps;
    int first, per;          // kv: first query tile and query tiles per head
    KeyTiles keys;           // dq: key tiles
};

// The 8 row warps: warp w has the TMEM lanes (resident rows) 32 (w % 4) .. and the columns 64 (w / 4) .. of
// every step.
template <typename T, int DP, bool KV>
DN8_DEV void bwd_rows(const dn8_attention_bwd_args& a, BwdShared& sh, const BwdWalk& wk, uint32_t tmem) {
    using C = BwdCfg<DP>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t quad = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + C::S + quad + half * 64, tp = tmem + C::DPC + quad + half * 64;
    volatile int* abort_flag = &sh.abort;
    const Sequence seq = sh.seq;
    const int off = seq.nk - seq.nq;
    const int left = a.left < 0 ? ATT_FAR : a.left, right = a.right < 0 ? ATT_FAR : a.right;
    const float sc = a.scale * ATT_LOG2E;
    const int r = wk.r0 + row;                                   // key j (KV) or query i
    const bool inside = r < (KV ? seq.nk : seq.nq);
    // KV: the key may be seen at all; dq: the row's statistics
    const bool keep = KV && inside && (a.keep == nullptr || a.keep[seq.k0 + r] != 0);
    float row_lse = INFINITY, row_delta = 0.0f;
    if (!KV && inside) {
        const float* w = static_cast<const float*>(a.work) + wk.h * a.Tq + seq.q0 + r;
        row_lse = w[0];
        row_delta = w[a.Hq * a.Tq];
    }
    const int rlast = min(wk.r0 + AT_TILE, KV ? seq.nk : seq.nq) - 1;
    bool ok = true;
    for (int u = 0; u < wk.steps; ++u) {
        const int st = u % C::ST;
        const int c0 = (KV ? wk.first + u % wk.per : wk.keys.tile(u)) * AT_TILE, cl = c0 + AT_TILE - 1;
        ok = mbar_wait_w(&sh.xok[st], (u / C::ST) & 1, a.err, abort_flag, ERR_WAIT_FULL | (80 << 4));
        if (!ok) break;
        uint32_t word[2] = {0xFFFFFFFFu, 0xFFFFFFFFu};
        bool masked;
        if (KV) {
            // columns are queries: seen from j - right - off on, up to j + left - off (first tokens: by all).
            // Queries behind the end are zero rows with lse2 = inf.
            masked = a.keep != nullptr || wk.r0 + AT_TILE > seq.nk || c0 + off < rlast - right ||
                     (cl + off > wk.r0 + left && rlast >= a.sinks);
            if (masked) {
                const int lo = r - right - off - c0, hi = r < a.sinks ? ATT_FAR : r + left - off - c0;
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    word[w] = keep ? bits_from(lo, 2 * half + w) & bits_upto(hi, 2 * half + w) : 0u;
            }
        } else {
            const int p = r + off;
            masked = a.keep != nullptr || cl > min(seq.nk - 1, wk.r0 + off + right) || (c0 < rlast + off - left && cl >= a.sinks);
            if (masked) {
                const int hi = min(seq.nk - 1, p + right) - c0, lo = p - left - c0;
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    word[w] = bits_upto(hi, 2 * half + w) & sh.words[st][2 * half + w] &
                              (bits_from(lo, 2 * half + w) | bits_upto(a.sinks - 1 - c0, 2 * half + w));
            }
        }
        ok = mbar_wait_w(&sh.sfull, u & 1, a.err, abort_flag, ERR_WAIT_ACC | (81 << 4));
        if (!ok) break;
        tc_fence_after();
        uint32_t pr[2][32];                                      // P of this thread's 64 columns, fp32
        tmem_ld32(ts, pr[0]);
        tmem_ld32(ts + 32, pr[1]);
        tmem_wait_ld(pr[0]);
        reg_bind(pr[1]);
        if (!KV) {                                               // S is in registers: the next one may come
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.pready);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (KV) {
                const float4* l4 = reinterpret_cast<const float4*>(sh.lse2[st] + half * 64 + c * 32);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float4 l = l4[e];
                    const float ls[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        pr[c][4 * e + x] = __float_as_uint(ex2(fmaf(__uint_as_float(pr[c][4 * e + x]), sc, -ls[x])));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    pr[c][e] = __float_as_uint(ex2(fmaf(__uint_as_float(pr[c][e]), sc, -row_lse)));
            }
            if (masked)
#pragma unroll
                for (int e = 0; e < 32; ++e) pr[c][e] = (word[c] >> e) & 1u ? pr[c][e] : 0u;
        }
        if (KV) {
            // P in [0, 1], rounded to the inputs' type for dv
            uint32_t pk[32];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    pk[16 * c + e] = pack2(T(), __uint_as_float(pr[c][2 * e]), __uint_as_float(pr[c][2 * e + 1]));
            tmem_st32(ts, pk);
            tmem_wait_st(pk);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.pready);
        }
        ok = mbar_wait_w(&sh.dpfull, u & 1, a.err, abort_flag, ERR_WAIT_ACC | (82 << 4));
        if (!ok) break;
        tc_fence_after();
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t dp[32];
            tmem_ld32(tp + 32 * c, dp);
            tmem_wait_ld(dp);
            float ds[32];
            if (KV) {
                const float4* d4 = reinterpret_cast<const float4*>(sh.delta[st] + half * 64 + c * 32);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float4 d = d4[e];
                    const float de[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        ds[4 * e + x] = __uint_as_float(pr[c][4 * e + x]) * ((__uint_as_float(dp[4 * e + x]) - de[x]) * a.scale);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    ds[e] = __uint_as_float(pr[c][e]) * ((__uint_as_float(dp[e]) - row_delta) * a.scale);
            }
            // (a masked pair's dP may be NaN, and 0 * NaN is not 0)
            if (masked)
#pragma unroll
                for (int e = 0; e < 32; ++e) ds[e] = (word[c] >> e) & 1u ? ds[e] : 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) pk[16 * c + e] = pack2(T(), ds[2 * e], ds[2 * e + 1]);
        }
        tmem_st32(tp, pk);
        tmem_wait_st(pk);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.dsready);
    }
    if (ok && wk.steps > 0) {
        ok = mbar_wait_w(&sh.fin, 0, a.err, abort_flag, ERR_WAIT_ACC | (83 << 4));
        tc_fence_after();
    }
    // the sums: half 0 writes dv and half 1 dk, or each half its columns of dq
    const int64_t at = static_cast<int64_t>(KV ? seq.k0 : seq.q0) + r;
    T* dst = KV ? (half == 0 ? static_cast<T*>(a.dv) + at * a.dv_stride_t + wk.h * a.dv_stride_h
                             : static_cast<T*>(a.dk) + at * a.dk_stride_t + wk.h * a.dk_stride_h)
                : static_cast<T*>(a.dq) + at * a.dq_stride_t + wk.h * a.dq_stride_h;
    const uint32_t acc = tmem + quad + (KV && half == 1 ? C::ACC1 : C::ACC0);
    const bool zero = wk.steps == 0 || (!KV && row_lse == INFINITY);
    constexpr int CHUNKS = DP / 32;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        if (!KV && (c < CHUNKS / 2) != (half == 0)) continue;
        uint32_t o[32];
        if (wk.steps > 0 && ok) {
            tmem_ld32(acc + 32 * c, o);
            tmem_wait_ld(o);
        }
        if (ok && inside)
#pragma unroll
            for (int e = 0; e < 32; e += 8)
                if (32 * c + e < a.D) {
                    float v[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) v[x] = zero ? 0.0f : __uint_as_float(o[e + x]);
                    store_f32(dst + 32 * c + e, v);
                }
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(AB_THREADS, 1)
attn_bwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo,
                const dn8_attention_bwd_args a, int kv_blocks) {
    using C = BwdCfg<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sr = smem;                                  // R0, R1
    uint8_t* sx = smem + 2 * C::TILE;                    // stages of X0, X1
    BwdShared& sh = *reinterpret_cast<BwdShared*>(sx + 2 * C::ST * C::TILE);
    volatile int* abort_flag = &sh.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.Hq / a.Hk;
    const bool kv = static_cast<int>(blockIdx.x) < kv_blocks;
    const int idx = kv ? blockIdx.x : blockIdx.x - kv_blocks, heads = kv ? a.Hk : a.Hq;
    if (warp == 8) {
        const Sequence f = kv ? find_block<true>(a, idx / heads, 1, AT_TILE) : find_block<false>(a, idx / heads, 1, AT_TILE);
        if (lane == 0) {
            sh.seq = f;
            mbar_init(&sh.rfull, 1);
            mbar_init(&sh.fin, 1);
            mbar_init(&sh.sfull, 1);
            mbar_init(&sh.dpfull, 1);
            mbar_init(&sh.pready, 8);
            mbar_init(&sh.dsready, 8);
            for (int s = 0; s < 3; ++s) {
                mbar_init(&sh.xfull[s], 1);
                mbar_init(&sh.xempty[s], 2);             // the last product and warp 10
                mbar_init(&sh.xok[s], 1);
            }
            sh.abort = 0;
            mbar_fence_init();
        }
        __syncwarp();
    }
    if (warp == 9) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const Sequence seq = sh.seq;
    const int off = seq.nk - seq.nq;
    const int left = a.left < 0 ? ATT_FAR : a.left, right = a.right < 0 ? ATT_FAR : a.right;
    BwdWalk wk;
    wk.kv = kv;
    wk.h = idx % heads;
    wk.steps = wk.first = wk.r0 = 0;
    wk.per = 1;
    wk.keys.count = wk.keys.first = wk.keys.start = 0;
    if (seq.b >= 0) {
        if (kv) {
            // first key tiles first: first tokens and open left sides make them the longest
            wk.r0 = seq.blk * AT_TILE;
            const int jl = min(wk.r0 + AT_TILE, seq.nk) - 1;
            const int lo = max(0, wk.r0 - right - off), hi = wk.r0 < a.sinks ? seq.nq - 1 : min(seq.nq - 1, jl + left - off);
            if (lo <= hi) {
                wk.first = lo / AT_TILE;
                wk.per = hi / AT_TILE - wk.first + 1;
                wk.steps = wk.per * G;
            }
        } else {
            wk.r0 = ((seq.nq - 1) / AT_TILE - seq.blk) * AT_TILE;
            wk.keys = key_tiles(wk.r0 + off, min(wk.r0 + AT_TILE, seq.nq) - 1 + off, seq.nk, left, right, a.sinks, AT_TILE);
            wk.steps = wk.keys.count;
        }
    }
    // tile and head of step u
    auto tile_of = [&](int u) -> int { return kv ? wk.first + u % wk.per : wk.keys.tile(u); };
    auto head_of = [&](int u) -> int { return kv ? wk.h * G + u / wk.per : wk.h / G; };
    griddep_wait();                                      // delta and lse2

    if (seq.b >= 0 && warp == 9) {
        // ---------------- TMA ----------------
        if (lane == 0 && wk.steps > 0) {
            const int r0 = (kv ? seq.k0 : seq.q0) + wk.r0;
            mbar_expect_tx(&sh.rfull, 2 * C::TILE);
            load_tile<DP>(sr, kv ? &mk : &mq, &sh.rfull, wk.h, r0);
            load_tile<DP>(sr + C::TILE, kv ? &mv : &mdo, &sh.rfull, wk.h, r0);
            for (int u = 0; u < wk.steps; ++u) {
                const int s = u % C::ST;
                if (!mbar_wait(&sh.xempty[s], ((u / C::ST) & 1) ^ 1, a.err, abort_flag, ERR_WAIT_EMPTY | (84 << 4))) break;
                const int x0 = (kv ? seq.q0 : seq.k0) + tile_of(u) * AT_TILE, hx = head_of(u);
                mbar_expect_tx(&sh.xfull[s], 2 * C::TILE);
                load_tile<DP>(sx + 2 * s * C::TILE, kv ? &mq : &mk, &sh.xfull[s], hx, x0);
                load_tile<DP>(sx + (2 * s + 1) * C::TILE, kv ? &mdo : &mv, &sh.xfull[s], hx, x0);
            }
        }
        __syncwarp();
    } else if (seq.b >= 0 && warp == 10) {
        // ---------------- masked rows of the streamed tiles, statistics of the query rows ----------------
        // Streamed rows are summed over: a row whose weights are all zero must not hold NaN.
        for (int u = 0; u < wk.steps; ++u) {
            const int s = u % C::ST, t0 = tile_of(u) * AT_TILE;
            uint32_t word[4];
            float l2[4], de[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int x = t0 + w * 32 + lane;
                bool live;
                if (kv) {
                    l2[w] = INFINITY;
                    de[w] = 0.0f;
                    if (x < seq.nq) {
                        const float* ws = static_cast<const float*>(a.work) + head_of(u) * a.Tq + seq.q0 + x;
                        l2[w] = ws[0];
                        de[w] = ws[a.Hq * a.Tq];
                    }
                    live = l2[w] != INFINITY;
                } else {
                    live = x < seq.nk && (a.keep == nullptr || a.keep[seq.k0 + x] != 0);
                }
                word[w] = __ballot_sync(0xffffffffu, live);
            }
            if (!mbar_wait_w(&sh.xfull[s], (u / C::ST) & 1, a.err, abort_flag, ERR_WAIT_FULL | (85 << 4))) break;
            const bool fix = (word[0] & word[1] & word[2] & word[3]) != 0xFFFFFFFFu;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if (kv) {
                    sh.lse2[s][w * 32 + lane] = l2[w];
                    sh.delta[s][w * 32 + lane] = de[w];
                } else if (lane == w) {
                    sh.words[s][w] = word[w];
                }
                if (fix && !((word[w] >> lane) & 1u)) {
                    // X0, and for dk, dv X1 too (dout): the tiles that are right operands of a sum over rows
                    const int blocks = (kv ? 2 : 1) * (DP / 64);
                    for (int b = 0; b < blocks; ++b) {
                        uint4* row = reinterpret_cast<uint4*>(sx + 2 * s * C::TILE + b * AT_BLOCK + (w * 32 + lane) * 128);
#pragma unroll
                        for (int c = 0; c < 8; ++c) row[c] = make_uint4(0u, 0u, 0u, 0u);
                    }
                }
            }
            if (fix) fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.xok[s]);
                mbar_arrive(&sh.xempty[s]);
            }
        }
    } else if (seq.b >= 0 && warp == 8 && wk.steps > 0) {
        // ---------------- tcgen05 issue ----------------
        const uint32_t r0 = smem_u32(sr), r1 = r0 + C::TILE, x = smem_u32(sx);
        auto wait_x = [&](int u) -> bool {
            const int s = u % C::ST;
            return mbar_wait_w(&sh.xfull[s], (u / C::ST) & 1, a.err, abort_flag, ERR_WAIT_FULL | (86 << 4)) &&
                   mbar_wait_w(&sh.xok[s], (u / C::ST) & 1, a.err, abort_flag, ERR_WAIT_FULL | (87 << 4));
        };
        bool ok = mbar_wait_w(&sh.rfull, 0, a.err, abort_flag, ERR_WAIT_FULL | (88 << 4)) && wait_x(0);
        if (ok) {
            tc_fence_after();
            mma_scores<T, DP>(tmem + C::S, r0, x);
            umma_commit_w(&sh.sfull);
            mma_scores<T, DP>(tmem + C::DPC, r1, x + C::TILE);
            umma_commit_w(&sh.dpfull);
        }
        for (int u = 0; ok && u < wk.steps; ++u) {
            const uint32_t x0 = x + 2 * (u % C::ST) * C::TILE, xn = x + 2 * ((u + 1) % C::ST) * C::TILE;
            ok = mbar_wait_w(&sh.pready, u & 1, a.err, abort_flag, ERR_WAIT_ACC | (89 << 4));
            if (!ok) break;
            tc_fence_after();
            if (kv) mma_values<T, DP>(tmem + C::ACC0, tmem + C::S, x0 + C::TILE, u > 0);
            if (u + 1 < wk.steps) {
                ok = wait_x(u + 1);
                if (!ok) break;
                tc_fence_after();
                mma_scores<T, DP>(tmem + C::S, r0, xn);
                umma_commit_w(&sh.sfull);
            }
            ok = mbar_wait_w(&sh.dsready, u & 1, a.err, abort_flag, ERR_WAIT_ACC | (90 << 4));
            if (!ok) break;
            tc_fence_after();
            mma_values<T, DP>(tmem + (kv ? C::ACC1 : C::ACC0), tmem + C::DPC, x0, u > 0);
            umma_commit_w(&sh.xempty[u % C::ST]);
            if (u + 1 < wk.steps) {
                mma_scores<T, DP>(tmem + C::DPC, r1, xn + C::TILE);
                umma_commit_w(&sh.dpfull);
            }
        }
        if (ok) umma_commit_w(&sh.fin);
        __syncwarp();
    } else if (seq.b >= 0 && warp < 8) {
        if (kv) bwd_rows<T, DP, true>(a, sh, wk, tmem);
        else bwd_rows<T, DP, false>(a, sh, wk, tmem);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

size_t attention_bwd_work(const dn8_attention_bwd_args& a) { return static_cast<size_t>(a.Tq) * a.Hq * 2 * sizeof(float); }

template <typename T, int DP> static cudaError_t bwd_go(const dn8_attention_bwd_args& a, cudaStream_t st) {
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
    e = cudaFuncSetAttribute(attn_bwd_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdCfg<DP>::SMEM);
    if (e != cudaSuccess) return e;
    // bounds on the tiles: every sequence may leave one unfilled
    const int64_t kt = (a.Tk / AT_TILE + (a.B < a.Tk ? a.B : a.Tk)) * a.Hk;
    const int64_t qt = (a.Tq / AT_TILE + (a.B < a.Tq ? a.B : a.Tq)) * a.Hq;
    if (kt + qt > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    if (a.Tq > 0) {
        e = launch_pdl(false, attn_bwd_prep_kernel<T, DP / 8>, dim3(static_cast<unsigned>((a.Tq + 31) / 32), a.Hq),
                       dim3(32 * (DP / 8)), 0, st, a);
        if (e != cudaSuccess) return e;
    }
    return launch_pdl(a.Tq > 0, attn_bwd_kernel<T, DP>, dim3(static_cast<unsigned>(kt + qt)), dim3(AB_THREADS),
                      BwdCfg<DP>::SMEM, st, mq, mk, mv, mdo, a, static_cast<int>(kt));
}

cudaError_t launch_attention_bwd(const dn8_attention_bwd_args& a, cudaStream_t st) {
    if (a.type == DN8_F16) return a.D <= 64 ? bwd_go<__half, 64>(a, st) : bwd_go<__half, 128>(a, st);
    return a.D <= 64 ? bwd_go<__nv_bfloat16, 64>(a, st) : bwd_go<__nv_bfloat16, 128>(a, st);
}

}  // namespace dn8
